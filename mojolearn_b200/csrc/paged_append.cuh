// Fresh q | k | v rows into their places: per-head norms, the rotation to each row's position, keys and values into the pages.
//
//   u = x * rsqrt(mean(x^2) + eps) * w      per head of q and k, where the model norms them (w, or 1 + w)
//   y_i = u_i cos_i - u_{i+r/2} sin_i,  y_{i+r/2} = u_{i+r/2} cos_i + u_i sin_i   for i < r/2, the columns from r on as they are
//
// Bound: HBM, each word read once and written once; a single token is one trip through memory and the launch.
// A head's columns go by units of 16 bytes of the row type; a lane takes a unit of the first half and its partner of the second, so that
// the rotation needs no other lane and the norm is one shuffle reduction over the lanes of the head (a power of two of them, some
// idle where the head has an odd number of units). Sums and products are in 32 bits, two words an instruction, and a word is rounded once, at
// its store. With many rows a warp takes several sets of heads of its row one after another, the next one's words asked for before this one's
// are worked on: 350 instructions a set, most of them to find its place, had taken 60 us where the bytes need 33.
// Measured: 16 prompts of 33 to 1024 tokens, 32 + 2 x 8 heads of 128, with norms, bfloat16: 45 us (0.72 of the HBM rate; 0.68 instructions a cycle).
#pragma once
#include <algorithm>

#include "paged.cuh"
#include "paged_async.cuh"

namespace b200i {

struct AppendCall {
    PagedCall c;
    const void *q, *k, *v;
    void *q_out, *k_cache, *v_cache;
    long long ldq, ldk, ldv;       // elements between rows
    const float *cosv, *sinv;      // [positions, rope_dim / 2], nullptr: no rotation
    const float *q_norm, *k_norm;  // [head_dim] each, nullptr: no norm
    int rope_dim, positions;
    float eps, norm_shift;         // norm_shift: added to the norm's weight (0 or 1)
    float part_of_head;            // 1 / head_dim
};

template <typename T>
struct Unit; // 16 bytes of a row; its words two by two
template <>
struct Unit<float> {
    static constexpr int N = 4;
    using Raw = float4;
    static __device__ __forceinline__ Raw ask(const float *p) { return __ldg(reinterpret_cast<const float4 *>(p)); }
    static __device__ __forceinline__ void words(unsigned long long *x, const Raw &r) { x[0] = pg_two(r.x, r.y), x[1] = pg_two(r.z, r.w); }
    static __device__ __forceinline__ void store(float *p, const unsigned long long *x) { *reinterpret_cast<ulonglong2 *>(p) = make_ulonglong2(x[0], x[1]); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const unsigned long long *x) {
        float w[4];
        pg_one(x[0], w[0], w[1]), pg_one(x[1], w[2], w[3]);
        *reinterpret_cast<uint2 *>(p) = make_uint2(pg_pack(w[0], w[1]), pg_pack(w[2], w[3]));
    }
};
template <>
struct Unit<__nv_bfloat16> {
    static constexpr int N = 8;
    using Raw = uint4;
    static __device__ __forceinline__ Raw ask(const __nv_bfloat16 *p) { return __ldg(reinterpret_cast<const uint4 *>(p)); }
    static __device__ __forceinline__ void words(unsigned long long *x, const Raw &r) {
        const unsigned v[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = pg_two(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xFFFF0000u));
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const unsigned long long *x) {
        unsigned v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float lo, hi;
            pg_one(x[i], lo, hi);
            v[i] = pg_pack(lo, hi);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(v[0], v[1], v[2], v[3]);
    }
};

// Where a row's head goes: the output row of q, or its page's place; false where it goes nowhere.
template <typename RT, typename CT>
__device__ __forceinline__ bool append_place(const AppendCall &a, long long t, int b, int pos, int part, int head, RT **dst_row, CT **dst_cache) {
    *dst_row = nullptr, *dst_cache = nullptr;
    if (part == 0) {
        *dst_row = static_cast<RT *>(a.q_out) + (t * a.c.heads + head) * a.c.hd;
        return true;
    }
    if (pos < 0) return false; // the lengths say that this row was cached before the sequence began
    const long long at = paged_offset(a.c, b, head, pos);
    if (at < 0) return false;
    *dst_cache = static_cast<CT *>(part == 1 ? a.k_cache : a.v_cache) + at;
    return true;
}

// Whether the rotation's table has no row for a position: nothing is written for the row then, and that is reported.
__device__ __forceinline__ bool append_past(const AppendCall &a, int pos) {
    if (!a.cosv || pos < a.positions) return false;
    atomicExch(a.c.status, PAGED_BAD_POSITION);
    return true;
}

// N words of 32 bits, 16-byte aligned, two by two.
template <int N>
__device__ __forceinline__ void append_words(unsigned long long *x, const float *p) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 v = __ldg(reinterpret_cast<const float4 *>(p + i));
        x[i / 2] = pg_two(v.x, v.y), x[i / 2 + 1] = pg_two(v.z, v.w);
    }
}

// blockIdx.x: the row; its heads in sets of 32 >> lanes_log2, a set a warp, by steps of the warps of gridDim.y blocks. A row's words are asked for
// before it is known whose they are.
template <typename RT, typename CT>
__global__ void __launch_bounds__(128) append_units_kernel(const AppendCall a, int lanes_log2, int sets) {
    constexpr int N = Unit<RT>::N;
    const long long t = blockIdx.x;
    const int lane = threadIdx.x & ((1 << lanes_log2) - 1), in_set = (threadIdx.x & 31) >> lanes_log2;
    // unit pairs of the rotated columns come first, pairs of neighbouring units of the others after them
    const int half = a.rope_dim / 2, pairs = half / N, rest = (a.c.hd - a.rope_dim) / N;
    const bool turned = lane < pairs;
    const int at0 = turned ? lane * N : a.rope_dim + (lane - pairs) * 2 * N, at1 = turned ? at0 + half : at0 + N;
    const bool some0 = lane < pairs + (rest + 1) / 2, some1 = some0 && (turned || (lane - pairs) * 2 + 1 < rest);
    const RT *const q = static_cast<const RT *>(a.q) + t * a.ldq, *const k = static_cast<const RT *>(a.k) + t * a.ldk, *const v = static_cast<const RT *>(a.v) + t * a.ldv;
    const int parts = a.c.heads + 2 * a.c.kv;

    typename Unit<RT>::Raw raw0, raw1;
    const auto ask = [&](int set) {
        const int head = (set << (5 - lanes_log2)) + in_set;
        const RT *src = head < a.c.heads ? q + head * a.c.hd : (head < a.c.heads + a.c.kv ? k + (head - a.c.heads) * a.c.hd : v + (head - a.c.heads - a.c.kv) * a.c.hd);
        raw0 = raw1 = typename Unit<RT>::Raw{};
        if (head < parts && some0) raw0 = Unit<RT>::ask(src + at0);
        if (head < parts && some1) raw1 = Unit<RT>::ask(src + at1);
    };
    int set = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int step = gridDim.y * 4;
    if (set < sets) ask(set);

    const int b = paged_row_seq(a.c, t);
    if (b < 0) return; // a row of no sequence: nothing is written for it
    const PagedSeq s = paged_seq_checked(a.c, b);
    if (s.n == 0) return; // its tables do not hold it
    const int pos = s.pos0 + (int)(t - s.first);
    if (append_past(a, pos)) return;
    // the position's place in the caches, of key head 0; -1: none
    const long long place = pos < 0 ? -1 : paged_offset(a.c, b, 0, pos);
    const int head_words = a.c.hd << a.c.page_shift;
    unsigned long long c[N / 2], sn[N / 2];
    const bool turns = turned && a.cosv != nullptr;
    if (turns) {
        const long long row = (long long)max(pos, 0) * half + at0;
        append_words<N>(c, a.cosv + row);
        append_words<N>(sn, a.sinv + row);
    }
    for (; set < sets; set += step) {
        const int head = (set << (5 - lanes_log2)) + in_set, part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2); // q, k, v
        unsigned long long x0[N / 2], x1[N / 2];
        Unit<RT>::words(x0, raw0), Unit<RT>::words(x1, raw1);
        if (set + step < sets) ask(set + step);
        if (a.q_norm || a.k_norm) { // uniform over the grid: the reduction is a warp's
            unsigned long long sums = 0;
#pragma unroll
            for (int i = 0; i < N / 2; i++) sums = pg_fma2(x0[i], x0[i], pg_fma2(x1[i], x1[i], sums));
            float sum, other;
            pg_one(sums, sum, other);
            sum += other;
            for (int o = (1 << lanes_log2) >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            const float *w = part == 0 ? a.q_norm : (part == 1 ? a.k_norm : nullptr);
            if (w) {
                const float r = rsqrtf(fmaf(sum, a.part_of_head, a.eps));
                const unsigned long long r2 = pg_two(r, r), shift2 = pg_two(a.norm_shift * r, a.norm_shift * r);
                unsigned long long weight[N / 2];
                if (some0) {
                    append_words<N>(weight, w + at0);
#pragma unroll
                    for (int i = 0; i < N / 2; i++) x0[i] = pg_mul2(x0[i], pg_fma2(weight[i], r2, shift2));
                }
                if (some1) {
                    append_words<N>(weight, w + at1);
#pragma unroll
                    for (int i = 0; i < N / 2; i++) x1[i] = pg_mul2(x1[i], pg_fma2(weight[i], r2, shift2));
                }
            }
        }
        if (head >= parts || !some0) continue;
        if (turns && part < 2) {
            const unsigned long long minus = pg_two(-1.0f, -1.0f);
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                const unsigned long long u = x0[i], y = x1[i];
                x0[i] = pg_fma2(u, c[i], pg_mul2(pg_mul2(y, sn[i]), minus));
                x1[i] = pg_fma2(y, c[i], pg_mul2(u, sn[i]));
            }
        }
        if (part == 0) {
            RT *dst = static_cast<RT *>(a.q_out) + (t * a.c.heads + head) * a.c.hd;
            Unit<RT>::store(dst + at0, x0);
            if (some1) Unit<RT>::store(dst + at1, x1);
        } else if (place >= 0) {
            CT *dst = static_cast<CT *>(part == 1 ? a.k_cache : a.v_cache) + place + (long long)(head - a.c.heads - (part == 1 ? 0 : a.c.kv)) * head_words;
            Unit<RT>::store(dst + at0, x0);
            if (some1) Unit<RT>::store(dst + at1, x1);
        }
    }
}

// Rotations whose halves are not whole units (a partial rotation of few columns), or tables and weights that are not 16-byte aligned: a warp a head, a
// column a lane.
template <typename RT, typename CT>
__global__ void __launch_bounds__(256) append_columns_kernel(const AppendCall a) {
    const long long t = blockIdx.x;
    const int lane = threadIdx.x & 31, b = paged_row_seq(a.c, t);
    int head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (b < 0 || head >= a.c.heads + 2 * a.c.kv) return;
    const PagedSeq s = paged_seq_checked(a.c, b);
    if (s.n == 0) return; // its tables do not hold it
    const int pos = s.pos0 + (int)(t - s.first), part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2);
    if (append_past(a, pos)) return;
    head -= part == 0 ? 0 : (part == 1 ? a.c.heads : a.c.heads + a.c.kv);
    const RT *src = part == 0 ? static_cast<const RT *>(a.q) + t * a.ldq : (part == 1 ? static_cast<const RT *>(a.k) + t * a.ldk : static_cast<const RT *>(a.v) + t * a.ldv);
    src += (long long)head * a.c.hd;
    const float *w = part == 0 ? a.q_norm : (part == 1 ? a.k_norm : nullptr);
    float r = 1.0f;
    if (w) {
        float sum = 0.0f;
        for (int i = lane; i < a.c.hd; i += 32) {
            const float x = paged_read(src + i);
            sum = fmaf(x, x, sum);
        }
        r = 1.0f / sqrtf(paged_warp_sum(sum) / (float)a.c.hd + a.eps);
    }
    RT *dst_row;
    CT *dst_cache;
    if (!append_place<RT, CT>(a, t, b, pos, part, head, &dst_row, &dst_cache)) return;
    const int half = a.rope_dim / 2;
    const long long row = (long long)max(pos, 0) * half;
    float out[PAGED_MAX_HD / 32];
#pragma unroll
    for (int k = 0; k < PAGED_MAX_HD / 32; k++) {
        const int i = lane + 32 * k;
        if (i >= a.c.hd) break;
        float x = paged_read(src + i);
        if (w) x = x * r * (w[i] + a.norm_shift);
        if (part < 2 && a.cosv && i < a.rope_dim) {
            const int j = i < half ? i : i - half, p = i < half ? i + half : i - half;
            float y = paged_read(src + p);
            if (w) y = y * r * (w[p] + a.norm_shift);
            const float c = a.cosv[row + j], sn = a.sinv[row + j];
            x = i < half ? fmaf(x, c, -(y * sn)) : fmaf(x, c, y * sn);
        }
        out[k] = x;
    }
    __syncwarp(); // all is read before any of it is written: the queries may be rotated in their place
#pragma unroll
    for (int k = 0; k < PAGED_MAX_HD / 32; k++) {
        const int i = lane + 32 * k;
        if (i >= a.c.hd) break;
        if (dst_row)
            paged_write(dst_row + i, out[k]);
        else
            paged_write(dst_cache + i, out[k]);
    }
}

template <typename RT, typename CT>
cudaError_t launch_append(const AppendCall &a, int sms, cudaStream_t st) {
    constexpr int N = Unit<RT>::N;
    const int parts = a.c.heads + 2 * a.c.kv;
    const uintptr_t words = reinterpret_cast<uintptr_t>(a.cosv) | reinterpret_cast<uintptr_t>(a.sinv) | reinterpret_cast<uintptr_t>(a.q_norm) | reinterpret_cast<uintptr_t>(a.k_norm);
    if ((a.rope_dim / 2) % N == 0 && (a.c.hd - a.rope_dim) % N == 0 && words % 16 == 0) {
        const int need = a.rope_dim / 2 / N + ((a.c.hd - a.rope_dim) / N + 1) / 2;
        int lg = 0;
        while ((1 << lg) < need) lg++;
        // with a few rows a warp takes one set of heads, so that none waits for another's; with many it takes all that the blocks of a row leave it
        const int per_set = 32 >> lg, sets = (parts + per_set - 1) / per_set, blocks = (sets + 3) / 4;
        const long long room = 8LL * sms; // blocks that fill the device
        const int y = (int)std::max<long long>(1, std::min<long long>(blocks, room / a.c.rows));
        append_units_kernel<RT, CT><<<dim3((unsigned)a.c.rows, (unsigned)y), 128, 0, st>>>(a, lg, sets);
    } else {
        append_columns_kernel<RT, CT><<<dim3((unsigned)a.c.rows, (unsigned)((parts + 7) / 8)), 256, 0, st>>>(a);
    }
    return cudaGetLastError();
}

} // namespace b200i

// Fresh q | k | v rows into their places: per-head norms, the rotation to each row's position, keys and values into the pages.
//
//   u = x * rsqrt(mean(x^2) + eps) * w      per head of q and k, where the model norms them (w, or 1 + w)
//   y_i = u_i cos_i - u_{i+r/2} sin_i,  y_{i+r/2} = u_{i+r/2} cos_i + u_i sin_i   for i < r/2, the columns from r on as they are
//
// Bound: HBM, each word read once and written once; a single token is one trip through memory and the launch.
// A head's columns go by units of 16 bytes of the row type; a lane takes a unit of the first half and its partner of the second, so that
// the rotation needs no other lane and the norm is one shuffle reduction over the lanes of the head (a power of two of them, some
// idle where the head has an odd number of units). Sums and products are in 32 bits, and a word is rounded once, at its store.
#pragma once
#include "paged.cuh"

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
};

template <typename T>
struct Unit; // 16 bytes of a row
template <>
struct Unit<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(float *x, const float *p) {
        const float4 w = *reinterpret_cast<const float4 *>(p);
        x[0] = w.x, x[1] = w.y, x[2] = w.z, x[3] = w.w;
    }
    static __device__ __forceinline__ void store(float *p, const float *x) { *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *x) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
        *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<const unsigned *>(&a), *reinterpret_cast<const unsigned *>(&b));
    }
};
template <>
struct Unit<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void load(float *x, const __nv_bfloat16 *p) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p);
        const unsigned v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float *x) {
        unsigned v[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            v[i] = *reinterpret_cast<const unsigned *>(&a);
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

// blockIdx.x: the row, blockIdx.y: a block of its heads; `lanes` of a warp (a power of two) to a head.
template <typename RT, typename CT>
__global__ void __launch_bounds__(256) append_units_kernel(const AppendCall a, int lanes_log2) {
    constexpr int N = Unit<RT>::N;
    const long long t = blockIdx.x;
    const int b = paged_row_seq(a.c, t);
    if (b < 0) return; // a row of no sequence: nothing is written for it
    const PagedSeq s = paged_seq(a.c, b);
    const int pos = s.pos0 + (int)(t - s.first);
    const int unit = blockIdx.y * 256 + threadIdx.x, lane = unit & ((1 << lanes_log2) - 1);
    int head = unit >> lanes_log2;
    const int part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2); // q, k, v
    const bool any = head < a.c.heads + 2 * a.c.kv;
    head -= part == 0 ? 0 : (part == 1 ? a.c.heads : a.c.heads + a.c.kv);
    const RT *src = part == 0 ? static_cast<const RT *>(a.q) + t * a.ldq : (part == 1 ? static_cast<const RT *>(a.k) + t * a.ldk : static_cast<const RT *>(a.v) + t * a.ldv);
    src += (long long)head * a.c.hd;

    // unit pairs of the rotated columns come first, pairs of neighbouring units of the others after them
    const int half = a.rope_dim / 2, pairs = half / N, rest = (a.c.hd - a.rope_dim) / N;
    const bool turned = lane < pairs;
    const int at0 = turned ? lane * N : a.rope_dim + (lane - pairs) * 2 * N, at1 = turned ? at0 + half : at0 + N;
    const bool has0 = any && lane < pairs + (rest + 1) / 2, has1 = has0 && (turned || (lane - pairs) * 2 + 1 < rest);
    float x0[N], x1[N];
#pragma unroll
    for (int i = 0; i < N; i++) x0[i] = x1[i] = 0.0f;
    if (has0) Unit<RT>::load(x0, src + at0);
    if (has1) Unit<RT>::load(x1, src + at1);

    const float *w = part == 0 ? a.q_norm : (part == 1 ? a.k_norm : nullptr);
    if (a.q_norm || a.k_norm) { // uniform over the grid: the reduction is a warp's
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) sum = fmaf(x0[i], x0[i], fmaf(x1[i], x1[i], sum));
        for (int o = (1 << lanes_log2) >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        if (w) {
            const float r = 1.0f / sqrtf(sum / (float)a.c.hd + a.eps);
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (has0) x0[i] = x0[i] * r * (w[at0 + i] + a.norm_shift);
                if (has1) x1[i] = x1[i] * r * (w[at1 + i] + a.norm_shift);
            }
        }
    }
    if (turned && part < 2 && a.cosv && any) {
        const long long row = (long long)min(max(pos, 0), a.positions - 1) * half + at0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float c = __ldg(a.cosv + row + i), sn = __ldg(a.sinv + row + i), u = x0[i], v = x1[i];
            x0[i] = fmaf(u, c, -(v * sn));
            x1[i] = fmaf(v, c, u * sn);
        }
    }
    RT *dst_row;
    CT *dst_cache;
    if (!has0 || !append_place<RT, CT>(a, t, b, pos, part, head, &dst_row, &dst_cache)) return;
    if (dst_row) {
        Unit<RT>::store(dst_row + at0, x0);
        if (has1) Unit<RT>::store(dst_row + at1, x1);
    } else {
        Unit<RT>::store(dst_cache + at0, x0);
        if (has1) Unit<RT>::store(dst_cache + at1, x1);
    }
}

// Rotations whose halves are not whole units (a partial rotation of few columns): a warp a head, a column a lane.
template <typename RT, typename CT>
__global__ void __launch_bounds__(256) append_columns_kernel(const AppendCall a) {
    const long long t = blockIdx.x;
    const int lane = threadIdx.x & 31, b = paged_row_seq(a.c, t);
    int head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (b < 0 || head >= a.c.heads + 2 * a.c.kv) return;
    const PagedSeq s = paged_seq(a.c, b);
    const int pos = s.pos0 + (int)(t - s.first), part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2);
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
    const long long row = (long long)min(max(pos, 0), a.positions - 1) * half;
    for (int i = lane; i < a.c.hd; i += 32) {
        float x = paged_read(src + i);
        if (w) x = x * r * (w[i] + a.norm_shift);
        if (part < 2 && a.cosv && i < a.rope_dim) {
            const int j = i < half ? i : i - half, p = i < half ? i + half : i - half;
            float y = paged_read(src + p);
            if (w) y = y * r * (w[p] + a.norm_shift);
            const float c = a.cosv[row + j], sn = a.sinv[row + j];
            x = i < half ? fmaf(x, c, -(y * sn)) : fmaf(x, c, y * sn);
        }
        if (dst_row)
            paged_write(dst_row + i, x);
        else
            paged_write(dst_cache + i, x);
    }
}

template <typename RT, typename CT>
cudaError_t launch_append(const AppendCall &a, cudaStream_t st) {
    constexpr int N = Unit<RT>::N;
    const int parts = a.c.heads + 2 * a.c.kv;
    if ((a.rope_dim / 2) % N == 0 && (a.c.hd - a.rope_dim) % N == 0) {
        const int need = a.rope_dim / 2 / N + ((a.c.hd - a.rope_dim) / N + 1) / 2;
        int lg = 0;
        while ((1 << lg) < need) lg++;
        const long long units = (long long)parts << lg;
        append_units_kernel<RT, CT><<<dim3((unsigned)a.c.rows, (unsigned)((units + 255) / 256)), 256, 0, st>>>(a, lg);
    } else {
        append_columns_kernel<RT, CT><<<dim3((unsigned)a.c.rows, (unsigned)((parts + 7) / 8)), 256, 0, st>>>(a);
    }
    return cudaGetLastError();
}

} // namespace b200i

// Fresh q | k | v rows into their places in a cache of 4 bits (paged_int4.cuh): norms, rotation and the queries as in paged_append.cuh, keys and values as codes.
//
// A code is what the definition says of the 64-bit value of its key. The kernel's 32-bit value is off by less than 2^-20 of the two words that the rotation makes
// it of (the norm's sum, root and products: 2^-21.4; the rotation's: 2^-23), so where the largest magnitude of a group, or a word, is nearer than that to a border between
// two scales or codes (about one group in 5000), the warp's keys are done again in 64 bits. Values, and keys without norm and rotation, have no such error: what a
// code leaves is computed exactly.
// Bound: HBM, and latency for a few rows. A lane takes four columns, eight lanes a group: its largest magnitude is three steps across lanes, and the partner of a rotated
// column is in the lane half a rotation away. Rotations whose halves are not whole lanes, and tables that are not on 16-byte boundaries, go by a warp a head with a column of
// each group a lane, keys and values in 64 bits.
#pragma once
#include "paged_append.cuh"
#include "paged_int4.cuh"

namespace b200i {

struct Append4Call {
    AppendCall a;
    double eps;
};

// Where the codes and scales of a row's position are, of key head 0, and what a key head is further on.
struct Append4Place {
    long long codes, scales, head;
};
__device__ __forceinline__ bool append4_place(Append4Place *at, const PagedCall &c, int b, int pos) {
    if (pos < 0) return false; // the lengths say that this row was cached before the sequence began
    const int row = paged_cache_row(c, b, 0, pos), groups = int4_groups(c.hd), in = pos & ((1 << c.page_shift) - 1);
    if (row < 0) return false;
    at->head = (long long)(INT4_BYTES * groups) << c.page_shift;
    const long long page = (long long)(row >> c.page_shift) * at->head;
    at->codes = page + in * 16 * groups, at->scales = page + ((16 * groups) << c.page_shift) + in * 2 * groups;
    return true;
}

template <typename T> struct Four4; // four columns of a row
template <> struct Four4<float> {
    using Raw = float4;
    static __device__ __forceinline__ float4 words(const Raw &r) { return r; }
    static __device__ __forceinline__ void store(float *p, const float (&x)[4]) { *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]); }
};
template <> struct Four4<__nv_bfloat16> {
    using Raw = uint2;
    static __device__ __forceinline__ float4 words(const Raw &r) { return PagedWords<__nv_bfloat16>::words(r); }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&x)[4]) { *reinterpret_cast<uint2 *>(p) = make_uint2(pg_pack(x[0], x[1]), pg_pack(x[2], x[3])); }
};

// Codes and scale of the lane's four columns by the 64-bit words of its key. All lanes; `lanes` of them a head.
struct Append4Exact {
    float x[4], w[4], c[4], sn[4];
    float shift;
    int lanes, from, sign; // the partner's lane, and whether the lane's columns are the rotation's first half (-1), its second (1) or none (0)
    bool normed;
    double eps;
    int hd;
};
struct Append4Codes {
    float n[4], scale;
};
static __device__ __noinline__ Append4Codes append4_exact(const Append4Exact &e) {
    double x[4], y[4];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = e.x[i], sum = fma(x[i], x[i], sum);
    if (e.normed) {
        for (int o = e.lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        const double r = sqrt(sum / (double)e.hd + e.eps);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = x[i] / r * ((double)e.w[i] + (double)e.shift);
    }
    double most = 0.0;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const double other = __shfl_sync(0xFFFFFFFFu, x[i], e.from);
        y[i] = e.sign == 0 ? x[i] : fma(x[i], (double)e.c[i], (double)e.sign * (other * (double)e.sn[i]));
        odd |= !(fabs(y[i]) <= 3.4e38);
        most = fmax(most, fabs(y[i]));
    }
    if (odd) most = INFINITY;
    for (int o = 1; o < 8; o <<= 1) most = fmax(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
    Append4Codes r;
    r.scale = int4_scale(most);
#pragma unroll
    for (int i = 0; i < 4; i++) r.n[i] = r.scale == r.scale ? int4_code(y[i], r.scale) : 0.0f;
    return r;
}

// blockIdx.x: the row; its heads in sets of 32 >> lanes_log2, a set a warp, by steps of the warps of gridDim.y blocks.
template <typename RT>
__global__ void __launch_bounds__(128) append_int4_kernel(const Append4Call f, int lanes_log2, int sets) {
    using W = Four4<RT>;
    const AppendCall &a = f.a;
    const long long t = blockIdx.x;
    const int all = threadIdx.x & 31, lane = all & ((1 << lanes_log2) - 1), in_set = all >> lanes_log2, col = 4 * lane;
    const bool some = col < a.c.hd;
    const int half = a.rope_dim / 2, parts = a.c.heads + 2 * a.c.kv;
    const RT *const q = static_cast<const RT *>(a.q) + t * a.ldq, *const k = static_cast<const RT *>(a.k) + t * a.ldk, *const v = static_cast<const RT *>(a.v) + t * a.ldv;
    typename W::Raw raw;
    const auto ask = [&](int set) {
        const int head = (set << (5 - lanes_log2)) + in_set;
        const RT *src = head < a.c.heads ? q + head * a.c.hd : (head < a.c.heads + a.c.kv ? k + (head - a.c.heads) * a.c.hd : v + (head - a.c.heads - a.c.kv) * a.c.hd);
        raw = {};
        if (head < parts && some) raw = __ldg(reinterpret_cast<const typename W::Raw *>(src + col));
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
    Append4Place place;
    const bool placed = append4_place(&place, a.c, b, pos);
    // The rotation: y = x c -+ other s, the other word being half a rotation of columns away.
    const bool turns = a.cosv != nullptr && col < a.rope_dim;
    const int sign = !turns ? 0 : (col < half ? -1 : 1), from = !turns ? all : (col < half ? all + half / 4 : all - half / 4);
    float4 c = make_float4(1.0f, 1.0f, 1.0f, 1.0f), sn = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (turns) {
        const long long row = (long long)max(pos, 0) * half + (col < half ? col : col - half);
        c = __ldg(reinterpret_cast<const float4 *>(a.cosv + row)), sn = __ldg(reinterpret_cast<const float4 *>(a.sinv + row));
    }
    for (; set < sets; set += step) {
        const int head = (set << (5 - lanes_log2)) + in_set, part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2); // q, k, v
        const float4 r4 = W::words(raw);
        float x[4] = {r4.x, r4.y, r4.z, r4.w}, y[4];
        if (set + step < sets) ask(set + step);
        Append4Exact e;
#pragma unroll
        for (int i = 0; i < 4; i++) e.x[i] = x[i], e.w[i] = 0.0f;
        const float *w = part == 0 ? a.q_norm : (part == 1 ? a.k_norm : nullptr);
        if (a.q_norm || a.k_norm) { // uniform over the grid: the reduction is a warp's
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; i++) sum = fmaf(x[i], x[i], sum);
            for (int o = (1 << lanes_log2) >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (w && some) {
                const float r = rsqrtf(fmaf(sum, a.part_of_head, a.eps));
                const float4 w4 = __ldg(reinterpret_cast<const float4 *>(w + col));
                e.w[0] = w4.x, e.w[1] = w4.y, e.w[2] = w4.z, e.w[3] = w4.w;
#pragma unroll
                for (int i = 0; i < 4; i++) x[i] *= (e.w[i] + a.norm_shift) * r;
            }
        }
        const bool turned = part < 2 && sign != 0;
        const float cs[4] = {c.x, c.y, c.z, c.w}, sns[4] = {sn.x, sn.y, sn.z, sn.w};
        float off[4]; // how far a word may be from its 64-bit value
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float other = __shfl_sync(0xFFFFFFFFu, x[i], from);
            y[i] = turned ? fmaf(x[i], cs[i], sign < 0 ? -(other * sns[i]) : other * sns[i]) : x[i];
            off[i] = part == 1 && (w || turned) ? 0x1p-20f * (fabsf(x[i]) + (turned ? fabsf(other) : 0.0f)) : 0.0f;
        }
        if (part == 0 && some) W::store(static_cast<RT *>(a.q_out) + (t * a.c.heads + head) * a.c.hd + col, y);
        if (!__any_sync(0xFFFFFFFFu, part > 0)) continue;
        // ---- the codes ----
        unsigned most = 0;
        float most_off = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) most = max(most, __float_as_uint(y[i]) & 0x7FFFFFFFu), most_off = fmaxf(most_off, off[i]); // (a NaN's bits are larger than an infinity's)
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            most = max(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
            most_off = fmaxf(most_off, __shfl_xor_sync(0xFFFFFFFFu, most_off, o));
        }
        Append4Codes n;
        n.scale = int4_scale(__uint_as_float(most));
        const float before = __uint_as_float(__float_as_uint(n.scale) - 0x80000u), inverse = 1.0f / n.scale;
        bool near = most_off > 0.0f && (7.0f * n.scale - __uint_as_float(most) <= most_off || __uint_as_float(most) - 7.0f * before <= most_off);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float left;
            n.n[i] = int4_code(y[i], n.scale, inverse, &left);
            near |= off[i] > 0.0f && fabsf(fabsf(left) - 0.5f * n.scale) <= off[i];
        }
        if (most >= 0x7F800000u) n.n[0] = n.n[1] = n.n[2] = n.n[3] = 0.0f, near = false;
        if (__any_sync(0xFFFFFFFFu, near)) {
#pragma unroll
            for (int i = 0; i < 4; i++) e.c[i] = cs[i], e.sn[i] = sns[i];
            e.shift = a.norm_shift, e.lanes = 1 << lanes_log2, e.from = from, e.sign = turned ? sign : 0, e.normed = a.k_norm != nullptr, e.eps = f.eps, e.hd = a.c.hd;
            const Append4Codes exact = append4_exact(e);
            if (part == 1) n = exact; // (of values nothing is normed)
        }
        // a lane has the first or the last four of a word's eight columns
        const unsigned shift = (lane & 1) * 8;
        unsigned word = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) word |= (unsigned)((int)n.n[i] + 8) << (shift + 4 * (i >> 1) + 16 * (i & 1));
        word |= __shfl_xor_sync(0xFFFFFFFFu, word, 1);
        if (part == 0 || head >= parts || !placed || lane >= 8 * int4_groups(a.c.hd)) continue;
        unsigned char *const cache = static_cast<unsigned char *>(part == 1 ? a.k_cache : a.v_cache) + place.head * (head - a.c.heads - (part == 1 ? 0 : a.c.kv));
        if ((lane & 1) == 0) *reinterpret_cast<unsigned *>(cache + place.codes + 2 * lane) = word;
        if ((lane & 7) == 0) *reinterpret_cast<unsigned short *>(cache + place.scales + 2 * (lane >> 3)) = (unsigned short)(__float_as_uint(n.scale) >> 16);
    }
}

// Any rotation: a warp a head, lane i the columns i, i + 32, ...: group by group.
template <typename RT>
__global__ void __launch_bounds__(256) append_int4_columns_kernel(const Append4Call f) {
    const AppendCall &a = f.a;
    const long long t = blockIdx.x;
    const int lane = threadIdx.x & 31, b = paged_row_seq(a.c, t);
    int head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (b < 0 || head >= a.c.heads + 2 * a.c.kv) return;
    const PagedSeq s = paged_seq_checked(a.c, b);
    if (s.n == 0) return; // its tables do not hold it
    const int pos = s.pos0 + (int)(t - s.first), part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2);
    if (append_past(a, pos)) return;
    head -= part == 0 ? 0 : (part == 1 ? a.c.heads : a.c.heads + a.c.kv);
    Append4Place place;
    if (part > 0 && !append4_place(&place, a.c, b, pos)) return;
    const RT *src = part == 0 ? static_cast<const RT *>(a.q) + t * a.ldq : (part == 1 ? static_cast<const RT *>(a.k) + t * a.ldk : static_cast<const RT *>(a.v) + t * a.ldv);
    src += (long long)head * a.c.hd;
    const float *w = part == 0 ? a.q_norm : (part == 1 ? a.k_norm : nullptr);
    double root = 1.0;
    if (w) {
        double sum = 0.0;
        for (int i = lane; i < a.c.hd; i += 32) {
            const double x = paged_read(src + i);
            sum = fma(x, x, sum);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        root = sqrt(sum / (double)a.c.hd + f.eps);
    }
    const int half = a.rope_dim / 2;
    const long long row = (long long)max(pos, 0) * half;
    const auto word = [&](int i) { return w ? (double)paged_read(src + i) / root * ((double)w[i] + (double)a.norm_shift) : (double)paged_read(src + i); };
    double out[PAGED_MAX_HD / 32];
#pragma unroll
    for (int k = 0; k < PAGED_MAX_HD / 32; k++) {
        const int i = lane + 32 * k;
        out[k] = 0.0;
        if (i >= a.c.hd) continue;
        out[k] = word(i);
        if (part < 2 && a.cosv && i < a.rope_dim) {
            const int j = i < half ? i : i - half;
            const double other = word(i < half ? i + half : i - half), c = a.cosv[row + j], sn = a.sinv[row + j];
            out[k] = i < half ? fma(out[k], c, -(other * sn)) : fma(out[k], c, other * sn);
        }
    }
    __syncwarp(); // all is read before any of it is written: the queries may be rotated in their place
    unsigned char *const cache = static_cast<unsigned char *>(part == 1 ? a.k_cache : a.v_cache) + (part > 0 ? place.head * head : 0);
#pragma unroll
    for (int k = 0; k < PAGED_MAX_HD / 32; k++) {
        if (32 * k >= a.c.hd) break;
        const int i = lane + 32 * k;
        if (part == 0) {
            if (i < a.c.hd) paged_write(static_cast<RT *>(a.q_out) + (t * a.c.heads + head) * a.c.hd + i, (float)out[k]);
            continue;
        }
        double most = fabs(out[k]) <= 3.4e38 ? fabs(out[k]) : INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmax(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
        const float scale = int4_scale(most);
        const unsigned n = (unsigned)((int)(scale == scale ? int4_code(out[k], scale) : 0.0f) + 8);
        unsigned word4 = n << (4 * ((lane & 7) >> 1) + 16 * (lane & 1));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) word4 |= __shfl_xor_sync(0xFFFFFFFFu, word4, o);
        if ((lane & 7) == 0) *reinterpret_cast<unsigned *>(cache + place.codes + 16 * k + lane / 2) = word4;
        if (lane == 0) *reinterpret_cast<unsigned short *>(cache + place.scales + 2 * k) = (unsigned short)(__float_as_uint(scale) >> 16);
    }
}

template <typename RT>
cudaError_t launch_append4(const AppendCall &a, double eps, int sms, cudaStream_t st) {
    const Append4Call f = {a, eps};
    const int parts = a.c.heads + 2 * a.c.kv, groups = int4_groups(a.c.hd);
    const uintptr_t words = reinterpret_cast<uintptr_t>(a.cosv) | reinterpret_cast<uintptr_t>(a.sinv) | reinterpret_cast<uintptr_t>(a.q_norm) | reinterpret_cast<uintptr_t>(a.k_norm);
    if ((a.rope_dim / 2) % 4 == 0 && words % 16 == 0) {
        const int lg = groups == 1 ? 3 : (groups == 2 ? 4 : 5), per_set = 32 >> lg, sets = (parts + per_set - 1) / per_set, blocks = (sets + 3) / 4;
        const int y = (int)std::max<long long>(1, std::min<long long>(blocks, 8LL * sms / a.c.rows)); // as in launch_append
        append_int4_kernel<RT><<<dim3((unsigned)a.c.rows, (unsigned)y), 128, 0, st>>>(f, lg, sets);
    } else {
        append_int4_columns_kernel<RT><<<dim3((unsigned)a.c.rows, (unsigned)((parts + 7) / 8)), 256, 0, st>>>(f);
    }
    return cudaGetLastError();
}

} // namespace b200i

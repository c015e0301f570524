// What the kernels of the paged cache share: the arguments of a call, where a position lives, and the plain walk of one row.
//
// A cache is [pages, n_kv, page, head_dim] (keys and values apart), `page` a power of two; page_table [batch, max_pages] names
// the pages of each sequence in the order of its positions. A call's rows are those of all sequences one after another:
// sequence b's are cu[b] .. cu[b + 1], and lengths[b] counts what its cache holds with them, so that its row i is at
// position lengths[b] - n + i. All three arrays live on the device and are read there; what they say is bounded by the
// extents of the tensors before it is used as an index, so that no table makes a kernel read or write outside of them: a page
// number outside the pool reads as zeros, is not written, and sets the library's status word to PAGED_BAD_PAGE; a sequence whose length
// its page table has no room for, or whose row offsets are not the call's, is left out and sets it to PAGED_BAD_TABLE.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "paged_place.cuh"

namespace b200i {

constexpr int PAGED_MAX_HD = 128;
constexpr int PAGED_BAD_PAGE = 11; // the status word: a page number outside the pool
constexpr int PAGED_BAD_BOUND = 12; // the status word: more new tokens in a sequence than the call's bound
constexpr int PAGED_BAD_TABLE = 14; // the status word: a length past the page table, or row offsets that are not the call's
constexpr int PAGED_BAD_POSITION = 15; // the status word: a position past the rotation's table
constexpr float PAGED_LOG2E = 1.4426950408889634f;

struct PagedCall {
    const int *table, *cu, *lengths;
    int *status;
    long long rows;        // of q: the extent cu is held to
    int batch, heads, kv, group, hd;
    int pages, page_shift, max_pages;
    unsigned group_part;   // 2^32 / group + 1, rounded down: the upper half of a product with it is a quotient
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedCall &c, int b) { return paged_place(c.cu[b], c.cu[b + 1], c.lengths[b], (int)c.rows, c.max_pages << c.page_shift); }

// The same, and the status word where the tables do not hold the sequence: each kernel looks at every sequence once in this way.
__device__ __forceinline__ PagedSeq paged_seq_checked(const PagedCall &c, int b) {
    const int lo = c.cu[b], hi = c.cu[b + 1], length = c.lengths[b], capacity = c.max_pages << c.page_shift;
    if (!paged_holds(lo, hi, length, (int)c.rows, capacity)) atomicExch(c.status, PAGED_BAD_TABLE);
    return paged_place(lo, hi, length, (int)c.rows, capacity);
}

// The sequence of row t, or -1: a warp looks at 32 entries of cu at a time. All lanes call it with one t.
__device__ __forceinline__ int paged_row_seq(const PagedCall &c, long long t) {
    const int lane = threadIdx.x & 31;
    for (int b0 = 0; b0 < c.batch; b0 += 32) {
        const int b = b0 + lane;
        const unsigned here = __ballot_sync(0xFFFFFFFFu, b < c.batch && t < (long long)c.cu[b + 1]);
        if (here) {
            const int found = b0 + __ffs(here) - 1;
            return t >= (long long)c.cu[found] ? found : -1;
        }
    }
    return -1;
}

// The row (of head_dim) of position `pos` of sequence b and head h in a cache, or -1 (and the status word) for a bad page.
__device__ __forceinline__ int paged_cache_row(const PagedCall &c, int b, int h, int pos) {
    const int id = c.table[(long long)b * c.max_pages + (pos >> c.page_shift)];
    if ((unsigned)id >= (unsigned)c.pages) {
        atomicExch(c.status, PAGED_BAD_PAGE);
        return -1;
    }
    return ((id * c.kv + h) << c.page_shift) + (pos & ((1 << c.page_shift) - 1));
}
// The same as an element.
__device__ __forceinline__ long long paged_offset(const PagedCall &c, int b, int h, int pos) {
    const int row = paged_cache_row(c, b, h, pos);
    return row < 0 ? -1 : (long long)row * c.hd;
}

__device__ __forceinline__ float paged_read(const float *p) { return *p; }
__device__ __forceinline__ float paged_read(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void paged_write(float *p, float v) { *p = v; }
__device__ __forceinline__ void paged_write(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float paged_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float paged_warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}

struct AttendCall {
    PagedCall c;
    const void *q, *k, *v;
    void *out;
    long long ldq;  // elements between rows of q
    float scale, softcap;  // scale > 0: a negative one is the queries' sign (flip)
    float cap_part;        // 1 / softcap
    int flip;
    float cap_inner, cap_outer, cap_near[4]; // of capped scores (paged_many.cuh): scale / softcap and its inverse, both within 32 bits; the polynomial's coefficients
    int cap_far;                             // 0: with the even powers of cap_inner in them
    int window;     // 0: none
    int max_new;    // a sequence's rows past these are not computed
};

// What an output's sum is multiplied by, l the sum of its weights: zero where the row, at position pos, sees nothing (a row that sees
// anything sees itself); NaN where all that it sees are scores of -infinity.
__device__ __forceinline__ float paged_share(float l, int pos) { return l != 0.0f ? 1.0f / l : (pos < 0 ? 0.0f : NAN); }

// Eight words of a row on a 16-byte boundary, and four on one of 8 or 16 bytes, as they are asked for and as 32-bit words.
template <typename T> struct PagedWords;
template <> struct PagedWords<float> {
    struct Eight { float4 lo, hi; };
    using Four = float4;
    static __device__ __forceinline__ Eight eight(const float *p) { return {*reinterpret_cast<const float4 *>(p), *reinterpret_cast<const float4 *>(p + 4)}; }
    static __device__ __forceinline__ Four four(const float *p) { return *reinterpret_cast<const float4 *>(p); }
    static __device__ __forceinline__ float4 lower(const Eight &x) { return x.lo; }
    static __device__ __forceinline__ float4 upper(const Eight &x) { return x.hi; }
    static __device__ __forceinline__ float4 words(const Four &x) { return x; }
};
template <> struct PagedWords<__nv_bfloat16> {
    using Eight = uint4;
    using Four = uint2;
    static __device__ __forceinline__ Eight eight(const __nv_bfloat16 *p) { return *reinterpret_cast<const uint4 *>(p); }
    static __device__ __forceinline__ Four four(const __nv_bfloat16 *p) { return *reinterpret_cast<const uint2 *>(p); }
    static __device__ __forceinline__ float4 two(unsigned x, unsigned y) { return make_float4(__uint_as_float(x << 16), __uint_as_float(x & 0xFFFF0000u), __uint_as_float(y << 16), __uint_as_float(y & 0xFFFF0000u)); }
    static __device__ __forceinline__ float4 lower(const Eight &x) { return two(x.x, x.y); }
    static __device__ __forceinline__ float4 upper(const Eight &x) { return two(x.z, x.w); }
    static __device__ __forceinline__ float4 words(const Four &x) { return two(x.x, x.y); }
};
__device__ __forceinline__ float paged_dot(const float4 &x, const float4 &y, float z) { return fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, fmaf(x.x, y.x, z)))); }

// A (row, head) over some of its keys: the largest score (-infinity: none), the weights' sum and four columns of the weighted sum of values,
// from 4 * lane on.
struct RowSums {
    float m, l, o[4];
};

// softmax(z) . V of one (row, head) by one warp, over the positions begin .. end - 1: z = scale * q.k, capped to softcap * tanh(z / softcap).
// A key that the row does not see is not read at all, so nothing that stands there (an infinity, a NaN) can reach the row.
// Every other path comes here with a row that did not come out finite: a masked key has weight zero there, but is multiplied.
// Bound: latency, and L2 where many rows are here (each reads its keys for itself). 32 keys at a time: eight lanes have a key's columns between them,
// eight rounds of four keys, and the rounds' sums are added up across the lanes so that each is left with one key; of the values a lane has four columns
// of each key. A score that is NaN or infinite ends it, since all of the row is NaN then. Few registers, since the kernels that call this
// have theirs counted with it. Measured, one NaN among the values: 32 rows of 131000 keys 6 ms (95 us without it), 16384 rows of 16000 to 16511 30 ms
// (178 us); a warp a key, with a trip to memory and a reduction for each, had taken 230 and 121.
template <typename RT, typename CT>
__device__ __noinline__ RowSums attend_keys_plain(const AttendCall &a, int b, int row, int h, int begin, int end) {
    using QW = PagedWords<RT>;
    using W = PagedWords<CT>;
    constexpr int ASK = sizeof(CT) == 2 ? 4 : 2, ASK_V = 2 * ASK; // keys a lane asks for at once
    // What the loop needs of the arguments is read before it: they are behind an address here, and read again after every store that might be to them.
    const PagedCall c = a.c;
    const CT *const keys = static_cast<const CT *>(a.k), *const values = static_cast<const CT *>(a.v);
    const float scale = a.flip ? -a.scale : a.scale, softcap = a.softcap;
    const int lane = threadIdx.x & 31, part = lane & 7, hd = c.hd, kvh = h / c.group, c0 = 4 * lane;
    const RT *q = static_cast<const RT *>(a.q) + (long long)row * a.ldq + (long long)h * hd;
    const auto place = [&](int j) { return j < end ? paged_cache_row(c, b, kvh, j) : -1; };
    RowSums r = {-INFINITY, 0.0f, {0.0f, 0.0f, 0.0f, 0.0f}};
    int next = place(begin + lane);
#pragma unroll 1
    for (int j0 = begin; j0 < end; j0 += 32) {
        const int here = min(32, end - j0), at = next;
        next = place(j0 + 32 + lane);
        float sums[8] = {};
#pragma unroll 1
        for (int col = 8 * part; col - 8 * part < hd; col += 64) { // alike in all lanes
            typename QW::Eight x = {};
            if (col < hd) x = QW::eight(q + col);
#pragma unroll
            for (int i0 = 0; i0 < 8; i0 += ASK) {
                typename W::Eight y[ASK];
#pragma unroll
                for (int i = 0; i < ASK; i++) {
                    const int key = __shfl_sync(0xFFFFFFFFu, at, 4 * (i0 + i) + (lane >> 3));
                    y[i] = {};
                    if (key >= 0 && col < hd) y[i] = W::eight(keys + (long long)key * hd + col);
                }
#pragma unroll
                for (int i = 0; i < ASK; i++) sums[i0 + i] = paged_dot(QW::upper(x), W::upper(y[i]), paged_dot(QW::lower(x), W::lower(y[i]), sums[i0 + i]));
            }
        }
#pragma unroll
        for (int w = 4; w > 0; w >>= 1) { // a lane keeps the rounds whose number has its own bit, and gives the others away
#pragma unroll
            for (int i = 0; i < w; i++) {
                const bool upper = part & w;
                const float give = upper ? sums[i] : sums[i + w], mine = upper ? sums[i + w] : sums[i];
                sums[i] = mine + __shfl_xor_sync(0xFFFFFFFFu, give, w);
            }
        }
        float z = sums[0] * scale;
        if (softcap > 0.0f) z = softcap * tanhf(z / softcap);
        if (4 * part + (lane >> 3) >= here) z = -INFINITY; // the lane's key
        if (__any_sync(0xFFFFFFFFu, !(z < INFINITY))) return {0.0f, NAN, {NAN, NAN, NAN, NAN}};
        float top = z;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const float m2 = fmaxf(r.m, top), base = m2 == -INFINITY ? 0.0f : m2;
        const float keep = r.m == -INFINITY ? 0.0f : paged_exp2((r.m - base) * PAGED_LOG2E), w = paged_exp2((z - base) * PAGED_LOG2E);
        r.m = m2, r.l = fmaf(r.l, keep, paged_warp_sum(w));
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
        for (int k0 = 0; k0 < here; k0 += ASK_V) {
            typename W::Four v[ASK_V]; // a key past the end has no place and no weight
#pragma unroll
            for (int k = 0; k < ASK_V; k++) {
                const int key = __shfl_sync(0xFFFFFFFFu, at, k0 + k);
                v[k] = {};
                if (key >= 0 && c0 < hd) v[k] = W::four(values + (long long)key * hd + c0);
            }
#pragma unroll
            for (int k = 0; k < ASK_V; k++) {
                const float wk = __shfl_sync(0xFFFFFFFFu, w, ((k0 + k) >> 2) | ((k0 + k) & 3) << 3);
                const float4 y = W::words(v[k]);
                sum.x = fmaf(wk, y.x, sum.x), sum.y = fmaf(wk, y.y, sum.y), sum.z = fmaf(wk, y.z, sum.z), sum.w = fmaf(wk, y.w, sum.w);
            }
        }
        r.o[0] = fmaf(r.o[0], keep, sum.x), r.o[1] = fmaf(r.o[1], keep, sum.y), r.o[2] = fmaf(r.o[2], keep, sum.z), r.o[3] = fmaf(r.o[3], keep, sum.w);
    }
    return r;
}
// The positions that a row at `pos` sees.
__device__ __forceinline__ int attend_begin(const AttendCall &a, int pos) { return a.window ? max(0, pos - a.window + 1) : 0; }
__device__ __forceinline__ int attend_end(int pos, int length) { return min(pos + 1, length); }

// Rows that see nothing are zero; scores that are all -infinity have no softmax: NaN.
template <typename RT, typename CT>
__device__ __noinline__ void attend_row_plain(const AttendCall &a, int b, int row, int pos, int length, int h) {
    const RowSums r = attend_keys_plain<RT, CT>(a, b, row, h, attend_begin(a, pos), attend_end(pos, length));
    RT *out = static_cast<RT *>(a.out) + ((long long)row * a.c.heads + h) * a.c.hd;
    const int c0 = 4 * (threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (c0 + i < a.c.hd) paged_write(out + c0 + i, r.l != 0.0f ? r.o[i] / r.l : paged_share(r.l, pos));
}

} // namespace b200i

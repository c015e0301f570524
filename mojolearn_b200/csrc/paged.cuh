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

// The first element of position `pos` of sequence b and head h in a cache, or -1 (and the status word) for a bad page.
__device__ __forceinline__ long long paged_offset(const PagedCall &c, int b, int h, int pos) {
    const int id = c.table[(long long)b * c.max_pages + (pos >> c.page_shift)];
    if ((unsigned)id >= (unsigned)c.pages) {
        atomicExch(c.status, PAGED_BAD_PAGE);
        return -1;
    }
    return ((((long long)id * c.kv + h) << c.page_shift) + (pos & ((1 << c.page_shift) - 1))) * c.hd;
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

// softmax(z) . V of one (row, head) by one warp, key by key: z = scale * q.k, capped to softcap * tanh(z / softcap).
// Rows that see nothing are zero; scores that are all -infinity have no softmax: NaN.
// A key that the row does not see is not read at all, so nothing that stands there (an infinity, a NaN) can reach the row.
// Every other path comes here with a row that did not come out finite: a masked key has weight zero there, but is multiplied.
template <typename RT, typename CT>
__device__ __noinline__ void attend_row_plain(const AttendCall &a, int b, int row, int pos, int length, int h) {
    const int lane = threadIdx.x & 31, hd = a.c.hd, kvh = h / a.c.group;
    const RT *q = static_cast<const RT *>(a.q) + (long long)row * a.ldq + (long long)h * hd;
    float qv[PAGED_MAX_HD / 32], acc[PAGED_MAX_HD / 32], part[PAGED_MAX_HD / 32]; // part: of the last up to 64 keys, so that long sums stay exact enough
#pragma unroll
    for (int i = 0; i < PAGED_MAX_HD / 32; i++) {
        qv[i] = lane + 32 * i < hd ? paged_read(q + lane + 32 * i) : 0.0f;
        acc[i] = part[i] = 0.0f;
    }
    const int end = min(pos + 1, length), begin = a.window ? max(0, pos - a.window + 1) : 0;
    float m = -INFINITY, l = 0.0f, lpart = 0.0f;
    for (int j = begin; j < end; j++) {
        const long long at = paged_offset(a.c, b, kvh, j);
        float kx[PAGED_MAX_HD / 32], dot = 0.0f;
#pragma unroll
        for (int i = 0; i < PAGED_MAX_HD / 32; i++) {
            kx[i] = at >= 0 && lane + 32 * i < hd ? paged_read(static_cast<const CT *>(a.k) + at + lane + 32 * i) : 0.0f;
            if (lane + 32 * i < hd) dot = fmaf(qv[i], kx[i], dot);
        }
        float z = paged_warp_sum(a.flip ? -dot : dot) * a.scale;
        if (a.softcap > 0.0f) z = a.softcap * tanhf(z / a.softcap);
        const float m2 = z > m || z != z ? z : m;
        if (m2 == -INFINITY) continue; // a weight of zero
        const float keep = paged_exp2((m - m2) * PAGED_LOG2E), w = paged_exp2((z - m2) * PAGED_LOG2E);
        m = m2;
        const bool full = ((j - begin) & 63) == 63;
        lpart = fmaf(lpart, keep, w);
        l = full ? fmaf(l, keep, lpart) : l * keep;
        if (full) lpart = 0.0f;
#pragma unroll
        for (int i = 0; i < PAGED_MAX_HD / 32; i++) {
            const float vx = at >= 0 && lane + 32 * i < hd ? paged_read(static_cast<const CT *>(a.v) + at + lane + 32 * i) : 0.0f;
            part[i] = fmaf(w, vx, part[i] * keep);
            acc[i] = full ? fmaf(acc[i], keep, part[i]) : acc[i] * keep;
            if (full) part[i] = 0.0f;
        }
    }
    l += lpart;
    RT *out = static_cast<RT *>(a.out) + ((long long)row * a.c.heads + h) * hd;
#pragma unroll
    for (int i = 0; i < PAGED_MAX_HD / 32; i++)
        if (lane + 32 * i < hd) paged_write(out + lane + 32 * i, l != 0.0f ? (acc[i] + part[i]) / l : paged_share(l, pos));
}

} // namespace b200i

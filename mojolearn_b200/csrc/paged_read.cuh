// Rows of a paged cache read back: keys and values of each sequence's rows as one array each.
//
// Bound: HBM, what is held read once and what it stands for written once. A block takes up to 32 rows: the lanes of one warp look up where they are, and a thread
// has a unit of eight columns of a head and takes it of several rows, keys and values alike, whose words are all asked for before the first is stored;
// neighbours write neighbouring bytes.
// 16 sequences of 90 to 4000 positions, 8 heads of 128, 4 bits as bfloat16: 48 us, 4.7 TB/s (55 with one row at a time). 16 of 2000: 43 us, of bfloat16 words 47.5 (5.5 TB/s),
// of float32 ones 91 (5.8). 10 rows of 2000 sequences, most of them without rows, in a call of 4096: 24 us (102 with offsets looked at one by one, row by row where they belong to nobody).
#pragma once
#include <algorithm>

#include "paged_int4.cuh"

namespace b200i {

struct ReadCall {
    PagedCall c;
    const void *k_cache, *v_cache;
    void *k_out, *v_out;
};

constexpr int READ_ROWS = 32, READ_THREADS = 256;

// Eight columns as they are written: what is not float32 is bfloat16 words already, or codes that become them.
__device__ __forceinline__ void read_store(float *p, const PagedWords<float>::Eight &x) { *reinterpret_cast<float4 *>(p) = x.lo, *reinterpret_cast<float4 *>(p + 4) = x.hi; }
__device__ __forceinline__ void read_store(__nv_bfloat16 *p, const uint4 &x) { *reinterpret_cast<uint4 *>(p) = x; }
__device__ __forceinline__ void read_store(float *p, const uint4 &x) {
    using W = PagedWords<__nv_bfloat16>;
    *reinterpret_cast<float4 *>(p) = W::lower(x), *reinterpret_cast<float4 *>(p + 4) = W::upper(x);
}
template <typename OT> __device__ __forceinline__ void read_store(OT *p, const PagedRows<Int4>::Eight &x) {
    unsigned v[4];
    const unsigned s = __float_as_uint(x.scale);
    int4_pairs(v, x.word, int4_factors(s | s >> 16)); // (a bfloat16 word above zeros)
    read_store(p, make_uint4(v[0], v[1], v[2], v[3]));
}

template <typename CT, typename OT>
__global__ void __launch_bounds__(READ_THREADS) read_kernel(const ReadCall a, int rows) {
    constexpr int ASK = 4; // rows that a thread asks for at once
    __shared__ int at[READ_ROWS]; // a row's place in the caches, of key head 0; -1: there is none, and it is zeros; -2: it belongs to no sequence
    const PagedCall &c = a.c;
    const long long t0 = (long long)blockIdx.x * rows;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        const long long t = t0 + lane;
        const bool mine = lane < rows && t < c.rows;
        int b0 = paged_seq_after(c, t0), row = -2;
        int b = b0 < c.batch && t < c.cu[b0 + 1] ? b0 : c.batch; // the first sequence that ends behind the lane's row: the first row's, or one after it
        for (; b0 < c.batch && __any_sync(0xFFFFFFFFu, mine && b == c.batch); b0 += 32) {
            int end = b0 + lane < c.batch ? c.cu[b0 + lane + 1] : -1, before = 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) { // the largest end up to the lane's: these never fall, whatever cu says
                const int lower = __shfl_up_sync(0xFFFFFFFFu, end, o);
                end = max(end, lane >= o ? lower : end);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) before += __shfl_sync(0xFFFFFFFFu, end, before + o - 1) <= t ? o : 0;
            const bool found = __shfl_sync(0xFFFFFFFFu, end, before) > t;
            if (b == c.batch && found) b = b0 + before;
        }
        if (mine && b < c.batch && t >= c.cu[b]) {
            const PagedSeq s = paged_seq_checked(c, b);
            const int pos = s.pos0 + (int)(t - s.first);
            if (s.n > 0) row = pos < 0 ? -1 : paged_cache_row(c, b, 0, pos);
        }
        at[lane] = row;
    }
    __syncthreads();
    const int units = c.kv * c.hd / 8, span = min(units, READ_THREADS), step = READ_THREADS / span, r0 = threadIdx.x / span; // units of a row; a thread's rows are step apart
    if (r0 >= step) return;
    const PagedRows<CT> keys(a.k_cache, c), values(a.v_cache, c);
    for (int u = threadIdx.x - r0 * span; u < units; u += span) {
        const int head = u * 8 / c.hd, col = u * 8 - head * c.hd;
        for (int first = r0; first < rows; first += ASK * step) {
            typename PagedRows<CT>::Eight k[ASK], v[ASK];
            int place[ASK];
#pragma unroll
            for (int i = 0; i < ASK; i++) {
                const int r = first + i * step;
                place[i] = r < rows ? at[r] : -2;
                k[i] = {}, v[i] = {};
                if (place[i] < 0) continue;
                const int of = place[i] + (head << c.page_shift);
                k[i] = keys.eight(of, col), v[i] = values.eight(of, col);
            }
#pragma unroll
            for (int i = 0; i < ASK; i++) {
                if (place[i] == -2) continue;
                const long long to = ((t0 + first + i * step) * c.kv + head) * c.hd + col;
                read_store(static_cast<OT *>(a.k_out) + to, k[i]);
                read_store(static_cast<OT *>(a.v_out) + to, v[i]);
            }
        }
    }
}

template <typename CT, typename OT>
cudaError_t launch_read(const ReadCall &a, int sms, cudaStream_t st) {
    const int rows = (int)std::max<long long>(1, std::min<long long>(READ_ROWS, a.c.rows / (4 * sms))); // with a few rows a block takes fewer
    read_kernel<CT, OT><<<(unsigned)((a.c.rows + rows - 1) / rows), READ_THREADS, 0, st>>>(a, rows);
    return cudaGetLastError();
}

} // namespace b200i

// Rows of a paged cache read back: keys and values of each sequence's rows as one array each.
//
// Bound: HBM, what is held read once and what it stands for written once. A block takes READ_ROWS rows: its warps look up where they are, one each, and its
// threads take units of eight columns of them, keys and values alike, so that neighbours write neighbouring bytes.
#pragma once
#include <algorithm>

#include "paged_int4.cuh"

namespace b200i {

struct ReadCall {
    PagedCall c;
    const void *k_cache, *v_cache;
    void *k_out, *v_out;
};

constexpr int READ_ROWS = 8;

template <typename OT> struct ReadStore;
template <> struct ReadStore<float> {
    static __device__ __forceinline__ void eight(float *p, const float4 &x, const float4 &y) { *reinterpret_cast<float4 *>(p) = x, *reinterpret_cast<float4 *>(p + 4) = y; }
};
template <> struct ReadStore<__nv_bfloat16> {
    static __device__ __forceinline__ void eight(__nv_bfloat16 *p, const float4 &x, const float4 &y) {
        *reinterpret_cast<uint4 *>(p) = make_uint4(pg_pack(x.x, x.y), pg_pack(x.z, x.w), pg_pack(y.x, y.y), pg_pack(y.z, y.w));
    }
};

template <typename CT, typename OT>
__global__ void __launch_bounds__(32 * READ_ROWS) read_kernel(const ReadCall a) {
    __shared__ int at[READ_ROWS]; // a row's place in the caches, of key head 0; -1: there is none, and it is zeros; -2: it belongs to no sequence
    const PagedCall &c = a.c;
    const int warp = threadIdx.x >> 5;
    const long long t0 = (long long)blockIdx.x * READ_ROWS, t = t0 + warp;
    int row = -2;
    if (t < c.rows) {
        const int b = paged_row_seq(c, t);
        if (b >= 0) {
            const PagedSeq s = paged_seq_checked(c, b);
            const int pos = s.pos0 + (int)(t - s.first);
            if (s.n > 0) row = pos < 0 ? -1 : paged_cache_row(c, b, 0, pos);
        }
    }
    if ((threadIdx.x & 31) == 0) at[warp] = row;
    __syncthreads();
    const int units = c.kv * c.hd / 8; // of a row
    const PagedRows<CT> keys(a.k_cache, c), values(a.v_cache, c);
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < READ_ROWS * units; i += gridDim.y * blockDim.x) {
        const int r = i / units, u = i - r * units, head = u * 8 / c.hd, col = u * 8 - head * c.hd, place = at[r];
        if (place == -2) continue;
        typename PagedRows<CT>::Eight k = {}, v = {};
        if (place >= 0) {
            const int of = place + (head << c.page_shift);
            k = keys.eight(of, col), v = values.eight(of, col);
        }
        const long long to = ((t0 + r) * c.kv + head) * c.hd + col;
        ReadStore<OT>::eight(static_cast<OT *>(a.k_out) + to, PagedRows<CT>::lower(k), PagedRows<CT>::upper(k));
        ReadStore<OT>::eight(static_cast<OT *>(a.v_out) + to, PagedRows<CT>::lower(v), PagedRows<CT>::upper(v));
    }
}

template <typename CT, typename OT>
cudaError_t launch_read(const ReadCall &a, int sms, cudaStream_t st) {
    const long long blocks = (a.c.rows + READ_ROWS - 1) / READ_ROWS, each = ((long long)READ_ROWS * a.c.kv * a.c.hd / 8 + 32 * READ_ROWS - 1) / (32 * READ_ROWS);
    const int y = (int)std::max<long long>(1, std::min<long long>(each, 8LL * sms / blocks)); // with a few rows a thread takes one unit
    read_kernel<CT, OT><<<dim3((unsigned)blocks, (unsigned)y), 32 * READ_ROWS, 0, st>>>(a);
    return cudaGetLastError();
}

} // namespace b200i

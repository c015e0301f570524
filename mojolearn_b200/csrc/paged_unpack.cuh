// A cache in 4 bits as one of bfloat16 words, for attention of so many rows that what makes words of codes in it would do so again and again.
//
// The words go to pages of a workspace, in the order of the sequences' positions: page i of sequence b is page b max_pages + i there, and the table says so. A word is the one
// that the codes stand for, so nothing is rounded. Bound: HBM and L2, 4.5 bits read and 16 written a word; pages that no row sees are left as they are.
// 2048 tokens behind 14336, 32 heads on 8 of 128: 560 to 600 us (at the power limit; by the box), some 20 of them here, and 862 with words made in the attention, where each of a key head's 32 blocks of 256
// rows makes them for itself.
#pragma once
#include "paged_int4.cuh"
#include "paged_read.cuh"

namespace b200i {

struct UnpackCall {
    AttendCall a;
    __nv_bfloat16 *k, *v;
    int *table;
    int at_once; // pages of a sequence that the grid has blocks for
};

// blockIdx.x: a page of a sequence, and every at_once-th after it; blockIdx.y: a key head.
static __global__ void __launch_bounds__(READ_THREADS) unpack_kernel(const UnpackCall u) {
    constexpr int ASK = 4; // units that a thread asks for at once
    const PagedCall &c = u.a.c;
    const int b = blockIdx.x / u.at_once, page = 1 << c.page_shift, kvh = blockIdx.y, units = c.hd / 8, all = units * page;
    const PagedSeq s = paged_seq(c, b);
    if (s.n == 0) return;
    const int low = u.a.window ? s.pos0 + 1 - u.a.window : 0; // no row sees what is below
    const PagedRows<Int4> keys(u.a.k, c), values(u.a.v, c);
    for (int i = blockIdx.x - b * u.at_once; i < c.max_pages && i * page < s.length; i += u.at_once) {
        const int at_page = b * c.max_pages + i;
        if (threadIdx.x == 0 && kvh == 0) u.table[at_page] = at_page;
        if ((i + 1) * page <= low) continue;
        const int id = c.table[at_page];
        const bool there = (unsigned)id < (unsigned)c.pages;
        if (!there && threadIdx.x == 0) atomicExch(c.status, PAGED_BAD_PAGE);
        const int from = there ? (id * c.kv + kvh) << c.page_shift : 0;
        const long long to = ((long long)at_page * c.kv + kvh) * page * c.hd;
        for (int first = threadIdx.x; first < all; first += ASK * READ_THREADS) {
            PagedRows<Int4>::Eight k[ASK], v[ASK];
#pragma unroll
            for (int j = 0; j < ASK; j++) {
                const int at = first + j * READ_THREADS, row = at / units, col = (at - row * units) * 8;
                k[j] = {}, v[j] = {};
                if (there && at < all) k[j] = keys.eight(from + row, col), v[j] = values.eight(from + row, col);
            }
#pragma unroll
            for (int j = 0; j < ASK; j++) {
                const int at = first + j * READ_THREADS;
                if (at >= all) continue;
                read_store(u.k + to + at * 8, k[j]);
                read_store(u.v + to + at * 8, v[j]);
            }
        }
    }
}

// Bytes of the workspace's pages and their table.
inline long long unpack_words(long long batch, long long positions, long long kv, long long hd) { return batch * positions * kv * hd * 2; }
inline long long unpack_bytes(long long batch, long long positions, long long kv, long long hd) { return 2 * unpack_words(batch, positions, kv, hd) + (batch * positions / 16 * 4 + 15) / 16 * 16; }

// `ws`: unpack_bytes of the call's page tables' positions. The call as one on the words. A block has one page of sequences of up to max_length positions, and more of longer ones, so that
// a table with room to grow costs no blocks.
inline cudaError_t launch_unpack(AttendCall *a, void *ws, long long max_length, cudaStream_t st) {
    const long long words = unpack_words(a->c.batch, (long long)a->c.max_pages << a->c.page_shift, a->c.kv, a->c.hd);
    UnpackCall u = {*a, static_cast<__nv_bfloat16 *>(ws), reinterpret_cast<__nv_bfloat16 *>(static_cast<unsigned char *>(ws) + words), reinterpret_cast<int *>(static_cast<unsigned char *>(ws) + 2 * words),
                    (int)std::min<long long>(a->c.max_pages, ((max_length - 1) >> a->c.page_shift) + 1)};
    unpack_kernel<<<dim3((unsigned)(a->c.batch * u.at_once), (unsigned)a->c.kv), READ_THREADS, 0, st>>>(u);
    a->k = u.k, a->v = u.v, a->c.table = u.table, a->c.pages = a->c.batch * a->c.max_pages;
    return cudaGetLastError();
}

} // namespace b200i

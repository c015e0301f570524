// Attention of few rows over a paged cache: a decode step's single tokens (and up to 16 rows a sequence and key head).
//
//   z_rj = scale q_r . k_j (capped),   o_r = sum_j 2^(z_rj log2 e - m_r) v_j / sum_j 2^(z_rj log2 e - m_r)
//
// Bound: HBM, every key and value read once: the rows of all heads that share a key head are taken together.
// Work. The keys of an item (sequence, key head) are cut into tiles of FEW_KEYS; all items' tiles form one line, and each block takes an
// equal piece of it whatever the lengths are, so ragged batches and one long sequence fill the device alike. A block
// that holds an item whole stores its rows; otherwise it leaves (m, l, o) of its part in the workspace, at most two of them, and
// attend_join_kernel joins an item's parts in the order of its keys: the same words for the same call.
// Block. One warp copies: tensor-map boxes of 128 bytes by a page's rows (128-byte swizzle) into a ring of tiles, running
// ahead over the ends of items. Four warps compute, each on 16 keys of a tile of its own with a maximum, a sum and an output of its
// own, which meet when the item ends: nothing in the loop waits for another warp. The products are m16n8k16 with the KEYS as rows, so
// that eight query rows fill an instruction: S^T = K Q^T, then O^T = V^T P^T, P^T being S^T turned by movmatrix.
// The tensor cores are fed by mma.sync here: eight rows need 1 / 16 of a tcgen05 tile, and the kernel waits for memory.
// 32-bit words go in as three bfloat16 pieces (24 bits), products of pieces down to 2^-24 of the whole kept; a weight has two
// pieces where the rows are bfloat16, so that the output's own rounding is the only one of 8 bits.
#pragma once
#include <algorithm>
#include <atomic>

#include "paged.cuh"
#include "paged_async.cuh"

namespace b200i {

constexpr int FEW_WARPS = 4, FEW_THREADS = 32 * (FEW_WARPS + 1);

// keys of a ring slot: 64 of bfloat16, 32 of float32, so that a slot is head_dim (padded) x 256 bytes of keys and values
template <typename CT> struct FewKeys { static constexpr int N = 64; };
template <> struct FewKeys<float> { static constexpr int N = 32; };

template <int HDP, int NT> struct FewShape {
    static constexpr int SLOT = HDP * 256;
    // two blocks on an SM: 113 KB each, of which the meeting of the four warps takes HDP * NT * 96
    static constexpr int SLOTS = (112 * 1024 - HDP * NT * 96 - 1536) / SLOT > 6 ? 6 : (112 * 1024 - HDP * NT * 96 - 1536) / SLOT;
    static constexpr int MEET = 3 * HDP * NT * 8 * 4;
    static constexpr int SMEM = 1024 + SLOTS * SLOT + MEET + 512;
};

struct FewCall {
    AttendCall a;
    float *part;       // [blocks][2][rows * HDP] outputs of parts, then [blocks][2][2 * rows] of m and l
    int *head;         // [blocks][8]: the item whose beginning a block left as a part: sequence (or -1), key head, tiles, tiles of the block before it, tiles a block
    int whole;         // a block takes whole items: no parts
};

// Tiles of a sequence's key heads: from the first key that a row sees; one where rows see nothing, which makes them zero.
__device__ __forceinline__ int few_tiles(const AttendCall &a, const PagedSeq &s, int keys, int *first_tile) {
    const int lo = a.window ? max(0, s.pos0 + 1 - a.window) : 0, t0 = min(lo, s.length) / keys;
    *first_tile = t0;
    return s.n == 0 ? 0 : max(1, (s.length + keys - 1) / keys - t0);
}

// A block's place on the line of all items' tiles.
struct LinePlace {
    int b, kvh;       // the sequence and key head in which it begins
    long long in;     // tiles of that sequence and key head before it
    long long size;   // tiles of the sequence and key head
    long long left;   // tiles of the block
    long long per;    // tiles a block
    long long start;  // where the block begins
};

// `size_of(b)`: the tiles of one key head of sequence b. All threads of the block call it; `sh` holds 32 words.
template <typename F>
__device__ __forceinline__ LinePlace line_place(const PagedCall &c, F size_of, int block, int blocks, long long *sh) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = (int)blockDim.x >> 5;
    long long mine = 0, sum = 0;
    for (int b = tid; b < c.batch; b += blockDim.x) sum += mine = size_of(b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    if (lane == 0) sh[warp] = sum;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < warps; w++) total += sh[w];
    total *= c.kv;
    const long long per = (total + blocks - 1) / blocks, start = per * block;
    __syncthreads();
    if (tid == 0) sh[28] = -1;
    long long before = 0; // of the sequences before this round's
    for (int b0 = 0; b0 < c.batch && start < total; b0 += blockDim.x) {
        const int b = b0 + tid;
        long long here = mine; // what the first loop left, where that saw the whole batch
        if (c.batch > (int)blockDim.x) here = b < c.batch ? size_of(b) : 0;
        long long scan = here;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xFFFFFFFFu, scan, o);
            if (lane >= o) scan += up;
        }
        if (lane == 31) sh[warp] = scan;
        __syncthreads();
        long long base = before;
        for (int w = 0; w < warps; w++) {
            if (w < warp) base += sh[w];
            before += sh[w];
        }
        const long long from = (base + scan - here) * c.kv, to = (base + scan) * c.kv;
        if (start >= from && start < to) { // one thread of one round
            const long long in = start - from;
            sh[28] = b, sh[29] = in / here, sh[30] = in % here, sh[31] = here;
        }
        __syncthreads();
    }
    __syncthreads();
    LinePlace p;
    p.per = per, p.start = start;
    p.left = sh[28] < 0 ? 0 : min(per, total - start);
    p.b = (int)sh[28], p.kvh = (int)sh[29], p.in = sh[30], p.size = sh[31];
    return p;
}

struct FewPlace {
    int b, kvh, tile, count; // a tile of an item of `count`
    long long left;          // tiles of the block from here (where items are whole: items)
    long long line;          // where on the line the item begins
    long long per;           // tiles a block
};
__device__ __forceinline__ FewPlace few_place(const AttendCall &a, int keys, bool whole, int block, int blocks, long long *sh) {
    const auto tiles = [&](int b) {
        int t0;
        return few_tiles(a, paged_seq(a.c, b), keys, &t0);
    };
    const LinePlace l = line_place(a.c, [&](int b) -> long long { return whole ? (long long)(tiles(b) > 0) : (long long)tiles(b); }, block, blocks, sh);
    FewPlace p;
    p.b = l.b, p.kvh = l.kvh, p.tile = whole ? 0 : (int)l.in, p.count = l.left > 0 ? (whole ? tiles(l.b) : (int)l.size) : 0;
    p.left = l.left, p.line = l.start - l.in, p.per = l.per;
    return p;
}

// The item after this one.
__device__ __forceinline__ void few_next(const AttendCall &a, int keys, FewPlace &p) {
    p.line += p.count;
    p.tile = 0;
    if (++p.kvh < a.c.kv) return;
    p.kvh = 0;
    int t0;
    do p.count = ++p.b < a.c.batch ? few_tiles(a, paged_seq(a.c, p.b), keys, &t0) : 1;
    while (p.count == 0);
}

// 16 keys by 16 columns of the tile as fragments, N pieces each: rows are keys.
__device__ __forceinline__ void few_keys(unsigned (&f)[1][4], const unsigned char *tile, int key0, int ks, int lane, const __nv_bfloat16 *) {
    const int mi = lane >> 3, row = key0 + (lane & 7) + (mi & 1) * 8, chunk = 2 * ks + (mi >> 1);
    pg_ldmatrix(f[0], pg_smem(tile) + (unsigned)((chunk >> 3) * (FewKeys<__nv_bfloat16>::N * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)));
}
__device__ __forceinline__ void few_keys(unsigned (&f)[3][4], const unsigned char *tile, int key0, int ks, int lane, const float *) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int row = key0 + (lane >> 2) + (i & 1) * 8, col = 16 * ks + (lane & 3) * 2 + (i >> 1) * 8, chunk = (col & 31) >> 2;
        const float2 x = *reinterpret_cast<const float2 *>(tile + (col >> 5) * (FewKeys<float>::N * 128) + row * 128 + ((chunk ^ (row & 7)) << 4) + (col & 3) * 4);
        unsigned piece[3];
        pg_split<3>(piece, x.x, x.y);
        f[0][i] = piece[0], f[1][i] = piece[1], f[2][i] = piece[2];
    }
}
// The same of the values, turned: rows are columns of the tile (16 of them), columns its keys. keep: which keys are to be read
// (bits of the 16); the others' words, which may be anything, become zeros.
__device__ __forceinline__ void few_values(unsigned (&f)[1][4], const unsigned char *tile, int key0, int mt, int lane, unsigned keep, const __nv_bfloat16 *) {
    const int mi = lane >> 3, row = key0 + (lane & 7) + (mi >> 1) * 8, chunk = 2 * mt + (mi & 1);
    pg_ldmatrix_t(f[0], pg_smem(tile) + (unsigned)((chunk >> 3) * (FewKeys<__nv_bfloat16>::N * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)));
    if (keep != 0xFFFFu) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const unsigned two = keep >> ((lane & 3) * 2 + (i >> 1) * 8);
            f[0][i] &= ((two & 1) ? 0xFFFFu : 0u) | ((two & 2) ? 0xFFFF0000u : 0u);
        }
    }
}
__device__ __forceinline__ void few_values(unsigned (&f)[3][4], const unsigned char *tile, int key0, int mt, int lane, unsigned keep, const float *) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int col = 16 * mt + (lane >> 2) + (i & 1) * 8, chunk = (col & 31) >> 2;
        float x[2];
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int k = (lane & 3) * 2 + e + (i >> 1) * 8, row = key0 + k;
            const float w = *reinterpret_cast<const float *>(tile + (col >> 5) * (FewKeys<float>::N * 128) + row * 128 + ((chunk ^ (row & 7)) << 4) + (col & 3) * 4);
            x[e] = (keep >> k) & 1 ? w : 0.0f;
        }
        unsigned piece[3];
        pg_split<3>(piece, x[0], x[1]);
        f[0][i] = piece[0], f[1][i] = piece[1], f[2][i] = piece[2];
    }
}

// d += A B over pieces of both: those whose places together are below three (2^-24 of the whole and up), the smallest first. The
// tensor cores cut their sums off instead of rounding them: with EXACT the product begins at zero and is added to d in 32-bit arithmetic
// (32 heads of 1250 float32 keys are off by 3.1e-6 without it).
template <bool EXACT, int PA, int PB>
__device__ __forceinline__ void few_mma(float (&d)[4], const unsigned (&a)[PA][4], const unsigned (&b0)[PB], const unsigned (&b1)[PB]) {
    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int places = 2; places >= 0; places--)
#pragma unroll
        for (int i = 0; i < PA; i++)
            if (places - i >= 0 && places - i < PB) pg_mma(EXACT ? part : d, a[i], b0[places - i], b1[places - i]);
    if (EXACT) {
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] += part[i];
    }
}

template <typename RT, typename CT, int HDP, int NT>
__global__ void __launch_bounds__(FEW_THREADS, 2) attend_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const FewCall f) {
    using Shape = FewShape<HDP, NT>;
    constexpr int KEYS = FewKeys<CT>::N, SLOTS = Shape::SLOTS, HALF = Shape::SLOT / 2, BOX_COLS = 128 / (int)sizeof(CT), BOXES = HDP / BOX_COLS;
    constexpr int QP = sizeof(RT) == 4 ? 3 : 1, CP = sizeof(CT) == 4 ? 3 : 1, PP = sizeof(RT) == 4 ? 3 : 2; // pieces of a query, of a key or value, of a weight
    constexpr bool EXACT = sizeof(RT) == 4;
    constexpr int GROUPS = KEYS / 16, KS = HDP / 16, ROWS = NT * 8;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char *ring = smem + ((1024u - (pg_smem(smem) & 1023u)) & 1023u);
    float *meet = reinterpret_cast<float *>(ring + SLOTS * Shape::SLOT);
    unsigned long long *full = reinterpret_cast<unsigned long long *>(meet + Shape::MEET / 4), *empty = full + SLOTS;
    __shared__ float ml[FEW_WARPS][2][ROWS];
    __shared__ long long place[32];
    __shared__ unsigned bad_rows;
    __shared__ int dead;
    const AttendCall &a = f.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < SLOTS; s++) {
            pg_bar_init(&full[s], 1);
            pg_bar_init(&empty[s], GROUPS);
        }
        bad_rows = 0, dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    FewPlace p = few_place(a, KEYS, f.whole != 0, blockIdx.x, gridDim.x, place);
    if (tid == 0 && !f.whole) f.head[blockIdx.x * 8] = -1;
    __syncthreads();
    const int page = 1 << a.c.page_shift, box_rows = min(page, KEYS), pieces = KEYS / box_rows;

    if (warp == FEW_WARPS) { // ---------------- the copies ----------------
        unsigned it = 0;
        bool alive = true;
        while (p.left > 0 && alive) {
            const PagedSeq s = paged_seq(a.c, p.b);
            int t0;
            few_tiles(a, s, KEYS, &t0);
            const int tiles = (int)min((long long)(p.count - p.tile), f.whole ? (long long)p.count : p.left);
            const int last_page = (s.length - 1) >> a.c.page_shift;
            const int *ids = a.c.table + (long long)p.b * a.c.max_pages;
            int base = ((t0 + p.tile) * KEYS) >> a.c.page_shift; // the first page that `id` holds, a lane each; `ahead` the 32 after
            int id = base + lane <= last_page ? ids[base + lane] : 0, ahead = base + 32 + lane <= last_page ? ids[base + 32 + lane] : 0;
            for (int t = 0; t < tiles; t++, it++) {
                const int slot = (int)(it % SLOTS), pos = (t0 + p.tile + t) * KEYS;
                if (!__all_sync(0xFFFFFFFFu, pg_bar_wait(&empty[slot], ((it / SLOTS) & 1u) ^ 1u))) { // a fresh barrier counts as released
                    if (lane == 0) atomicExch(a.c.status, PAGED_WAIT);
                    alive = false;
                    break;
                }
                const int there = min(pieces, max(0, (s.length - pos + box_rows - 1) / box_rows)); // pieces that hold positions of the sequence
                unsigned char *dst = ring + slot * Shape::SLOT;
                if (lane == 0) pg_bar_expect(&full[slot], (unsigned)(there * box_rows * 128 * BOXES * 2));
                __syncwarp();
                const int first = (pos >> a.c.page_shift);
                if (first + pieces - 1 >= base + 32 && there > 0) { // a tile's pages (at most four) lie in one set of 32: sets begin at its own
                    base += 32;
                    id = ahead;
                    ahead = base + 32 + lane <= last_page ? ids[base + 32 + lane] : 0;
                }
                for (int u = 0; u < there * 2 * BOXES; u += 32) {
                    const int v = u + lane, piece = v / (2 * BOXES), box = v % (2 * BOXES);
                    const int mine = __shfl_sync(0xFFFFFFFFu, id, (first + min(piece, there - 1) - base) & 31);
                    if (piece < there) {
                        const int at = pos + piece * box_rows;
                        int row = a.c.pages * a.c.kv * page; // past the pool: zeros
                        if ((unsigned)mine < (unsigned)a.c.pages)
                            row = ((mine * a.c.kv + p.kvh) << a.c.page_shift) + (at & (page - 1));
                        else
                            atomicExch(a.c.status, PAGED_BAD_PAGE);
                        const bool is_v = box >= BOXES;
                        const int cb = is_v ? box - BOXES : box;
                        pg_tma_load(dst + (is_v ? HALF : 0) + cb * (KEYS * 128) + piece * (box_rows * 128), is_v ? &map_v : &map_k, &full[slot], cb * BOX_COLS, row);
                    }
                }
            }
            p.left -= f.whole ? 1 : tiles;
            if (p.left > 0) few_next(a, KEYS, p);
        }
        if (!alive) { // copies in flight end before the block does
            for (unsigned i = it > (unsigned)SLOTS ? it - SLOTS : 0; i < it; i++) pg_bar_wait(&full[i % SLOTS], (i / SLOTS) & 1u);
        }
        return;
    }

    // ---------------- the products ----------------
    const float unit = (a.softcap > 0.0f ? a.softcap : a.scale) * PAGED_LOG2E, inner = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;
    unsigned it = 0;
    bool alive = true, first_part = true;
    while (p.left > 0) {
        const PagedSeq s = paged_seq(a.c, p.b);
        int t0;
        few_tiles(a, s, KEYS, &t0);
        const int tiles = (int)min((long long)(p.count - p.tile), f.whole ? (long long)p.count : p.left);
        const int n = min(s.n, a.max_new), rows = min(n * a.c.group, ROWS);
        if (s.n > a.max_new && tid == 0) atomicExch(a.c.status, PAGED_BAD_BOUND);

        unsigned q0[NT][KS][QP], q1[NT][KS][QP]; // the rows as fragments: columns (lane % 4) * 2 and the next, and eight further on
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 8 + (lane >> 2);
            const RT *src = static_cast<const RT *>(a.q) + (long long)(s.first + r / a.c.group) * a.ldq + (long long)(p.kvh * a.c.group + r % a.c.group) * a.c.hd;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int col = ks * 16 + h * 8 + (lane & 3) * 2;
                    if (r < rows && col < a.c.hd) x[2 * h] = paged_read(src + col), x[2 * h + 1] = paged_read(src + col + 1);
                }
                if (a.flip) x[0] = -x[0], x[1] = -x[1], x[2] = -x[2], x[3] = -x[3];
                pg_split<QP>(q0[nt][ks], x[0], x[1]);
                pg_split<QP>(q1[nt][ks], x[2], x[3]);
            }
        }
        int hi[NT][2], lo[NT][2]; // what a row sees: positions lo .. hi - 1, of the lane's rows (lane % 4) * 2 and the next
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = nt * 8 + (lane & 3) * 2 + e;
                hi[nt][e] = r < rows ? s.pos0 + r / a.c.group + 1 : 0;
                lo[nt][e] = a.window ? hi[nt][e] - a.window : 0;
            }
        const int all_lo = a.window ? s.pos0 + n - a.window : 0; // every row sees positions all_lo .. pos0

        float o[NT][KS][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < KS; mt++) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f;
        }
        for (int t = 0; t < tiles; t++, it++) {
            const int group = (warp - (int)(it * GROUPS % FEW_WARPS) + FEW_WARPS) % FEW_WARPS; // which 16 keys of the tile are this warp's
            if (group >= GROUPS) continue;
            const int slot = (int)(it % SLOTS);
            if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&full[slot], (it / SLOTS) & 1u))) {
                if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
                alive = false; // it goes on without waiting, so that the others meet it; nothing of the block is stored from here on
            }
            const int key0 = group * 16, j0 = (t0 + p.tile + t) * KEYS + key0;
            if (alive && j0 < s.length) {
                const unsigned char *kt = ring + slot * Shape::SLOT, *vt = kt + HALF;
                float z[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) z[nt][0] = z[nt][1] = z[nt][2] = z[nt][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    unsigned k[CP][4];
                    few_keys(k, kt, key0, ks, lane, static_cast<const CT *>(nullptr));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) few_mma<EXACT>(z[nt], k, q0[nt][ks], q1[nt][ks]);
                }
                const bool edge = j0 + 16 > s.pos0 + 1 || j0 < all_lo;
                unsigned w0[NT][PP], w1[NT][PP];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = z[nt][i];
                        x = unit * (a.softcap > 0.0f ? tanhf(x * inner) : x);
                        if (edge) {
                            const int j = j0 + (lane >> 2) + (i >> 1) * 8;
                            if (j >= hi[nt][i & 1] || j < lo[nt][i & 1]) x = -INFINITY;
                        }
                        z[nt][i] = x;
                    }
                    float top[2] = {fmaxf(z[nt][0], z[nt][2]), fmaxf(z[nt][1], z[nt][3])};
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        top[0] = fmaxf(top[0], __shfl_xor_sync(0xFFFFFFFFu, top[0], d));
                        top[1] = fmaxf(top[1], __shfl_xor_sync(0xFFFFFFFFu, top[1], d));
                    }
                    if (__any_sync(0xFFFFFFFFu, top[0] > m[nt][0] || top[1] > m[nt][1])) {
                        float keep[2];
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const float next = fmaxf(m[nt][e], top[e]);
                            keep[e] = m[nt][e] == -INFINITY ? 0.0f : paged_exp2(m[nt][e] - next);
                            m[nt][e] = next;
                            l[nt][e] *= keep[e];
                        }
#pragma unroll
                        for (int mt = 0; mt < KS; mt++)
                            o[nt][mt][0] *= keep[0], o[nt][mt][1] *= keep[1], o[nt][mt][2] *= keep[0], o[nt][mt][3] *= keep[1];
                    }
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        w[i] = paged_exp2(z[nt][i] - (m[nt][i & 1] == -INFINITY ? 0.0f : m[nt][i & 1]));
                        l[nt][i & 1] += w[i];
                    }
                    pg_split<PP>(w0[nt], w[0], w[1]);
                    pg_split<PP>(w1[nt], w[2], w[3]);
#pragma unroll
                    for (int i = 0; i < PP; i++) w0[nt][i] = pg_transpose(w0[nt][i]), w1[nt][i] = pg_transpose(w1[nt][i]);
                }
                unsigned keep = 0xFFFFu; // positions of the sequence that some row sees; what stands in the others is not multiplied
                if (edge) {
                    const int low = a.window ? s.pos0 + 1 - a.window : 0;
                    keep = j0 + 16 > s.length ? 0xFFFFu >> (j0 + 16 - s.length) : 0xFFFFu;
                    if (j0 < low) keep &= low - j0 < 16 ? 0xFFFFu << (low - j0) : 0u;
                }
#pragma unroll
                for (int mt = 0; mt < KS; mt++) {
                    unsigned v[CP][4];
                    few_values(v, vt, key0, mt, lane, keep, static_cast<const CT *>(nullptr));
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) few_mma<EXACT>(o[nt][mt], v, w0[nt], w1[nt]);
                }
            }
            __syncwarp();
            if (lane == 0) pg_bar_arrive(&empty[slot]);
        }

        // ---- the item's (or its part's) end: the four warps' results meet ----
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[nt][e] += __shfl_xor_sync(0xFFFFFFFFu, l[nt][e], d);
                if (lane < 4) ml[warp][0][nt * 8 + lane * 2 + e] = m[nt][e], ml[warp][1][nt * 8 + lane * 2 + e] = l[nt][e];
            }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory");
        float mm[NT][2], ll[NT][2];
        constexpr int MINE = KS / FEW_WARPS; // a warp joins this many of the 16-column pieces
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = nt * 8 + (lane & 3) * 2 + e;
                float top = ml[0][0][r];
#pragma unroll
                for (int w = 1; w < FEW_WARPS; w++) top = fmaxf(top, ml[w][0][r]);
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < FEW_WARPS; w++) sum += ml[w][0][r] == -INFINITY ? 0.0f : ml[w][1][r] * paged_exp2(ml[w][0][r] - top);
                mm[nt][e] = top, ll[nt][e] = sum;
            }
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const float keep[2] = {m[nt][0] == -INFINITY ? 0.0f : paged_exp2(m[nt][0] - mm[nt][0]), m[nt][1] == -INFINITY ? 0.0f : paged_exp2(m[nt][1] - mm[nt][1])};
#pragma unroll
            for (int mt = 0; mt < KS; mt++) {
#pragma unroll
                for (int i = 0; i < 4; i++) o[nt][mt][i] *= keep[i & 1];
                const int owner = mt / MINE;
                if (owner != warp) { // [owner][the three others][piece of the owner][lane], 16 bytes a lane
                    const int k = warp < owner ? warp : warp - 1;
                    reinterpret_cast<float4 *>(meet)[(((owner * 3 + k) * MINE + mt % MINE) * NT + nt) * 32 + lane] = make_float4(o[nt][mt][0], o[nt][mt][1], o[nt][mt][2], o[nt][mt][3]);
                }
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory");
        const bool is_whole = p.tile == 0 && tiles == p.count;
        const long long slot = (long long)blockIdx.x * 2 + (first_part && p.tile > 0 ? 0 : 1);
        unsigned wrong = 0;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mt = 0; mt < KS; mt++) {
                if (mt / MINE != warp) continue;
                float x[4] = {o[nt][mt][0], o[nt][mt][1], o[nt][mt][2], o[nt][mt][3]};
#pragma unroll
                for (int k = 0; k < 3; k++) { // in the order of the warps, whichever this is
                    const float4 y = reinterpret_cast<const float4 *>(meet)[(((warp * 3 + k) * MINE + mt % MINE) * NT + nt) * 32 + lane];
                    x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int r = nt * 8 + (lane & 3) * 2 + (i & 1), col = mt * 16 + (lane >> 2) + (i >> 1) * 8;
                    if (is_whole) {
                        const float y = ll[nt][i & 1] == 0.0f ? 0.0f : x[i] / ll[nt][i & 1];
                        if (r < rows && col < a.c.hd && !dead) {
                            paged_write(static_cast<RT *>(a.out) + ((long long)(s.first + r / a.c.group) * a.c.heads + p.kvh * a.c.group + r % a.c.group) * a.c.hd + col, y);
                            if (!isfinite(y)) wrong |= 1u << r;
                        }
                    } else if (r < rows) {
                        f.part[(slot * ROWS + r) * HDP + col] = x[i];
                    }
                }
            }
        if (!is_whole) {
            float *stats = f.part + (long long)gridDim.x * 2 * ROWS * HDP + slot * 2 * ROWS;
            if (warp == 0 && lane < 4)
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 2; e++) stats[nt * 8 + lane * 2 + e] = mm[nt][e], stats[ROWS + nt * 8 + lane * 2 + e] = ll[nt][e];
            if (tid == 0 && p.tile == 0 && !dead) {
                int *head = f.head + blockIdx.x * 8;
                head[0] = p.b, head[1] = p.kvh, head[2] = p.count, head[3] = (int)(p.line - p.per * blockIdx.x), head[4] = (int)p.per;
            }
        }
        if (wrong) atomicOr(&bad_rows, wrong);
        asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory"); // `meet`, `ml` are read, `bad_rows` is whole
        if (bad_rows) { // a masked key's zero weight met a value that is not finite, or a 32-bit word left bfloat16's range
            const unsigned rest = bad_rows;
            asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory");
            if (tid == 0) bad_rows = 0;
            for (int r = warp; r < rows; r += FEW_WARPS)
                if (rest >> r & 1) attend_row_plain<RT, CT>(a, p.b, s.first + r / a.c.group, s.pos0 + r / a.c.group, s.length, p.kvh * a.c.group + r % a.c.group);
            asm volatile("bar.sync 1, %0;" ::"n"(32 * FEW_WARPS) : "memory");
        }
        first_part = false;
        p.left -= f.whole ? 1 : tiles;
        if (p.left > 0) few_next(a, KEYS, p);
    }
}

// The parts of an item that several blocks share. blockIdx.x: the block that began it; blockIdx.y: the row.
template <typename RT, typename CT, int HDP, int NT>
__global__ void __launch_bounds__(HDP) attend_join_kernel(const FewCall f) {
    constexpr int ROWS = NT * 8;
    const AttendCall &a = f.a;
    const int c0 = blockIdx.x, r = blockIdx.y, col = threadIdx.x;
    const int b = f.head[c0 * 8];
    if (b < 0) return;
    const int kvh = f.head[c0 * 8 + 1], count = f.head[c0 * 8 + 2], from = f.head[c0 * 8 + 3], per = f.head[c0 * 8 + 4];
    const PagedSeq s = paged_seq(a.c, b);
    if (r >= min(s.n, a.max_new) * a.c.group) return;
    const int parts = min(1 + (int)((from + (long long)count - 1) / per), (int)gridDim.x - c0);
    const float *stats = f.part + (long long)gridDim.x * 2 * ROWS * HDP;
    float top = -INFINITY;
    for (int i = 0; i < parts; i++) top = fmaxf(top, stats[((long long)(c0 + i) * 2 + (i == 0)) * 2 * ROWS + r]);
    float l = 0.0f, o = 0.0f;
    for (int i = 0; i < parts; i++) {
        const long long slot = (long long)(c0 + i) * 2 + (i == 0);
        const float m = stats[slot * 2 * ROWS + r], keep = m == -INFINITY ? 0.0f : paged_exp2(m - top);
        l = fmaf(stats[slot * 2 * ROWS + ROWS + r], keep, l);
        o = fmaf(f.part[(slot * ROWS + r) * HDP + col], keep, o);
    }
    const int row = s.first + r / a.c.group, h = kvh * a.c.group + r % a.c.group;
    const float y = l == 0.0f ? 0.0f : o / l;
    if (col < a.c.hd) paged_write(static_cast<RT *>(a.out) + ((long long)row * a.c.heads + h) * a.c.hd + col, y);
    if (__syncthreads_or(col < a.c.hd && !isfinite(y)) && threadIdx.x < 32) attend_row_plain<RT, CT>(a, b, row, s.pos0 + r / a.c.group, s.length, h);
}

// ---- host side ----

// How a call is cut: from what the host knows of the lengths, so nothing waits for the device.
struct FewPlan {
    int blocks, whole;
    long long part_floats, bytes; // of the workspace
};
constexpr int FEW_LEAST = 4;  // tiles that a block takes at least
constexpr int FEW_WHOLE = 8;  // items of up to as many tiles are not cut

inline FewPlan few_plan(int sms, int batch, int kv, int hdp, int nt, int keys, long long max_new, long long max_length, int window) {
    FewPlan p;
    long long span = max_length;
    if (window > 0) span = std::min(span, (long long)window + max_new + keys);
    const long long items = (long long)batch * kv, tiles = (span + keys - 1) / keys;
    p.whole = tiles <= FEW_WHOLE;
    const long long want = p.whole ? items : (items * tiles + FEW_LEAST - 1) / FEW_LEAST;
    p.blocks = (int)std::min<long long>(2LL * sms, want);
    p.part_floats = p.whole ? 0 : (long long)p.blocks * 2 * nt * 8 * (hdp + 2);
    p.bytes = p.whole ? 0 : p.part_floats * 4 + (long long)p.blocks * 32;
    return p;
}

template <typename RT, typename CT, int HDP, int NT>
cudaError_t launch_few_as(const AttendCall &a, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    using Shape = FewShape<HDP, NT>;
    constexpr int KEYS = FewKeys<CT>::N;
    FewCall f;
    f.a = a, f.whole = p.whole, f.part = static_cast<float *>(ws), f.head = p.whole ? nullptr : reinterpret_cast<int *>(static_cast<float *>(ws) + p.part_floats);
    alignas(64) CUtensorMap map_k, map_v;
    const long long rows = ((long long)a.c.pages * a.c.kv) << a.c.page_shift;
    const int box = std::min(1 << a.c.page_shift, KEYS);
    if (!paged_map(&map_k, a.k, rows, a.c.hd, sizeof(CT) == 4, box) || !paged_map(&map_v, a.v, rows, a.c.hd, sizeof(CT) == 4, box)) return cudaErrorNotSupported;
    static std::atomic<bool> known[64];
    if (device >= 64 || !known[device].load()) {
        const cudaError_t e = cudaFuncSetAttribute(attend_few_kernel<RT, CT, HDP, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
        if (e != cudaSuccess) return e;
        if (device < 64) known[device].store(true);
    }
    attend_few_kernel<RT, CT, HDP, NT><<<p.blocks, FEW_THREADS, Shape::SMEM, st>>>(map_k, map_v, f);
    *launches += 1;
    if (!p.whole) {
        attend_join_kernel<RT, CT, HDP, NT><<<dim3(p.blocks, NT * 8), HDP, 0, st>>>(f);
        *launches += 1;
    }
    return cudaGetLastError();
}
template <typename RT, typename CT>
cudaError_t launch_few(const AttendCall &a, const FewPlan &p, int hdp, int nt, void *ws, int device, cudaStream_t st, int *launches) {
    if (hdp == 64) return nt == 1 ? launch_few_as<RT, CT, 64, 1>(a, p, ws, device, st, launches) : launch_few_as<RT, CT, 64, 2>(a, p, ws, device, st, launches);
    return nt == 1 ? launch_few_as<RT, CT, 128, 1>(a, p, ws, device, st, launches) : launch_few_as<RT, CT, 128, 2>(a, p, ws, device, st, launches);
}

} // namespace b200i

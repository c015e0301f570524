// Attention of few rows over a paged cache: a decode step's single tokens (and up to 16 rows a sequence and key head).
//
//   z_rj = scale q_r . k_j (capped),   o_r = sum_j 2^(z_rj log2 e - m_r) v_j / sum_j 2^(z_rj log2 e - m_r)
//
// Bound: HBM, every key and value read once: the rows of all heads that share a key head are taken together.
// Work. The keys of an item (sequence, key head) are cut into tiles; all items' tiles form one line, and each block takes an
// equal piece of it whatever the lengths are, so ragged batches and one long sequence fill the device alike. A block
// that holds an item whole stores its rows; otherwise it leaves (m, l, o) of its part in the workspace, at most two of them, and
// attend_join_kernel joins an item's parts in the order of its keys: the same words for the same call.
// Block. One warp copies: tensor-map boxes of 128 bytes by a page's rows (128-byte swizzle) into a ring of tiles, and before an item's
// tiles its queries and what the others need to know of it, running ahead over the ends of items. Four warps compute, each on
// keys of a tile of its own with a maximum, a sum and an output of its own, which meet when the item ends: nothing in the loop
// waits for another warp.
// bfloat16 rows (attend_few_kernel): m16n8k16 with the KEYS as rows, so that eight query rows fill an instruction: S^T = K Q^T, then
// O^T = V^T P^T, P^T being S^T turned by movmatrix. The tensor cores are fed by mma.sync here: eight rows need 1 / 16 of a tcgen05 tile,
// and the kernel waits for memory. A weight goes in as two bfloat16 pieces, so that the output's own rounding is the only one of 8 bits.
// float32 rows (attend_few_fma_kernel): two or four lanes a key for the scores, a lane four columns for the values, in fused multiply-adds. Products of
// three bfloat16 pieces on the tensor cores took 5000 cycles for 16 keys of a float32 cache, of which splitting was most.
// Measured, kernel and join, of the HBM rate: 32 sequences of 1216 to 1279 float32 keys, 16 heads, 111 us (0.90); 64 of 91 to 8192 bfloat16 keys, 32
// heads on 8, 202 us (0.86); one of 131000, 95 us (0.87); one of 200 keys 8.5 us a call.
#pragma once
#include <algorithm>
#include <atomic>

#include "paged.cuh"
#include "paged_async.cuh"

namespace b200i {

constexpr int FEW_WARPS = 4, FEW_THREADS = 32 * (FEW_WARPS + 1), FEW_ITEMS = 2; // items whose queries are held

// keys of a ring slot, which is 32 KB of keys and values: 64 of bfloat16 and 32 of float32 at head_dim 128, twice as many at 64
constexpr int FEW_SLOT = 32 * 1024;
template <typename CT, int HDP> struct FewKeys { static constexpr int N = FEW_SLOT / (2 * HDP * (int)sizeof(CT)); };

// Shared memory of a block: the ring, `meet` bytes for the warps' results, the queries, barriers. Two blocks on an SM (113 KB each) where
// that leaves two slots.
template <int HDP, int MEET_BYTES, int QUERY_BYTES> struct FewShape {
    static constexpr int WARPS = FEW_WARPS, SLOT = FEW_SLOT, MEET = MEET_BYTES, QUERY = QUERY_BYTES;
    static constexpr int REST = 1024 + 512 + MEET + FEW_ITEMS * QUERY;
    static constexpr int BLOCKS = (110 * 1024 - REST) / SLOT >= 2 ? 2 : 1;
    static constexpr int ROOM = ((BLOCKS == 2 ? 112 : 220) * 1024 - REST) / SLOT;
    static constexpr int SLOTS = ROOM > 6 ? 6 : ROOM;
    static constexpr int SMEM = REST + SLOTS * SLOT;
    static_assert(SLOTS >= 2, "shared memory");
};

struct FewCall {
    AttendCall a;
    float *part;       // [blocks][2][rows * HDP] outputs of parts, then [blocks][2][2 * rows] of m and l
    int *head;         // [blocks][8]: the item whose beginning a block left as a part: sequence (or -1), key head, tiles, tiles of the block before it, tiles a block
    int whole;         // a block takes whole items, by steps of the grid: no parts
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

// 64-bit quotients cost hundreds of cycles; almost all are of 32-bit words.
__device__ __forceinline__ long long line_div(long long x, long long y) { return ((x | y) >> 32) == 0 ? (long long)((unsigned)x / (unsigned)y) : x / y; }

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
    const long long per = line_div(total + blocks - 1, blocks), start = per * block;
    __syncthreads();
    if (tid == 0) sh[28] = -1;
    long long before = 0; // of the sequences before those that the block looks at
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
            const long long in = start - from, head = line_div(in, here);
            sh[28] = b, sh[29] = head, sh[30] = in - head * here, sh[31] = here;
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

// What the copying warp tells the others of an item, or of the block's part of it.
struct FewItem {
    int kvh, b;
    PagedSeq s;
    int n;             // tokens whose rows are computed
    int pos;           // position of its first key
    int tiles, before; // tiles of the block; tiles of the item in the blocks before
    int count;         // tiles of the item
    int line;          // where on the line the item begins, from where the block does (negative where another block began it)
    int per;           // tiles a block
    int more;          // 0: this is no item, and the block is done
};

// The block's shared memory.
template <typename Shape> struct FewMemory {
    unsigned char *ring, *query;
    float *meet;
    unsigned long long *full, *empty, *item_full, *item_empty;
    __device__ __forceinline__ FewMemory(unsigned char *smem) {
        ring = smem + ((1024u - (pg_smem(smem) & 1023u)) & 1023u);
        query = ring + Shape::SLOTS * Shape::SLOT;
        meet = reinterpret_cast<float *>(query + FEW_ITEMS * Shape::QUERY);
        full = reinterpret_cast<unsigned long long *>(reinterpret_cast<unsigned char *>(meet) + Shape::MEET), empty = full + Shape::SLOTS;
        item_full = empty + Shape::SLOTS, item_empty = item_full + FEW_ITEMS;
    }
};

// The copying warp. `items`: FEW_ITEMS of them in shared memory. `bring(to, full, pos, there, low, kvh, page_of)`, all lanes, asks for the `there` pieces (of
// min(page, KEYS) positions) of a tile that begins at pos, as bytes that `full` counts: page_of(piece) is a piece's page, and positions below low are seen by no row.
template <typename RT, int KEYS, typename Shape, typename F>
__device__ __forceinline__ void few_copies(const FewCall &f, const FewMemory<Shape> &sm, FewItem *items, const LinePlace &p, F bring) {
    constexpr int SLOTS = Shape::SLOTS;
    const AttendCall &a = f.a;
    const int lane = threadIdx.x & 31, page = 1 << a.c.page_shift, box_rows = min(page, KEYS), pieces = KEYS / box_rows;
    unsigned it = 0, number = 0, sent = 0; // tiles, items looked at, phases of item_full that were begun
    bool alive = true;
    const auto wait = [&](unsigned long long *bar, unsigned parity) {
        if (!__all_sync(0xFFFFFFFFu, pg_bar_wait(bar, parity))) {
            if (lane == 0) atomicExch(a.c.status, PAGED_WAIT);
            alive = false;
        }
        return alive;
    };
    int b = p.b, kvh = p.kvh, before = (int)p.in, line = -before;
    long long left = p.left;
    PagedSeq s = {};
    int t0 = 0, count = 0;
    const auto settle = [&] { // whole items: the first from (b, kvh) on, by steps of the grid, that has rows
        for (; b < a.c.batch; kvh += gridDim.x, b += kvh / a.c.kv, kvh %= a.c.kv) {
            s = paged_seq_checked(a.c, b), count = few_tiles(a, s, KEYS, &t0);
            if (count > 0) return;
        }
        left = 0;
    };
    if (f.whole)
        settle();
    else if (left > 0)
        s = paged_seq(a.c, b), count = few_tiles(a, s, KEYS, &t0);
    for (; alive; number++) {
        const int at = number % FEW_ITEMS;
        if (!wait(&sm.item_empty[at], ((number / FEW_ITEMS) & 1u) ^ 1u)) break; // a fresh barrier counts as released
        if (left <= 0) { // the others are told that there is no more
            if (lane == 0) {
                items[at].more = 0;
                pg_bar_arrive(&sm.item_full[at]);
            }
            sent++;
            break;
        }
        const int tiles = f.whole ? count : (int)min((long long)(count - before), left), n = min(s.n, a.max_new);
        const unsigned row_bytes = (unsigned)(a.c.group * a.c.hd * (int)sizeof(RT)); // of a token's rows, which stand side by side
        if (lane == 0) {
            items[at] = FewItem{kvh, b, s, n, (t0 + before) * KEYS, tiles, before, count, line, (int)p.per, 1};
            if (s.n > a.max_new) atomicExch(a.c.status, PAGED_BAD_BOUND);
            pg_bar_expect(&sm.item_full[at], row_bytes * (unsigned)n);
        }
        sent++;
        __syncwarp();
        for (int i = lane; i < n; i += 32) {
            const RT *src = static_cast<const RT *>(a.q) + (long long)(s.first + i) * a.ldq + (long long)kvh * a.c.group * a.c.hd;
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(pg_smem(sm.query + at * Shape::QUERY) + i * row_bytes), "l"(src),
                         "r"(row_bytes), "r"(pg_smem(&sm.item_full[at]))
                         : "memory");
        }
        const int last_page = (s.length - 1) >> a.c.page_shift, low = a.window ? max(0, s.pos0 + 1 - a.window) : 0; // no row sees what is below
        const int *ids = a.c.table + (long long)b * a.c.max_pages;
        int base = ((t0 + before) * KEYS) >> a.c.page_shift; // the first page that `id` holds, a lane each; `ahead` the 32 after
        int id = base + lane <= last_page ? ids[base + lane] : 0, ahead = base + 32 + lane <= last_page ? ids[base + 32 + lane] : 0;
        // what follows is asked for while this item's tiles come in
        const int b1 = kvh + 1 < a.c.kv ? b : b + 1;
        PagedSeq s1 = s;
        if (!f.whole && b1 != b && b1 < a.c.batch) s1 = paged_seq(a.c, b1);
        for (int t = 0; t < tiles; t++, it++) {
            const int slot = (int)(it % SLOTS), pos = (t0 + before + t) * KEYS;
            if (!wait(&sm.empty[slot], ((it / SLOTS) & 1u) ^ 1u)) break;
            const int there = min(pieces, max(0, (s.length - pos + box_rows - 1) / box_rows)); // pieces that hold positions of the sequence
            const int first = pos >> a.c.page_shift;
            if (first + pieces - 1 >= base + 32 && there > 0) { // a tile's pages (at most sixteen) lie in one set of 32: sets begin at its own
                base += 32;
                id = ahead;
                ahead = base + 32 + lane <= last_page ? ids[base + 32 + lane] : 0;
            }
            bring(sm.ring + slot * Shape::SLOT, &sm.full[slot], pos, there, low, kvh, [&](int piece) { return __shfl_sync(0xFFFFFFFFu, id, (first + min(piece, there - 1) - base) & 31); });
        }
        if (f.whole) {
            kvh += gridDim.x, b += kvh / a.c.kv, kvh %= a.c.kv;
            settle();
            continue;
        }
        left -= tiles;
        line += count, before = 0;
        if (left <= 0) continue;
        if (++kvh >= a.c.kv) {
            kvh = 0, b++, s = s1, count = few_tiles(a, s, KEYS, &t0);
            while (count == 0 && b + 1 < a.c.batch) s = paged_seq(a.c, ++b), count = few_tiles(a, s, KEYS, &t0);
        }
    }
    // copies in flight end before the block does, whoever has given up
    for (unsigned i = it > (unsigned)SLOTS ? it - SLOTS : 0; i < it; i++) pg_bar_wait(&sm.full[i % SLOTS], (i / SLOTS) & 1u);
    for (unsigned i = sent > FEW_ITEMS ? sent - FEW_ITEMS : 0; i < sent; i++) pg_bar_wait(&sm.item_full[i % FEW_ITEMS], (i / FEW_ITEMS) & 1u);
}

// What brings tiles of float32 or bfloat16 caches: boxes of 128 bytes by a piece's rows.
template <typename CT, int HDP, typename Shape>
__device__ __forceinline__ auto few_boxes(const CUtensorMap *map_k, const CUtensorMap *map_v, const PagedCall &c) {
    return [map_k, map_v, &c](unsigned char *dst, unsigned long long *full, int pos, int there, int low, int kvh, auto page_of) {
        constexpr int KEYS = FewKeys<CT, HDP>::N, HALF = Shape::SLOT / 2, BOX_COLS = 128 / (int)sizeof(CT), BOXES = HDP / BOX_COLS;
        const int lane = threadIdx.x & 31, page = 1 << c.page_shift, box_rows = min(page, KEYS);
        if (lane == 0) pg_bar_expect(full, (unsigned)(there * box_rows * 128 * BOXES * 2));
        __syncwarp();
        for (int u = 0; u < there * 2 * BOXES; u += 32) {
            const int v = u + lane, piece = v / (2 * BOXES), box = v % (2 * BOXES);
            const int mine = page_of(piece);
            if (piece < there) {
                int row = c.pages * c.kv * page; // past the pool: zeros
                if (low - pos < (piece + 1) * box_rows) { // a page that nobody sees any more may be anyone's
                    if ((unsigned)mine < (unsigned)c.pages)
                        row = ((mine * c.kv + kvh) << c.page_shift) + ((pos + piece * box_rows) & (page - 1));
                    else
                        atomicExch(c.status, PAGED_BAD_PAGE);
                }
                const bool is_v = box >= BOXES;
                const int cb = is_v ? box - BOXES : box;
                pg_tma_load(dst + (is_v ? HALF : 0) + cb * (KEYS * 128) + piece * (box_rows * 128), is_v ? map_v : map_k, full, cb * BOX_COLS, row);
            }
        }
    };
}

// The beginning of a block: barriers, and its place on the line.
template <int KEYS, typename Shape, typename Bits>
__device__ __forceinline__ LinePlace few_begin(const FewCall &f, const FewMemory<Shape> &sm, long long *place, Bits *bad_rows, int *dead) {
    if (threadIdx.x == 0) {
        for (int s = 0; s < Shape::SLOTS; s++) {
            pg_bar_init(&sm.full[s], 1);
            pg_bar_init(&sm.empty[s], Shape::WARPS);
        }
        for (int i = 0; i < FEW_ITEMS; i++) {
            pg_bar_init(&sm.item_full[i], 1);
            pg_bar_init(&sm.item_empty[i], Shape::WARPS);
        }
        *bad_rows = 0, *dead = 0;
        if (!f.whole) f.head[blockIdx.x * 8] = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    LinePlace p;
    if (!f.whole) pg_follow_early();
    if (f.whole) {
        p.b = (int)blockIdx.x / f.a.c.kv, p.kvh = (int)blockIdx.x % f.a.c.kv, p.in = 0, p.left = 1, p.per = 0;
    } else {
        p = line_place(
            f.a.c,
            [&](int b) -> long long {
                int t0;
                return few_tiles(f.a, paged_seq_checked(f.a.c, b), KEYS, &t0);
            },
            blockIdx.x, gridDim.x, place);
    }
    __syncthreads();
    return p;
}

// A part's statistics and, where it begins the item, the item.
__device__ __forceinline__ void few_head(const FewCall &f, const FewItem &i) {
    int *head = f.head + blockIdx.x * 8;
    head[0] = i.b, head[1] = i.kvh, head[2] = i.count, head[3] = i.line, head[4] = i.per;
}
template <int WARPS = FEW_WARPS> __device__ __forceinline__ void few_meet() { asm volatile("bar.sync 1, %0;" ::"n"(32 * WARPS) : "memory"); } // the computing warps
// They meet, and know alike whether one of them brings a yes: a word in shared memory could change before the slower ones have read it.
template <int WARPS = FEW_WARPS> __device__ __forceinline__ bool few_vote(bool yes) {
    unsigned some;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(some) : "r"((unsigned)yes), "n"(32 * WARPS) : "memory");
    return some != 0;
}
// Rows that did not come out finite, done again: a masked key's zero weight met a value that is not finite.
template <typename RT, typename CT, int WARPS = FEW_WARPS, typename Bits>
__device__ __forceinline__ void few_again(const AttendCall &a, const FewItem &i, Bits *bad_rows, int rows) {
    const Bits rest = *bad_rows;
    few_meet<WARPS>();
    if (threadIdx.x == 0) *bad_rows = 0;
    for (int r = threadIdx.x >> 5; r < rows; r += WARPS)
        if (rest >> r & 1) attend_row_plain<RT, CT>(a, i.b, i.s.first + r / a.c.group, i.s.pos0 + r / a.c.group, i.s.length, i.kvh * a.c.group + r % a.c.group);
    few_meet<WARPS>();
}

// ---- bfloat16 rows ----

// 16 keys by 16 columns of the tile as a fragment: rows are keys.
template <int KEYS>
__device__ __forceinline__ void few_keys(unsigned (&f)[4], const unsigned char *tile, int key0, int ks, int lane) {
    const int mi = lane >> 3, row = key0 + (lane & 7) + (mi & 1) * 8, chunk = 2 * ks + (mi >> 1);
    pg_ldmatrix(f, pg_smem(tile) + (unsigned)((chunk >> 3) * (KEYS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)));
}
// The same of the values, turned: rows are columns of the tile (16 of them), columns its keys.
template <int KEYS>
__device__ __forceinline__ void few_values(unsigned (&f)[4], const unsigned char *tile, int key0, int mt, int lane) {
    const int mi = lane >> 3, row = key0 + (lane & 7) + (mi >> 1) * 8, chunk = 2 * mt + (mi & 1);
    pg_ldmatrix_t(f, pg_smem(tile) + (unsigned)((chunk >> 3) * (KEYS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)));
}

template <int HDP, int NT>
using FewMmaShape = FewShape<HDP, 3 * HDP * NT * 8 * 4, NT * 8 * HDP * 2>;

template <int HDP, int NT>
__global__ void __launch_bounds__(FEW_THREADS, FewMmaShape<HDP, NT>::BLOCKS) attend_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ FewCall f) {
    using T = __nv_bfloat16;
    using Shape = FewMmaShape<HDP, NT>;
    constexpr int KEYS = FewKeys<T, HDP>::N, SLOTS = Shape::SLOTS, HALF = Shape::SLOT / 2, KS = HDP / 16, ROWS = NT * 8;
    extern __shared__ __align__(128) unsigned char smem[];
    const FewMemory<Shape> sm(smem);
    __shared__ float ml[FEW_WARPS][2][ROWS];
    __shared__ long long place[32];
    __shared__ FewItem items[FEW_ITEMS];
    __shared__ unsigned bad_rows;
    __shared__ int dead;
    const AttendCall &a = f.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const LinePlace p = few_begin<KEYS>(f, sm, place, &bad_rows, &dead);
    if (warp == FEW_WARPS) {
        few_copies<T, KEYS>(f, sm, items, p, few_boxes<T, HDP, Shape>(&map_k, &map_v, f.a.c));
        return;
    }

    const float unit = a.softcap > 0.0f ? a.softcap * PAGED_LOG2E : a.scale * PAGED_LOG2E;
    unsigned it = 0;
    bool alive = true, first_part = true;
    const auto give_up = [&] {
        if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
        alive = false; // it goes on without waiting, so that the others meet it; nothing of the block is stored from here on
    };
    for (unsigned number = 0;; number++) {
        const int which = number % FEW_ITEMS;
        if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&sm.item_full[which], (number / FEW_ITEMS) & 1u))) give_up();
        if (few_vote(!alive)) break; // nobody goes on where one has given up: what the item is would not be known
        const FewItem item = items[which];
        if (!item.more) break;
        const PagedSeq s = item.s;
        const int rows = min(item.n * a.c.group, ROWS);

        unsigned q0[NT][KS], q1[NT][KS]; // the rows as fragments: columns (lane % 4) * 2 and the next, and eight further on
        const unsigned flip = a.flip ? 0x80008000u : 0u;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 8 + (lane >> 2);
            const unsigned char *src = sm.query + which * Shape::QUERY + r * a.c.hd * 2;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                const int col = ks * 16 + (lane & 3) * 2;
                q0[nt][ks] = r < rows && col < a.c.hd ? *reinterpret_cast<const unsigned *>(src + col * 2) ^ flip : 0u;
                q1[nt][ks] = r < rows && col + 8 < a.c.hd ? *reinterpret_cast<const unsigned *>(src + col * 2 + 16) ^ flip : 0u;
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
        const int all_lo = a.window ? s.pos0 + item.n - a.window : 0; // every row sees positions all_lo .. pos0

        float o[NT][KS][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int mt = 0; mt < KS; mt++) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f;
        }
        for (int t = 0; t < item.tiles; t++, it++) {
            const int slot = (int)(it % SLOTS);
            if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&sm.full[slot], (it / SLOTS) & 1u))) give_up();
#pragma unroll 1
            for (int key0 = warp * 16; key0 < KEYS; key0 += 16 * FEW_WARPS) {
                const int j0 = item.pos + t * KEYS + key0;
                if (!alive || j0 >= s.length) break;
                const unsigned char *kt = sm.ring + slot * Shape::SLOT, *vt = kt + HALF;
                float z[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++) z[nt][0] = z[nt][1] = z[nt][2] = z[nt][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ks++) {
                    unsigned k[4];
                    few_keys<KEYS>(k, kt, key0, ks, lane);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) pg_mma(z[nt], k, q0[nt][ks], q1[nt][ks]);
                }
                const bool edge = j0 + 16 > s.pos0 + 1 || j0 < all_lo;
                unsigned w0[NT][2], w1[NT][2]; // two pieces of the weights
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = z[nt][i];
                        x = unit * (a.softcap > 0.0f ? tanhf(x * a.scale * a.cap_part) : x); // (scale / softcap may leave 32 bits)
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
                    pg_split<2>(w0[nt], w[0], w[1]);
                    pg_split<2>(w1[nt], w[2], w[3]);
#pragma unroll
                    for (int i = 0; i < 2; i++) w0[nt][i] = pg_transpose(w0[nt][i]), w1[nt][i] = pg_transpose(w1[nt][i]);
                }
                unsigned mask[2] = {0xFFFFFFFFu, 0xFFFFFFFFu}; // what stands in positions that no row sees, or of no sequence, is not multiplied
                if (edge) {
                    const int low = a.window ? s.pos0 + 1 - a.window : 0;
                    unsigned keep = j0 + 16 > s.length ? 0xFFFFu >> (j0 + 16 - s.length) : 0xFFFFu;
                    if (j0 < low) keep &= low - j0 < 16 ? 0xFFFFu << (low - j0) : 0u;
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const unsigned two = keep >> ((lane & 3) * 2 + i * 8);
                        mask[i] = ((two & 1) ? 0xFFFFu : 0u) | ((two & 2) ? 0xFFFF0000u : 0u);
                    }
                }
#pragma unroll
                for (int mt = 0; mt < KS; mt++) {
                    unsigned v[4];
                    few_values<KEYS>(v, vt, key0, mt, lane);
                    v[0] &= mask[0], v[1] &= mask[0], v[2] &= mask[1], v[3] &= mask[1];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        pg_mma(o[nt][mt], v, w0[nt][1], w1[nt][1]);
                        pg_mma(o[nt][mt], v, w0[nt][0], w1[nt][0]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && alive) pg_bar_arrive(&sm.empty[slot]); // (what it has not waited for is not given back)
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
        few_meet();
        if (lane == 0 && alive) pg_bar_arrive(&sm.item_empty[which]);
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
        const bool is_whole = item.before == 0 && item.tiles == item.count;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float keep[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                keep[e] = m[nt][e] == -INFINITY ? 0.0f : paged_exp2(m[nt][e] - mm[nt][e]);
                if (is_whole) keep[e] *= paged_share(ll[nt][e], s.pos0 + (nt * 8 + (lane & 3) * 2 + e) / a.c.group);
            }
#pragma unroll
            for (int mt = 0; mt < KS; mt++) {
#pragma unroll
                for (int i = 0; i < 4; i++) o[nt][mt][i] *= keep[i & 1];
                const int owner = mt / MINE;
                if (owner != warp) { // [owner][the three others][piece of the owner][lane], 16 bytes a lane
                    const int k = warp < owner ? warp : warp - 1;
                    reinterpret_cast<float4 *>(sm.meet)[(((owner * 3 + k) * MINE + mt % MINE) * NT + nt) * 32 + lane] = make_float4(o[nt][mt][0], o[nt][mt][1], o[nt][mt][2], o[nt][mt][3]);
                }
            }
        }
        few_meet();
        const long long slot = (long long)blockIdx.x * 2 + (first_part && item.before > 0 ? 0 : 1);
        unsigned wrong = 0;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float *part[2];
            T *out[2];
            bool in[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = nt * 8 + (lane & 3) * 2 + e, token = r / a.c.group;
                in[e] = r < rows && !dead;
                part[e] = f.part + (slot * ROWS + r) * HDP;
                out[e] = static_cast<T *>(a.out) + ((long long)(s.first + token) * a.c.heads + item.kvh * a.c.group + r - token * a.c.group) * a.c.hd;
            }
#pragma unroll
            for (int mt = 0; mt < KS; mt++) {
                if (mt / MINE != warp) continue;
                float x[4] = {o[nt][mt][0], o[nt][mt][1], o[nt][mt][2], o[nt][mt][3]};
#pragma unroll
                for (int k = 0; k < 3; k++) { // in the order of the warps, whichever this is
                    const float4 y = reinterpret_cast<const float4 *>(sm.meet)[(((warp * 3 + k) * MINE + mt % MINE) * NT + nt) * 32 + lane];
                    x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int col = mt * 16 + (lane >> 2) + (i >> 1) * 8;
                    if (!in[i & 1]) continue;
                    if (is_whole) {
                        if (col < a.c.hd) out[i & 1][col] = __float2bfloat16_rn(x[i]);
                        if (!(x[i] * 0.0f == 0.0f)) wrong |= 1u << (nt * 8 + (lane & 3) * 2 + (i & 1)); // (past head_dim there are zeros)
                    } else {
                        part[i & 1][col] = x[i];
                    }
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
            if (tid == 0 && item.before == 0 && !dead) few_head(f, item);
        }
        if (wrong) atomicOr(&bad_rows, wrong);
        few_meet(); // what met is read, `bad_rows` is whole
        if (bad_rows) few_again<T, T>(a, item, &bad_rows, rows);
        first_part = false;
    }
}

// ---- float32 rows ----

template <typename CT, int HDP, int R>
using FewFmaShape = FewShape<HDP, FEW_WARPS * R * HDP * 4, R * HDP * 4>;

// Four 32-bit words of a key at 16-byte chunk c of its row (a row's chunks are permuted by its number: the tensor maps' swizzle); of bfloat16
// eight.
template <typename CT, int KEYS> struct FewRow;
template <int KEYS> struct FewRow<float, KEYS> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void load(float *x, const unsigned char *tile, int row, int c) {
        const float4 v = *reinterpret_cast<const float4 *>(tile + (c >> 3) * (KEYS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    }
    template <int COLS> // COLS columns from lane * COLS on
    static __device__ __forceinline__ void columns(float *x, const unsigned char *tile, int row, int lane) {
        const int c = lane * COLS / 4;
        const unsigned char *at = tile + (c >> 3) * (KEYS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        if constexpr (COLS == 4) {
            const float4 v = *reinterpret_cast<const float4 *>(at);
            x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
        } else {
            const float2 v = *reinterpret_cast<const float2 *>(at + (lane & 1) * 8);
            x[0] = v.x, x[1] = v.y;
        }
    }
};
template <int KEYS> struct FewRow<__nv_bfloat16, KEYS> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void two(float *x, unsigned v) { x[0] = __uint_as_float(v << 16), x[1] = __uint_as_float(v & 0xFFFF0000u); }
    static __device__ __forceinline__ void load(float *x, const unsigned char *tile, int row, int c) {
        const uint4 v = *reinterpret_cast<const uint4 *>(tile + (c >> 3) * (KEYS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
        two(x, v.x), two(x + 2, v.y), two(x + 4, v.z), two(x + 6, v.w);
    }
    template <int COLS>
    static __device__ __forceinline__ void columns(float *x, const unsigned char *tile, int row, int lane) {
        const int c = lane * COLS / 8;
        const unsigned char *at = tile + (c >> 3) * (KEYS * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
        if constexpr (COLS == 4) {
            const uint2 v = *reinterpret_cast<const uint2 *>(at + (lane & 1) * 8);
            two(x, v.x), two(x + 2, v.y);
        } else {
            two(x, *reinterpret_cast<const unsigned *>(at + (lane & 3) * 4));
        }
    }
};

template <typename CT, int HDP, int R>
__global__ void __launch_bounds__(FEW_THREADS, FewFmaShape<CT, HDP, R>::BLOCKS)
    attend_few_fma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ FewCall f) {
    using Shape = FewFmaShape<CT, HDP, R>;
    constexpr int KEYS = FewKeys<CT, HDP>::N, SLOTS = Shape::SLOTS, HALF = Shape::SLOT / 2, MINE = KEYS / FEW_WARPS, SPLIT = 32 / MINE, COLS = HDP / 32, N = FewRow<CT, KEYS>::N;
    extern __shared__ __align__(128) unsigned char smem[];
    const FewMemory<Shape> sm(smem);
    __shared__ float ml[FEW_WARPS][2][R];
    __shared__ long long place[32];
    __shared__ FewItem items[FEW_ITEMS];
    __shared__ unsigned bad_rows;
    __shared__ int dead;
    const AttendCall &a = f.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const LinePlace p = few_begin<KEYS>(f, sm, place, &bad_rows, &dead);
    if (warp == FEW_WARPS) {
        few_copies<float, KEYS>(f, sm, items, p, few_boxes<CT, HDP, Shape>(&map_k, &map_v, f.a.c));
        return;
    }

    float *const weights = sm.meet + warp * R * HDP; // [R][MINE], where this warp's results will be
    const int key = lane % MINE, share = lane / MINE;  // of a tile a warp takes MINE keys; SPLIT lanes have a key's columns between them
    const float sign = a.flip ? -1.0f : 1.0f, unit = sign * (a.softcap > 0.0f ? a.softcap * PAGED_LOG2E : a.scale * PAGED_LOG2E);
    unsigned it = 0;
    bool alive = true, first_part = true;
    const auto give_up = [&] {
        if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
        alive = false; // it goes on without waiting, so that the others meet it; nothing of the block is stored from here on
    };
    for (unsigned number = 0;; number++) {
        const int which = number % FEW_ITEMS;
        if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&sm.item_full[which], (number / FEW_ITEMS) & 1u))) give_up();
        if (few_vote(!alive)) break; // nobody goes on where one has given up: what the item is would not be known
        const FewItem item = items[which];
        if (!item.more) break;
        const PagedSeq s = item.s;
        const int rows = min(item.n * a.c.group, R), chunks = a.c.hd / N;
        const float *query = reinterpret_cast<const float *>(sm.query + which * Shape::QUERY);
        const int all_lo = a.window ? s.pos0 + item.n - a.window : 0, low = a.window ? s.pos0 + 1 - a.window : 0; // every row sees all_lo .. pos0; none sees what is below low

        float o[R][COLS], m[R], l[R]; // l: of the lane's keys, in the first share of lanes
#pragma unroll
        for (int r = 0; r < R; r++) {
            m[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
            for (int c = 0; c < COLS; c++) o[r][c] = 0.0f;
        }
        for (int t = 0; t < item.tiles; t++, it++) {
            // every warp waits for every tile: a wait for a phase whose predecessor it has not seen end may return at once
            const int slot = (int)(it % SLOTS), key0 = warp * MINE, j0 = item.pos + t * KEYS + key0, j = j0 + key;
            if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&sm.full[slot], (it / SLOTS) & 1u))) give_up();
            if (alive && j0 < s.length) {
                const unsigned char *kt = sm.ring + slot * Shape::SLOT, *vt = kt + HALF;
                unsigned long long z2[R];
#pragma unroll
                for (int r = 0; r < R; r++) z2[r] = 0;
#pragma unroll 4
                for (int c = share; c < chunks; c += SPLIT) {
                    float k[N];
                    FewRow<CT, KEYS>::load(k, kt, key0 + key, c);
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int e = 0; e < N; e += 4) {
                            const float4 q = *reinterpret_cast<const float4 *>(query + r * a.c.hd + c * N + e); // the same for all lanes of a share
                            z2[r] = pg_fma2(pg_two(k[e], k[e + 1]), pg_two(q.x, q.y), z2[r]);
                            z2[r] = pg_fma2(pg_two(k[e + 2], k[e + 3]), pg_two(q.z, q.w), z2[r]);
                        }
                }
                const bool edge = j0 + MINE > s.pos0 + 1 || j0 < all_lo;
#pragma unroll
                for (int r = 0; r < R; r++) {
                    float z, z1;
                    pg_one(z2[r], z, z1);
                    z += z1;
#pragma unroll
                    for (int d = MINE; d < 32; d <<= 1) z += __shfl_xor_sync(0xFFFFFFFFu, z, d);
                    z = unit * (a.softcap > 0.0f ? tanhf(z * a.scale * a.cap_part) : z);
                    if (edge) {
                        const int seen = s.pos0 + r / a.c.group;
                        if (j > seen || (a.window && j <= seen - a.window)) z = -INFINITY;
                    }
                    float top = z;
#pragma unroll
                    for (int d = 1; d < MINE; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                    if (top > m[r]) { // alike in all lanes
                        const float keep = m[r] == -INFINITY ? 0.0f : paged_exp2(m[r] - top);
                        m[r] = top, l[r] *= keep;
#pragma unroll
                        for (int c = 0; c < COLS; c++) o[r][c] *= keep;
                    }
                    const float w = paged_exp2(z - (m[r] == -INFINITY ? 0.0f : m[r]));
                    if (share == 0) {
                        l[r] += w;
                        weights[r * MINE + key] = w;
                    }
                }
                __syncwarp();
                const auto add = [&](int k, const float (&w)[R]) {
                    float v[COLS];
                    FewRow<CT, KEYS>::template columns<COLS>(v, vt, key0 + k, lane);
#pragma unroll
                    for (int r = 0; r < R; r++)
#pragma unroll
                        for (int c = 0; c < COLS; c++) o[r][c] = fmaf(w[r], v[c], o[r][c]);
                };
                if (!edge) {
#pragma unroll(R <= 4 ? 2 : 1)
                    for (int k = 0; k < MINE; k += 4) {
                        float4 w[R];
#pragma unroll
                        for (int r = 0; r < R; r++) w[r] = *reinterpret_cast<const float4 *>(weights + r * MINE + k);
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float one[R];
#pragma unroll
                            for (int r = 0; r < R; r++) one[r] = e == 0 ? w[r].x : (e == 1 ? w[r].y : (e == 2 ? w[r].z : w[r].w));
                            add(k + e, one);
                        }
                    }
                } else { // what stands in positions that no row sees, or of no sequence, is not read
#pragma unroll 1
                    for (int k = max(0, low - j0); k < min(MINE, s.length - j0); k++) {
                        float one[R];
#pragma unroll
                        for (int r = 0; r < R; r++) one[r] = weights[r * MINE + k];
                        add(k, one);
                    }
                }
            }
            __syncwarp();
            if (lane == 0 && alive) pg_bar_arrive(&sm.empty[slot]); // (what it has not waited for is not given back)
        }

        // ---- the item's (or its part's) end: the four warps' results meet, [warp][row][column] ----
#pragma unroll
        for (int r = 0; r < R; r++) {
            l[r] = paged_warp_sum(l[r]);
            if (lane == 0) ml[warp][0][r] = m[r], ml[warp][1][r] = l[r];
            float *to = sm.meet + (warp * R + r) * HDP + lane * COLS;
            if constexpr (COLS == 4)
                *reinterpret_cast<float4 *>(to) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
            else
                *reinterpret_cast<float2 *>(to) = make_float2(o[r][0], o[r][1]);
        }
        few_meet();
        if (lane == 0 && alive) pg_bar_arrive(&sm.item_empty[which]);
        const bool is_whole = item.before == 0 && item.tiles == item.count;
        const long long slot = (long long)blockIdx.x * 2 + (first_part && item.before > 0 ? 0 : 1);
        constexpr int AT_ONCE = 32 * FEW_WARPS / HDP; // rows that the threads take at once, a column each
        unsigned wrong = 0;
#pragma unroll 1
        for (int r = tid / HDP; r < rows; r += AT_ONCE) {
            const int col = tid % HDP, token = r / a.c.group;
            float top = ml[0][0][r];
#pragma unroll
            for (int w = 1; w < FEW_WARPS; w++) top = fmaxf(top, ml[w][0][r]);
            float sum = 0.0f, x = 0.0f;
#pragma unroll
            for (int w = 0; w < FEW_WARPS; w++) {
                const float keep = ml[w][0][r] == -INFINITY ? 0.0f : paged_exp2(ml[w][0][r] - top);
                sum = fmaf(ml[w][1][r], keep, sum);
                x = fmaf(sm.meet[(w * R + r) * HDP + col], keep, x);
            }
            if (dead) continue;
            if (is_whole) {
                x *= paged_share(sum, s.pos0 + token);
                if (col < a.c.hd) static_cast<float *>(a.out)[((long long)(s.first + token) * a.c.heads + item.kvh * a.c.group + r - token * a.c.group) * a.c.hd + col] = x;
                if (!(x * 0.0f == 0.0f)) wrong |= 1u << r; // (past head_dim there are zeros)
            } else {
                f.part[(slot * R + r) * HDP + col] = x;
                if (col == 0) {
                    float *stats = f.part + (long long)gridDim.x * 2 * R * HDP + slot * 2 * R;
                    stats[r] = top, stats[R + r] = sum;
                }
            }
        }
        if (!is_whole && tid == 0 && item.before == 0 && !dead) few_head(f, item);
        if (wrong) atomicOr(&bad_rows, wrong);
        few_meet(); // what met is read, `bad_rows` is whole
        if (bad_rows) few_again<float, CT>(a, item, &bad_rows, rows);
        first_part = false;
    }
}

// The parts of an item that several blocks share, in the order of its keys: a block a row, a warp every eighth part, a lane the statistics of a part
// and HDP / 32 columns of its output. blockIdx.x: the block that began the item; blockIdx.y: the row. What it costs is the way there: code that
// is fetched from L2, and a chain of loads.
template <typename RT, typename CT, int HDP, int ROWS>
__global__ void __launch_bounds__(256, 4) attend_join_kernel(const __grid_constant__ FewCall f) {
    constexpr int N = HDP / 32;
    __shared__ float met[8][HDP];
    const AttendCall &a = f.a;
    const int c0 = blockIdx.x, r = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int token = a.c.group == 1 ? r : (int)__umulhi((unsigned)r, a.c.group_part);
    pg_follow();
    const int4 head = *reinterpret_cast<const int4 *>(f.head + c0 * 8);
    const int per = f.head[c0 * 8 + 4], b = head.x;
    if (b < 0) return;
    const PagedSeq s = paged_seq(a.c, b);
    if (token >= min(s.n, a.max_new)) return;
    const int parts = min(1 + (int)((unsigned)(head.w + head.z - 1) / (unsigned)per), (int)gridDim.x - c0);
    const float *stats = f.part + (long long)gridDim.x * 2 * ROWS * HDP + r, *outputs = f.part + r * HDP + lane * N;
    const auto slot = [&](int i) { return (unsigned)((c0 + i) * 2 + (i == 0)); };
    float top = -INFINITY, l = 0.0f, o[N] = {};
#pragma unroll 1
    for (int i = lane; i < parts; i += 32) top = fmaxf(top, stats[slot(i) * (2 * ROWS)]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
#pragma unroll 1
    for (int i0 = 0; i0 < parts; i0 += 32) {
        float keep = 0.0f;
        if (i0 + lane < parts) {
            const float *at = stats + slot(i0 + lane) * (2 * ROWS);
            keep = *at == -INFINITY ? 0.0f : paged_exp2(*at - top);
            l = fmaf(at[ROWS], keep, l);
        }
        const int here = min(32, parts - i0);
#pragma unroll 2
        for (int i = warp; i < here; i += 8) {
            const float k = __shfl_sync(0xFFFFFFFFu, keep, i);
            const float *at = outputs + (long long)slot(i0 + i) * (ROWS * HDP);
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const float2 v = *reinterpret_cast<const float2 *>(at + e);
                o[e] = fmaf(v.x, k, o[e]), o[e + 1] = fmaf(v.y, k, o[e + 1]);
            }
        }
    }
    l = paged_warp_sum(l);
#pragma unroll
    for (int k = 0; k < N; k++) met[warp][lane * N + k] = o[k];
    __syncthreads();
    const int col = threadIdx.x, h = (head.y - token) * a.c.group + r;
    float y = 0.0f;
    if (col < a.c.hd) {
#pragma unroll
        for (int w = 0; w < 8; w++) y += met[w][col];
        y *= l != 0.0f ? __frcp_rn(l) : paged_share(l, s.pos0 + token);
        paged_write(static_cast<RT *>(a.out) + ((long long)(s.first + token) * a.c.heads + h) * a.c.hd + col, y);
    }
    if (!__syncthreads_or(!(y * 0.0f == 0.0f))) return;
    // done again, an eighth of its keys a warp
    __shared__ float again[8][2];
    const int pos = s.pos0 + token, begin = attend_begin(a, pos), end = attend_end(pos, s.length), step = (max(end - begin, 0) + 255) / 256 * 32;
    const RowSums sums = attend_keys_plain<RT, CT>(a, b, s.first + token, h, begin + warp * step, min(begin + (warp + 1) * step, end));
    if (lane == 0) again[warp][0] = sums.m, again[warp][1] = sums.l;
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (4 * lane + k < HDP) met[warp][4 * lane + k] = sums.o[k];
    __syncthreads();
    if (col >= a.c.hd) return;
    top = again[0][0];
    for (int w = 1; w < 8; w++) top = fmaxf(top, again[w][0]);
    l = y = 0.0f;
    for (int w = 0; w < 8; w++) {
        const float keep = again[w][0] == -INFINITY ? 0.0f : paged_exp2((again[w][0] - top) * PAGED_LOG2E);
        l = fmaf(again[w][1], keep, l), y = fmaf(met[w][col], keep, y);
    }
    paged_write(static_cast<RT *>(a.out) + ((long long)(s.first + token) * a.c.heads + h) * a.c.hd + col, l != 0.0f ? y / l : paged_share(l, pos));
}

// ---- host side ----

// How a call is cut: from what the host knows of the lengths, so nothing waits for the device.
struct FewPlan {
    int blocks, whole, most, rows; // most rows of an item; what it is laid out for
    long long part_floats, bytes; // of the workspace
};
constexpr int FEW_LEAST = 4;  // tiles that a block takes at least
constexpr int FEW_WHOLE = 8;  // items of up to as many tiles are not cut
constexpr int FEW_MOST = 16;  // rows of an item

template <bool F32, typename CT, int HDP, int R> constexpr int few_blocks_per_sm() { return F32 ? FewFmaShape<CT, HDP, R>::BLOCKS : FewMmaShape<HDP, R <= 8 ? 1 : 2>::BLOCKS; }

// Of at most `room` blocks at a time and tiles of `keys` keys, items of up to `whole` tiles uncut; p->rows is set.
inline void few_cut(FewPlan *p, int room, int keys, int batch, int kv, int hdp, long long max_new, long long max_length, int window, int whole = FEW_WHOLE) {
    long long span = max_length;
    if (window > 0) span = std::min(span, (long long)window + max_new + keys);
    const long long items = (long long)batch * kv, tiles = (span + keys - 1) / keys;
    p->whole = tiles <= whole;
    const long long want = p->whole ? items : (items * tiles + FEW_LEAST - 1) / FEW_LEAST;
    p->blocks = (int)std::min<long long>(room, want);
    p->part_floats = p->whole ? 0 : (long long)p->blocks * 2 * p->rows * (hdp + 2);
    p->bytes = p->whole ? 0 : p->part_floats * 4 + (long long)p->blocks * 32;
}

inline FewPlan few_plan(int sms, bool f32_rows, bool f32_cache, int batch, int kv, int hdp, int rows, long long max_new, long long max_length, int window) {
    FewPlan p;
    const int keys = FEW_SLOT / (2 * hdp * (f32_cache ? 4 : 2));
    p.most = rows, p.rows = f32_rows ? 1 : 8; // laid out for 1, 2, 4, 8 or 16 float32 rows, for 8 or 16 of bfloat16
    while (p.rows < rows) p.rows *= 2;
    const int per_sm = p.rows < 16 ? 2 : (!f32_rows ? few_blocks_per_sm<false, __nv_bfloat16, 128, 16>() : (hdp == 64 ? few_blocks_per_sm<true, float, 64, 16>() : few_blocks_per_sm<true, float, 128, 16>()));
    few_cut(&p, per_sm * sms, keys, batch, kv, hdp, max_new, max_length, window);
    return p;
}

template <typename RT, typename CT, int HDP, int R>
cudaError_t launch_few_as(const AttendCall &a, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    constexpr bool F32 = sizeof(RT) == 4;
    constexpr int KEYS = FewKeys<CT, HDP>::N;
    FewCall f;
    f.a = a, f.whole = p.whole, f.part = static_cast<float *>(ws), f.head = p.whole ? nullptr : reinterpret_cast<int *>(static_cast<float *>(ws) + p.part_floats);
    alignas(64) CUtensorMap map_k, map_v;
    const long long rows = ((long long)a.c.pages * a.c.kv) << a.c.page_shift;
    const int box = std::min(1 << a.c.page_shift, KEYS);
    if (!paged_map(&map_k, a.k, rows, a.c.hd, sizeof(CT) == 4, box) || !paged_map(&map_v, a.v, rows, a.c.hd, sizeof(CT) == 4, box)) return cudaErrorNotSupported;
    void (*kernel)(const CUtensorMap, const CUtensorMap, const FewCall);
    int smem;
    if constexpr (F32)
        kernel = attend_few_fma_kernel<CT, HDP, R>, smem = FewFmaShape<CT, HDP, R>::SMEM;
    else
        kernel = attend_few_kernel<HDP, R / 8>, smem = FewMmaShape<HDP, R / 8>::SMEM;
    static std::atomic<bool> known[64];
    if (device >= 64 || !known[device].load()) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (device < 64) known[device].store(true);
    }
    kernel<<<p.blocks, FEW_THREADS, smem, st>>>(map_k, map_v, f);
    *launches += 1;
    if (!p.whole) {
        *launches += 1;
        return launch_following<FewCall>(attend_join_kernel<RT, CT, HDP, R>, dim3(p.blocks, p.most), 256, st, f);
    }
    return cudaGetLastError();
}
template <typename RT, typename CT, int HDP>
cudaError_t launch_few_rows(const AttendCall &a, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    if constexpr (sizeof(RT) == 4) {
        if (p.rows == 1) return launch_few_as<RT, CT, HDP, 1>(a, p, ws, device, st, launches);
        if (p.rows == 2) return launch_few_as<RT, CT, HDP, 2>(a, p, ws, device, st, launches);
        if (p.rows == 4) return launch_few_as<RT, CT, HDP, 4>(a, p, ws, device, st, launches);
    }
    return p.rows == 8 ? launch_few_as<RT, CT, HDP, 8>(a, p, ws, device, st, launches) : launch_few_as<RT, CT, HDP, 16>(a, p, ws, device, st, launches);
}
template <typename RT, typename CT>
cudaError_t launch_few(const AttendCall &a, const FewPlan &p, int hdp, void *ws, int device, cudaStream_t st, int *launches) {
    return hdp == 64 ? launch_few_rows<RT, CT, 64>(a, p, ws, device, st, launches) : launch_few_rows<RT, CT, 128>(a, p, ws, device, st, launches);
}

} // namespace b200i

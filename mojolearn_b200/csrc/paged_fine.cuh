// Attention of many float32 rows over a paged cache on the tcgen05 tensor cores, to 32-bit accuracy.
//
// A 32-bit word is the sum of three bfloat16 pieces of 8 bits each, and a product of two words the sum of the products of their
// pieces; those down to 2^-24 of the whole are taken (three of them where the cache is bfloat16, which is one piece; six where it is
// float32), each exact, the small ones first. Weights go in as three pieces too: two leave 2.4e-6 of an output out (9000 keys).
// The tensor pipe cuts its sums off where it adds to a large one (an output summed there over all keys was off by 2.2e-6 to 4.3e-6, by 1e-6 or less
// this way): a tile's P V begins at zero, and the softmax threads add it to their row's 32-bit registers, rounding to nearest.
//
// Bound: the tensor pipe at 6 (bfloat16 cache) or 12 (float32) times head_dim x 2 operations a (row, key) against 71 TFLOP/s of fma:
// 270 to 135 TFLOP/s of 4 head_dim operations at the measured bfloat16 rate. Rows, items, parts and the line are those of paged_many.cuh; a block
// has 128 rows and one stream of 64-key tiles, and two S in tensor memory, so that the softmax of one tile runs under the products of its
// neighbours; the output of a tile is read while the next score is made. The pieces of Q are in tensor memory (192 columns of 512 at head_dim 128) beside O (128) and two S that their P is
// written over (96 each): the products read only keys and values from shared memory, whose 64 rows a product would not pay for Q's.
// A bfloat16 cache comes in by tensor-map copies; of a float32 one four warps read the rows and write their pieces. An item's rows come in by bulk
// copies while the item before is worked on, are cut into pieces as soon as that one's last score is made, and its output goes out by bulk copies
// from the same place: rows read and written by their threads, 512 bytes apart, had taken 16000 of 35000 cycles of an item of 1024 keys.
// Measured, with what follows it: 4 prompts of 1024 tokens, 16 heads of 128: 142 us on a bfloat16 cache, 223 on a float32 one (32 and 64 at the tensor rate
// of their products):
// the issuing thread waits, three barriers between two products, and a product of 64 columns takes 45 cycles, not 32.
// Of a cache in 4 bits the four warps write the codes' words, which are one piece as bfloat16 ones are: 12 chunks of up to 509 tokens behind up to 4000, 429 us (391 on words).
#pragma once
#include "paged_many.cuh"

namespace b200i {

constexpr int FINE_THREADS = 384, FINE_KEYS = 64, FINE_ROWS = 128; // four warps of softmax, four that bring keys and values, and a group of which one issues
constexpr int FINE_REGS = 232, FINE_REGS_LOAD = 144, FINE_REGS_LESS = 128; // a thread: together 504 = 3 x 168, what the block is launched with

template <typename CT, int HDP> struct FineShape {
    static constexpr int PIECES = std::is_same_v<CT, float> ? 3 : 1;
    static constexpr int TILE = HDP * 128;               // bytes of 64 rows of bfloat16
    static constexpr int SLOT = PIECES * TILE;
    static constexpr int PITCH = HDP * 4 + 16;           // of a row's words on their way in and out: eight rows' 16 bytes fall into different banks
    static constexpr int STAGE = FINE_ROWS * PITCH;
    static constexpr int ROOM = (224 * 1024 - STAGE) / SLOT;
    static constexpr int SLOTS = ROOM > 8 ? 8 : ROOM;
    static constexpr int SMEM = 1024 + SLOTS * SLOT + STAGE + 256;
    static_assert(SLOTS >= 3, "two keys and a value");
};

template <typename CT, int HDP>
__global__ void __launch_bounds__(FINE_THREADS, 1) attend_fine_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ManyCall f) {
    using Shape = FineShape<CT, HDP>;
    using Walk = ManyWalk<FINE_ROWS, FINE_KEYS, 1>;
    constexpr int SLOTS = Shape::SLOTS, SLOT = Shape::SLOT, TILE = Shape::TILE, CP = Shape::PIECES, LOADERS = std::is_same_v<CT, __nv_bfloat16> ? 1 : 128, BOXES = HDP / 64, HALF_COLS = FINE_KEYS * 128, BR = FINE_ROWS;
    constexpr int Q_COLS = HDP / 2, O_AT = 3 * Q_COLS, S_AT = O_AT + HDP, S_COLS = 96; // columns of tensor memory
    static_assert(S_AT + 2 * S_COLS <= 512, "tensor memory");
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char *ring = smem + ((1024u - (pg_smem(smem) & 1023u)) & 1023u), *stage = ring + SLOTS * SLOT;
    unsigned long long *full = reinterpret_cast<unsigned long long *>(stage + Shape::STAGE), *empty = full + SLOTS;
    unsigned long long *s_full = empty + SLOTS, *p_full = s_full + 2, *o_full = p_full + 2, *o_free = o_full + 1, *q_full = o_free + 1, *tail = q_full + 1, *stage_full = tail + 1, *stage_empty = stage_full + 1, *done = stage_empty + 1; // 2 SLOTS + 11 <= 32 words
    __shared__ long long place[32];
    __shared__ unsigned tmem_slot;
    __shared__ int dead;
    const AttendCall &a = f.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < SLOTS; s++) {
            pg_bar_init(&full[s], LOADERS);
            pg_bar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            pg_bar_init(&s_full[i], 1);
            pg_bar_init(&p_full[i], 128);
        }
        pg_bar_init(o_full, 1);
        pg_bar_init(o_free, 128);
        pg_bar_init(q_full, 128);
        pg_bar_init(tail, 1);
        pg_bar_init(stage_full, 1);
        pg_bar_init(stage_empty, 128);
        pg_bar_init(done, 1);
        dead = 0;
        f.head[blockIdx.x * 8] = -1, f.head[blockIdx.x * 8 + 6] = 0x7FFFFFFF, f.head[blockIdx.x * 8 + 7] = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pg_smem(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pg_follow_early();
    const LinePlace line = line_place(a.c, [&](int b) { return Walk::steps_of(a, b); }, blockIdx.x, gridDim.x, place);
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const unsigned tmem = tmem_slot;
    const int page = 1 << a.c.page_shift;
    Walk w;
    w.begin(a, line);

    if (warp >= 4 && warp < 8) { // ---------------- keys and values ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FINE_REGS_LOAD));
        // in the order of their first use: K0 K1 V0 K2 V1 K3 ...
        const auto load_of = [](int u, int tiles, bool *is_v) {
            const int lead = min(2, tiles), v = u - lead;
            const bool mixed = v < 2 * (tiles - lead);
            *is_v = v >= 0 && (!mixed || (v & 1) == 0);
            return v < 0 ? u : (mixed ? (*is_v ? v / 2 : v / 2 + lead) : (tiles - lead) + (v - 2 * (tiles - lead)));
        };
        unsigned ld = 0;
        bool alive = true;
        if (LOADERS == 1 && warp == 4) {
            unsigned tails = 0;
            bool tail_lost = false;
            const int box_rows = min(page, FINE_KEYS);
            while (w.left > 0 && alive) {
                const ManyItem item = w.item(a, paged_seq(a.c, w.b));
                const int tiles = w.tiles(item), first = w.first(item), last_page = (item.high - 1) >> a.c.page_shift;
                const int *ids = a.c.table + (long long)w.b * a.c.max_pages;
                for (int u = 0; u < 2 * tiles; u++, ld++) {
                    bool is_v;
                    const int tile = load_of(u, tiles, &is_v), slot = (int)(ld % SLOTS), pos = (item.t0 + first + tile) * FINE_KEYS;
                    if (!__all_sync(0xFFFFFFFFu, pg_bar_wait(&empty[slot], ((ld / SLOTS) & 1u) ^ 1u))) {
                        alive = false;
                        break;
                    }
                    const int there = min(FINE_KEYS / box_rows, max(0, (item.high - pos + box_rows - 1) / box_rows)); // pieces that hold positions that some row sees
                    unsigned char *dst = ring + slot * SLOT;
                    const bool clean = is_v && (pos + FINE_KEYS > item.high || pos < item.low); // rows of values that no row sees are to be zero
                    unsigned long long *bar = clean ? tail : &full[slot];
                    if (lane == 0) pg_bar_expect(bar, (unsigned)(there * box_rows * 128 * BOXES));
                    __syncwarp();
                    for (int x = lane; x < there * BOXES; x += 32) {
                        const int piece = x / BOXES, box = x % BOXES, at = pos + piece * box_rows, index = at >> a.c.page_shift;
                        int row = a.c.pages * a.c.kv * page; // past the pool: zeros
                        if (item.low - at < box_rows) { // a page that nobody sees any more may be anyone's
                            const int id = index <= last_page ? ids[index] : -1;
                            if ((unsigned)id < (unsigned)a.c.pages)
                                row = ((id * a.c.kv + w.kvh) << a.c.page_shift) + (at & (page - 1));
                            else
                                atomicExch(a.c.status, PAGED_BAD_PAGE);
                        }
                        pg_tma_load(dst + box * HALF_COLS + piece * (box_rows * 128), is_v ? &map_v : &map_k, bar, box * 64, row);
                    }
                    if (clean) {
                        if (!__all_sync(0xFFFFFFFFu, pg_bar_wait(tail, tails & 1u))) {
                            alive = false, tail_lost = true;
                            break;
                        }
                        tails++;
                        for (int x = lane; x < FINE_KEYS * 8 * BOXES; x += 32) { // 16 bytes each; a row's are in one swizzle atom, so their order does not matter
                            const int at = pos + ((x >> 3) & (FINE_KEYS - 1));
                            if (at >= item.high || at < item.low) *reinterpret_cast<uint4 *>(dst + x * 16) = make_uint4(0, 0, 0, 0);
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) pg_bar_arrive(&full[slot]);
                    }
                }
                if (alive) w.next(a);
            }
            if (!alive && lane == 0) atomicExch(a.c.status, PAGED_WAIT);
            // copies in flight end before the block does, whoever has given up
            if (tail_lost) pg_bar_wait(tail, tails & 1u);
            for (unsigned i = ld > (unsigned)SLOTS ? ld - SLOTS : 0; i < ld; i++) pg_bar_wait(&full[i % SLOTS], (i / SLOTS) & 1u);
        } else if constexpr (std::is_same_v<CT, float>) {
            constexpr int CHUNKS = HDP / 8, ROWS_AT_ONCE = 128 / CHUNKS, N = FINE_KEYS / ROWS_AT_ONCE; // a thread: N pieces of 8 columns, of rows ROWS_AT_ONCE apart
            const int mine = tid - 128, chunk = mine % CHUNKS, row0 = mine / CHUNKS;
            while (w.left > 0) {
                const ManyItem item = w.item(a, paged_seq(a.c, w.b));
                const int tiles = w.tiles(item), first = w.first(item);
                const int *ids = a.c.table + (long long)w.b * a.c.max_pages;
                const auto page_ids = [&](int (&id)[N], int u) { // the pages of a load's rows; -1: nothing to read
                    bool is_v;
                    const int pos = (item.t0 + first + load_of(u, tiles, &is_v)) * FINE_KEYS + row0;
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const int at = pos + i * ROWS_AT_ONCE;
                        id[i] = at >= item.low && at < item.high ? ids[at >> a.c.page_shift] : -1;
                        if (at >= item.low && at < item.high && (unsigned)id[i] >= (unsigned)a.c.pages) {
                            atomicExch(a.c.status, PAGED_BAD_PAGE);
                            id[i] = -1;
                        }
                    }
                };
                int id[N];
                page_ids(id, 0);
                for (int u = 0; u < 2 * tiles; u++, ld++) {
                    bool is_v;
                    const int tile = load_of(u, tiles, &is_v), slot = (int)(ld % SLOTS), pos = (item.t0 + first + tile) * FINE_KEYS + row0;
                    const float *from = static_cast<const float *>(is_v ? a.v : a.k);
                    float4 x[N][2];
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        x[i][0] = x[i][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (id[i] >= 0 && chunk * 8 < a.c.hd) {
                            const long long at = ((((long long)id[i] * a.c.kv + w.kvh) << a.c.page_shift) + ((pos + i * ROWS_AT_ONCE) & (page - 1))) * a.c.hd + chunk * 8;
                            x[i][0] = __ldg(reinterpret_cast<const float4 *>(from + at)), x[i][1] = __ldg(reinterpret_cast<const float4 *>(from + at + 4));
                        }
                    }
                    if (u + 1 < 2 * tiles) page_ids(id, u + 1);
                    if (alive && !pg_bar_wait(&empty[slot], ((ld / SLOTS) & 1u) ^ 1u)) {
                        atomicExch(a.c.status, PAGED_WAIT);
                        alive = false; // it goes on without waiting and without writing
                    }
                    if (!alive) continue;
                    unsigned char *dst = ring + slot * SLOT + (chunk >> 3) * HALF_COLS;
#pragma unroll
                    for (int i = 0; i < N; i++) {
                        const int row = row0 + i * ROWS_AT_ONCE;
                        unsigned p[4][3];
                        pg_split<3>(p[0], x[i][0].x, x[i][0].y), pg_split<3>(p[1], x[i][0].z, x[i][0].w);
                        pg_split<3>(p[2], x[i][1].x, x[i][1].y), pg_split<3>(p[3], x[i][1].z, x[i][1].w);
#pragma unroll
                        for (int k = 0; k < 3; k++)
                            *reinterpret_cast<uint4 *>(dst + k * TILE + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = make_uint4(p[0][k], p[1][k], p[2][k], p[3][k]);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    pg_bar_arrive(&full[slot]);
                }
                w.next(a);
            }
        } else if constexpr (std::is_same_v<CT, Int4>) { // the codes, written as bfloat16 words
            using Tile = Int4Tile<HDP, FINE_KEYS, 4, 1>;
            const Tile mine(warp - 4, lane);
            while (w.left > 0) {
                const ManyItem item = w.item(a, paged_seq(a.c, w.b));
                const int tiles = w.tiles(item), begin = (item.t0 + w.first(item)) * FINE_KEYS;
                int id[Tile::N], next_pos;
                typename Tile::Codes next;
                bool next_v;
                const auto look = [&](int p) { // the pages of part p of the item's loads
                    next_pos = begin + load_of(p / Tile::PARTS, tiles, &next_v) * FINE_KEYS + p % Tile::PARTS * (FINE_KEYS / Tile::PARTS);
                    mine.pages(id, a.c, w.b, next_pos, item.low, item.high);
                };
                look(0);
                mine.ask(next, id, a.c, w.kvh, next_v ? a.v : a.k, next_pos, item.low, item.high);
                look(1);
                const int all = 2 * tiles * Tile::PARTS;
                for (int p = 0; p < all; p++) {
                    const int slot = (int)(ld % SLOTS), part = p % Tile::PARTS;
                    const typename Tile::Codes codes = next;
                    if (p + 1 < all) mine.ask(next, id, a.c, w.kvh, next_v ? a.v : a.k, next_pos, item.low, item.high);
                    if (p + 2 < all) look(p + 2);
                    if (part == 0 && alive && !pg_bar_wait(&empty[slot], ((ld / SLOTS) & 1u) ^ 1u)) {
                        atomicExch(a.c.status, PAGED_WAIT);
                        alive = false; // it goes on without waiting and without writing
                    }
                    if (alive) mine.put(ring + slot * SLOT, part, codes);
                    if (part < Tile::PARTS - 1) continue;
                    ld++;
                    if (!alive) continue;
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    pg_bar_arrive(&full[slot]);
                }
                w.next(a);
            }
        }
    } else if (warp >= 8) { // ---------------- the products ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FINE_REGS_LESS));
        if (tid == 256) {
            unsigned ld = 0, items = 0, tile_count = 0;
            bool alive = true;
            const unsigned r0 = pg_smem(ring);
            const auto here = [&](unsigned long long *bar, unsigned parity) {
                if (alive && !pg_bar_wait(bar, parity)) alive = false;
                pg_fence_after();
                return alive;
            };
            const auto score = [&](unsigned i, unsigned buffer) { // S = Q K^T, K being load i
                const unsigned d = tmem + S_AT + buffer * S_COLS;
                bool add = false;
#pragma unroll 1
                for (int places = 2; places >= 0; places--) // of the pieces of both together: the smallest products first
#pragma unroll 1
                    for (int k = 0; k < CP && k <= places; k++) {
                        const unsigned kd = pg_desc_low(r0 + (i % SLOTS) * SLOT + k * TILE), qa = tmem + (places - k) * Q_COLS;
#pragma unroll
                        for (int ks = 0; ks < HDP / 16; ks++) {
                            pg_mma_ts(d, qa + ks * 8, pg_desc(kd + ((ks >> 2) * HALF_COLS + (ks & 3) * 32) / 16), pg_idesc(FINE_KEYS, false), add);
                            add = true;
                        }
                    }
                pg_commit(&empty[i % SLOTS]);
                pg_commit(&s_full[buffer]);
            };
            const auto value = [&](unsigned i, unsigned buffer) { // O = P V, V being load i
                bool add = false;
#pragma unroll 1
                for (int places = 2; places >= 0; places--)
#pragma unroll 1
                    for (int k = 0; k < CP && k <= places; k++) {
                        const int piece = places - k, next = piece < 2 ? 32 : 16; // columns from 32 keys' piece to the next 32 keys'
                        const unsigned vd = pg_desc_low(r0 + (i % SLOTS) * SLOT + k * TILE, HALF_COLS), pa = tmem + S_AT + buffer * S_COLS + (piece < 2 ? piece * 16 : 64);
#pragma unroll
                        for (int ks = 0; ks < FINE_KEYS / 16; ks++) {
                            pg_mma_ts(tmem + O_AT, pa + (ks >> 1) * next + (ks & 1) * 8, pg_desc(vd + ks * 2048 / 16), pg_idesc(HDP, true), add);
                            add = true;
                        }
                    }
                pg_commit(&empty[i % SLOTS]);
                pg_commit(o_full);
            };
            while (w.left > 0 && alive) {
                const int tiles = w.tiles(w.item(a, paged_seq(a.c, w.b)));
                here(q_full, items & 1u);
                items++;
                const unsigned t0 = tile_count; // tiles done before the item: the buffers and barriers go on from item to item
                for (int j = 0; j < min(2, tiles) && alive; j++)
                    if (here(&full[ld % SLOTS], (ld / SLOTS) & 1u)) score(ld++, (t0 + j) & 1u);
                for (int j = 0; j < tiles && alive; j++) {
                    const unsigned t = t0 + j;
                    if (!here(&full[ld % SLOTS], (ld / SLOTS) & 1u) || !here(&p_full[t & 1u], (t >> 1) & 1u) || !here(o_free, (t & 1u) ^ 1u)) break; // O of the tile before is read
                    value(ld++, t & 1u);
                    if (j + 2 < tiles && here(&full[ld % SLOTS], (ld / SLOTS) & 1u)) score(ld++, t & 1u);
                }
                tile_count += tiles;
                if (alive) w.next(a);
            }
            if (!alive) { // products in flight end before their tensor memory is given back
                atomicExch(a.c.status, PAGED_WAIT);
                pg_commit(done);
                pg_bar_wait(done, 0);
            }
        }
        if (warp == 9) { // ---------------- the queries of the next item, while this one's keys are worked on ----------------
            unsigned items = 0;
            while (w.left > 0) {
                const PagedSeq s = paged_seq(a.c, w.b);
                const ManyItem item = w.item(a, s);
                if (!__all_sync(0xFFFFFFFFu, pg_bar_wait(stage_empty, (items & 1u) ^ 1u))) {
                    if (lane == 0) atomicExch(a.c.status, PAGED_WAIT);
                    break;
                }
                if (lane == 0) pg_bar_expect(stage_full, (unsigned)(item.rows * a.c.hd * 4));
                __syncwarp();
                for (int r = lane; r < item.rows; r += 32) {
                    const int2 at = many_row(a, item, r);
                    const float *src = static_cast<const float *>(a.q) + (long long)(s.first + at.x) * a.ldq + (w.kvh * a.c.group + at.y) * a.c.hd;
                    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(pg_smem(stage + r * Shape::PITCH)), "l"(src),
                                 "r"(a.c.hd * 4), "r"(pg_smem(stage_full))
                                 : "memory");
                }
                items++;
                w.next(a);
            }
            if (items > 0) pg_bar_wait(stage_full, (items - 1) & 1u); // copies in flight end before the block does, whoever has given up
        }
        __syncwarp();
    } else { // ---------------- the softmax: a thread a row ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FINE_REGS));
        const unsigned at = tmem + ((unsigned)(warp * 32) << 16);
        const float unit = a.scale * PAGED_LOG2E;
        unsigned tile_count = 0;
        bool alive = true, first_part = true;
        const auto give_up = [&] {
            if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
            alive = false; // it goes on without waiting; nothing of the block is stored from here on
        };
        unsigned char *const mine = stage + tid * Shape::PITCH;
        unsigned items = 0;
        const auto queries = [&](int rows) { // an item's rows from where they were brought to, as pieces into tensor memory: a thread its own
            if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(stage_full, items & 1u))) give_up();
            items++;
            if (!alive) return;
            const bool valid = tid < rows;
#pragma unroll 1
            for (int c = 0; c < HDP; c += 16) {
                unsigned p[3][8];
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (valid && c + i < a.c.hd) x = *reinterpret_cast<const float4 *>(mine + (c + i) * 4);
                    if (a.flip) x = make_float4(-x.x, -x.y, -x.z, -x.w);
                    unsigned lo[3], hi[3];
                    pg_split<3>(lo, x.x, x.y);
                    pg_split<3>(hi, x.z, x.w);
#pragma unroll
                    for (int k = 0; k < 3; k++) p[k][i / 2] = lo[k], p[k][i / 2 + 1] = hi[k];
                }
#pragma unroll
                for (int k = 0; k < 3; k++) pg_st8(at + k * Q_COLS + c / 2, p[k]);
            }
            pg_wait_st();
            pg_fence_before();
            pg_bar_arrive(q_full);
        };
        if (w.left > 0) {
            queries(w.item(a, paged_seq(a.c, w.b)).rows);
            if (alive) pg_bar_arrive(stage_empty); // for the second item's; the place is free again for the one after next when an item's output has left it
        }
        while (w.left > 0) {
            const PagedSeq s = paged_seq(a.c, w.b);
            const ManyItem item = w.item(a, s);
            const int tiles = w.tiles(item), first = w.first(item);
            const bool valid = tid < item.rows;
            const int2 place = many_row(a, item, tid);
            if (s.n > a.max_new && tid == 0) atomicExch(a.c.status, PAGED_BAD_BOUND);
            const int hi = valid ? s.pos0 + place.x + 1 : 0, lo = a.window ? hi - a.window : 0;
            float m = -INFINITY, l = 0.0f;
            unsigned long long o[HDP / 2]; // two columns each
#pragma unroll
            for (int c = 0; c < HDP / 2; c++) o[c] = 0;
            const auto take = [&](unsigned t) { // o += the output of tile t
                if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(o_full, t & 1u))) give_up();
                if (!alive) return;
                pg_fence_after();
#pragma unroll
                for (int c = 0; c < HDP; c += 32) {
                    unsigned v[32];
                    pg_ld32(v, at + O_AT + c);
                    pg_wait_ld(v);
#pragma unroll
                    for (int i = 0; i < 32; i += 2) o[(c + i) / 2] = pg_add2(o[(c + i) / 2], pg_two(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
                }
                pg_fence_before();
                pg_bar_arrive(o_free);
            };
            for (int j = 0; j < tiles; j++) {
                const unsigned t = tile_count + j, s_at = at + S_AT + (t & 1u) * S_COLS;
                const int pos = (item.t0 + first + j) * FINE_KEYS;
                if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&s_full[t & 1u], (t >> 1) & 1u))) give_up();
                if (!alive) continue;
                pg_fence_after();
                const bool edge = __any_sync(0xFFFFFFFFu, valid && (pos + FINE_KEYS > hi || pos < lo));
                unsigned z[32];
                float *x = reinterpret_cast<float *>(z), top[2] = {-INFINITY, -INFINITY};
                const auto hide = [&](int c) {
                    if (!edge) return;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (pos + c + i >= hi || pos + c + i < lo) x[i] = -INFINITY;
                };
#pragma unroll
                for (int c = 32; c >= 0; c -= 32) { // the largest score; the first columns come last and stay for their weights
                    pg_ld32(z, s_at + c);
                    pg_wait_ld(z);
                    hide(c);
#pragma unroll
                    for (int i = 0; i < 32; i += 4) top[0] = pg_max3(top[0], x[i], x[i + 1]), top[1] = pg_max3(top[1], x[i + 2], x[i + 3]);
                }
                float most = fmaxf(top[0], top[1]);
                if (a.softcap > 0.0f) pg_cap_fine<2>(top, a), most = max(lo, pos) < min(hi, pos + FINE_KEYS) ? fmaxf(top[0], top[1]) : -INFINITY; // (nothing is seen)
                most *= unit;
                const float to = most > m ? most : m, keep = m == -INFINITY ? 0.0f : paged_exp2(m - to), base = to == -INFINITY ? 0.0f : to;
                const unsigned long long unit2 = pg_two(unit, unit), base2 = pg_two(-base, -base);
                unsigned long long sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 64; c += 32) {
                    if (c) {
                        pg_ld32(z, s_at + c);
                        pg_wait_ld(z);
                    }
                    if (a.softcap > 0.0f) pg_cap_fine<32>(x, a);
                    if (c || a.softcap > 0.0f) hide(c);
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        unsigned p[3][8];
#pragma unroll
                        for (int i = 0; i < 16; i += 2) {
                            float w0, w1;
                            pg_one(pg_fma2(pg_two(x[16 * h + i], x[16 * h + i + 1]), unit2, base2), w0, w1);
                            w0 = paged_exp2(w0), w1 = paged_exp2(w1);
                            sum[(i / 2) & 1] = pg_add2(sum[(i / 2) & 1], pg_two(w0, w1));
                            unsigned piece[3];
                            pg_split<3>(piece, w0, w1);
#pragma unroll
                            for (int k = 0; k < 3; k++) p[k][i / 2] = piece[k];
                        }
                        // over columns of S that have been read, and the 32 behind it: 32 keys' pieces at c, c + 16 and 64 + c / 2
                        pg_st8(s_at + c + 8 * h, p[0]), pg_st8(s_at + c + 16 + 8 * h, p[1]), pg_st8(s_at + 64 + c / 2 + 8 * h, p[2]);
                    }
                }
                pg_wait_st();
                pg_fence_before();
                pg_bar_arrive(&p_full[t & 1u]);
                float s0, s1;
                pg_one(pg_add2(sum[0], sum[1]), s0, s1);
                l = fmaf(l, keep, s0 + s1);
                if (j > 0) take(t - 1);
                if (__any_sync(0xFFFFFFFFu, to > m)) {
#pragma unroll
                    for (int c = 0; c < HDP / 2; c++) o[c] = pg_mul2(o[c], pg_two(keep, keep));
                }
                m = to;
            }
            tile_count += tiles;
            const bool is_whole = w.skip == 0 && w.steps(item) == item.steps;
            const long long slot = (long long)blockIdx.x * 2 + (first_part && w.skip > 0 ? 0 : 1);
            if (!is_whole && valid) {
                float *ml = f.part + (long long)gridDim.x * 2 * BR * HDP + slot * 2 * BR;
                ml[tid] = m, ml[BR + tid] = l;
            }
            if (!is_whole && tid == 0 && w.skip == 0 && alive && !dead) {
                int *head = f.head + blockIdx.x * 8;
                head[0] = w.b, head[1] = w.kvh, head[2] = w.block, head[3] = item.steps, head[4] = w.line, head[5] = (int)line.per;
            }
            const int kvh = w.kvh;
            w.next(a);
            if (w.left > 0) queries(w.item(a, paged_seq(a.c, w.b)).rows); // the scores that read the last ones are done: the next item's begin under what follows
            take(tile_count - 1);

            // ---- the item's (or its part's) end: the row goes out the way its query came ----
            const float share = !is_whole ? 1.0f : paged_share(l, s.pos0 + place.x); // (where nothing is seen, O is zero, or not finite and done again)
            unsigned long long odd = 0; // zero times what is stored: NaN where that is not finite
            const unsigned long long share2 = pg_two(share, share);
#pragma unroll
            for (int c = 0; c < HDP; c += 4) {
                const unsigned long long y0 = pg_mul2(o[c / 2], share2), y1 = pg_mul2(o[c / 2 + 1], share2);
                odd = pg_fma2(y0, 0, odd), odd = pg_fma2(y1, 0, odd);
                *reinterpret_cast<ulonglong2 *>(mine + c * 4) = make_ulonglong2(y0, y1);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            const bool store = valid && alive && !dead;
            if (store) {
                float *to = is_whole ? static_cast<float *>(a.out) + ((long long)(s.first + place.x) * a.c.heads + kvh * a.c.group + place.y) * a.c.hd : f.part + (slot * BR + tid) * HDP;
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(to), "r"(pg_smem(mine)), "r"(is_whole ? a.c.hd * 4 : HDP * 4) : "memory");
            }
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            if (alive) pg_bar_arrive(stage_empty); // (a place whose rows it has not waited for is not given back)
            float odd0, odd1;
            pg_one(odd, odd0, odd1);
            unsigned rest = __ballot_sync(0xFFFFFFFFu, store && is_whole && !(odd0 + odd1 == 0.0f));
            // A masked key's zero weight met a value that is not finite, or a 32-bit word left bfloat16's range: the row is done again after this kernel. Row by
            // row with its place: where a thread only stores a word, the compiler's code for the softmax of float32 caches takes 293 us for 222.
            while (rest) {
                const int k = __ffs(rest) - 1, token = __shfl_sync(0xFFFFFFFFu, place.x, k), head = __shfl_sync(0xFFFFFFFFu, place.y, k);
                rest &= rest - 1;
                many_mark(f.head + blockIdx.x * 8 + 6, (s.first + token) * a.c.heads + kvh * a.c.group + head);
            }
            first_part = false;
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); // what leaves shared memory has left it
    }
    pg_fence_before();
    __syncthreads();
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// ---- host side ----
template <typename CT, int HDP>
cudaError_t launch_fine_as(const AttendCall &a, const ManyPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    using Shape = FineShape<CT, HDP>;
    ManyCall f;
    f.a = a, f.part = static_cast<float *>(ws), f.head = reinterpret_cast<int *>(static_cast<float *>(ws) + p.part_floats);
    alignas(64) CUtensorMap map_k = {}, map_v = {}; // (of a cache in 4 bits nothing is copied by them)
    const long long rows = ((long long)a.c.pages * a.c.kv) << a.c.page_shift;
    const int box = std::min(1 << a.c.page_shift, FINE_KEYS);
    constexpr bool f32 = std::is_same_v<CT, float>;
    if constexpr (!std::is_same_v<CT, Int4>)
        if (!paged_map(&map_k, a.k, rows, a.c.hd, f32, box) || !paged_map(&map_v, a.v, rows, a.c.hd, f32, box)) return cudaErrorNotSupported;
    static std::atomic<bool> known[64];
    if (device >= 64 || !known[device].load()) {
        const cudaError_t e = cudaFuncSetAttribute(attend_fine_kernel<CT, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
        if (e != cudaSuccess) return e;
        if (device < 64) known[device].store(true);
    }
    attend_fine_kernel<CT, HDP><<<p.blocks, FINE_THREADS, Shape::SMEM, st>>>(map_k, map_v, f);
    return many_after<float, CT, HDP, FINE_ROWS, FINE_KEYS, 1>(f, p.blocks, st, launches);
}

} // namespace b200i

// Attention of many rows over a paged cache on the tcgen05 tensor cores: prompts, and chunks of new tokens behind what is cached.
//
//   z = scale Q K^T (capped),   O = 2^(z log2 e - m) V / sum 2^(z log2 e - m),   128 rows by 128 keys at a time
//
// Bound: the tensor pipe, 4 head_dim operations a (row, key), and beside it the exponentials: 16 a clock on an SM against 8192
// operations, so at head_dim 128 the two pipes need the same time and neither may wait for the other.
// Rows. A row is a (token, head of the key head's group), so grouped heads share the keys that are brought in.
// Block. Two streams, each of four softmax warps (a thread a row), an S of 128 columns and an O of head_dim columns in tensor memory: while one
// stream's softmax runs, the other's products do. A block of more than 128 rows gives each stream 128 of them and the same keys; one
// of up to 128 gives both streams the rows, and every other tile of keys each, and joins the two at the end. One thread issues
// the products: S = Q K^T from shared memory, O += P V with P (bfloat16, over the columns of S that it came from) read from tensor
// memory and V as it lies, keys down. One warp copies keys and values: tensor-map boxes of 128 bytes by a page's rows into a ring.
// The running maximum is moved, and O multiplied by what that costs, only when a row's maximum has grown by more than 2^8: weights
// up to 2^8 are as exact, and a product of O by one is saved. S of the next tile is signalled after the products before it are done,
// so O stands still while a softmax warp has an S in hand.
// Work is cut as in paged_few.cuh: all items' steps on one line, an equal piece a block, parts joined by attend_join_rows_kernel.
#pragma once
#include "paged_few.cuh"

namespace b200i {

constexpr int MANY_THREADS = 384, MANY_KEYS = 128; // two streams' softmax, and a group of warps of which one copies and one issues
constexpr int MANY_REGS = 208, MANY_REGS_LESS = 88;  // a thread: 2 x 208 + 88 = 504 = 3 x 168, what the block is launched with

template <int HDP> struct ManyShape {
    static constexpr int TILE = HDP * 256;     // bytes of 128 rows of bfloat16
    static constexpr int QUERY = 2 * TILE;     // a stream each; the streams' meeting place too
    static constexpr int BLOCK_ROWS = 256;
    static constexpr int ROOM = (226 * 1024 - 1024 - 4096 - QUERY) / TILE;
    static constexpr int SLOTS = ROOM > 8 ? 8 : ROOM;
    static constexpr int SMEM = 1024 + QUERY + SLOTS * TILE + 256;
};

// A descriptor of a tile of 128-byte swizzled rows (groups of eight 1024 bytes apart) from the lower word that pg_desc_low makes of its
// address; steps within the tile are added to that, in units of 16 bytes. K-major, or with its rows as the contraction, where
// `next` are the bytes from 64 columns to the next 64.
__device__ __forceinline__ unsigned pg_desc_low(unsigned addr, unsigned next = 16) { return ((addr & 0x3FFFFu) >> 4) | ((next >> 4) << 16); }
__device__ __forceinline__ unsigned long long pg_desc(unsigned low) {
    unsigned long long d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "n"((1024 >> 4) | (1 << 14) | (2 << 29)));
    return d;
}
// 32-bit sums of bfloat16 products, 128 rows; turned: B's rows are the contraction
__host__ __device__ constexpr unsigned pg_idesc(int n, bool turned) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (turned ? 1u << 16 : 0u) | ((unsigned)(n >> 3) << 17) | (8u << 24);
}
__device__ __forceinline__ void pg_mma_ss(unsigned d, unsigned long long a, unsigned long long b, unsigned idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
                 : "memory");
}
__device__ __forceinline__ void pg_mma_ts(unsigned d, unsigned a, unsigned long long b, unsigned idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((unsigned)add)
                 : "memory");
}
__device__ __forceinline__ void pg_commit(unsigned long long *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(pg_smem(bar)) : "memory");
}
__device__ __forceinline__ void pg_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pg_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void pg_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pg_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define PG_R8(v, i) "r"((v)[i]), "r"((v)[i + 1]), "r"((v)[i + 2]), "r"((v)[i + 3]), "r"((v)[i + 4]), "r"((v)[i + 5]), "r"((v)[i + 6]), "r"((v)[i + 7])
#define PG_W8(v, i) "=r"((v)[i]), "=r"((v)[i + 1]), "=r"((v)[i + 2]), "=r"((v)[i + 3]), "=r"((v)[i + 4]), "=r"((v)[i + 5]), "=r"((v)[i + 6]), "=r"((v)[i + 7])
// 32 columns of a lane's row
__device__ __forceinline__ void pg_ld32(unsigned *v, unsigned taddr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, "
        "%27, %28, %29, %30, %31}, [%32];"
        : PG_W8(v, 0), PG_W8(v, 8), PG_W8(v, 16), PG_W8(v, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void pg_st32(unsigned taddr, const unsigned *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, "
        "%27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        PG_R8(v, 0), PG_R8(v, 8), PG_R8(v, 16), PG_R8(v, 24)
        : "memory");
}
__device__ __forceinline__ void pg_st16(unsigned taddr, const unsigned *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), PG_R8(v, 0), PG_R8(v, 8)
        : "memory");
}
__device__ __forceinline__ void pg_st8(unsigned taddr, const unsigned *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), PG_R8(v, 0) : "memory");
}

// x = tanh(x inner) of a row's N scores. Where all of a warp's are within 0.35, as capped scores mostly are, by the series x - x^3 / 3 + 2 x^5 / 15
// - 17 x^7 / 315 + 62 x^9 / 2835 - 1382 x^11 / 155925, whose next term is 1.2e-8 of x there; elsewhere sign(x) (1 - 2 / (1 + e^{2 |x|})).
template <int N>
__device__ __forceinline__ void pg_tanh(float *x, float inner) {
    float most = 0.0f;
#pragma unroll
    for (int c = 0; c < N; c++) {
        x[c] *= inner;
        most = fmaxf(most, fabsf(x[c]));
    }
    const auto series = [](float v) {
        const float q = v * v;
        float s = fmaf(q, -1382.0f / 155925.0f, 62.0f / 2835.0f);
        s = fmaf(q, s, -17.0f / 315.0f), s = fmaf(q, s, 2.0f / 15.0f), s = fmaf(q, s, -1.0f / 3.0f);
        return fmaf(v * q, s, v);
    };
    if (!__any_sync(0xFFFFFFFFu, most > 0.35f)) {
#pragma unroll
        for (int c = 0; c < N; c++) x[c] = series(x[c]);
    } else {
#pragma unroll
        for (int c = 0; c < N; c++) {
            const float e = paged_exp2(fabsf(x[c]) * (2.0f * PAGED_LOG2E)), far = copysignf(1.0f - __fdividef(2.0f, 1.0f + e), x[c]);
            x[c] = fabsf(x[c]) > 0.35f ? (e > 1e30f ? copysignf(1.0f, x[c]) : far) : series(x[c]);
        }
    }
}

// An item: up to BR rows of one sequence and key head, over tiles of KEYS keys.
struct ManyItem {
    int row0, rows;    // of the sequence and key head
    int t0, tiles;     // tiles that some row sees
    int low, high;     // and positions
    bool pair;         // a step is a tile; else (two streams, and rows for one) two tiles, one a stream
    int steps;
};
template <int BR, int KEYS, int STREAMS>
__device__ __forceinline__ ManyItem many_item(const AttendCall &a, const PagedSeq &s, int n, int block) {
    ManyItem i;
    i.row0 = block * BR, i.rows = min(n * a.c.group - i.row0, BR);
    const int first = i.row0 / a.c.group, last = (i.row0 + i.rows - 1) / a.c.group;
    i.high = min(s.length, max(s.pos0 + last + 1, 0));
    i.low = a.window ? min(max(s.pos0 + first + 1 - a.window, 0), i.high) : 0;
    i.t0 = i.low / KEYS;
    i.tiles = max(1, (i.high + KEYS - 1) / KEYS - i.t0); // rows that see nothing: one tile, masked
    i.pair = STREAMS == 1 || i.rows > BR / 2;
    i.steps = i.pair ? i.tiles : (i.tiles + 1) / 2;
    return i;
}
__device__ __forceinline__ int many_blocks(const AttendCall &a, int n, int block_rows) { return (int)(((long long)n * a.c.group + block_rows - 1) / block_rows); }

// A block's way along the line of all items' steps; every warp of the block goes it by itself.
template <int BR, int KEYS, int STREAMS> struct ManyWalk {
    int b, kvh, block, blocks, n;
    PagedSeq s;
    ManyItem item;
    int skip;          // steps of the item that other blocks do before this one
    long long left;    // steps of the block from here
    long long line;    // where on the line the item begins

    static __device__ __forceinline__ long long steps_of(const AttendCall &a, int b) {
        const PagedSeq s = paged_seq(a.c, b);
        const int n = min(s.n, a.max_new), blocks = many_blocks(a, n, BR);
        long long sum = 0;
        for (int i = 0; i < blocks; i++) sum += many_item<BR, KEYS, STREAMS>(a, s, n, i).steps;
        return sum;
    }
    __device__ __forceinline__ void begin(const AttendCall &a, const LinePlace &p) {
        b = p.b, kvh = p.kvh, block = 0, left = p.left, line = p.start - p.in, skip = 0;
        if (left <= 0) return;
        long long in = p.in;
        sequence(a);
        item = many_item<BR, KEYS, STREAMS>(a, s, n, 0);
        while (in >= item.steps) in -= item.steps, line += item.steps, item = many_item<BR, KEYS, STREAMS>(a, s, n, ++block);
        skip = (int)in;
    }
    __device__ __forceinline__ void sequence(const AttendCall &a) { s = paged_seq(a.c, b), n = min(s.n, a.max_new), blocks = many_blocks(a, n, BR); }
    __device__ __forceinline__ int steps() const { return (int)min((long long)(item.steps - skip), left); } // that the block does of the item
    __device__ __forceinline__ int first() const { return item.pair ? skip : 2 * skip; }                    // its first tile
    __device__ __forceinline__ int tiles() const { return min(item.pair ? skip + steps() : 2 * (skip + steps()), item.tiles) - first(); }
    __device__ __forceinline__ void next(const AttendCall &a) {
        left -= steps();
        if (left <= 0) return;
        line += item.steps, skip = 0;
        if (++block >= blocks) {
            block = 0;
            if (++kvh >= a.c.kv) {
                kvh = 0, b++;
                while (b + 1 < a.c.batch && paged_seq(a.c, b).n == 0) b++;
                sequence(a);
            }
        }
        item = many_item<BR, KEYS, STREAMS>(a, s, n, block);
    }
};

struct ManyCall {
    AttendCall a;
    float *part; // [blocks][2][BLOCK_ROWS][HDP], then [blocks][2][2][BLOCK_ROWS] of m and l
    int *head;   // [blocks][8]: sequence (or -1), key head, block of rows, steps, steps of the block before it, steps a block
};

template <int HDP>
__global__ void __launch_bounds__(MANY_THREADS, 1) attend_many_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const ManyCall f) {
    using Shape = ManyShape<HDP>;
    constexpr int SLOTS = Shape::SLOTS, TILE = Shape::TILE, BOXES = HDP / 64, BR = Shape::BLOCK_ROWS, HALF_COLS = 128 * 128; // bytes of a tile's 64 columns
    using T = __nv_bfloat16; // of rows and cache
    using Walk = ManyWalk<BR, MANY_KEYS, 2>;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char *query = smem + ((1024u - (pg_smem(smem) & 1023u)) & 1023u), *ring = query + Shape::QUERY;
    unsigned long long *full = reinterpret_cast<unsigned long long *>(ring + SLOTS * TILE), *empty = full + SLOTS;
    unsigned long long *s_full = empty + SLOTS, *p_full = s_full + 2, *o_full = p_full + 2, *q_full = o_full + 2, *tail = q_full + 1; // 2 SLOTS + 8 <= 32 words
    __shared__ float stats[2][2][128];
    __shared__ long long place[16];
    __shared__ unsigned tmem_slot;
    __shared__ int dead;
    const AttendCall &a = f.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < SLOTS; s++) {
            pg_bar_init(&full[s], 1);
            pg_bar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            pg_bar_init(&s_full[i], 1);
            pg_bar_init(&p_full[i], 128);
            pg_bar_init(&o_full[i], 1);
        }
        pg_bar_init(q_full, 256);
        pg_bar_init(tail, 1);
        dead = 0;
        f.head[blockIdx.x * 8] = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pg_smem(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const LinePlace line = line_place(a.c, [&](int b) { return Walk::steps_of(a, b); }, blockIdx.x, gridDim.x, place);
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const unsigned tmem = tmem_slot;
    const int page = 1 << a.c.page_shift, box_rows = min(page, MANY_KEYS);
    Walk w;
    w.begin(a, line);
    const ManyItem &item = w.item;

    if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(MANY_REGS_LESS));
    if (warp == 8) { // ---------------- the copies ----------------
        unsigned ld = 0, tails = 0;
        bool alive = true;
        while (w.left > 0 && alive) {
            const int tiles = w.tiles(), first = w.first();
            const int last_page = (item.high - 1) >> a.c.page_shift;
            const int *ids = a.c.table + (long long)w.b * a.c.max_pages;
            // in the order of their first use: K0 V0 K1 V1 ..., or K0 K1 V0 K2 V1 K3 ... where the streams have tiles of their own
            const int lead = min(item.pair ? 1 : 2, tiles);
            for (int u = 0; u < 2 * tiles && alive; u++, ld++) {
                const int v = u - lead; // after the first keys: values, then keys, as long as there are any
                const bool paired = v < 2 * (tiles - lead);
                const bool is_v = v >= 0 && (paired ? (v & 1) == 0 : true);
                const int tile = v < 0 ? u : (paired ? (is_v ? v / 2 : v / 2 + lead) : (tiles - lead) + (v - 2 * (tiles - lead)));
                const int slot = (int)(ld % SLOTS), pos = (item.t0 + first + tile) * MANY_KEYS;
                if (!__all_sync(0xFFFFFFFFu, pg_bar_wait(&empty[slot], ((ld / SLOTS) & 1u) ^ 1u))) {
                    if (lane == 0) atomicExch(a.c.status, PAGED_WAIT);
                    alive = false;
                    break;
                }
                const int there = min(MANY_KEYS / box_rows, max(0, (item.high - pos + box_rows - 1) / box_rows)); // pieces that hold positions that some row sees
                unsigned char *dst = ring + slot * TILE;
                const bool clean = is_v && (pos + MANY_KEYS > item.high || pos < item.low); // rows of values that no row sees are to be zero
                unsigned long long *bar = clean ? tail : &full[slot];
                if (lane == 0) pg_bar_expect(bar, (unsigned)(there * box_rows * 128 * BOXES));
                __syncwarp();
                for (int x = lane; x < there * BOXES; x += 32) {
                    const int piece = x / BOXES, box = x % BOXES, at = pos + piece * box_rows, index = at >> a.c.page_shift;
                    int row = a.c.pages * a.c.kv * page; // past the pool: zeros
                    const int id = index <= last_page ? ids[index] : -1;
                    if ((unsigned)id < (unsigned)a.c.pages)
                        row = ((id * a.c.kv + w.kvh) << a.c.page_shift) + (at & (page - 1));
                    else
                        atomicExch(a.c.status, PAGED_BAD_PAGE);
                    pg_tma_load(dst + box * HALF_COLS + piece * (box_rows * 128), is_v ? &map_v : &map_k, bar, box * 64, row);
                }
                if (clean) {
                    if (!__all_sync(0xFFFFFFFFu, pg_bar_wait(tail, tails & 1u))) {
                        if (lane == 0) atomicExch(a.c.status, PAGED_WAIT);
                        alive = false;
                        break;
                    }
                    tails++;
                    for (int x = lane; x < 128 * 8 * BOXES; x += 32) { // 16 bytes each; a row's are in one swizzle atom, so their order does not matter
                        const int at = pos + ((x >> 3) & 127);
                        if (at >= item.high || at < item.low) *reinterpret_cast<uint4 *>(dst + (x >> 10) * HALF_COLS + (x & 1023) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) pg_bar_arrive(&full[slot]);
                }
            }
            if (alive) w.next(a);
        }
        if (!alive) // copies in flight end before the block does
            for (unsigned i = ld > (unsigned)SLOTS ? ld - SLOTS : 0; i < ld; i++) pg_bar_wait(&full[i % SLOTS], (i / SLOTS) & 1u);
    } else if (warp == 9) { // ---------------- the products ----------------
        if (lane == 0) {
            unsigned ld = 0, items = 0, p_count[2] = {0, 0};
            bool alive = true;
            const unsigned q0 = pg_smem(query), r0 = pg_smem(ring);
            const auto here = [&](unsigned i) { // a load is there
                if (alive && !pg_bar_wait(&full[i % SLOTS], (i / SLOTS) & 1u)) alive = false;
                pg_fence_after();
            };
            const auto score = [&](int stream, unsigned i, bool pair) { // S = Q K^T, K being load i
                const unsigned k = pg_desc_low(r0 + (i % SLOTS) * TILE), d = tmem + stream * 128;
                const unsigned q = pg_desc_low(q0 + (pair ? stream : 0) * TILE);
#pragma unroll
                for (int ks = 0; ks < HDP / 16; ks++)
                    pg_mma_ss(d, pg_desc(q + ((ks >> 2) * HALF_COLS + (ks & 3) * 32) / 16), pg_desc(k + ((ks >> 2) * HALF_COLS + (ks & 3) * 32) / 16), pg_idesc(128, false), ks > 0);
                pg_commit(&s_full[stream]);
            };
            const auto value = [&](int stream, unsigned i, bool add) { // O += P V, V being load i
                const unsigned v = pg_desc_low(r0 + (i % SLOTS) * TILE, HALF_COLS), d = tmem + 256 + stream * 128;
#pragma unroll
                for (int ks = 0; ks < 8; ks++) pg_mma_ts(d, tmem + stream * 128 + ks * 8, pg_desc(v + ks * 2048 / 16), pg_idesc(HDP, true), add || ks > 0);
            };
            const auto weights = [&](int stream) { // the stream's P is there
                if (alive && !pg_bar_wait(&p_full[stream], p_count[stream] & 1u)) alive = false;
                p_count[stream]++;
                pg_fence_after();
            };
            while (w.left > 0 && alive) {
                const int tiles = w.tiles(), first = w.first();
                if (!pg_bar_wait(q_full, items & 1u)) alive = false;
                items++;
                pg_fence_after();
                if (item.pair) {
                    unsigned k = ld++, v;
                    here(k);
                    if (alive) score(0, k, true), score(1, k, true), pg_commit(&empty[k % SLOTS]);
                    for (int j = 0; j < tiles && alive; j++) {
                        v = ld++;
                        here(v);
                        if (j + 1 < tiles) k = ld++;
                        for (int stream = 0; stream < 2 && alive; stream++) {
                            weights(stream);
                            if (!alive) break;
                            value(stream, v, j > 0);
                            if (stream == 1) pg_commit(&empty[v % SLOTS]);
                            if (j + 1 < tiles) {
                                if (stream == 0) here(k);
                                if (!alive) break;
                                score(stream, k, true);
                                if (stream == 1) pg_commit(&empty[k % SLOTS]);
                            } else {
                                pg_commit(&o_full[stream]);
                            }
                        }
                    }
                } else {
                    for (int j = 0; j < min(2, tiles) && alive; j++, ld++) {
                        here(ld);
                        if (alive) score(j, ld, false), pg_commit(&empty[ld % SLOTS]);
                    }
                    for (int j = 0; j < tiles && alive; j++) {
                        const int stream = j & 1;
                        here(ld);
                        weights(stream);
                        if (!alive) break;
                        value(stream, ld, j > 1);
                        pg_commit(&empty[ld % SLOTS]);
                        ld++;
                        if (j + 2 < tiles) {
                            here(ld);
                            if (!alive) break;
                            score(stream, ld, false);
                            pg_commit(&empty[ld % SLOTS]);
                            ld++;
                        } else {
                            pg_commit(&o_full[stream]);
                        }
                    }
                }
                if (alive) w.next(a);
            }
            if (!alive) atomicExch(a.c.status, PAGED_WAIT);
        }
        __syncwarp();
    }
    } else { // ---------------- the softmax of a stream: a thread a row ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY_REGS));
        const int stream = warp >> 2, r = tid & 127;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, s_at = tmem + lanes + stream * 128, o_at = tmem + lanes + 256 + stream * 128;
        const float unit = a.softcap > 0.0f ? a.softcap * PAGED_LOG2E : a.scale * PAGED_LOG2E, inner = a.softcap > 0.0f ? a.scale / a.softcap : 0.0f;
        unsigned s_count = 0, o_count = 0;
        bool alive = true, first_part = true;
        while (w.left > 0) {
            const int tiles = w.tiles(), first = w.first();
            if (w.s.n > a.max_new && tid == 0) atomicExch(a.c.status, PAGED_BAD_BOUND);
            // the rows into shared memory, K-major and swizzled; a stream its own rows, or half of the columns of the shared ones
            {
                constexpr int CHUNKS = HDP / 8; // 16 bytes of bfloat16
                const int tile = item.pair ? stream : 0;
                for (int u = r; u < 128 * CHUNKS; u += 128) {
                    const int row = u / CHUNKS, chunk = u % CHUNKS, at = item.row0 + tile * 128 + row;
                    if (!item.pair && (chunk & 1) != stream) continue;
                    const T *src = static_cast<const T *>(a.q) + (long long)(w.s.first + at / a.c.group) * a.ldq + (long long)(w.kvh * a.c.group + at % a.c.group) * a.c.hd + chunk * 8;
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (tile * 128 + row < item.rows && chunk * 8 < a.c.hd) x = *reinterpret_cast<const uint4 *>(src);
                    *reinterpret_cast<uint4 *>(query + tile * TILE + (chunk >> 3) * HALF_COLS + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) = x;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                pg_bar_arrive(q_full);
            }
            const int mine = (item.pair ? stream * 128 : 0) + r, row = item.row0 + mine;
            const bool valid = mine < item.rows;
            const int hi = valid ? w.s.pos0 + row / a.c.group + 1 : 0, lo = a.window ? hi - a.window : 0;
            float m = -INFINITY, l = 0.0f;
            int taken = 0;
            for (int j = item.pair ? 0 : stream; j < tiles; j += item.pair ? 1 : 2, taken++) {
                const int pos = (item.t0 + first + j) * MANY_KEYS;
                if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&s_full[stream], s_count & 1u))) {
                    if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
                    alive = false; // it goes on without waiting, so that the others meet it; nothing of the block is stored from here on
                }
                s_count++;
                if (!alive) continue;
                pg_fence_after();
                unsigned z[128];
#pragma unroll
                for (int c = 0; c < 4; c++) pg_ld32(z + 32 * c, s_at + 32 * c);
                pg_wait_ld();
                float *x = reinterpret_cast<float *>(z);
                if (a.softcap > 0.0f) pg_tanh<128>(x, inner);
                if (unit <= 0.0f) { // a negative scale turns the order of the scores around, none makes them all alike
#pragma unroll
                    for (int c = 0; c < 128; c++) x[c] = unit < 0.0f ? -x[c] : 0.0f;
                }
                const float size = unit == 0.0f ? 1.0f : fabsf(unit);
                if (__any_sync(0xFFFFFFFFu, valid && (pos + MANY_KEYS > hi || pos < lo))) {
#pragma unroll
                    for (int c = 0; c < 128; c++)
                        if (pos + c >= hi || pos + c < lo) x[c] = -INFINITY;
                }
                float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
                for (int c = 4; c < 128; c += 4)
#pragma unroll
                    for (int e = 0; e < 4; e++) top[e] = fmaxf(top[e], x[c + e]);
                const float most = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * size;
                if (__any_sync(0xFFFFFFFFu, most > m + 8.0f)) {
                    const float to = most > m ? most : m, keep = m == -INFINITY ? 0.0f : paged_exp2(m - to);
                    m = to, l *= keep;
                    if (taken > 0) {
#pragma unroll 1
                        for (int c = 0; c < HDP; c += 32) {
                            unsigned o[32];
                            pg_ld32(o, o_at + c);
                            pg_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                            pg_st32(o_at + c, o);
                        }
                    }
                }
                const float base = m == -INFINITY ? 0.0f : m;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < 128; c += 32) {
                    unsigned p[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float w0 = paged_exp2(fmaf(x[c + i], size, -base)), w1 = paged_exp2(fmaf(x[c + i + 1], size, -base));
                        sum[i & 2] += w0, sum[(i & 2) + 1] += w1;
                        p[i / 2] = pg_pack(w0, w1);
                    }
                    pg_st16(s_at + c / 2, p);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                pg_wait_st();
                pg_fence_before();
                pg_bar_arrive(&p_full[stream]);
            }

            // ---- the item's (or its part's) end ----
            if (taken > 0) {
                if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&o_full[stream], o_count & 1u))) {
                    if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
                    alive = false;
                }
                o_count++;
                pg_fence_after();
            }
            const bool is_whole = w.skip == 0 && w.steps() == item.steps;
            const long long slot = (long long)blockIdx.x * 2 + (first_part && w.skip > 0 ? 0 : 1);
            float keep = 1.0f;
            int from = 0, to = HDP; // the columns that this stream finishes
            if (!item.pair) { // the streams' results meet where the queries were: each finishes half of the columns
                stats[stream][0][r] = m, stats[stream][1][r] = l;
                asm volatile("bar.sync 1, 256;" ::: "memory"); // both streams are done with their products, so with the queries too
                const float other_m = stats[1 - stream][0][r], other_l = stats[1 - stream][1][r], top = fmaxf(m, other_m);
                keep = m == -INFINITY ? 0.0f : paged_exp2(m - top);
                l = l * keep + (other_m == -INFINITY ? 0.0f : other_l * paged_exp2(other_m - top));
                m = top;
                from = stream * (HDP / 2), to = from + HDP / 2;
#pragma unroll 1
                for (int c = (1 - stream) * (HDP / 2); c < (2 - stream) * (HDP / 2); c += 32) {
                    unsigned o[32];
                    if (taken > 0 && alive) {
                        pg_ld32(o, o_at + c);
                        pg_wait_ld();
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; i++) o[i] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        reinterpret_cast<float4 *>(query)[((c + i) / 4) * 128 + r] = make_float4(__uint_as_float(o[i]) * keep, __uint_as_float(o[i + 1]) * keep, __uint_as_float(o[i + 2]) * keep,
                                                                                                __uint_as_float(o[i + 3]) * keep);
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            bool wrong = false;
            const float share = l == 0.0f ? 0.0f : 1.0f / l;
            T *out = static_cast<T *>(a.out) + ((long long)(w.s.first + row / a.c.group) * a.c.heads + w.kvh * a.c.group + row % a.c.group) * a.c.hd;
#pragma unroll 1
            for (int c = from; c < to; c += 32) {
                unsigned o[32];
                if (taken > 0 && alive) {
                    pg_ld32(o, o_at + c);
                    pg_wait_ld();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) o[i] = 0;
                }
                float y[32];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const float4 z = item.pair ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : reinterpret_cast<const float4 *>(query)[((c + i) / 4) * 128 + r];
                    y[i] = __uint_as_float(o[i]) * keep + z.x, y[i + 1] = __uint_as_float(o[i + 1]) * keep + z.y;
                    y[i + 2] = __uint_as_float(o[i + 2]) * keep + z.z, y[i + 3] = __uint_as_float(o[i + 3]) * keep + z.w;
                }
                if (!valid) continue;
                if (!is_whole) {
                    float4 *dst = reinterpret_cast<float4 *>(f.part + (slot * BR + mine) * HDP + c);
#pragma unroll
                    for (int i = 0; i < 8; i++) dst[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                    continue;
                }
#pragma unroll
                for (int i = 0; i < 32; i++) {
                    y[i] = l == 0.0f ? 0.0f : y[i] * share;
                    wrong |= !isfinite(y[i]);
                }
                if (dead) continue;
#pragma unroll
                for (int i = 0; i < 32; i += 8)
                    if (c + i < a.c.hd)
                        *reinterpret_cast<uint4 *>(out + c + i) = make_uint4(pg_pack(y[i], y[i + 1]), pg_pack(y[i + 2], y[i + 3]), pg_pack(y[i + 4], y[i + 5]), pg_pack(y[i + 6], y[i + 7]));
            }
            if (!is_whole) {
                float *ml = f.part + (long long)gridDim.x * 2 * BR * HDP + slot * 2 * BR;
                if (valid && from == 0) ml[mine] = m, ml[BR + mine] = l;
                if (tid == 0 && w.skip == 0 && !dead) {
                    int *head = f.head + blockIdx.x * 8;
                    head[0] = w.b, head[1] = w.kvh, head[2] = w.block, head[3] = item.steps, head[4] = (int)(w.line - line.start), head[5] = (int)line.per;
                }
            }
            unsigned rest = __ballot_sync(0xFFFFFFFFu, wrong);
            while (rest) { // a masked key's zero weight met a value that is not finite
                const int k = __ffs(rest) - 1, at = __shfl_sync(0xFFFFFFFFu, row, k);
                rest &= rest - 1;
                attend_row_plain<T, T>(a, w.b, w.s.first + at / a.c.group, w.s.pos0 + at / a.c.group, w.s.length, w.kvh * a.c.group + at % a.c.group);
            }
            pg_fence_before();
            asm volatile("bar.sync 1, 256;" ::: "memory"); // `query` and `stats` are read
            first_part = false;
            w.next(a);
        }
    }
    pg_fence_before();
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// The parts of an item that several blocks share: a warp a row. blockIdx.x: the block that began it.
template <typename RT, typename CT, int HDP, int BR>
__global__ void __launch_bounds__(256) attend_join_rows_kernel(const ManyCall f) {
    const AttendCall &a = f.a;
    const int c0 = blockIdx.x, mine = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int *head = f.head + c0 * 8;
    const int b = head[0];
    if (b < 0) return;
    const int kvh = head[1], block = head[2], count = head[3], from = head[4], per = head[5];
    const PagedSeq s = paged_seq(a.c, b);
    const int row = block * BR + mine;
    if (row >= min(s.n, a.max_new) * a.c.group) return;
    const int parts = min(1 + (int)((from + (long long)count - 1) / per), (int)gridDim.x - c0);
    const float *ml = f.part + (long long)gridDim.x * 2 * BR * HDP;
    constexpr int N = HDP / 32;
    float top = -INFINITY;
    for (int i = 0; i < parts; i++) top = fmaxf(top, ml[((long long)(c0 + i) * 2 + (i == 0)) * 2 * BR + mine]);
    float l = 0.0f, o[N];
#pragma unroll
    for (int k = 0; k < N; k++) o[k] = 0.0f;
    for (int i = 0; i < parts; i++) {
        const long long slot = (long long)(c0 + i) * 2 + (i == 0);
        const float m = ml[slot * 2 * BR + mine], keep = m == -INFINITY ? 0.0f : paged_exp2(m - top);
        l = fmaf(ml[slot * 2 * BR + BR + mine], keep, l);
#pragma unroll
        for (int k = 0; k < N; k++) o[k] = fmaf(f.part[(slot * BR + mine) * HDP + lane * N + k], keep, o[k]);
    }
    const int token = row / a.c.group, h = kvh * a.c.group + row % a.c.group;
    RT *out = static_cast<RT *>(a.out) + ((long long)(s.first + token) * a.c.heads + h) * a.c.hd;
    bool wrong = false;
#pragma unroll
    for (int k = 0; k < N; k++) {
        const float y = l == 0.0f ? 0.0f : o[k] / l;
        if (lane * N + k < a.c.hd) {
            paged_write(out + lane * N + k, y);
            wrong |= !isfinite(y);
        }
    }
    if (__any_sync(0xFFFFFFFFu, wrong)) attend_row_plain<RT, CT>(a, b, s.first + token, s.pos0 + token, s.length, h);
}

// ---- host side ----
struct ManyPlan {
    int blocks;
    long long part_floats, bytes;
};
inline ManyPlan many_plan(int sms, int block_rows, int hdp) {
    ManyPlan p;
    p.blocks = sms;
    p.part_floats = (long long)p.blocks * 2 * block_rows * (hdp + 2);
    p.bytes = p.part_floats * 4 + (long long)p.blocks * 32;
    return p;
}

template <int HDP>
cudaError_t launch_many_as(const AttendCall &a, const ManyPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    using Shape = ManyShape<HDP>;
    ManyCall f;
    f.a = a, f.part = static_cast<float *>(ws), f.head = reinterpret_cast<int *>(static_cast<float *>(ws) + p.part_floats);
    alignas(64) CUtensorMap map_k, map_v;
    const long long rows = ((long long)a.c.pages * a.c.kv) << a.c.page_shift;
    const int box = std::min(1 << a.c.page_shift, MANY_KEYS);
    if (!paged_map(&map_k, a.k, rows, a.c.hd, false, box) || !paged_map(&map_v, a.v, rows, a.c.hd, false, box)) return cudaErrorNotSupported;
    static std::atomic<bool> known[64];
    if (device >= 64 || !known[device].load()) {
        const cudaError_t e = cudaFuncSetAttribute(attend_many_kernel<HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
        if (e != cudaSuccess) return e;
        if (device < 64) known[device].store(true);
    }
    attend_many_kernel<HDP><<<p.blocks, MANY_THREADS, Shape::SMEM, st>>>(map_k, map_v, f);
    attend_join_rows_kernel<__nv_bfloat16, __nv_bfloat16, HDP, Shape::BLOCK_ROWS><<<dim3(p.blocks, Shape::BLOCK_ROWS / 8), 256, 0, st>>>(f);
    *launches += 2;
    return cudaGetLastError();
}

} // namespace b200i

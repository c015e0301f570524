// Attention of many rows over a paged cache on the tcgen05 tensor cores: prompts, and chunks of new tokens behind what is cached.
//
//   z = scale Q K^T (capped),   O = 2^(z log2 e - m) V / sum 2^(z log2 e - m),   128 rows by 128 keys at a time
//
// Bound: the tensor pipe, 4 head_dim operations a (row, key), and beside it the exponentials: 16 a clock on an SM against 8192
// operations, so at head_dim 128 the two pipes need the same time and neither may wait for the other.
// Rows. A row is a (token, head of the key head's group), so grouped heads share the keys that are brought in.
// Block. Two streams, each of eight softmax warps (two threads a row, for half of a tile's columns each), an S of 128 columns and an O of head_dim columns in tensor memory: while one
// stream's softmax runs, the other's products do. A block of more than 128 rows gives each stream 128 of them and the same keys; one
// of up to 128 gives both streams the rows, and every other tile of keys each, and joins the two at the end. One thread issues
// the products: S = Q K^T from shared memory, O += P V with P (bfloat16, over the columns of S that it came from) read from tensor
// memory and V as it lies, keys down. One warp copies keys and values: tensor-map boxes of 128 bytes by a page's rows into a ring.
// A row's weights are taken from the largest score of the tiles before, and that is moved, O multiplied by what it costs, only when it has grown
// by more than 2^8: larger weights are as exact (up to 2^100, from where the row is done again), the scores are read once, and nothing is
// exchanged between their reading and P. S of the next tile is signalled after the products before it are done, and this tile's products begin
// when the first half of P has been stored AND both halves of O have been multiplied, so O stands still while it is.
// P's one rounding, to 8 bits: an output's terms are off independently of one another, and its norm by 2.2e-3 to 2.4e-3 where its own rounding alone makes 1.7e-3. A second
// piece would be half as many products again, and the products are what bounds long calls. (Weights' sums are taken before the rounding, in 32 bits.)
// Work is cut as in paged_few.cuh: all items' steps on one line, an equal piece a block, parts joined by attend_join_rows_kernel.
// Measured, with what follows it: 2048 tokens behind 14336, 32 heads on 8 of 128, 588 us (876 TFLOP/s of 1627, at 990 of 1000 W); each stream's score,
// softmax and sum follow one another, and two streams fill the tensor pipe to 0.54. 12 chunks of up to 509 tokens, window 1024, capped, 194 us.
// A cache in 4 bits: three warps of the fifth group read codes and write their bfloat16 words into the ring where the copies would (paged_int4.cuh). They are
// the block's first warps, which the scheduler favours: as the last ones they starved beside the softmax (2048 tokens behind 14336: 976 us, 861 so; such calls unpack the cache
// first). Five drafted tokens of 24 sequences, 28 heads on 4, window 4096, capped: 90 us (80 on bfloat16 words). Seven such warps in blocks of 768 threads spill (1430 us for the
// first), and copies of codes far ahead into shared memory were slower too (975, and 98 for the drafted ones).
#pragma once
#include <type_traits>

#include "paged_few.cuh"
#include "paged_int4.cuh"

namespace b200i {

constexpr int MANY_THREADS = 640, MANY_KEYS = 128, MANY_LOAD_WARPS = 3; // two groups of four warps a stream, and one of which one warp copies and one issues

template <int HDP> struct ManyShape {
    static constexpr int TILE = HDP * 256;     // bytes of 128 rows of bfloat16
    static constexpr int QUERY = 2 * TILE;     // a stream each; the streams' meeting place too
    static constexpr int BLOCK_ROWS = 256;
    static constexpr int ROOM = (226 * 1024 - 1024 - 2560 - QUERY) / TILE;
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
__device__ __forceinline__ void pg_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define PG_R8(v, i) "r"((v)[i]), "r"((v)[i + 1]), "r"((v)[i + 2]), "r"((v)[i + 3]), "r"((v)[i + 4]), "r"((v)[i + 5]), "r"((v)[i + 6]), "r"((v)[i + 7])
#define PG_W8(v, i) "=r"((v)[i]), "=r"((v)[i + 1]), "=r"((v)[i + 2]), "=r"((v)[i + 3]), "=r"((v)[i + 4]), "=r"((v)[i + 5]), "=r"((v)[i + 6]), "=r"((v)[i + 7])
#define PG_RW8(v, i) "+r"((v)[i]), "+r"((v)[i + 1]), "+r"((v)[i + 2]), "+r"((v)[i + 3]), "+r"((v)[i + 4]), "+r"((v)[i + 5]), "+r"((v)[i + 6]), "+r"((v)[i + 7])
// Waits for the loads so far; `v` are words of the last of them, which nothing may use before.
__device__ __forceinline__ void pg_wait_ld(unsigned *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : PG_RW8(v, 0), PG_RW8(v, 8), PG_RW8(v, 16), PG_RW8(v, 24)::"memory");
}
// 32 columns of a lane's row
__device__ __forceinline__ void pg_ld32(unsigned *v, unsigned taddr) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, "
        "%27, %28, %29, %30, %31}, [%32];"
        : PG_W8(v, 0), PG_W8(v, 8), PG_W8(v, 16), PG_W8(v, 24)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void pg_ld16(unsigned *v, unsigned taddr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : PG_W8(v, 0), PG_W8(v, 8)
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void pg_wait_ld16(unsigned *v) { asm volatile("tcgen05.wait::ld.sync.aligned;" : PG_RW8(v, 0), PG_RW8(v, 8)::"memory"); }
__device__ __forceinline__ void pg_st16(unsigned taddr, const unsigned *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), PG_R8(v, 0), PG_R8(v, 8)
        : "memory");
}
__device__ __forceinline__ void pg_st8(unsigned taddr, const unsigned *v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), PG_R8(v, 0) : "memory");
}

__device__ __forceinline__ float pg_max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
// Capped scores before their scale: x = tanh(x inner) / inner, inner = scale / softcap, so that the scale that follows is the uncapped one's.
// Far from zero as sign(x) (1 - 2 / (1 + e^{2 |x inner|})); both forms for every score where one of the warp's is far, and no branch between them.
__device__ __forceinline__ float pg_cap_far(float x, float inner, float outer) {
    const float e = paged_exp2(fabsf(x) * (inner * 2.0f * PAGED_LOG2E));
    return copysignf((1.0f - __fdividef(2.0f, 1.0f + e)) * outer, x); // (the quotient of a huge or infinite e is zero)
}
// Up to |y| = 1, y = x inner, as x + x q P(q), q = y^2: for weights of 8 bits P has four coefficients, the largest error being 4.5e-6 of the cap; they
// were chosen by least maximum among those that meet tanh(1), so that there is no step between the two forms that large caps would turn into a step of
// a score. Which form a score takes goes by y alone, so a small score under a large cap stays as exact as it is. A warp whose scores are all
// below the cap, as they mostly are, does only this one. With inner's powers in the coefficients (cap_near, in AttendCall) the product y is saved:
// 12 capped chunks 191 us against 194. FAR has it, for an inner whose eighth power would leave 32 bits.
constexpr float CAP_NEAR[4] = {-0.33295240f, 0.13005409f, -0.04421596f, 0.00870843f};
template <int N, bool FAR>
__device__ __forceinline__ void pg_cap(float *x, const AttendCall &a) {
    float most = 0.0f;
#pragma unroll
    for (int c = 0; c < N; c += 2) most = pg_max3(most, fabsf(x[c]), fabsf(x[c + 1]));
    unsigned long long k[4];
#pragma unroll
    for (int i = 0; i < 4; i++) k[i] = pg_two(a.cap_near[i], a.cap_near[i]);
    const unsigned long long inner = pg_two(a.cap_inner, a.cap_inner);
    const auto near = [&](int c, float &y0, float &y1) {
        const unsigned long long v = pg_two(x[c], x[c + 1]), y = FAR ? pg_mul2(v, inner) : v, q = pg_mul2(y, y);
        unsigned long long p = pg_fma2(q, k[3], k[2]);
        p = pg_fma2(q, p, k[1]), p = pg_fma2(q, p, k[0]);
        pg_one(pg_fma2(pg_mul2(v, q), p, v), y0, y1);
    };
    if (!__any_sync(0xFFFFFFFFu, most > a.cap_outer)) {
#pragma unroll
        for (int c = 0; c < N; c += 2) near(c, x[c], x[c + 1]);
    } else {
#pragma unroll
        for (int c = 0; c < N; c += 2) {
            float y0, y1;
            near(c, y0, y1);
            const float f0 = pg_cap_far(x[c], a.cap_inner, a.cap_outer), f1 = pg_cap_far(x[c + 1], a.cap_inner, a.cap_outer);
            x[c] = fabsf(x[c]) > a.cap_outer ? f0 : y0, x[c + 1] = fabsf(x[c + 1]) > a.cap_outer ? f1 : y1;
        }
    }
}
// To 32-bit accuracy by the series x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 + 62 x^9 / 2835 - 1382 x^11 / 155925 within 0.35, whose next term is 1.2e-8 of x there.
template <int N>
__device__ __forceinline__ void pg_cap_fine(float *x, const AttendCall &a) {
    float most = 0.0f;
#pragma unroll
    for (int c = 0; c < N; c++) most = fmaxf(most, fabsf(x[c]));
    const auto near = [&](float y) {
        const float v = y * a.cap_inner, q = v * v;
        float s = fmaf(q, -1382.0f / 155925.0f, 62.0f / 2835.0f);
        s = fmaf(q, s, -17.0f / 315.0f), s = fmaf(q, s, 2.0f / 15.0f), s = fmaf(q, s, -1.0f / 3.0f);
        return fmaf(y * q, s, y);
    };
    if (!__any_sync(0xFFFFFFFFu, most * a.cap_inner > 0.35f)) {
#pragma unroll
        for (int c = 0; c < N; c++) x[c] = near(x[c]);
    } else {
#pragma unroll
        for (int c = 0; c < N; c++) {
            const float y = near(x[c]), f = pg_cap_far(x[c], a.cap_inner, a.cap_outer);
            x[c] = fabsf(x[c]) * a.cap_inner > 0.35f ? f : y;
        }
    }
}

// An item: up to BR rows of one sequence and key head, over tiles of KEYS keys.
struct ManyItem {
    int row0, rows;    // of the sequence and key head
    int token0, head0; // of the first of them
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
    i.token0 = first, i.head0 = i.row0 - first * a.c.group;
    i.high = min(s.length, max(s.pos0 + last + 1, 0));
    i.low = a.window ? min(max(s.pos0 + first + 1 - a.window, 0), i.high) : 0;
    i.t0 = i.low / KEYS;
    i.tiles = max(1, (i.high + KEYS - 1) / KEYS - i.t0); // rows that see nothing: one tile, masked
    i.pair = STREAMS == 1 || i.rows > BR / 2;
    i.steps = i.pair ? i.tiles : (i.tiles + 1) / 2;
    return i;
}
// The token and the head (of the key head's group) of an item's row r.
__device__ __forceinline__ int2 many_row(const AttendCall &a, const ManyItem &i, int r) {
    const unsigned n = (unsigned)(i.head0 + r), t = a.c.group == 1 ? n : __umulhi(n, a.c.group_part); // n / group: n group < 2^32
    return make_int2(i.token0 + (int)t, (int)(n - t * (unsigned)a.c.group));
}
__device__ __forceinline__ int many_blocks(const AttendCall &a, int n, int block_rows) { return (int)(((long long)n * a.c.group + block_rows - 1) / block_rows); }

// A block's way along the line of all items' steps; every warp of the block goes it by itself. Only the place is kept from item
// to item: what follows from it is read again.
template <int BR, int KEYS, int STREAMS> struct ManyWalk {
    int b, kvh, block;
    int skip;  // steps of the item that other blocks do before this one
    int left;  // steps of the block from here
    int line;  // where on the line the item begins, from where the block does

    static __device__ __forceinline__ int rows_of(const AttendCall &a, const PagedSeq &s) { return min(s.n, a.max_new); } // tokens that are computed
    static __device__ __forceinline__ long long steps_of(const AttendCall &a, int b) {
        const PagedSeq s = paged_seq_checked(a.c, b);
        const int n = rows_of(a, s), blocks = many_blocks(a, n, BR);
        long long sum = 0;
        for (int i = 0; i < blocks; i++) sum += many_item<BR, KEYS, STREAMS>(a, s, n, i).steps;
        return sum;
    }
    __device__ __forceinline__ void begin(const AttendCall &a, const LinePlace &p) {
        b = p.b, kvh = p.kvh, block = 0, left = (int)p.left, line = 0, skip = 0;
        if (left <= 0) return;
        const PagedSeq s = paged_seq(a.c, b);
        const int n = rows_of(a, s);
        long long in = p.in;
        for (;; block++) {
            const int steps = many_item<BR, KEYS, STREAMS>(a, s, n, block).steps;
            if (in < steps) break;
            in -= steps;
        }
        skip = (int)in, line = -skip;
    }
    __device__ __forceinline__ ManyItem item(const AttendCall &a, const PagedSeq &s) const { return many_item<BR, KEYS, STREAMS>(a, s, rows_of(a, s), block); }
    __device__ __forceinline__ int steps(const ManyItem &i) const { return min(i.steps - skip, left); } // that the block does of the item
    __device__ __forceinline__ int first(const ManyItem &i) const { return i.pair ? skip : 2 * skip; }  // its first tile
    __device__ __forceinline__ int tiles(const ManyItem &i) const { return min(i.pair ? skip + steps(i) : 2 * (skip + steps(i)), i.tiles) - first(i); }
    __device__ __forceinline__ void next(const AttendCall &a) {
        const PagedSeq s = paged_seq(a.c, b);
        const ManyItem i = item(a, s);
        left -= steps(i), line += i.steps, skip = 0;
        if (left <= 0 || ++block < many_blocks(a, rows_of(a, s), BR)) return;
        block = 0;
        if (++kvh < a.c.kv) return;
        kvh = 0, b++;
        while (b + 1 < a.c.batch && paged_seq(a.c, b).n == 0) b++;
    }
};

// 64 scores of a row, in tensor memory at s_at: their largest, and then their weights, of which the sum is returned and the bfloat16 words put
// over them. Apart by what a tile needs, so that the common one is a straight run of instructions (scores that are capped; keys that are not
// seen: the row sees columns lo .. hi - 1), and loops of 32 columns, so that the code of a tile that comes seldom is not long: fetched from L2 it
// took 8000 cycles where all columns were written out. A quarter of the exponentials by a cubic beside the unit that
// makes them (16 a clock) cost 8 %: 2048 tokens over 16384 keys 558 -> 601 us.
template <bool EDGE>
__device__ __forceinline__ float many_largest(unsigned s_at, int lo, int hi) {
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
    for (int h = 0; h < 2; h++, lo -= 32, hi -= 32) {
        unsigned z[32];
        const float *x = reinterpret_cast<const float *>(z);
        pg_ld32(z, s_at + 32 * h);
        pg_wait_ld(z);
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = EDGE && (i + e >= hi || i + e < lo) ? -INFINITY : x[i + e];
            top[0] = pg_max3(top[0], y[0], y[1]), top[1] = pg_max3(top[1], y[2], y[3]);
        }
    }
    return fmaxf(top[0], top[1]);
}
template <int CAP, bool EDGE> // CAP: 0 none, 1 capped, 2 capped with FAR
__device__ __forceinline__ float many_weights(const AttendCall &a, unsigned s_at, float unit, float base, int lo, int hi, float &largest) {
    const unsigned long long unit2 = pg_two(unit, unit), base2 = pg_two(-base, -base);
    float top[2] = {-INFINITY, -INFINITY};
    unsigned long long sum[2] = {0, 0};
    unsigned z[2][16]; // 16 columns, and the next 16 on their way
    pg_ld16(z[0], s_at);
    pg_wait_ld16(z[0]);
#pragma unroll(CAP || EDGE ? 1 : 2)
    for (int h = 0; h < 2; h++, lo -= 32, hi -= 32) {
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
            float *x = reinterpret_cast<float *>(z[c / 16]);
            unsigned p[8];
            if (c == 0 || h == 0) pg_ld16(z[1 - c / 16], s_at + 32 * h + c + 16);
            if (CAP) {
                if (EDGE) { // what is not seen may be anything
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (c + i >= hi || c + i < lo) x[i] = 0.0f;
                }
                pg_cap<16, CAP == 2>(x, a);
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
                if (EDGE) {
                    if (c + i >= hi || c + i < lo) x[i] = -INFINITY;
                    if (c + i + 1 >= hi || c + i + 1 < lo) x[i + 1] = -INFINITY;
                }
                top[(i / 2) & 1] = pg_max3(top[(i / 2) & 1], x[i], x[i + 1]);
                const unsigned long long v = pg_fma2(pg_two(x[i], x[i + 1]), unit2, base2);
                float w0, w1;
                pg_one(v, w0, w1);
                w0 = paged_exp2(w0), w1 = paged_exp2(w1);
                sum[(i / 2) & 1] = pg_add2(sum[(i / 2) & 1], pg_two(w0, w1));
                p[i / 2] = pg_pack(w0, w1);
            }
            if (c == 0 || h == 0) pg_wait_ld16(z[1 - c / 16]);
            pg_st8(s_at + 16 * h + c / 2, p); // over columns that have been read
        }
    }
    largest = fmaxf(top[0], top[1]);
    float s0, s1;
    pg_one(pg_add2(sum[0], sum[1]), s0, s1);
    return s0 + s1;
}

struct ManyCall {
    AttendCall a;
    float *part; // [blocks][2][BLOCK_ROWS][HDP], then [blocks][2][2][BLOCK_ROWS] of m and l
    int *head;   // [blocks][8]: sequence (or -1), key head, block of rows, steps, steps of the block before it, steps a block, the first and the last row that did not come out finite
};

// A row did not come out finite: it is done again by attend_again_kernel.
static __device__ __noinline__ void many_mark(int *at, int row) { atomicMin(at, row), atomicMax(at + 1, row); } // rows and heads of the output, one after another

// 16 columns of an output that is there, or zeros.
__device__ __forceinline__ void many_output(unsigned *o, unsigned at, bool some) {
    if (some) {
        pg_ld16(o, at);
        pg_wait_ld16(o);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) o[i] = 0;
    }
}

template <typename CT, int HDP>
__global__ void __launch_bounds__(MANY_THREADS, 1) attend_many_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ ManyCall f) {
    using Shape = ManyShape<HDP>;
    constexpr int SLOTS = Shape::SLOTS, TILE = Shape::TILE, BOXES = HDP / 64, BR = Shape::BLOCK_ROWS, HALF_COLS = 128 * 128; // bytes of a tile's 64 columns
    using T = __nv_bfloat16; // of rows, and of keys and values in shared memory
    constexpr bool FOUR = std::is_same_v<CT, Int4>;
    using Walk = ManyWalk<BR, MANY_KEYS, 2>;
    extern __shared__ __align__(128) unsigned char smem[];
    unsigned char *query = smem + ((1024u - (pg_smem(smem) & 1023u)) & 1023u), *ring = query + Shape::QUERY;
    unsigned long long *full = reinterpret_cast<unsigned long long *>(ring + SLOTS * TILE), *empty = full + SLOTS;
    unsigned long long *s_full = empty + SLOTS, *p_full = s_full + 2, *o_full = p_full + 4, *q_full = o_full + 2, *tail = q_full + 1, *done = tail + 1; // 2 SLOTS + 11 <= 32 words
    __shared__ float stats[2][2][128], half_stat[3][2][2][128]; // m and l of a stream's rows; what the two threads of a row tell each other
    __shared__ long long place[32];
    __shared__ unsigned long long pair_bars[8];
    __shared__ unsigned tmem_slot;
    __shared__ int dead;
    const AttendCall &a = f.a;
    // Where codes become words, that group is the first: the others have the scheduler's favour else, and wait for it.
    const int tid = FOUR ? (threadIdx.x + 512) % 640 : threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int i = 0; i < 8; i++) pg_bar_init(&pair_bars[i], 64);
        for (int s = 0; s < SLOTS; s++) {
            pg_bar_init(&full[s], FOUR ? 32 * MANY_LOAD_WARPS : 1);
            pg_bar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            pg_bar_init(&s_full[i], 1);
            pg_bar_init(&p_full[2 * i], 256), pg_bar_init(&p_full[2 * i + 1], 128);
            pg_bar_init(&o_full[i], 1);
        }
        pg_bar_init(q_full, 512);
        pg_bar_init(tail, 1);
        pg_bar_init(done, 1);
        dead = 0;
        f.head[blockIdx.x * 8] = -1, f.head[blockIdx.x * 8 + 6] = 0x7FFFFFFF, f.head[blockIdx.x * 8 + 7] = -1;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 17) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(pg_smem(&tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pg_follow_early();
    const LinePlace line = line_place(a.c, [&](int b) { return Walk::steps_of(a, b); }, blockIdx.x, gridDim.x, place);
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const unsigned tmem = tmem_slot;
    const int page = 1 << a.c.page_shift, box_rows = min(page, MANY_KEYS);
    Walk w;
    w.begin(a, line);

    if (warp >= 16) { // apart in this order: with the three as one chain of conditions the compiler's code took 190 us for 186 (12 chunks, capped)
        // keys and values in the order of their first use: K0 V0 K1 V1 ..., or K0 K1 V0 K2 V1 K3 ... where the streams have tiles of their own
        const auto load_of = [](int u, int tiles, int lead, bool *is_v) {
            const int v = u - lead; // after the first keys: values, then keys, as long as there are any
            const bool paired = v < 2 * (tiles - lead);
            *is_v = v >= 0 && (paired ? (v & 1) == 0 : true);
            return v < 0 ? u : (paired ? (*is_v ? v / 2 : v / 2 + lead) : (tiles - lead) + (v - 2 * (tiles - lead)));
        };
        if (FOUR && warp != 17) { // ---------------- the cache's codes, written as bfloat16 words ----------------
            if constexpr (FOUR) {
                using Tile = Int4Tile<HDP, MANY_KEYS, MANY_LOAD_WARPS, HDP / 64>;
                const Tile mine(warp == 16 ? 0 : warp - 17, lane);
                unsigned ld = 0;
                bool alive = true;
                while (w.left > 0) {
                    const ManyItem item = w.item(a, paged_seq(a.c, w.b));
                    const int tiles = w.tiles(item), begin = (item.t0 + w.first(item)) * MANY_KEYS, lead = min(item.pair ? 1 : 2, tiles);
                    int id[Tile::N], next_pos;
                    typename Tile::Codes next;
                    bool next_v;
                    const auto look = [&](int p) { // the pages of part p of the item's loads
                        next_pos = begin + load_of(p / Tile::PARTS, tiles, lead, &next_v) * MANY_KEYS + p % Tile::PARTS * (MANY_KEYS / Tile::PARTS);
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
                        if (alive) mine.put(ring + slot * TILE, part, codes);
                        if (part < Tile::PARTS - 1) continue;
                        ld++;
                        if (!alive) continue;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        pg_bar_arrive(&full[slot]);
                    }
                    w.next(a);
                }
                __syncwarp();
            }
        } else if (warp == 16) { // ---------------- the copies ----------------
            unsigned ld = 0, tails = 0;
            bool alive = true, tail_lost = false;
            while (w.left > 0 && alive) {
                const ManyItem item = w.item(a, paged_seq(a.c, w.b));
                const int tiles = w.tiles(item), first = w.first(item), last_page = (item.high - 1) >> a.c.page_shift;
                const int *ids = a.c.table + (long long)w.b * a.c.max_pages;
                const int lead = min(item.pair ? 1 : 2, tiles);
                for (int u = 0; u < 2 * tiles && alive; u++, ld++) {
                    bool is_v;
                    const int tile = load_of(u, tiles, lead, &is_v);
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
                            if (lane == 0) atomicExch(a.c.status, PAGED_WAIT);
                            alive = false, tail_lost = true;
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
            // copies in flight end before the block does, whoever has given up
            if (tail_lost) pg_bar_wait(tail, tails & 1u);
            for (unsigned i = ld > (unsigned)SLOTS ? ld - SLOTS : 0; i < ld; i++) pg_bar_wait(&full[i % SLOTS], (i / SLOTS) & 1u);
        } else if (warp == 17) { // ---------------- the products ----------------
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
                const auto value = [&](int stream, unsigned i, bool add) { // O += P V, V being load i, as the two halves of P come (the first with word from both that O may be added to); false where they do not
                    const unsigned v = pg_desc_low(r0 + (i % SLOTS) * TILE, HALF_COLS), d = tmem + 256 + stream * 128;
                    for (int half = 0; half < 2; half++) {
                        if (alive && !pg_bar_wait(&p_full[2 * stream + half], p_count[stream] & 1u)) alive = false;
                        if (!alive) return false;
                        pg_fence_after();
#pragma unroll
                        for (int ks = 0; ks < 4; ks++)
                            pg_mma_ts(d, tmem + stream * 128 + half * 64 + ks * 8, pg_desc(v + half * (64 * 128 / 16) + ks * 2048 / 16), pg_idesc(HDP, true), add || half > 0 || ks > 0);
                    }
                    p_count[stream]++;
                    return true;
                };
                while (w.left > 0 && alive) {
                    const ManyItem item = w.item(a, paged_seq(a.c, w.b));
                    const int tiles = w.tiles(item);
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
                                if (!value(stream, v, j > 0)) break;
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
                            if (!value(stream, ld, j > 1)) break;
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
                if (!alive) { // products in flight end before their tensor memory is given back
                    atomicExch(a.c.status, PAGED_WAIT);
                    pg_commit(done);
                    pg_bar_wait(done, 0);
                }
            }
            __syncwarp();
        }
    } else { // ---------------- the softmax of a stream: two threads a row, 64 columns of a tile each ----------------
        const int stream = warp >> 3, half = (warp >> 2) & 1, r = tid & 127;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, s_at = tmem + lanes + stream * 128 + 64 * half, o_at = tmem + lanes + 256 + stream * 128;
        const float unit = a.scale * PAGED_LOG2E;
        unsigned s_count = 0, o_count = 0, items = 0;
        bool alive = true;
        unsigned told = 0;
        const auto tell = [&] { // the same within the loop, where one of the two may have given up: with a bound
            unsigned long long *bar = &pair_bars[stream * 4 + (warp & 3)];
            pg_bar_arrive(bar);
            if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(bar, told & 1u))) {
                if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
                alive = false;
            }
            told++;
        };
        const auto meet = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + stream * 4 + (warp & 3)) : "memory"); }; // of the two warps of the same rows: each comes here once an item, whatever happened
        while (w.left > 0) {
            const PagedSeq s = paged_seq(a.c, w.b);
            const ManyItem item = w.item(a, s);
            const int tiles = w.tiles(item);
            if (s.n > a.max_new && tid == 0) atomicExch(a.c.status, PAGED_BAD_BOUND);
            // the rows into shared memory, K-major and swizzled: a stream its own, or both the shared ones
            {
                constexpr int CHUNKS = HDP / 8, N = CHUNKS / 2; // of 16 bytes; that a thread brings where its stream has rows of its own, all asked for at once
                const int tile = item.pair ? stream : 0, chunk = tid % CHUNKS, row0 = (item.pair ? tid & 255 : tid) / CHUNKS, step = (item.pair ? 256 : 512) / CHUNKS;
                const unsigned flip = a.flip ? 0x80008000u : 0u;
                uint4 x[N];
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int row = row0 + i * step;
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (row < 128 && tile * 128 + row < item.rows && chunk * 8 < a.c.hd) {
                        const int2 at = many_row(a, item, tile * 128 + row);
                        x[i] = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (long long)(s.first + at.x) * a.ldq + (w.kvh * a.c.group + at.y) * a.c.hd + chunk * 8);
                    }
                }
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int row = row0 + i * step;
                    if (row < 128)
                        *reinterpret_cast<uint4 *>(query + tile * TILE + (chunk >> 3) * HALF_COLS + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)) =
                            make_uint4(x[i].x ^ flip, x[i].y ^ flip, x[i].z ^ flip, x[i].w ^ flip);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                pg_bar_arrive(q_full);
            }
            const int mine = (item.pair ? stream * 128 : 0) + r;
            const bool valid = mine < item.rows;
            const int2 place = many_row(a, item, mine);
            // of the first tile's columns of this thread, those that the row sees
            int hi = valid ? s.pos0 + place.x + 1 : 0, lo = a.window ? hi - a.window : 0;
            const int begin = (item.t0 + w.first(item) + (item.pair ? 0 : stream)) * MANY_KEYS + 64 * half, step = (item.pair ? 1 : 2) * MANY_KEYS;
            hi -= begin, lo -= begin;
            float m = -INFINITY, l = 0.0f, known = -INFINITY; // known: the largest score of the tile before, of this thread's columns
            const int all = item.pair ? tiles : (tiles + 1 - stream) / 2;
            for (int j = 0; j < all; j++, hi -= step, lo -= step) {
                if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&s_full[stream], s_count & 1u))) {
                    if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
                    alive = false; // it goes on without waiting, so that the others meet it; nothing of the block is stored from here on
                }
                s_count++;
                pg_fence_after();
                if (!alive) continue;
                const bool edge = __any_sync(0xFFFFFFFFu, valid && (hi < 64 || lo > 0));
                // The largest score of the tiles before this one, of both halves, is what a row's weights are taken from, so that the scores are read
                // once and nobody waits: a tile's own may exceed it, which costs range and no exactness. Rows that have seen nothing yet have none:
                // there the two threads of each row look for this tile's first (alike in both halves: they hold the same rows and the same m).
                float most = -INFINITY;
                if (__any_sync(0xFFFFFFFFu, valid && m == -INFINITY)) {
                    most = edge ? many_largest<true>(s_at, lo, hi) : many_largest<false>(s_at, lo, hi);
                    half_stat[0][stream][half][r] = most;
                    tell();
                    most = fmaxf(most, half_stat[0][stream][1 - half][r]);
                    tell(); // read, before it is written again
                    if (!alive) continue;
                    if (a.softcap > 0.0f) {
                        float capped[2] = {most, 0.0f};
                        a.cap_far ? pg_cap<2, true>(capped, a) : pg_cap<2, false>(capped, a);
                        const int at = 64 * half; // a score of -infinity is capped as well; a row that sees nothing of the tile stays without
                        most = max(lo + at, 0) < min(hi + at, MANY_KEYS) ? capped[0] : -INFINITY;
                    }
                    most *= unit;
                }
                if (j > 0) most = fmaxf(most, fmaxf(known, half_stat[1 + ((j - 1) & 1)][stream][1 - half][r])); // (this tile's scores come after both have left them)
                if (__any_sync(0xFFFFFFFFu, most > m + 8.0f)) { // alike in both halves
                    const float to = most > m ? most : m, keep = m == -INFINITY ? 0.0f : paged_exp2(m - to);
                    m = to, l *= keep;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = half * (HDP / 2); c < (half + 1) * (HDP / 2); c += 16) {
                            unsigned o[16];
                            pg_ld16(o, o_at + c);
                            pg_wait_ld16(o);
#pragma unroll
                            for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
                            pg_st16(o_at + c, o);
                        }
                        pg_wait_st();
                    }
                }
                if (half) { // the first half's products add to all columns of O, so they wait for this half's too to be multiplied
                    pg_fence_before();
                    pg_bar_arrive(&p_full[2 * stream]);
                }
                const float base = m == -INFINITY ? 0.0f : m;
                float largest;
                if (a.softcap > 0.0f && !a.cap_far)
                    l += edge ? many_weights<1, true>(a, s_at, unit, base, lo, hi, largest) : many_weights<1, false>(a, s_at, unit, base, lo, hi, largest);
                else if (a.softcap > 0.0f)
                    l += many_weights<2, true>(a, s_at, unit, base, lo, hi, largest);
                else
                    l += edge ? many_weights<0, true>(a, s_at, unit, base, lo, hi, largest) : many_weights<0, false>(a, s_at, unit, base, lo, hi, largest);
                known = largest * unit;
                if (known > base + 100.0f && valid) l = NAN; // weights out of range: the row is done again like one that is not finite
                half_stat[1 + (j & 1)][stream][half][r] = known;
                pg_wait_st();
                pg_fence_before();
                pg_bar_arrive(&p_full[2 * stream + half]);
            }

            // ---- the item's (or its part's) end ----
            if (all > 0) {
                if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&o_full[stream], o_count & 1u))) {
                    if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
                    alive = false;
                }
                o_count++;
                pg_fence_after();
            }
            half_stat[0][stream][half][r] = l;
            meet();
            l = half_stat[0][stream][0][r] + half_stat[0][stream][1][r];
            const bool is_whole = w.skip == 0 && w.steps(item) == item.steps, some = all > 0 && alive;
            const long long slot = (long long)blockIdx.x * 2 + (items == 0 && w.skip > 0 ? 0 : 1);
            // the columns that this thread finishes: half of its row's, or where the streams share rows a quarter
            constexpr int Q4 = HDP / 4;
            const int from = item.pair ? half * (HDP / 2) : (stream * 2 + half) * Q4, to = from + (item.pair ? HDP / 2 : Q4);
            float keep = 1.0f;
            if (!item.pair) { // the streams' results meet where the queries were
                if (half == 0) stats[stream][0][r] = m, stats[stream][1][r] = l;
                asm volatile("bar.sync 9, 512;" ::: "memory"); // both streams are done with their products, so with the queries too
                const float other_m = stats[1 - stream][0][r], other_l = stats[1 - stream][1][r], top = fmaxf(m, other_m);
                keep = m == -INFINITY ? 0.0f : paged_exp2(m - top);
                l = l * keep + (other_m == -INFINITY ? 0.0f : other_l * paged_exp2(other_m - top));
                m = top;
                const int theirs = ((1 - stream) * 2 + half) * Q4;
#pragma unroll 1
                for (int c = theirs; c < theirs + Q4; c += 16) {
                    unsigned o[16];
                    many_output(o, o_at + c, some);
#pragma unroll
                    for (int i = 0; i < 16; i += 4)
                        reinterpret_cast<float4 *>(query)[((c + i) / 4) * 128 + r] = make_float4(__uint_as_float(o[i]) * keep, __uint_as_float(o[i + 1]) * keep, __uint_as_float(o[i + 2]) * keep,
                                                                                                __uint_as_float(o[i + 3]) * keep);
                }
                asm volatile("bar.sync 9, 512;" ::: "memory");
            }
            const float share = !is_whole ? 1.0f : paged_share(l, s.pos0 + place.x); // (where nothing is seen, O is zero, or not finite and done again)
            const unsigned long long keep2 = pg_two(keep * share, keep * share), share2 = pg_two(share, share);
            unsigned long long odd = 0; // zero times what is stored: NaN where that is not finite
            T *out = static_cast<T *>(a.out) + ((long long)(s.first + place.x) * a.c.heads + w.kvh * a.c.group + place.y) * a.c.hd;
            float *part = f.part + (slot * BR + mine) * HDP;
            const bool store = valid && !dead;
#pragma unroll 1
            for (int c = from; c < to; c += 16) {
                unsigned o[16];
                many_output(o, o_at + c, some);
                float y[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    unsigned long long v = pg_mul2(pg_two(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), keep2);
                    if (!item.pair) {
                        const float2 z = reinterpret_cast<const float2 *>(query)[(((c + i) / 4) * 128 + r) * 2 + (i / 2) % 2];
                        v = pg_fma2(pg_two(z.x, z.y), share2, v);
                    }
                    odd = pg_fma2(v, 0, odd);
                    pg_one(v, y[i], y[i + 1]);
                }
                if (!store) continue;
                if (is_whole) {
#pragma unroll
                    for (int i = 0; i < 16; i += 8)
                        if (c + i < a.c.hd)
                            *reinterpret_cast<uint4 *>(out + c + i) = make_uint4(pg_pack(y[i], y[i + 1]), pg_pack(y[i + 2], y[i + 3]), pg_pack(y[i + 4], y[i + 5]), pg_pack(y[i + 6], y[i + 7]));
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4 *>(part + c + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                }
            }
            if (!is_whole) {
                float *ml = f.part + (long long)gridDim.x * 2 * BR * HDP + slot * 2 * BR;
                if (valid && from == 0) ml[mine] = m, ml[BR + mine] = l;
                if (tid == 0 && w.skip == 0 && !dead) {
                    int *head = f.head + blockIdx.x * 8;
                    head[0] = w.b, head[1] = w.kvh, head[2] = w.block, head[3] = item.steps, head[4] = w.line, head[5] = (int)line.per;
                }
            }
            float odd0, odd1;
            pg_one(odd, odd0, odd1);
            // a masked key's zero weight met a value that is not finite, or the weights left their range: the row is done again after this kernel
            if (store && is_whole && !(odd0 + odd1 == 0.0f)) many_mark(f.head + blockIdx.x * 8 + 6, (s.first + place.x) * a.c.heads + w.kvh * a.c.group + place.y);
            pg_fence_before();
            asm volatile("bar.sync 9, 512;" ::: "memory"); // `query` and the statistics are read
            items++;
            w.next(a);
        }
    }
    pg_fence_before();
    __syncthreads();
    if (warp == 17) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// The parts of an item that several blocks share, in the order of its keys: a warp four rows, a lane the statistics of a part and HDP / 32 columns.
// blockIdx.x: the block that began the item; blockIdx.y: 32 rows of it.
template <typename RT, typename CT, int HDP, int BR>
__global__ void __launch_bounds__(256) attend_join_rows_kernel(const __grid_constant__ ManyCall f) {
    constexpr int ROWS = 4, N = HDP / 32;
    const AttendCall &a = f.a;
    const int c0 = blockIdx.x, lane = threadIdx.x & 31, mine = (blockIdx.y * 8 + (threadIdx.x >> 5)) * ROWS;
    pg_follow();
    int *head = f.head + c0 * 8;
    const int b = head[0], kvh = head[1], block = head[2], count = head[3], from = head[4], per = head[5];
    if (b < 0) return;
    const PagedSeq s = paged_seq(a.c, b);
    const int rows = min(min(s.n, a.max_new) * a.c.group - block * BR, BR);
    if (mine >= rows) return;
    const int parts = min(1 + (int)((from + (long long)count - 1) / per), (int)gridDim.x - c0);
    const float *ml = f.part + (long long)gridDim.x * 2 * BR * HDP;
    const auto slot = [&](int i) { return (long long)(c0 + i) * 2 + (i == 0); };
    float top[ROWS], l[ROWS], o[ROWS][N];
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
        top[r] = -INFINITY, l[r] = 0.0f;
#pragma unroll
        for (int k = 0; k < N; k++) o[r][k] = 0.0f;
    }
    for (int i = lane; i < parts; i += 32) {
        const float4 m = *reinterpret_cast<const float4 *>(ml + slot(i) * 2 * BR + mine); // (rows past the item's hold anything, and are not stored)
        top[0] = fmaxf(top[0], m.x), top[1] = fmaxf(top[1], m.y), top[2] = fmaxf(top[2], m.z), top[3] = fmaxf(top[3], m.w);
    }
#pragma unroll
    for (int r = 0; r < ROWS; r++)
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top[r] = fmaxf(top[r], __shfl_xor_sync(0xFFFFFFFFu, top[r], d));
    for (int i0 = 0; i0 < parts; i0 += 32) {
        float keep[ROWS] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (i0 + lane < parts) {
            const float *at = ml + slot(i0 + lane) * 2 * BR + mine;
            const float4 m = *reinterpret_cast<const float4 *>(at), sums = *reinterpret_cast<const float4 *>(at + BR);
            const float ms[ROWS] = {m.x, m.y, m.z, m.w}, ls[ROWS] = {sums.x, sums.y, sums.z, sums.w};
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                keep[r] = ms[r] == -INFINITY ? 0.0f : paged_exp2(ms[r] - top[r]);
                l[r] = fmaf(ls[r], keep[r], l[r]);
            }
        }
        const int here = min(32, parts - i0);
#pragma unroll 2
        for (int i = 0; i < here; i++) {
            const float *at = f.part + (slot(i0 + i) * BR + mine) * HDP + lane * N;
#pragma unroll
            for (int r = 0; r < ROWS; r++) {
                const float k = __shfl_sync(0xFFFFFFFFu, keep[r], i);
                float x[N];
                if constexpr (N == 4) {
                    const float4 v = *reinterpret_cast<const float4 *>(at + r * HDP);
                    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
                } else {
                    const float2 v = *reinterpret_cast<const float2 *>(at + r * HDP);
                    x[0] = v.x, x[1] = v.y;
                }
#pragma unroll
                for (int e = 0; e < N; e++) o[r][e] = fmaf(x[e], k, o[r][e]);
            }
        }
    }
    const unsigned first = (unsigned)(block * BR), token0 = first / (unsigned)a.c.group, head0 = first - token0 * (unsigned)a.c.group;
    const bool mine_columns = lane * N < a.c.hd;
#pragma unroll
    for (int r = 0; r < ROWS; r++) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) l[r] += __shfl_xor_sync(0xFFFFFFFFu, l[r], d);
        if (mine + r >= rows) continue;
        const unsigned n = head0 + (unsigned)(mine + r), t = a.c.group == 1 ? n : __umulhi(n, a.c.group_part);
        const int token = (int)(token0 + t), h = kvh * a.c.group + (int)(n - t * (unsigned)a.c.group);
        const float share = paged_share(l[r], s.pos0 + token);
        float odd = 0.0f; // zero times what is stored: NaN where that is not finite
#pragma unroll
        for (int k = 0; k < N; k++) {
            o[r][k] *= share;
            odd = fmaf(o[r][k], 0.0f, odd);
        }
        RT *out = static_cast<RT *>(a.out) + ((long long)(s.first + token) * a.c.heads + h) * a.c.hd + lane * N;
        if (mine_columns) {
            if constexpr (sizeof(RT) == 2 && N == 4)
                *reinterpret_cast<uint2 *>(out) = make_uint2(pg_pack(o[r][0], o[r][1]), pg_pack(o[r][2], o[r][3]));
            else if constexpr (sizeof(RT) == 2)
                *reinterpret_cast<unsigned *>(out) = pg_pack(o[r][0], o[r][1]);
            else if constexpr (N == 4)
                *reinterpret_cast<float4 *>(out) = make_float4(o[r][0], o[r][1], o[r][2], o[r][3]);
            else
                *reinterpret_cast<float2 *>(out) = make_float2(o[r][0], o[r][1]);
        }
        if (mine_columns && !(odd == 0.0f)) many_mark(head + 6, (s.first + token) * a.c.heads + h);
    }
}

// The rows that did not come out finite, done again: of each block's items, whose way along the line is gone once more, those between the first and the
// last that were marked are looked at. A kernel by itself: in the one that makes the parts the other warps' waits (about a second at most) ran while
// rows were done again, and its registers would be this one's. Where no row is marked it costs 2 to 6 us of a call.
// blockIdx.x: the block whose items these are; blockIdx.y: eight rows of them, by steps of 8 gridDim.y.
template <typename RT, typename CT, int BR, int KEYS, int STREAMS>
__global__ void __launch_bounds__(256) attend_again_kernel(const __grid_constant__ ManyCall f) {
    using Walk = ManyWalk<BR, KEYS, STREAMS>;
    __shared__ long long place[32];
    const AttendCall &a = f.a;
    const int lane = threadIdx.x & 31;
    pg_follow();
    const int first = f.head[blockIdx.x * 8 + 6], last = f.head[blockIdx.x * 8 + 7];
    if (last < first) return;
    const LinePlace line = line_place(a.c, [&](int b) { return Walk::steps_of(a, b); }, blockIdx.x, gridDim.x, place);
    Walk w;
    for (w.begin(a, line); w.left > 0; w.next(a)) {
        const PagedSeq s = paged_seq(a.c, w.b);
        if (w.skip > 0 || (s.first + s.n) * a.c.heads <= first || s.first * a.c.heads > last) continue; // another block began it, or none of its rows is marked
        const ManyItem item = w.item(a, s);
        for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < item.rows; r += gridDim.y * 8) {
            const int2 at = many_row(a, item, r);
            const int h = w.kvh * a.c.group + at.y;
            const RT *out = static_cast<const RT *>(a.out) + ((long long)(s.first + at.x) * a.c.heads + h) * a.c.hd;
            bool odd = false;
            for (int c = lane; c < a.c.hd; c += 32) odd |= !(paged_read(out + c) * 0.0f == 0.0f);
            if (__any_sync(0xFFFFFFFFu, odd)) attend_row_plain<RT, CT>(a, w.b, s.first + at.x, s.pos0 + at.x, s.length, h);
        }
    }
}

// ---- host side ----
struct ManyPlan {
    int blocks;
    long long part_floats, bytes;
};
// No more blocks than the call can have steps, from what the host knows of it, so that the workspace of a short call is short: a block's parts are 266 KB
// at 256 rows and head_dim 128, and 39 MB on 148.
inline ManyPlan many_plan(int sms, int block_rows, int hdp, int keys, long long rows, long long batch, long long kv, long long group, long long max_new, long long max_length) {
    ManyPlan p;
    const long long of_all = rows * group / block_rows + batch, of_each = batch * ((std::min(max_new, rows) * group + block_rows - 1) / block_rows);
    const long long items = kv * std::min(of_all, of_each), steps = (max_length + keys - 1) / keys + 1; // (one more where a window begins inside a tile)
    p.blocks = (int)std::max(1LL, std::min((long long)sms, items > sms ? (long long)sms : items * steps));
    p.part_floats = (long long)p.blocks * 2 * block_rows * (hdp + 2);
    p.bytes = p.part_floats * 4 + (long long)p.blocks * 32;
    return p;
}

// What follows the kernel that makes the parts.
template <typename RT, typename CT, int HDP, int BR, int KEYS, int STREAMS>
cudaError_t many_after(const ManyCall &f, int blocks, cudaStream_t st, int *launches) {
    *launches += 3;
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess) e = launch_following<ManyCall>(attend_join_rows_kernel<RT, CT, HDP, BR>, dim3(blocks, BR / 32), 256, st, f);
    return e != cudaSuccess ? e : launch_following<ManyCall>(attend_again_kernel<RT, CT, BR, KEYS, STREAMS>, dim3(blocks, 8), 256, st, f);
}

template <typename CT, int HDP>
cudaError_t launch_many_as(const AttendCall &a, const ManyPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    using Shape = ManyShape<HDP>;
    ManyCall f;
    f.a = a, f.part = static_cast<float *>(ws), f.head = reinterpret_cast<int *>(static_cast<float *>(ws) + p.part_floats);
    alignas(64) CUtensorMap map_k = {}, map_v = {}; // (of a cache in 4 bits nothing is copied by them)
    const long long rows = ((long long)a.c.pages * a.c.kv) << a.c.page_shift;
    const int box = std::min(1 << a.c.page_shift, MANY_KEYS);
    if constexpr (!std::is_same_v<CT, Int4>)
        if (!paged_map(&map_k, a.k, rows, a.c.hd, false, box) || !paged_map(&map_v, a.v, rows, a.c.hd, false, box)) return cudaErrorNotSupported;
    static std::atomic<bool> known[64];
    if (device >= 64 || !known[device].load()) {
        const cudaError_t e = cudaFuncSetAttribute(attend_many_kernel<CT, HDP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
        if (e != cudaSuccess) return e;
        if (device < 64) known[device].store(true);
    }
    attend_many_kernel<CT, HDP><<<p.blocks, MANY_THREADS, Shape::SMEM, st>>>(map_k, map_v, f);
    return many_after<__nv_bfloat16, CT, HDP, Shape::BLOCK_ROWS, MANY_KEYS, 2>(f, p.blocks, st, launches);
}

} // namespace b200i

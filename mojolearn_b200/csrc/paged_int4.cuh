// Keys and values of a paged cache in 4 bits.
//
// A head's columns go by groups of 32, the last one filled up with zeros. A column is a code n of 4 bits, a group has a bfloat16 scale s:
//
//   x = s (n - 8),   s the smallest number of five significant bits, from 2^-100 on, with 7 s >= max |x|;   n - 8 = x / s to the nearest, ties to even
//
// Five bits times three are eight: what a code stands for is a bfloat16 word, so that the tensor cores multiply the cached values themselves and nothing
// is rounded a second time on any way through them. s ends at 2^90 (words beyond 7 s are cut to it), so that with weights of at most one no sum over 2^31 keys leaves 32 bits.
// Kernels whose weights exceed one for a while (by 2^8 with few rows, up to 2^100 with many) may overflow: such a row does not come out finite and is done again with
// weights of at most one, like a row that met an infinity. The scale
// of a group with a word that is not finite is NaN, as are all its words then. A page and head are one run of bytes: the codes of its positions, 16 bytes a
// group, then their scales, 2 bytes a group. A 32-bit word of codes holds eight columns, 2 i in its i-th four bits and 2 i + 1 in the (i + 4)-th: a shift and a mask make
// a pair of neighbouring columns as two 16-bit words.
//
// A code in the lowest bits of a 16-bit word is the bfloat16 word n 2^-133, and in the next four bits 2^-129 n: below 2^-125 these words lie evenly. Times 2^127, which is exact, and
// then one multiply-add by 2^6 s (or 2^2 s) and -8 s, exact as a whole: eight columns are one shift, four masks and eight multiply-adds for two. With 16 + n made by a mask and
// an or, and s (16 + n) - 24 s, they are four shifts, four of (mask, or) and four multiply-adds; masks and shifts run at half the rate, and attention of 64 grouped single tokens
// took 121 us so and 112 this way.
#pragma once
#include "paged.cuh"
#include "paged_async.cuh"

namespace b200i {

struct Int4 {}; // the type of such a cache
constexpr int INT4_GROUP = 32, INT4_BYTES = 18; // columns of a group, and its bytes

__host__ __device__ __forceinline__ int int4_groups(int hd) { return (hd + INT4_GROUP - 1) / INT4_GROUP; }

// Where the codes of a cache's row (of paged_cache_row) begin, and where its scales do.
__device__ __forceinline__ const unsigned char *int4_page(const void *base, int page, int groups, int page_shift) {
    return static_cast<const unsigned char *>(base) + (((long long)page * (INT4_BYTES * groups)) << page_shift);
}
__device__ __forceinline__ const unsigned char *int4_codes(const void *base, int row, int groups, int page_shift) {
    return int4_page(base, row >> page_shift, groups, page_shift) + (row & ((1 << page_shift) - 1)) * (16 * groups);
}
__device__ __forceinline__ const unsigned short *int4_scales(const void *base, int row, int groups, int page_shift) {
    return reinterpret_cast<const unsigned short *>(int4_page(base, row >> page_shift, groups, page_shift) + ((16 * groups) << page_shift)) + (row & ((1 << page_shift) - 1)) * groups;
}
__device__ __forceinline__ float int4_word(unsigned word, int column, float scale) { return (float)((int)(word >> (4 * (column >> 1) + 16 * (column & 1)) & 15u) - 8) * scale; }

__device__ __forceinline__ unsigned pg_fma_bf16(unsigned x, unsigned y, unsigned z) { // two bfloat16 words at a time
    unsigned r;
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(y), "r"(z));
    return r;
}
// What two scales, of a pair of codes, are multiplied in as.
struct Int4Factors {
    unsigned first, second, shift; // 2^6 s, 2^2 s, -8 s
};
__device__ __forceinline__ Int4Factors int4_factors(unsigned two_scales) {
    return {pg_fma_bf16(two_scales, 0x42804280u, 0x80008000u), pg_fma_bf16(two_scales, 0x40804080u, 0x80008000u), pg_fma_bf16(two_scales, 0xC100C100u, 0x80008000u)};
}
// The four codes of each half of a word, as pairs (lower half, upper half) of words.
__device__ __forceinline__ void int4_pairs(unsigned (&x)[4], unsigned word, const Int4Factors &f) {
    const unsigned far = word >> 8, up = 0x7F007F00u, zero = 0x80008000u; // 2^127, -0
    x[0] = pg_fma_bf16(pg_fma_bf16(word & 0x000F000Fu, up, zero), f.first, f.shift);
    x[1] = pg_fma_bf16(pg_fma_bf16(word & 0x00F000F0u, up, zero), f.second, f.shift);
    x[2] = pg_fma_bf16(pg_fma_bf16(far & 0x000F000Fu, up, zero), f.first, f.shift);
    x[3] = pg_fma_bf16(pg_fma_bf16(far & 0x00F000F0u, up, zero), f.second, f.shift);
}

template <> struct PagedRows<Int4> {
    const void *base;
    int groups, page_shift;
    struct Eight { unsigned word; float scale; };
    struct Four { unsigned word; float scale; }; // the word shifted so that the four columns are its first
    __device__ __forceinline__ PagedRows(const void *p, const PagedCall &c) : base(p), groups(int4_groups(c.hd)), page_shift(c.page_shift) {}
    __device__ __forceinline__ Eight eight(int row, int col) const {
        return {*reinterpret_cast<const unsigned *>(int4_codes(base, row, groups, page_shift) + col / 2),
                __uint_as_float((unsigned)int4_scales(base, row, groups, page_shift)[col / INT4_GROUP] << 16)};
    }
    __device__ __forceinline__ Four four(int row, int col) const {
        const Eight e = eight(row, col & ~7);
        return {e.word >> (col & 4) * 2, e.scale};
    }
    static __device__ __forceinline__ float4 words(unsigned w, float s) { return make_float4(int4_word(w, 0, s), int4_word(w, 1, s), int4_word(w, 2, s), int4_word(w, 3, s)); }
    static __device__ __forceinline__ float4 lower(const Eight &x) { return words(x.word, x.scale); }
    static __device__ __forceinline__ float4 upper(const Eight &x) { return words(x.word >> 8, x.scale); }
    static __device__ __forceinline__ float4 words(const Four &x) { return words(x.word, x.scale); }
};

// Keys or values of a tile of KEYS positions on their way into shared memory as rows of bfloat16 in 128-byte swizzled halves of 64 columns, by WARPS warps:
// a lane a group of a key, in PARTS of KEYS / PARTS keys. What a part takes is asked for one part ahead, and the pages it lies in two ahead.
template <int HDP, int KEYS, int WARPS, int PARTS_> struct Int4Tile {
    static constexpr int PARTS = PARTS_, GROUPS = HDP / INT4_GROUP, AT_ONCE = 32 / GROUPS, ALL = KEYS / PARTS / AT_ONCE, N = (ALL + WARPS - 1) / WARPS;
    struct Codes {
        uint4 word[N];
        unsigned scale[N]; // a bfloat16 word
    };
    int warp, key, group; // of the warp's first keys, the lane's
    __device__ __forceinline__ Int4Tile(int warp_, int lane) : warp(warp_), key(warp_ * AT_ONCE + lane / GROUPS), group(lane % GROUPS) {}
    __device__ __forceinline__ bool mine(int i) const { return ALL % WARPS == 0 || warp + i * WARPS < ALL; }
    // the lane's i-th key of a part that begins at pos, and whether a row sees it: positions low .. high - 1
    __device__ __forceinline__ int place(int i, int pos) const { return pos + key + i * (WARPS * AT_ONCE); }
    __device__ __forceinline__ bool some(int i, int pos, int low, int high) const { return mine(i) && place(i, pos) >= low && place(i, pos) < high; }
    __device__ __forceinline__ void pages(int (&id)[N], const PagedCall &c, int b, int pos, int low, int high) const {
#pragma unroll
        for (int i = 0; i < N; i++) id[i] = some(i, pos, low, high) ? __ldg(c.table + (long long)b * c.max_pages + (place(i, pos) >> c.page_shift)) : 0;
    }
    __device__ __forceinline__ void ask(Codes &x, const int (&id)[N], const PagedCall &c, int kvh, const void *cache, int pos, int low, int high) const {
        const int groups = int4_groups(c.hd);
#pragma unroll
        for (int i = 0; i < N; i++) {
            x.word[i] = make_uint4(0, 0, 0, 0), x.scale[i] = 0;
            if (group >= groups || !some(i, pos, low, high)) continue;
            if ((unsigned)id[i] >= (unsigned)c.pages) {
                atomicExch(c.status, PAGED_BAD_PAGE);
                continue;
            }
            const int in = place(i, pos) & ((1 << c.page_shift) - 1);
            const unsigned char *page = int4_page(cache, id[i] * c.kv + kvh, groups, c.page_shift);
            x.word[i] = __ldg(reinterpret_cast<const uint4 *>(page + (in * groups + group) * 16));
            x.scale[i] = __ldg(reinterpret_cast<const unsigned short *>(page + ((16 * groups) << c.page_shift)) + in * groups + group);
        }
    }
    // Zeros where nothing was read. The lanes of eight 16-byte stores have two keys and four groups (four and two): the groups' chunks are taken in another
    // order in the upper half, so that they fall into different banks.
    __device__ __forceinline__ void put(unsigned char *tile, int part, const Codes &x) const {
        const int turn = GROUPS == 4 ? group & 2 : 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (!mine(i)) continue;
            const int row = part * (KEYS / PARTS) + key + i * (WARPS * AT_ONCE);
            const Int4Factors f = int4_factors(x.scale[i] * 0x10001u);
            unsigned w[4] = {x.word[i].x, x.word[i].y, x.word[i].z, x.word[i].w};
            if (turn) {
                unsigned t = w[0];
                w[0] = w[2], w[2] = t, t = w[1], w[1] = w[3], w[3] = t;
            }
            unsigned char *dst = tile + (group >> 1) * (KEYS * 128) + row * 128;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                unsigned v[4];
                int4_pairs(v, w[k], f);
                *reinterpret_cast<uint4 *>(dst + ((((group & 1) * 4 + (k ^ turn)) ^ (row & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
            }
        }
    }
};

// ---- writing ----

// The scale of a group whose largest magnitude is `most`, a 32-bit or 64-bit word; NaN where that is not finite.
template <typename F> __device__ __forceinline__ float int4_scale(F most) {
    if (!(most < (F)INFINITY)) return __uint_as_float(0x7FFF0000u);
    float s = __uint_as_float(__float_as_uint((float)most * (1.0f / 7.0f)) & 0xFFF80000u); // cut off to five bits: it, or one of the next two
    if ((F)(7.0f * s) < most) s = __uint_as_float(__float_as_uint(s) + 0x80000u);
    if ((F)(7.0f * s) < most) s = __uint_as_float(__float_as_uint(s) + 0x80000u);
    return fminf(fmaxf(s, 0x1p-100f), 0x1p90f);
}
// x / s to the nearest, ties to even, from -7 to 7
__device__ __forceinline__ float int4_code(double x, float s) {
    return (float)fmin(fmax(rint(x / (double)s), -7.0), 7.0);
}

} // namespace b200i

// Fresh q | k | v rows into their places in a cache of 4 bits (paged_int4.cuh): norms, rotation and the queries as in paged_append.cuh, keys and values as codes.
//
// A code is what the definition says of the 64-bit value of its key. The kernel's 32-bit value is off by less than 2^-20 of itself where it is normed (the squares' sum by
// 14 roundings of 2^-24, halved by the root, the root by 2 of 2^-23, three products), and a rotated one by less than 2^-19 of the larger of the two words that it is made of, 2^-22 where
// they were not normed (three roundings). Where the largest magnitude of a group, or a word, is nearer than that to a border between two scales or codes (one head of 128 in 250, or 2000),
// or the squares' mean is not between 2^-60 and 2^60, the head is done again in 64 bits, by the whole warp. Values, and keys without norm and rotation, have no such error.
// Bound: HBM, and latency for a few rows. A lane takes the unit pairs of paged_append.cuh; the units of a group are in neighbouring lanes where half a rotation is
// whole groups, and looked up else. What is not a warp's units goes by a warp a head, a column of each group a lane, in 64 bits: rotations whose halves are not whole
// units, tables that are not on 16-byte boundaries, and the keys that are done again.
// 16 prompts of 33 to 1024 tokens, 32 heads on 8 of 128, norms: 70 us (45 into a cache of bfloat16 words), 60 without the second look and the heads that are done again for it; those in a kernel of their own took 16 us or more, those of a row gathered behind its loop 72.5 in all.
#pragma once
#include "paged_append.cuh"
#include "paged_int4.cuh"

namespace b200i {

struct Append4Call {
    AppendCall a;
    double eps;
};

// Where the codes and scales of a row's position are, of key head 0, and what a key head is further on.
struct Append4Place {
    long long codes, scales, head;
};
__device__ __forceinline__ bool append4_place(Append4Place *at, const PagedCall &c, int b, int pos) {
    if (pos < 0) return false; // the lengths say that this row was cached before the sequence began
    const int row = paged_cache_row(c, b, 0, pos), groups = int4_groups(c.hd), in = pos & ((1 << c.page_shift) - 1);
    if (row < 0) return false;
    at->head = (long long)(INT4_BYTES * groups) << c.page_shift;
    const long long page = (long long)(row >> c.page_shift) * at->head;
    at->codes = page + in * 16 * groups, at->scales = page + ((16 * groups) << c.page_shift) + in * 2 * groups;
    return true;
}

// A row's head of keys or values (part 1 or 2) by a warp, in 64 bits: lane i has columns i, i + 32, ...
template <typename RT>
__device__ __noinline__ void append4_head(const Append4Call &f, long long t, int part, int head, int pos, const Append4Place &place) {
    const AppendCall &a = f.a;
    const int lane = threadIdx.x & 31;
    const RT *src = (part == 1 ? static_cast<const RT *>(a.k) + t * a.ldk : static_cast<const RT *>(a.v) + t * a.ldv) + (long long)head * a.c.hd;
    const float *w = part == 1 ? a.k_norm : nullptr;
    double root = 1.0;
    if (w) {
        double sum = 0.0;
        for (int i = lane; i < a.c.hd; i += 32) {
            const double x = paged_read(src + i);
            sum = fma(x, x, sum);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
        root = sqrt(sum / (double)a.c.hd + f.eps);
    }
    const int half = a.rope_dim / 2;
    const long long row = (long long)max(pos, 0) * half;
    const auto word = [&](int i) { return w ? (double)paged_read(src + i) / root * ((double)w[i] + (double)a.norm_shift) : (double)paged_read(src + i); };
    unsigned char *const cache = static_cast<unsigned char *>(part == 1 ? a.k_cache : a.v_cache) + place.head * head;
#pragma unroll 1
    for (int k = 0; 32 * k < a.c.hd; k++) {
        const int i = lane + 32 * k;
        double y = 0.0;
        if (i < a.c.hd) {
            y = word(i);
            if (part == 1 && a.cosv && i < a.rope_dim) {
                const int j = i < half ? i : i - half;
                const double other = word(i < half ? i + half : i - half), c = a.cosv[row + j], sn = a.sinv[row + j];
                y = i < half ? fma(y, c, -(other * sn)) : fma(y, c, other * sn);
            }
        }
        double most = y == y ? fabs(y) : INFINITY; // (the largest of two leaves NaN out)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmax(most, __shfl_xor_sync(0xFFFFFFFFu, most, o));
        const float scale = int4_scale(most);
        unsigned n = (unsigned)((int)(scale == scale ? int4_code(y, scale) : 0.0f) + 8) << (4 * ((lane & 7) >> 1) + 16 * (lane & 1));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) n |= __shfl_xor_sync(0xFFFFFFFFu, n, o);
        if ((lane & 7) == 0) *reinterpret_cast<unsigned *>(cache + place.codes + 16 * k + lane / 2) = n;
        if (lane == 0) *reinterpret_cast<unsigned short *>(cache + place.scales + 2 * k) = (unsigned short)(__float_as_uint(scale) >> 16);
    }
}

// The largest of three magnitudes; NaN where one is.
__device__ __forceinline__ float append4_most(float x, float y, float z) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
template <int N> __device__ __forceinline__ float append4_largest(const unsigned long long (&x)[N]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < N; i++) {
        float lo, hi;
        pg_one(x[i], lo, hi);
        m = append4_most(m, lo, hi);
    }
    return m;
}

// The codes of a unit's columns, as their four bits in two halves of 16: those of even columns and of odd ones. *nearest: how near the nearest word is to a
// border between two codes, where LOOK asks for that.
template <bool LOOK, int N>
__device__ __forceinline__ uint2 append4_codes(const unsigned long long (&x)[N / 2], float s, float inverse, float *nearest) {
    float q[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        float two[2];
        pg_one(x[i / 2], two[0], two[1]);
        const float y = two[i & 1];
        // the quotient to nearest: one of eight bits by five is a tie if and only if it says so, and one of 24 that says so is one where it leaves nothing
        float p = y * inverse;
        p = fmaf(fmaf(-p, s, y), inverse, p);
        q[i] = (p + 12582912.0f) - 12582912.0f;
        if (N == 4) {
            const float left = fmaf(-p, s, y);
            if (fabsf(p - q[i]) == 0.5f && left != 0.0f) q[i] = p + copysignf(0.5f, left);
        }
        if (LOOK) *nearest = fminf(*nearest, fabsf(fabsf(fmaf(-q[i], s, y)) - 0.5f * s));
    }
    float half[2]; // 8388608 and the codes (each eight more than q) as digits of sixteen
#pragma unroll
    for (int e = 0; e < 2; e++) {
        half[e] = q[e] + (N == 8 ? 8388608.0f + 34952.0f : 8388608.0f + 136.0f);
#pragma unroll
        for (int i = 1; i < N / 2; i++) half[e] = fmaf(q[2 * i + e], (float)(1 << (4 * i)), half[e]);
    }
    return make_uint2(__float_as_uint(half[0]), __float_as_uint(half[1]));
}

// blockIdx.x: the row; its heads in sets of 32 >> lanes_log2, a set a warp, by steps of the warps of gridDim.y blocks. (Queries, norms and rotation as in
// append_units_kernel.)
template <typename RT>
__global__ void __launch_bounds__(128) append_int4_kernel(const __grid_constant__ Append4Call f, int lanes_log2, int sets) {
    constexpr int N = Unit<RT>::N, OF = INT4_GROUP / N; // units of a group
    const AppendCall &a = f.a;
    const long long t = blockIdx.x;
    const int all = threadIdx.x & 31, lane = all & ((1 << lanes_log2) - 1), in_set = all >> lanes_log2;
    const int half = a.rope_dim / 2, pairs = half / N, rest = (a.c.hd - a.rope_dim) / N;
    const bool turned = lane < pairs;
    const int at0 = turned ? lane * N : a.rope_dim + (lane - pairs) * 2 * N, at1 = turned ? at0 + half : at0 + N;
    const bool some0 = lane < pairs + (rest + 1) / 2, some1 = some0 && (turned || (lane - pairs) * 2 + 1 < rest);
    const bool straight = rest == 0 && pairs % OF == 0; // a group's units are OF neighbouring lanes' first, or second
    const RT *const q = static_cast<const RT *>(a.q) + t * a.ldq, *const k = static_cast<const RT *>(a.k) + t * a.ldk, *const v = static_cast<const RT *>(a.v) + t * a.ldv;
    const int parts = a.c.heads + 2 * a.c.kv, groups = int4_groups(a.c.hd);

    typename Unit<RT>::Raw raw0, raw1;
    const auto ask = [&](int set) {
        const int head = (set << (5 - lanes_log2)) + in_set;
        const RT *src = head < a.c.heads ? q + head * a.c.hd : (head < a.c.heads + a.c.kv ? k + (head - a.c.heads) * a.c.hd : v + (head - a.c.heads - a.c.kv) * a.c.hd);
        raw0 = raw1 = typename Unit<RT>::Raw{};
        if (head < parts && some0) raw0 = Unit<RT>::ask(src + at0);
        if (head < parts && some1) raw1 = Unit<RT>::ask(src + at1);
    };
    int set = blockIdx.y * 4 + (threadIdx.x >> 5);
    const int step = gridDim.y * 4;
    if (set < sets) ask(set);

    const int b = paged_row_seq(a.c, t);
    if (b < 0) return; // a row of no sequence: nothing is written for it
    const PagedSeq s = paged_seq_checked(a.c, b);
    if (s.n == 0) return; // its tables do not hold it
    const int pos = s.pos0 + (int)(t - s.first);
    if (append_past(a, pos)) return;
    Append4Place place;
    const bool placed = append4_place(&place, a.c, b, pos);
    unsigned long long c[N / 2], sn[N / 2];
    const bool turns = turned && a.cosv != nullptr;
    float turn_off = 0.0f; // of a rotated word, in units of the largest one that it is made of
    bool still = true;     // the rotation leaves the lane's words as they are, ties too: position 0
    if (turns) {
        const long long row = (long long)max(pos, 0) * half + at0;
        append_words<N>(c, a.cosv + row);
        append_words<N>(sn, a.sinv + row);
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            float u[4];
            pg_one(c[i], u[0], u[1]), pg_one(sn[i], u[2], u[3]);
            turn_off = fmaxf(turn_off, fmaxf(fmaxf(fabsf(u[0]), fabsf(u[1])), fmaxf(fabsf(u[2]), fabsf(u[3]))));
            still &= u[0] == 1.0f && u[1] == 1.0f && u[2] == 0.0f && u[3] == 0.0f;
        }
        turn_off *= a.k_norm ? 0x1p-19f : (still ? 0.0f : 0x1p-22f);
    }
    for (; set < sets; set += step) {
        const int head = (set << (5 - lanes_log2)) + in_set, part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2); // q, k, v
        unsigned long long x0[N / 2], x1[N / 2];
        Unit<RT>::words(x0, raw0), Unit<RT>::words(x1, raw1);
        if (set + step < sets) ask(set + step);
        const float *w = part == 0 ? a.q_norm : (part == 1 ? a.k_norm : nullptr);
        bool exact = true; // the squares' mean is known to 2^-20 of itself: none of them left 32 bits
        if (a.q_norm || a.k_norm) { // uniform over the grid: the reduction is a warp's
            unsigned long long sums = 0;
#pragma unroll
            for (int i = 0; i < N / 2; i++) sums = pg_fma2(x0[i], x0[i], pg_fma2(x1[i], x1[i], sums));
            float sum, other;
            pg_one(sums, sum, other);
            sum += other;
            for (int o = (1 << lanes_log2) >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
            if (w) {
                const float mean = fmaf(sum, a.part_of_head, a.eps), r = rsqrtf(mean);
                exact = mean >= 0x1p-60f && mean <= 0x1p60f;
                const unsigned long long r2 = pg_two(r, r), shift2 = pg_two(a.norm_shift * r, a.norm_shift * r);
                unsigned long long weight[N / 2];
                if (some0) {
                    append_words<N>(weight, w + at0);
#pragma unroll
                    for (int i = 0; i < N / 2; i++) x0[i] = pg_mul2(x0[i], pg_fma2(weight[i], r2, shift2));
                }
                if (some1) {
                    append_words<N>(weight, w + at1);
#pragma unroll
                    for (int i = 0; i < N / 2; i++) x1[i] = pg_mul2(x1[i], pg_fma2(weight[i], r2, shift2));
                }
            }
        }
        const bool held = __any_sync(0xFFFFFFFFu, part > 0); // keys or values among the warp's heads
        // How far a word may be from its 64-bit value: by the largest words that it is made of; negative where it is that value.
        const bool moved = part == 1 && (w || (turns && turn_off != 0.0f));
        float off = -1.0f;
        if (held && moved) {
            const float most = append4_most(append4_largest(x0), append4_largest(x1), 0.0f);
            off = most * (turns ? turn_off : 0x1p-20f);
            if (w) off = exact ? off + 0x1p-110f : INFINITY; // (the products with the weight may be denormal: 2^-150 of a word of up to 2^34)
        }
        if (turns && part < 2) {
            const unsigned long long minus = pg_two(-1.0f, -1.0f);
#pragma unroll
            for (int i = 0; i < N / 2; i++) {
                const unsigned long long u = x0[i], y = x1[i];
                x0[i] = pg_fma2(u, c[i], pg_mul2(pg_mul2(y, sn[i]), minus));
                x1[i] = pg_fma2(y, c[i], pg_mul2(u, sn[i]));
            }
        }
        if (part == 0 && some0) {
            RT *dst = static_cast<RT *>(a.q_out) + (t * a.c.heads + head) * a.c.hd;
            Unit<RT>::store(dst + at0, x0);
            if (some1) Unit<RT>::store(dst + at1, x1);
        }
        if (!held) continue;
        // ---- the codes ----
        float most0 = append4_largest(x0), most1 = append4_largest(x1), far0 = off, far1 = off;
        if (straight) {
#pragma unroll
            for (int o = 1; o < OF; o <<= 1) {
                most0 = append4_most(most0, __shfl_xor_sync(0xFFFFFFFFu, most0, o), 0.0f), most1 = append4_most(most1, __shfl_xor_sync(0xFFFFFFFFu, most1, o), 0.0f);
                far0 = fmaxf(far0, __shfl_xor_sync(0xFFFFFFFFu, far0, o));
            }
            far1 = far0;
        } else { // unit u of a head is lane u's first, lane u - pairs' second, or one of two neighbours behind the rotation
            float m0 = 0.0f, m1 = 0.0f, f0 = off, f1 = off;
#pragma unroll 1
            for (int i = 0; i < 2 * OF; i++) {
                const int u = (i < OF ? at0 : at1) / N / OF * OF + i % OF, r = u - 2 * pairs;
                const int from = (all - lane) + (r < 0 ? (u < pairs ? u : u - pairs) : pairs + r / 2);
                const bool second = r < 0 ? u >= pairs : (r & 1) != 0, there = u * N < a.c.hd;
                const float p0 = __shfl_sync(0xFFFFFFFFu, most0, from), p1 = __shfl_sync(0xFFFFFFFFu, most1, from);
                const float g = __shfl_sync(0xFFFFFFFFu, off, from);
                if (there && i < OF) m0 = append4_most(m0, second ? p1 : p0, 0.0f), f0 = fmaxf(f0, g);
                if (there && i >= OF) m1 = append4_most(m1, second ? p1 : p0, 0.0f), f1 = fmaxf(f1, g);
            }
            most0 = m0, most1 = m1, far0 = f0, far1 = f1;
        }
        bool near = false;
        const bool look = __any_sync(0xFFFFFFFFu, off >= 0.0f);
        float scale[2];
        uint2 code[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float top = h ? most1 : most0, s5 = int4_scale(top), before = __uint_as_float(__float_as_uint(s5) - 0x80000u), far = h ? far1 : far0;
            float inverse, nearest = INFINITY;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(s5));
            scale[h] = s5;
            code[h] = look ? append4_codes<true, N>(h ? x1 : x0, s5, inverse, &nearest) : append4_codes<false, N>(h ? x1 : x0, s5, inverse, &nearest);
            near |= nearest <= off;
            if (moved) near |= 7.0f * s5 - top <= far || (s5 > 0x1p-100f && top - 7.0f * before <= far);
            if (!(top <= 7.0f * s5)) near = true; // words that are cut, or not finite
        }
        near &= part > 0 && head < parts && some0 && placed; // (a lane without a second unit has zeros there, which are near nothing)
        const unsigned again = __ballot_sync(0xFFFFFFFFu, near), mine = again >> (all - lane) & (unsigned)((1ull << (1 << lanes_log2)) - 1);
        if (part > 0 && head < parts && placed && mine == 0) {
            unsigned char *const cache = static_cast<unsigned char *>(part == 1 ? a.k_cache : a.v_cache) + place.head * (head - a.c.heads - (part == 1 ? 0 : a.c.kv));
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int at = h ? at1 : at0;
                if (!(h ? some1 : some0)) continue;
                if constexpr (N == 8) {
                    *reinterpret_cast<unsigned *>(cache + place.codes + at / 2) = __byte_perm(code[h].x, code[h].y, 0x5410);
                } else { // half a word: its first bytes, or its second ones
                    unsigned char *const to = cache + place.codes + at / 8 * 4 + (at / 4 & 1);
                    to[0] = (unsigned char)code[h].x, to[2] = (unsigned char)code[h].y;
                }
                if (at % INT4_GROUP == 0) *reinterpret_cast<unsigned short *>(cache + place.scales + at / INT4_GROUP * 2) = (unsigned short)(__float_as_uint(scale[h]) >> 16);
            }
            for (int at = a.c.hd + 8 * lane; at < INT4_GROUP * groups; at += 8 << lanes_log2) *reinterpret_cast<unsigned *>(cache + place.codes + at / 2) = 0x88888888u; // the last group's zeros
        }
        for (unsigned rest_of = again; rest_of;) { // the heads that are done again, one after another
            const int first = (__ffs(rest_of) - 1) >> lanes_log2 << lanes_log2, which = (set << (5 - lanes_log2)) + (first >> lanes_log2);
            rest_of &= ~(unsigned)(((1ull << (1 << lanes_log2)) - 1) << first);
            const int of = which < a.c.heads + a.c.kv ? 1 : 2;
            append4_head<RT>(f, t, of, which - a.c.heads - (of == 1 ? 0 : a.c.kv), pos, place);
        }
    }
}

// A warp a head: queries column by column, keys and values by append4_head.
template <typename RT>
__global__ void __launch_bounds__(256) append_int4_columns_kernel(const __grid_constant__ Append4Call f) {
    const AppendCall &a = f.a;
    const long long t = blockIdx.x;
    const int head = blockIdx.y * 8 + (threadIdx.x >> 5), b = paged_row_seq(a.c, t);
    if (b < 0 || head >= a.c.heads + 2 * a.c.kv) return;
    const PagedSeq s = paged_seq_checked(a.c, b);
    if (s.n == 0) return; // its tables do not hold it
    const int pos = s.pos0 + (int)(t - s.first), part = head < a.c.heads ? 0 : (head < a.c.heads + a.c.kv ? 1 : 2);
    if (append_past(a, pos)) return;
    if (part > 0) {
        Append4Place place;
        if (append4_place(&place, a.c, b, pos)) append4_head<RT>(f, t, part, head - a.c.heads - (part == 1 ? 0 : a.c.kv), pos, place);
        return;
    }
    append_columns<RT, RT>(a, static_cast<const RT *>(a.q) + t * a.ldq + (long long)head * a.c.hd, a.q_norm, pos, true,
                           static_cast<RT *>(a.q_out) + (t * a.c.heads + head) * a.c.hd);
}

template <typename RT>
cudaError_t launch_append4(const AppendCall &a, double eps, int sms, cudaStream_t st) {
    constexpr int N = Unit<RT>::N;
    const Append4Call f = {a, eps};
    const int parts = a.c.heads + 2 * a.c.kv;
    if (append_by_units<N>(a)) {
        const AppendCut cut = append_cut<N>(a, parts, sms);
        append_int4_kernel<RT><<<dim3((unsigned)a.c.rows, (unsigned)cut.blocks), 128, 0, st>>>(f, cut.lanes_log2, cut.sets);
    } else {
        append_int4_columns_kernel<RT><<<dim3((unsigned)a.c.rows, (unsigned)((parts + 7) / 8)), 256, 0, st>>>(f);
    }
    return cudaGetLastError();
}

} // namespace b200i

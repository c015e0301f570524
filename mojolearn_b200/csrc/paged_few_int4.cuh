// Attention of few rows over a paged cache in 4 bits: a decode step's single tokens (and up to 24 rows a sequence and key head).
//
// The sums, the line of tiles, the copying warp and the join are those of paged_few.cuh. Bound: HBM, 4.5 bits a word of keys and values; next to that the
// instructions that make bfloat16 words of codes (paged_int4.cuh), one and a half a word, of which an SM has 42 words a clock to do at the HBM rate. So a word is made once
// and meets all rows of its key head in one instruction: m16n8k16 with the KEYS as rows, S^T = K Q^T and O^T = V^T P^T, the eight columns being rows. What a word's place is in an
// instruction is free where both factors agree on it: of a key a lane takes a quarter of its columns, which is one group and one 16-byte load; of the values an eighth of the columns
// of four keys, whose codes become pairs along the keys by one byte permutation for eight words.
// PACK: up to four bfloat16 rows or two of float32 leave columns of the eight free. A weight is then two pieces of 8 bits in neighbouring columns (three in four
// columns; and so are float32 queries), and one product serves where the others need one for each piece.
// A tensor core cuts its 32-bit sums off where it adds to a large one: with float32 rows each 16 keys begin at zero and are added to the output to nearest.
// Weights are taken from the largest score so far as it was when one last exceeded it by 2^8: larger ones are as exact, and the usual tile needs one vote.
//
// Warps. Up to 16 rows, two blocks of four computing warps and one that copies: the registers of eight warps (96 a thread) spill, those of four (168) hold the sums and
// several chains of 16 keys, each of which hides the others' latency: four chains and tiles of 256 keys with PACK, two else (one for 16 float32 rows). More rows: one block of eight
// warps, two of which share keys and halve the columns. Measured, 64 sequences of 2000 to 8000 keys, 32 heads on 8 of 128: eight warps 106 us, four of two chains 98, of four 95
// (2.8 TB/s of 4.5-bit words; 167 us on a cache of bfloat16 words). One of 131000 keys with pages of 64: 47.5 us (3.2 TB/s; with pages of 16, 53; of words 94).
// 32 float32 tokens, 16 heads, up to 1250 keys a sequence: 35 us (of words 62; eight warps 47). One token at 200 keys: 8 us. Three blocks an SM (72 registers) spill: 144 us
// for the first. Scores worked out one step ahead of the weights gained nothing. SMs are active for 0.81 to 0.87 of these calls and then issue in half of their cycles: two to three
// warps a scheduler wait together, for loads first.
#pragma once
#include <type_traits>

#include "paged_int4.cuh"
#include "paged_many.cuh"

namespace b200i {

constexpr int few4_keys(bool pack) { return pack ? 256 : 128; } // of a tile

template <typename RT, int GROUPS, int NT, bool PACK> struct Few4Shape {
    static constexpr bool F32 = std::is_same_v<RT, float>;
    static constexpr int HDP = GROUPS <= 2 ? 64 : 128; // head_dim as it is laid out for the products: a lane's quarter (eighth) of it lies in one group
    static constexpr int WARPS = NT <= 2 ? 4 : 8, THREADS = 32 * (WARPS + 1), ROWS = PACK ? (F32 ? 2 : 4) : 8 * NT;
    static constexpr int BLOCKS = NT > 2 ? 1 : 2;                        // on an SM
    static constexpr int SPLIT = NT > 2 && HDP == 128 ? 2 : 1;           // warps that share keys, each for its part of the values' columns
    static constexpr int SLICES = WARPS / SPLIT, KEYS = few4_keys(PACK), CHUNKS = KEYS / 16 / SLICES; // a tile's keys go to so many warps, by so many times 16
    static constexpr int CH = PACK ? 4 : (NT == 1 || (NT == 2 && !F32) ? 2 : 1);                          // of which it works on so many at once
    static constexpr int HALF = KEYS * GROUPS * INT4_BYTES, SLOT = 2 * HALF; // keys, then values
    static constexpr int Q_PIECES = F32 ? 3 : 1, W_PIECES = F32 ? 3 : 2; // of 8 bits: what two leave of a weight, 2^-16, is far below a bfloat16 output's own rounding
    static constexpr bool HELD = PACK || (!F32 && NT == 1); // the queries stay in registers; else they lie as fragments where the warps' results meet
    static constexpr int PITCH = HDP + 8;                   // floats of a row of those
    static constexpr int MEET = 4 * ROWS * PITCH * 4, QUERY = ROWS * HDP * (int)sizeof(RT);
    static constexpr int REST = 1024 + 512 + MEET + FEW_ITEMS * QUERY;
    static constexpr int ROOM = ((BLOCKS == 2 ? 112 : 220) * 1024 - REST) / SLOT, SLOTS = ROOM > 8 ? 8 : ROOM;
    static constexpr int SMEM = REST + SLOTS * SLOT;
    static_assert(SLOTS >= 2 && (HELD || Q_PIECES * NT * HDP / 16 * 256 <= MEET), "shared memory");
};

// What brings a tile: two lanes a piece, its keys and its values, whose codes and scales follow one another in the cache as in the slot. Of a page larger than a tile
// they do not, and four lanes bring them.
template <typename Shape>
__device__ __forceinline__ auto few4_runs(const AttendCall &a) {
    return [&a](unsigned char *dst, unsigned long long *full, int pos, int there, int low, int kvh, auto page_of) {
        const PagedCall &c = a.c;
        const int lane = threadIdx.x & 31, page = 1 << c.page_shift, rows = min(page, Shape::KEYS), groups = int4_groups(c.hd), split = page > Shape::KEYS;
        const int values = lane & 1, scales = (lane >> 1) & split, piece = lane >> (1 + split); // this lane's
        const int id = page_of(piece), first = piece * rows;
        const bool want = piece < there && low - pos < first + rows; // a page that nobody sees any more may be anyone's
        const bool some = want && (unsigned)id < (unsigned)c.pages;
        unsigned char *const to = dst + (values ? Shape::HALF : 0) + first * groups * INT4_BYTES;
        if (want && !some) { // a page of zeros: scales of zero
            atomicExch(c.status, PAGED_BAD_PAGE);
            for (int i = 0; i < rows * groups * 2; i += 16) *reinterpret_cast<uint4 *>(to + rows * groups * 16 + i) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        const unsigned all = __ballot_sync(0xFFFFFFFFu, some);
        __syncwarp(); // the zeros are there before lane 0 arrives for all
        if (lane == 0) pg_bar_expect(full, (unsigned)((__popc(all) >> split) * rows * groups * INT4_BYTES));
        __syncwarp();
        if (!some) return;
        const unsigned char *src = int4_page(values ? a.v : a.k, id * c.kv + kvh, groups, c.page_shift);
        const int in = (pos + first) & (page - 1), codes = rows * groups * 16, bytes = !split ? rows * groups * INT4_BYTES : (scales ? rows * groups * 2 : codes);
        src += !split ? 0 : (scales ? ((16 * groups) << c.page_shift) + in * groups * 2 : in * groups * 16);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(pg_smem(to + scales * codes)), "l"(src), "r"(bytes), "r"(pg_smem(full)) : "memory");
    };
}

template <typename RT, int GROUPS, int NT, bool PACK>
__global__ void __launch_bounds__(Few4Shape<RT, GROUPS, NT, PACK>::THREADS, Few4Shape<RT, GROUPS, NT, PACK>::BLOCKS) attend_few_int4_kernel(const __grid_constant__ FewCall f) {
    using Shape = Few4Shape<RT, GROUPS, NT, PACK>;
    constexpr bool F32 = Shape::F32, HELD = Shape::HELD;
    constexpr int HDP = Shape::HDP, KEYS = Shape::KEYS, SLOTS = Shape::SLOTS, KS = HDP / 16, ROWS = Shape::ROWS, WARPS = Shape::WARPS, CH = Shape::CH, QP = Shape::Q_PIECES, WP = Shape::W_PIECES;
    constexpr int SPLIT = Shape::SPLIT, SLICES = Shape::SLICES, CHUNKS = Shape::CHUNKS, MT = KS / SPLIT; // MT: pieces of 16 columns of the output that a warp has
    constexpr int E = PACK ? 1 : 2 * NT;                          // rows of a lane's scores
    constexpr int K_WORDS = HDP / 32, V_WORDS = HDP / 64 / SPLIT; // of codes, of a key: a quarter of its columns, an eighth (of the warp's)
    constexpr int STRIDE = 16 * GROUPS;                           // bytes of a key's codes
    extern __shared__ __align__(128) unsigned char smem[];
    const FewMemory<Shape> sm(smem);
    __shared__ float ml[SLICES][2][ROWS], joined[2][ROWS];
    __shared__ long long place[32];
    __shared__ FewItem items[FEW_ITEMS];
    __shared__ unsigned long long bad_rows;
    __shared__ int dead;
    const AttendCall &a = f.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
    const LinePlace p = few_begin<KEYS>(f, sm, place, &bad_rows, &dead);
    if (warp == WARPS) {
        few_copies<RT, KEYS>(f, sm, items, p, few4_runs<Shape>(a));
        return;
    }

    // of the lane's columns: of a key's quarters and of its eighths, those that are in no group of the head's count as zeros
    const int slice = warp / SPLIT, side = warp % SPLIT, key0 = slice * 16 * CHUNKS; // the warp's keys of a tile
    const int k_group = t4 * (HDP / 4) / INT4_GROUP, v_group = g * (HDP / 8) / INT4_GROUP;
    const bool k_some = k_group < GROUPS, v_some = v_group < GROUPS;
    // in a slot, of 16 of its keys: the lane's codes and scales of keys g (and g + 8), and of values 2 t4 (and 1, 8 and 9 further on)
    const int box_rows = min(1 << a.c.page_shift, KEYS); // of the piece that they lie in
    int k_at[CHUNKS], k_scale[CHUNKS], v_at[CHUNKS], v_scale[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; c++) {
        const int key = key0 + 16 * c, in = key & (box_rows - 1), piece = (key - in) * (GROUPS * INT4_BYTES), scales = piece + box_rows * STRIDE;
        k_at[c] = piece + (in + g) * STRIDE + (k_some ? t4 * (HDP / 8) : 0), k_scale[c] = scales + (in + g) * (2 * GROUPS) + (k_some ? 2 * k_group : 0);
        v_at[c] = Shape::HALF + piece + (in + 2 * t4) * STRIDE + (v_some ? g * (HDP / 16) + side * (V_WORDS * 4) : 0);
        v_scale[c] = Shape::HALF + scales + (in + 2 * t4) * (2 * GROUPS) + (v_some ? 2 * v_group : 0);
    }
    const float unit = a.scale * PAGED_LOG2E, part_of_unit = 1.0f / unit; // (capped scores are still to be scaled: paged_many.cuh)
    const auto row_of = [&](int e) { return PACK ? (F32 ? t4 >> 1 : t4) : (e >> 1) * 8 + 2 * t4 + (e & 1); };
    const auto token_of = [&](int r) { return a.c.group == 1 ? r : (int)__umulhi((unsigned)r, a.c.group_part); };
    uint2 *const fragments = reinterpret_cast<uint2 *>(sm.meet);
    unsigned slot_at = 0, parity = 0; // of the next tile
    bool alive = true, first_part = true;
    const auto give_up = [&] {
        if (lane == 0) atomicExch(a.c.status, PAGED_WAIT), dead = 1;
        alive = false; // it goes on without waiting, so that the others meet it; nothing of the block is stored from here on
    };
    for (unsigned number = 0;; number++) {
        const int which = number % FEW_ITEMS;
        if (alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&sm.item_full[which], (number / FEW_ITEMS) & 1u))) give_up();
        if (few_vote<WARPS>(!alive)) break; // nobody goes on where one has given up: what the item is would not be known
        const FewItem &item = items[which]; // what the loop over the tiles does not need is read again after it
        if (!item.more) break;
        const int length = item.s.length, pos0 = item.s.pos0, tiles = item.tiles, begin = item.pos + key0;
        const auto rows_of = [&] { return min(item.n * a.c.group, ROWS); };

        // The rows as fragments: column n of row `row`, words col .. col + 3 of it, piece by piece.
        const auto words = [&, rows = rows_of()](uint2 (&q)[QP], int row, int col) {
#pragma unroll
            for (int k = 0; k < QP; k++) q[k] = make_uint2(0, 0);
            if (row >= rows || col >= a.c.hd) return;
            const unsigned char *src = sm.query + which * Shape::QUERY + (row * a.c.hd + col) * (int)sizeof(RT);
            if constexpr (F32) {
                float4 x = *reinterpret_cast<const float4 *>(src);
                if (a.flip) x = make_float4(-x.x, -x.y, -x.z, -x.w);
                unsigned lo[3], hi[3];
                pg_split<3>(lo, x.x, x.y), pg_split<3>(hi, x.z, x.w);
#pragma unroll
                for (int k = 0; k < 3; k++) q[k] = make_uint2(lo[k], hi[k]);
            } else {
                const unsigned flip = a.flip ? 0x80008000u : 0u;
                q[0] = *reinterpret_cast<const uint2 *>(src);
                q[0].x ^= flip, q[0].y ^= flip;
            }
        };
        uint2 held[HELD ? KS : 1];
        if constexpr (HELD) {
            const int row = !PACK ? g : (F32 ? g >> 2 : g >> 1), piece = !PACK ? 0 : (F32 ? g & 3 : g & 1);
#pragma unroll
            for (int ks = 0; ks < KS; ks++) {
                uint2 q[QP];
                words(q, row, t4 * (HDP / 4) + 4 * ks);
                held[ks] = piece == 0 ? q[0] : make_uint2(0, 0);
                if constexpr (F32) held[ks] = piece == 1 ? q[1] : (piece == 2 ? q[2] : held[ks]);
            }
        } else {
            for (int i = tid; i < NT * KS * 32; i += 32 * WARPS) {
                const int of = i & 31, ks = (i >> 5) % KS, nt = (i >> 5) / KS;
                uint2 q[QP];
                words(q, nt * 8 + (of >> 2), (of & 3) * (HDP / 4) + 4 * ks);
#pragma unroll
                for (int k = 0; k < QP; k++) fragments[k * (NT * KS * 32) + i] = q[k];
            }
            few_meet<WARPS>();
        }
        // every row sees positions all_lo .. pos0; none sees what is below low
        const int all_lo = a.window ? pos0 + item.n - a.window : 0, low = a.window ? pos0 + 1 - a.window : 0;

        float o[NT][MT][4], m[E], l[E], high[E]; // high: the score that m is to be moved for
#pragma unroll
        for (int e = 0; e < E; e++) m[e] = high[e] = -INFINITY, l[e] = 0.0f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int mt = 0; mt < MT; mt++) o[nt][mt][0] = o[nt][mt][1] = o[nt][mt][2] = o[nt][mt][3] = 0.0f;
        // Scores of 16 keys of a tile, the warp's chunk c of them.
        constexpr int ZS = F32 && !PACK ? 2 : 1; // large and small products apart
        float z[CH][ZS][NT][4];
        const auto scores = [&](const unsigned char *slot, int c, float (&z)[ZS][NT][4]) {
            unsigned code[2][K_WORDS];
            Int4Factors factors[2];
#pragma unroll
            for (int h = 0; h < 2; h++) { // keys g and g + 8
                const unsigned char *at = slot + k_at[c] + h * 8 * STRIDE;
                if constexpr (K_WORDS == 4) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(at);
                    code[h][0] = w.x, code[h][1] = w.y, code[h][2] = w.z, code[h][3] = w.w;
                } else {
                    const uint2 w = *reinterpret_cast<const uint2 *>(at);
                    code[h][0] = w.x, code[h][1] = w.y;
                }
                unsigned scale = *reinterpret_cast<const unsigned short *>(slot + k_scale[c] + h * 16 * GROUPS);
                if (GROUPS % 2 && !k_some) scale = 0;
                factors[h] = int4_factors(scale * 0x10001u);
            }
#pragma unroll
            for (int w = 0; w < K_WORDS; w++) {
                unsigned x[2][4];
#pragma unroll
                for (int h = 0; h < 2; h++) int4_pairs(x[h], code[h][w], factors[h]);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const unsigned k[4] = {x[0][2 * i], x[1][2 * i], x[0][2 * i + 1], x[1][2 * i + 1]};
                    const int ks = 2 * w + i;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                        for (int piece = HELD ? 0 : QP - 1; piece >= 0; piece--) {
                            const uint2 q = HELD ? held[HELD ? ks : 0] : fragments[piece * (NT * KS * 32) + (nt * KS + ks) * 32 + lane];
                            float(&sum)[4] = z[!HELD && piece > 0 ? ZS - 1 : 0][nt];
                            if (ks == 0 && (piece == 0 || piece == QP - 1))
                                pg_mma_first(sum, k, q.x, q.y);
                            else
                                pg_mma(sum, k, q.x, q.y);
                        }
                    }
                }
            }
        };
        for (int i = 0; i < tiles * (CHUNKS / CH); i++) {
            const int c0 = CHUNKS == CH ? 0 : i % (CHUNKS / CH) * CH, j0 = begin + i / (CHUNKS / CH) * KEYS + 16 * c0; // the step's first key: it has 16 CH
            const unsigned char *const slot = sm.ring + slot_at * Shape::SLOT;
            if (c0 == 0 && alive && !__all_sync(0xFFFFFFFFu, pg_bar_wait(&sm.full[slot_at], parity))) give_up();
            const auto leave = [&] {
                if (c0 + CH < CHUNKS) return;
                __syncwarp();
                if (lane == 0 && alive) pg_bar_arrive(&sm.empty[slot_at]); // (what it has not waited for is not given back)
                if (++slot_at == SLOTS) slot_at = 0, parity ^= 1;
            };
            if (!alive || j0 >= length || j0 + 16 * CH <= low) {
                leave();
                continue;
            }
#pragma unroll
            for (int c = 0; c < CH; c++) scores(slot, c0 + c, z[c]);
            float x[CH][E][2]; // keys g and g + 8
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        if constexpr (PACK) {
                            x[c][e][h] = z[c][0][0][2 * h];
                            if constexpr (F32) {
                                x[c][e][h] += z[c][0][0][2 * h + 1]; // two pieces here, the third beside it
                                x[c][e][h] += __shfl_xor_sync(0xFFFFFFFFu, x[c][e][h], 1);
                            }
                        } else {
                            x[c][e][h] = z[c][0][e >> 1][2 * h + (e & 1)];
                            if constexpr (F32) x[c][e][h] += z[c][ZS - 1][e >> 1][2 * h + (e & 1)];
                        }
                    }
            if (a.softcap > 0.0f) { // (what is not seen may be anything, and goes after this)
                if constexpr (F32)
                    pg_cap_fine<2 * E * CH>(&x[0][0][0], a);
                else if (a.cap_far)
                    pg_cap<2 * E * CH, true>(&x[0][0][0], a);
                else
                    pg_cap<2 * E * CH, false>(&x[0][0][0], a);
            }
            const bool edge = j0 + 16 * CH > pos0 + 1 || j0 < all_lo;
            unsigned counts[CH][2]; // the scales of values
#pragma unroll
            for (int c = 0; c < CH; c++) counts[c][0] = counts[c][1] = 0xFFFFFFFFu;
            if (edge) { // a row sees positions up to its own, and with a window the last so many of them
#pragma unroll
                for (int c = 0; c < CH; c++) {
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const int r = row_of(e), hi = r < rows_of() ? pos0 + token_of(r) + 1 : 0, lo = a.window ? hi - a.window : 0;
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const int j = j0 + 16 * c + g + h * 8;
                            if (j >= hi || j < lo) x[c][e][h] = -INFINITY;
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) { // what stands in positions that no row sees, or of no sequence, counts as zero
                        const int j = j0 + 16 * c + 2 * t4 + (k & 1) + (k >> 1) * 8;
                        if (j >= length || j < low) counts[c][k >> 1] &= k & 1 ? 0xFFFFu : 0xFFFF0000u;
                    }
                }
            }
            bool more = false;
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int e = 0; e < E; e++) more |= x[c][e][0] > high[e] || x[c][e][1] > high[e];
            if (__any_sync(0xFFFFFFFFu, more)) {
                float keep[E];
#pragma unroll
                for (int e = 0; e < E; e++) {
                    float top = fmaxf(x[0][e][0], x[0][e][1]);
#pragma unroll
                    for (int c = 1; c < CH; c++) top = pg_max3(top, x[c][e][0], x[c][e][1]);
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, d));
                    top = fmaxf(m[e], top * unit);
                    keep[e] = m[e] == -INFINITY ? 0.0f : paged_exp2(m[e] - top);
                    m[e] = top, l[e] *= keep[e], high[e] = (top + 8.0f) * part_of_unit;
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int mt = 0; mt < MT; mt++)
#pragma unroll
                        for (int i = 0; i < 4; i++) o[nt][mt][i] *= keep[PACK ? 0 : 2 * nt + (i & 1)];
            }
            // ---- weights ----
            unsigned w[CH][NT][PACK ? 1 : WP][2]; // as pieces and turned, keys down
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float base = m[e] == -INFINITY ? 0.0f : -m[e];
#pragma unroll
                for (int c = 0; c < CH; c++)
#pragma unroll
                    for (int h = 0; h < 2; h++) x[c][e][h] = paged_exp2(fmaf(x[c][e][h], unit, base)), l[e] += x[c][e][h];
            }
#pragma unroll
            for (int c = 0; c < CH; c++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (PACK) {
                        const float rest = x[c][0][h] - __uint_as_float(pg_pack(x[c][0][h], 0.0f) << 16);
                        unsigned two = pg_pack(x[c][0][h], rest);
                        if constexpr (F32) {
                            const float last = rest - __uint_as_float(two & 0xFFFF0000u);
                            if (t4 & 1) two = pg_pack(last, 0.0f);
                        }
                        w[c][0][0][h] = pg_transpose(two);
                    } else {
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            unsigned piece[WP];
                            pg_split<WP>(piece, x[c][2 * nt][h], x[c][2 * nt + 1][h]);
#pragma unroll
                            for (int k = 0; k < WP; k++) w[c][nt][k][h] = pg_transpose(piece[k]);
                        }
                    }
                }
            // ---- values ----
            unsigned code[CH][4][V_WORDS];
            Int4Factors factors[CH][2];
#pragma unroll
            for (int c = 0; c < CH; c++) {
                unsigned scale[4];
#pragma unroll
                for (int k = 0; k < 4; k++) { // keys 2 t4, 2 t4 + 1, and eight further on
                    const int key = (k & 1) + (k >> 1) * 8;
                    const unsigned char *at = slot + v_at[c0 + c] + key * STRIDE;
                    if constexpr (V_WORDS == 2) {
                        const uint2 v = *reinterpret_cast<const uint2 *>(at);
                        code[c][k][0] = v.x, code[c][k][1] = v.y;
                    } else {
                        code[c][k][0] = *reinterpret_cast<const unsigned *>(at);
                    }
                    scale[k] = *reinterpret_cast<const unsigned short *>(slot + v_scale[c0 + c] + key * GROUPS * 2);
                }
#pragma unroll
                for (int h = 0; h < 2; h++) factors[c][h] = int4_factors(GROUPS % 2 && !v_some ? 0u : (scale[2 * h] | scale[2 * h + 1] << 16) & counts[c][h]);
            }
#pragma unroll
            for (int v = 0; v < V_WORDS; v++)
#pragma unroll
                for (int c = 0; c < CH; c++) {
                    unsigned even[2][4], odd[2][4]; // columns 2 i and 2 i + 1, of two keys each
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        int4_pairs(even[h], __byte_perm(code[c][2 * h][v], code[c][2 * h + 1][v], 0x5410), factors[c][h]);
                        int4_pairs(odd[h], __byte_perm(code[c][2 * h][v], code[c][2 * h + 1][v], 0x7632), factors[c][h]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const unsigned x4[4] = {even[0][i], odd[0][i], even[1][i], odd[1][i]};
                        const int mt = 4 * v + i;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            if constexpr (F32) {
                                constexpr int LAST = (PACK ? 1 : WP) - 1;
                                float d[4];
                                pg_mma_first(d, x4, w[c][nt][LAST][0], w[c][nt][LAST][1]);
#pragma unroll
                                for (int k = LAST - 1; k >= 0; k--) pg_mma(d, x4, w[c][nt][k][0], w[c][nt][k][1]);
#pragma unroll
                                for (int k = 0; k < 4; k++) o[nt][mt][k] += d[k];
                            } else {
#pragma unroll
                                for (int k = (PACK ? 1 : WP) - 1; k >= 0; k--) pg_mma(o[nt][mt], x4, w[c][nt][k][0], w[c][nt][k][1]);
                            }
                        }
                    }
                }
            leave();
        }

        // ---- the item's (or its part's) end: the warps' results meet, [four places][row][column] ----
#pragma unroll
        for (int e = 0; e < E; e++) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xFFFFFFFFu, l[e], d);
            if (side == 0 && g == 0 && !(PACK && F32 && (t4 & 1))) ml[slice][0][row_of(e)] = m[e], ml[slice][1][row_of(e)] = l[e];
        }
        few_meet<WARPS>();
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int r = row_of(e);
            float top = ml[0][0][r], sum = 0.0f;
#pragma unroll
            for (int k = 1; k < SLICES; k++) top = fmaxf(top, ml[k][0][r]);
            if (warp == 0) { // alike in all lanes that have the row
#pragma unroll
                for (int k = 0; k < SLICES; k++) sum = fmaf(ml[k][1][r], ml[k][0][r] == -INFINITY ? 0.0f : paged_exp2(ml[k][0][r] - top), sum);
                joined[0][r] = top, joined[1][r] = sum;
            }
            const float keep = m[e] == -INFINITY ? 0.0f : paged_exp2(m[e] - top);
#pragma unroll
            for (int mt = 0; mt < MT; mt++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (PACK || (i & 1) == (e & 1)) o[PACK ? 0 : e >> 1][mt][i] *= keep;
        }
        const auto share_out = [&](int to, bool add) { // four neighbouring columns at a time
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int mt = 0; mt < MT; mt += 2) {
                    float4 y;
                    const float(&u)[4] = o[PACK ? 0 : e >> 1][mt], (&v)[4] = o[PACK ? 0 : e >> 1][mt + 1];
                    if constexpr (PACK) {
                        y = make_float4(u[0] + u[1], u[2] + u[3], v[0] + v[1], v[2] + v[3]); // the pieces
                        if constexpr (F32) {
                            y.x += __shfl_xor_sync(0xFFFFFFFFu, y.x, 1), y.y += __shfl_xor_sync(0xFFFFFFFFu, y.y, 1);
                            y.z += __shfl_xor_sync(0xFFFFFFFFu, y.z, 1), y.w += __shfl_xor_sync(0xFFFFFFFFu, y.w, 1);
                            if (t4 & 1) continue;
                        }
                    } else {
                        y = make_float4(u[e & 1], u[2 + (e & 1)], v[e & 1], v[2 + (e & 1)]);
                    }
                    float4 *const at = reinterpret_cast<float4 *>(sm.meet + (to * ROWS + row_of(e)) * Shape::PITCH + g * (HDP / 8) + 2 * (side * MT + mt));
                    if (add) {
                        const float4 x4 = *at;
                        y.x += x4.x, y.y += x4.y, y.z += x4.z, y.w += x4.w;
                    }
                    *at = y;
                }
        };
        if constexpr (SLICES == 4) {
            share_out(slice, false);
        } else { // four of the eight add to the others'
            if (slice >= 4) share_out(slice - 4, false);
            few_meet<WARPS>();
            if (slice < 4) share_out(slice, true);
        }
        few_meet<WARPS>();
        const bool is_whole = item.before == 0 && item.tiles == item.count;
        const long long part_slot = (long long)blockIdx.x * 2 + (first_part && item.before > 0 ? 0 : 1);
        const PagedSeq s = item.s;
        const int rows = rows_of();
        unsigned long long wrong = 0;
#pragma unroll 1
        for (int r = tid / HDP; r < rows && !dead; r += 32 * WARPS / HDP) {
            const int col = tid % HDP, token = token_of(r);
            const float *at = sm.meet + r * Shape::PITCH + col;
            float y = (at[0] + at[ROWS * Shape::PITCH]) + (at[2 * ROWS * Shape::PITCH] + at[3 * ROWS * Shape::PITCH]);
            if (is_whole) {
                y *= paged_share(joined[1][r], s.pos0 + token);
                if (col < a.c.hd) paged_write(static_cast<RT *>(a.out) + ((long long)(s.first + token) * a.c.heads + item.kvh * a.c.group + r - token * a.c.group) * a.c.hd + col, y);
                if (col < a.c.hd && !(y * 0.0f == 0.0f)) wrong |= 1ull << r;
            } else {
                f.part[(part_slot * ROWS + r) * HDP + col] = y;
                if (col == 0) {
                    float *stats = f.part + (long long)gridDim.x * 2 * ROWS * HDP + part_slot * 2 * ROWS;
                    stats[r] = joined[0][r], stats[ROWS + r] = joined[1][r];
                }
            }
        }
        if (!is_whole && tid == 0 && item.before == 0 && !dead) few_head(f, item);
        if (wrong) atomicOr(&bad_rows, wrong);
        few_meet<WARPS>(); // what met is read, `bad_rows` is whole
        if (bad_rows) few_again<RT, Int4, WARPS>(a, item, &bad_rows, rows);
        if (lane == 0 && alive) pg_bar_arrive(&sm.item_empty[which]); // each warp for itself: it has read the item
        first_part = false;
    }
}

// ---- host side ----
// Rows of an item. 32 sequences of 5000 keys, 28 heads on 4, 3 tokens (21 rows): 97 us here, 157 by the kernel for many; of float32 146 and 190. 32 heads on 8, 6 tokens (24 rows): 172
// and 285, of float32 270 and 347. Five drafted tokens of 24 sequences (35 rows, window 4096, capped) took 117 to 122 us in this kernel and 90 in the one for many.
constexpr int FEW4_MOST = 24;

inline FewPlan few4_plan(int sms, bool f32_rows, int batch, int kv, int hdp, int rows, long long max_new, long long max_length, int window) {
    FewPlan p;
    p.most = rows, p.rows = rows <= (f32_rows ? 2 : 4) ? (f32_rows ? 2 : 4) : (rows <= 8 ? 8 : (rows <= 16 ? 16 : FEW4_MOST));
    // Wide tiles: items of up to eight are not cut where there are as many as blocks (32 sequences of 1250 keys, 16 heads: 35 us), of up to four where there are fewer.
    const int room = (p.rows > 16 ? 1 : 2) * sms;
    const bool pack = p.rows < 8;
    few_cut(&p, room, few4_keys(pack), batch, kv, hdp, max_new, max_length, window, pack && (long long)batch * kv < room ? FEW_WHOLE / 2 : FEW_WHOLE);
    return p;
}

template <typename RT, int GROUPS, int NT, bool PACK>
cudaError_t launch_few4_as(const AttendCall &a, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    using Shape = Few4Shape<RT, GROUPS, NT, PACK>;
    FewCall f;
    f.a = a, f.whole = p.whole, f.part = static_cast<float *>(ws), f.head = p.whole ? nullptr : reinterpret_cast<int *>(static_cast<float *>(ws) + p.part_floats);
    const auto kernel = attend_few_int4_kernel<RT, GROUPS, NT, PACK>;
    static std::atomic<bool> known[64];
    if (device >= 64 || !known[device].load()) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM);
        if (e != cudaSuccess) return e;
        if (device < 64) known[device].store(true);
    }
    kernel<<<p.blocks, Shape::THREADS, Shape::SMEM, st>>>(f);
    *launches += 1;
    if (!p.whole) {
        *launches += 1;
        return launch_following<FewCall>(attend_join_kernel<RT, Int4, Shape::HDP, Shape::ROWS>, dim3(p.blocks, p.most), 256, st, f);
    }
    return cudaGetLastError();
}
template <typename RT, int GROUPS>
cudaError_t launch_few4_rows(const AttendCall &a, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    if (p.rows < 8) return launch_few4_as<RT, GROUPS, 1, true>(a, p, ws, device, st, launches);
    if (p.rows == FEW4_MOST) return launch_few4_as<RT, GROUPS, 3, false>(a, p, ws, device, st, launches);
    return p.rows == 8 ? launch_few4_as<RT, GROUPS, 1, false>(a, p, ws, device, st, launches) : launch_few4_as<RT, GROUPS, 2, false>(a, p, ws, device, st, launches);
}
template <typename RT>
cudaError_t launch_few4(const AttendCall &a, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    switch (int4_groups(a.c.hd)) {
    case 1: return launch_few4_rows<RT, 1>(a, p, ws, device, st, launches);
    case 2: return launch_few4_rows<RT, 2>(a, p, ws, device, st, launches);
    case 3: return launch_few4_rows<RT, 3>(a, p, ws, device, st, launches);
    default: return launch_few4_rows<RT, 4>(a, p, ws, device, st, launches);
    }
}

} // namespace b200i

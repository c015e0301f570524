// The paged cache's entry points of the C ABI: argument checks, choice of kernel, launches. Declared in include/b200i.h.
#include <algorithm>
#include <cmath>

#include "../../include/b200i.h"
#include "library.h"
#include "paged.cuh"
#include "paged_append.cuh"
#include "paged_few.cuh"
#include "paged_fine.cuh"
#include "paged_int4.h"
#include "paged_many.cuh"
#include "paged_read.cuh"
#include "paged_unpack.cuh"

using namespace b200i;
using b200i_library::refuse;

namespace {

constexpr int64_t MOST = 0x7FFFFFFF;

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether `bytes` from `at` on meet one of the rows of `width` bytes, `pitch` apart, from `row` on.
bool meets_rows(const void *at, long long bytes, const void *row, long long width, long long pitch, long long rows) {
    const long long off = (long long)reinterpret_cast<uintptr_t>(at) - (long long)reinterpret_cast<uintptr_t>(row); // of the region from the first row
    const long long first = off < width ? 0 : (off - width) / pitch + 1;                                            // the first row that ends behind its beginning
    return first < rows && first * pitch < off + bytes;
}

// What both calls check, and the part of the arguments that they share. `who` names the call in messages.
int64_t shared_part(PagedCall *c, const char *who, int64_t row_type, int64_t cache_type, const void *page_table, const void *cu, const void *lengths, int64_t rows,
                    int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t pages, int64_t page, int64_t max_pages, char *err, int64_t err_cap) {
    if (rows <= 0 || batch <= 0 || n_heads <= 0 || n_kv <= 0 || head_dim <= 0 || pages <= 0 || page <= 0 || max_pages <= 0)
        return refuse(err, err_cap, "%s: extents must be positive", who);
    if (rows > MOST / 2 || batch > MOST / 2 || pages > MOST || max_pages > MOST || max_pages * page > MOST)
        return refuse(err, err_cap, "%s: rows, sequences, pages and positions are counted in 31 bits", who);
    if (rows * n_heads > MOST) return refuse(err, err_cap, "%s: rows times heads are counted in 31 bits", who);
    if (n_heads % n_kv != 0 || n_heads > 32767) return refuse(err, err_cap, "%s: n_heads must be a multiple of n_kv and below 32768", who);
    if (head_dim % 8 != 0 || head_dim > PAGED_MAX_HD) return refuse(err, err_cap, "%s: head_dim must be a multiple of 8 up to %d", who, PAGED_MAX_HD);
    if (page < 16 || page > 256 || (page & (page - 1)) != 0) return refuse(err, err_cap, "%s: a page holds a power of two from 16 to 256 positions", who);
    if ((row_type != B200I_T_F32 && row_type != B200I_T_BF16) || (cache_type != B200I_T_F32 && cache_type != B200I_T_BF16 && cache_type != B200I_T_INT4) ||
        (row_type == B200I_T_BF16 && cache_type == B200I_T_F32))
        return refuse(err, err_cap, "%s: rows and cache are float32 and float32, float32 and bfloat16, bfloat16 and bfloat16, or either and 4 bits", who);
    if (pages * n_kv * page > MOST) return refuse(err, err_cap, "%s: a pool of more than 2^31 - 1 rows of head_dim", who);
    if (!page_table || !cu || !lengths) return refuse(err, err_cap, "%s: null page table, row offsets or lengths", who);
    int shift = 0;
    while ((1 << shift) < page) shift++;
    c->table = static_cast<const int *>(page_table), c->cu = static_cast<const int *>(cu), c->lengths = static_cast<const int *>(lengths);
    c->rows = rows, c->batch = (int)batch, c->heads = (int)n_heads, c->kv = (int)n_kv, c->group = (int)(n_heads / n_kv), c->hd = (int)head_dim;
    c->group_part = (unsigned)((1ull << 32) / (unsigned long long)c->group + 1);
    c->pages = (int)pages, c->page_shift = shift, c->max_pages = (int)max_pages;
    return 0;
}

// After the arguments: the device and its status word.
int64_t enter(PagedCall *c, const char *who, int64_t device, int *dev, char *err, int64_t err_cap) {
    if (b200i_library::enter_device(device, err, err_cap, dev)) return 1;
    c->status = b200i_library::status_word(*dev);
    return c->status ? 0 : refuse(err, err_cap, "%s: the device has no status word", who);
}

// The kernel of a call and how its work is cut.
struct AttendPlan {
    int few;      // rows of a sequence and key head, where they are few (else 0)
    int hdp;      // head_dim as it is laid out in shared memory
    FewPlan cut;
    ManyPlan cut_many; // where they are many
    int64_t unpacked_bytes; // behind the parts, for a cache in 4 bits as bfloat16 words; 0: it is read as it is
    int64_t bytes() const { return few ? cut.bytes : (unpacked_bytes ? unpacked_at() + unpacked_bytes : cut_many.bytes); }
    int64_t unpacked_at() const { return (cut_many.bytes + 15) / 16 * 16; }
};

// A cache in 4 bits is made one of words first where a sequence's rows are more than UNPACK_BLOCKS blocks of rows, each of which would make the words for itself, and where the
// words of all positions that the page table has room for take at most UNPACK_MOST bytes. Measured, 16384 keys, 8 heads: 500 rows a key head 89 us without and 100 with it, 600 rows
// 141 and 109, 800 rows 191 and 134. It is done for the whole call: of a mixed one the single tokens' sequences are unpacked too, which still gains (a chunk of 1024 tokens behind 3000
// beside 12 single ones at 4000, 32 heads on 8: 218 us, 288 without; 512 tokens 170 and 200; 150 behind 7000 beside 6 at 7000: 152 and 151) or takes the call past UNPACK_MOST. Short
// calls lose 3 to 6 us, up to some 2000 positions: 1024 tokens behind nothing 62 us and 57 without, behind 300 68 and 69.
constexpr int64_t UNPACK_BLOCKS = 2, UNPACK_MOST = 256 << 20;

// `positions`: of the page table, max_pages * page. What a call does and what room it asks for go by the same plan.
AttendPlan attend_plan(int device, int64_t row_type, int64_t cache_type, int64_t rows, int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t max_new, int64_t max_length, int64_t window,
                       int64_t positions) {
    AttendPlan p = {};
    p.hdp = head_dim <= 64 ? 64 : 128;
    const int64_t group = n_heads / n_kv;
    const int64_t most = cache_type == B200I_T_INT4 ? int4_few_most() : FEW_MOST;
    if (max_new <= most && max_new * group <= most) {
        p.few = (int)(max_new * group);
        if (cache_type == B200I_T_INT4)
            p.cut = int4_few_plan(b200i_library::device_sms(device), row_type == B200I_T_F32, (int)batch, (int)n_kv, p.hdp, p.few, max_new, max_length, (int)std::min(window, MOST));
        else
            p.cut = few_plan(b200i_library::device_sms(device), row_type == B200I_T_F32, cache_type == B200I_T_F32, (int)batch, (int)n_kv, p.hdp, p.few, max_new, max_length,
                         (int)std::min(window, MOST));
    } else {
        const bool wide = row_type == B200I_T_BF16;
        p.cut_many = many_plan(b200i_library::device_sms(device), wide ? ManyShape<128>::BLOCK_ROWS : FINE_ROWS, p.hdp, wide ? MANY_KEYS : FINE_KEYS, rows, batch, n_kv, group, max_new,
                               std::min(max_length, MOST));
        if (cache_type == B200I_T_INT4 && wide && std::min(max_new, rows) * group > UNPACK_BLOCKS * ManyShape<128>::BLOCK_ROWS && positions > 0 &&
            4.0 * (double)batch * (double)n_kv * (double)head_dim * (double)positions <= (double)UNPACK_MOST)
            p.unpacked_bytes = unpack_bytes(batch, positions, n_kv, head_dim); // (and the table, a thousandth of it)
    }
    return p;
}

// Bytes of a position of a head.
long long cache_row_bytes(int64_t type, int64_t head_dim) { return type == B200I_T_INT4 ? INT4_BYTES * int4_groups((int)head_dim) : head_dim * (type == B200I_T_F32 ? 4 : 2); }

bool rows_fit(int64_t ld, int64_t width, int64_t type) { return ld >= width && (ld * (type == B200I_T_F32 ? 4 : 2)) % 16 == 0; }

} // namespace

extern "C" {

int64_t b200i_paged_append(int64_t device, void *stream, void *q_out, void *k_cache, void *v_cache, const void *q, const void *k, const void *v, int64_t ldq, int64_t ldk,
                           int64_t ldv, int64_t row_type, int64_t cache_type, const float *cosv, const float *sinv, int64_t rope_dim, int64_t positions, const float *q_norm,
                           const float *k_norm, double eps, int64_t norm_kind, const int32_t *page_table, const int32_t *cu, const int32_t *lengths, int64_t rows, int64_t batch,
                           int64_t n_heads, int64_t n_kv, int64_t head_dim, int64_t pages, int64_t page, int64_t max_pages, char *err, int64_t err_cap) {
    AppendCall a;
    if (shared_part(&a.c, "paged_append", row_type, cache_type, page_table, cu, lengths, rows, batch, n_heads, n_kv, head_dim, pages, page, max_pages, err, err_cap)) return 1;
    if (!q_out || !k_cache || !v_cache || !q || !k || !v) return refuse(err, err_cap, "paged_append: null storage");
    if (!aligned16(q_out) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(q) || !aligned16(k) || !aligned16(v) ||
        !rows_fit(ldq, n_heads * head_dim, row_type) || !rows_fit(ldk, n_kv * head_dim, row_type) || !rows_fit(ldv, n_kv * head_dim, row_type))
        return refuse(err, err_cap, "paged_append: rows must start on 16-byte boundaries and hold their heads side by side");
    const long long es = row_type == B200I_T_F32 ? 4 : 2, q_bytes = n_heads * head_dim * es, kv_bytes = n_kv * head_dim * es;
    const bool in_place = q_out == q && (ldq == n_heads * head_dim || rows == 1); // a head's words are read and written by one warp
    if ((!in_place && meets_rows(q_out, rows * q_bytes, q, q_bytes, ldq * es, rows)) || meets_rows(q_out, rows * q_bytes, k, kv_bytes, ldk * es, rows) ||
        meets_rows(q_out, rows * q_bytes, v, kv_bytes, ldv * es, rows))
        return refuse(err, err_cap, "paged_append: the output lies over rows that are read, other than queries in their very place");
    if ((cosv == nullptr) != (sinv == nullptr)) return refuse(err, err_cap, "paged_append: cos without sin, or sin without cos");
    if (rope_dim == 0 || !cosv) rope_dim = head_dim;
    if (rope_dim < 0 || rope_dim > head_dim || rope_dim % 2 != 0) return refuse(err, err_cap, "paged_append: rope_dim %lld does not fit head_dim %lld", (long long)rope_dim, (long long)head_dim);
    if (cosv && (positions <= 0 || positions > MOST)) return refuse(err, err_cap, "paged_append: the rotation table holds no position");
    if (norm_kind != 0 && norm_kind != 2) return refuse(err, err_cap, "paged_append: norm kind %lld is not 0 (weight w) or 2 (weight 1 + w)", (long long)norm_kind);
    a.q = q, a.k = k, a.v = v, a.q_out = q_out, a.k_cache = k_cache, a.v_cache = v_cache, a.ldq = ldq, a.ldk = ldk, a.ldv = ldv;
    a.cosv = cosv, a.sinv = sinv, a.q_norm = q_norm, a.k_norm = k_norm, a.rope_dim = (int)rope_dim, a.positions = (int)positions;
    a.part_of_head = 1.0f / (float)head_dim, a.eps = (float)eps, a.norm_shift = norm_kind == 2 ? 1.0f : 0.0f;
    int dev;
    if (enter(&a.c, "paged_append", device, &dev, err, err_cap)) return 1;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (cache_type == B200I_T_INT4)
        LIBRARY_CUDA_TRY(int4_append(a, row_type == B200I_T_F32, eps, b200i_library::device_sms(dev), st));
    else if (row_type == B200I_T_BF16)
        LIBRARY_CUDA_TRY((launch_append<__nv_bfloat16, __nv_bfloat16>(a, b200i_library::device_sms(dev), st)));
    else if (cache_type == B200I_T_BF16)
        LIBRARY_CUDA_TRY((launch_append<float, __nv_bfloat16>(a, b200i_library::device_sms(dev), st)));
    else
        LIBRARY_CUDA_TRY((launch_append<float, float>(a, b200i_library::device_sms(dev), st)));
    b200i_library::count_launches(1);
    b200i_library::accept(err, err_cap);
    return 0;
}

int64_t b200i_paged_read(int64_t device, void *stream, void *k_out, void *v_out, const void *k_cache, const void *v_cache, int64_t out_type, int64_t cache_type, const int32_t *page_table,
                         const int32_t *cu, const int32_t *lengths, int64_t rows, int64_t batch, int64_t n_kv, int64_t head_dim, int64_t pages, int64_t page, int64_t max_pages, char *err,
                         int64_t err_cap) {
    ReadCall a;
    if (shared_part(&a.c, "paged_read", out_type, cache_type, page_table, cu, lengths, rows, batch, n_kv, n_kv, head_dim, pages, page, max_pages, err, err_cap)) return 1;
    if (!k_out || !v_out || !k_cache || !v_cache) return refuse(err, err_cap, "paged_read: null storage");
    if (!aligned16(k_out) || !aligned16(v_out) || !aligned16(k_cache) || !aligned16(v_cache)) return refuse(err, err_cap, "paged_read: storage must start on 16-byte boundaries");
    const long long bytes = rows * n_kv * head_dim * (out_type == B200I_T_F32 ? 4 : 2), held = pages * n_kv * page * cache_row_bytes(cache_type, head_dim);
    if (meets_rows(k_out, bytes, v_out, bytes, bytes, 1) || meets_rows(k_out, bytes, k_cache, held, held, 1) || meets_rows(k_out, bytes, v_cache, held, held, 1) ||
        meets_rows(v_out, bytes, k_cache, held, held, 1) || meets_rows(v_out, bytes, v_cache, held, held, 1))
        return refuse(err, err_cap, "paged_read: the outputs may lie neither over one another nor over the caches");
    a.k_cache = k_cache, a.v_cache = v_cache, a.k_out = k_out, a.v_out = v_out;
    int dev;
    if (enter(&a.c, "paged_read", device, &dev, err, err_cap)) return 1;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int sms = b200i_library::device_sms(dev);
    if (cache_type == B200I_T_INT4)
        LIBRARY_CUDA_TRY((out_type == B200I_T_F32 ? launch_read<Int4, float>(a, sms, st) : launch_read<Int4, __nv_bfloat16>(a, sms, st)));
    else if (cache_type == B200I_T_BF16)
        LIBRARY_CUDA_TRY((out_type == B200I_T_F32 ? launch_read<__nv_bfloat16, float>(a, sms, st) : launch_read<__nv_bfloat16, __nv_bfloat16>(a, sms, st)));
    else
        LIBRARY_CUDA_TRY((launch_read<float, float>(a, sms, st)));
    b200i_library::count_launches(1);
    b200i_library::accept(err, err_cap);
    return 0;
}

int64_t b200i_paged_attention_table_workspace_bytes(int64_t device, int64_t row_type, int64_t cache_type, int64_t rows, int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                                                    int64_t max_new, int64_t max_length, int64_t window, int64_t positions) {
    if (rows <= 0 || batch <= 0 || n_kv <= 0 || n_heads < n_kv || head_dim <= 0 || max_new <= 0 || max_length <= 0 || window < 0) return 0;
    int dev = (int)device;
    if (device < 0 && cudaGetDevice(&dev) != cudaSuccess) { cudaGetLastError(); dev = -1; }
    return attend_plan(dev, row_type, cache_type, rows, batch, n_heads, n_kv, head_dim, max_new, max_length, window, positions).bytes();
}

int64_t b200i_paged_attention_workspace_bytes(int64_t device, int64_t row_type, int64_t cache_type, int64_t rows, int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                                              int64_t max_new, int64_t max_length, int64_t window) {
    const int64_t positions = max_length <= MOST ? (max_length + 255) / 256 * 256 : 0; // of whole pages of any size
    return b200i_paged_attention_table_workspace_bytes(device, row_type, cache_type, rows, batch, n_heads, n_kv, head_dim, max_new, max_length, window, positions);
}

int64_t b200i_paged_attention(int64_t device, void *stream, void *out, const void *q, int64_t ldq, const void *k_cache, const void *v_cache, int64_t row_type, int64_t cache_type,
                              const int32_t *page_table, const int32_t *cu, const int32_t *lengths, int64_t rows, int64_t batch, int64_t n_heads, int64_t n_kv, int64_t head_dim,
                              int64_t pages, int64_t page, int64_t max_pages, int64_t max_new, int64_t max_length, double scale, int64_t window, double softcap, void *ws,
                              int64_t ws_bytes, char *err, int64_t err_cap) {
    AttendCall a;
    if (shared_part(&a.c, "paged_attention", row_type, cache_type, page_table, cu, lengths, rows, batch, n_heads, n_kv, head_dim, pages, page, max_pages, err, err_cap)) return 1;
    if (!out || !q || !k_cache || !v_cache) return refuse(err, err_cap, "paged_attention: null storage");
    if (!aligned16(out) || !aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || !rows_fit(ldq, n_heads * head_dim, row_type))
        return refuse(err, err_cap, "paged_attention: rows must start on 16-byte boundaries and hold their heads side by side");
    const long long row_bytes = n_heads * head_dim * (row_type == B200I_T_F32 ? 4 : 2);
    if (meets_rows(out, rows * row_bytes, q, row_bytes, ldq * (row_type == B200I_T_F32 ? 4 : 2), rows))
        return refuse(err, err_cap, "paged_attention: the output may not lie over the queries, which may be read again");
    if (max_new <= 0 || max_length <= 0) return refuse(err, err_cap, "paged_attention: the bounds on new tokens and lengths must be positive");
    if (window < 0 || !(softcap >= 0.0) || softcap > 1e30 || !(scale > -1e30 && scale < 1e30)) return refuse(err, err_cap, "paged_attention: window, softcap or scale is out of range");
    if (ws_bytes < 0 || (ws_bytes > 0 && !ws)) return refuse(err, err_cap, "paged_attention: a workspace size without a workspace");
    if (ws_bytes > 0 && !aligned16(ws)) return refuse(err, err_cap, "paged_attention: the workspace must start on a 16-byte boundary");
    a.q = q, a.k = k_cache, a.v = v_cache, a.out = out, a.ldq = ldq, a.flip = scale < 0.0;
    a.softcap = softcap > 0.0 ? std::max((float)softcap, 1e-30f) : 0.0f; // (a cap of next to nothing is still one: all weights alike)
    a.scale = std::max(fabsf((float)scale), 1e-30f); // none makes all weights alike, as does next to none
    // scale / softcap and its inverse, held to what 32 bits have: there next to every score is far below the cap, or far above it
    const auto within = [](double x) { return (float)std::min(std::max(x, 1.2e-38), 3.4e38); };
    a.cap_part = a.softcap > 0.0f ? 1.0f / a.softcap : 0.0f;
    a.cap_inner = a.softcap > 0.0f ? within((double)a.scale / a.softcap) : 0.0f, a.cap_outer = a.softcap > 0.0f ? within((double)a.softcap / a.scale) : 0.0f;
    a.cap_far = !(a.cap_inner > 1e-4f && a.cap_inner < 1e4f);
    float power = 1.0f;
    for (int i = 0; i < 4; i++) power *= a.cap_far ? 1.0f : a.cap_inner * a.cap_inner, a.cap_near[i] = CAP_NEAR[i] * power;
    // a window as wide as the table is none; so a position and a window's difference stays in 32 bits
    a.window = window < max_pages * page ? (int)window : 0, a.max_new = (int)std::min(max_new, MOST);
    int dev, launches = 0;
    if (enter(&a.c, "paged_attention", device, &dev, err, err_cap)) return 1;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    AttendPlan p = attend_plan(dev, row_type, cache_type, rows, batch, n_heads, n_kv, head_dim, max_new, max_length, window, max_pages * page);
    if (ws_bytes < p.bytes()) p.unpacked_bytes = 0; // there is no room for words
    if (ws_bytes < p.bytes()) return refuse(err, err_cap, "paged_attention: the workspace holds %lld bytes of %lld", (long long)ws_bytes, (long long)p.bytes());
    if (p.unpacked_bytes) {
        LIBRARY_CUDA_TRY(launch_unpack(&a, static_cast<unsigned char *>(ws) + p.unpacked_at(), max_length, st));
        launches++;
        LIBRARY_CUDA_TRY((p.hdp == 64 ? launch_many_as<__nv_bfloat16, 64>(a, p.cut_many, ws, dev, st, &launches) : launch_many_as<__nv_bfloat16, 128>(a, p.cut_many, ws, dev, st, &launches)));
    } else if (cache_type == B200I_T_INT4) {
        LIBRARY_CUDA_TRY(p.few ? int4_few(a, row_type == B200I_T_F32, p.cut, ws, dev, st, &launches) : int4_many(a, row_type == B200I_T_F32, p.cut_many, p.hdp, ws, dev, st, &launches));
    } else if (p.few) {
        if (row_type == B200I_T_BF16)
            LIBRARY_CUDA_TRY((launch_few<__nv_bfloat16, __nv_bfloat16>(a, p.cut, p.hdp, ws, dev, st, &launches)));
        else if (cache_type == B200I_T_BF16)
            LIBRARY_CUDA_TRY((launch_few<float, __nv_bfloat16>(a, p.cut, p.hdp, ws, dev, st, &launches)));
        else
            LIBRARY_CUDA_TRY((launch_few<float, float>(a, p.cut, p.hdp, ws, dev, st, &launches)));
    } else {
        if (row_type == B200I_T_BF16)
            LIBRARY_CUDA_TRY((p.hdp == 64 ? launch_many_as<__nv_bfloat16, 64>(a, p.cut_many, ws, dev, st, &launches) : launch_many_as<__nv_bfloat16, 128>(a, p.cut_many, ws, dev, st, &launches)));
        else if (cache_type == B200I_T_BF16)
            LIBRARY_CUDA_TRY((p.hdp == 64 ? launch_fine_as<__nv_bfloat16, 64>(a, p.cut_many, ws, dev, st, &launches) : launch_fine_as<__nv_bfloat16, 128>(a, p.cut_many, ws, dev, st, &launches)));
        else
            LIBRARY_CUDA_TRY((p.hdp == 64 ? launch_fine_as<float, 64>(a, p.cut_many, ws, dev, st, &launches) : launch_fine_as<float, 128>(a, p.cut_many, ws, dev, st, &launches)));
    }
    b200i_library::count_launches(launches);
    b200i_library::accept(err, err_cap);
    return 0;
}

} // extern "C"

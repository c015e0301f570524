// Barriers, tensor-map copies and matrix fragments of the paged kernels.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace b200i {

constexpr int PAGED_WAIT = 13;                   // the status word: a bounded wait ran out
constexpr unsigned PAGED_SPIN_LIMIT = 1u << 22;  // tries of a wait; each suspends the thread for a while

__device__ __forceinline__ unsigned pg_smem(const void *p) { return (unsigned)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void pg_bar_init(unsigned long long *bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(pg_smem(bar)), "r"(count));
}
__device__ __forceinline__ void pg_bar_expect(unsigned long long *bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(pg_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void pg_bar_arrive(unsigned long long *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pg_smem(bar)) : "memory");
}
// Waits for the phase of the given parity to end; false where the limit ran out.
__device__ __forceinline__ bool pg_bar_wait(unsigned long long *bar, unsigned parity) {
    for (unsigned spin = 0; spin < PAGED_SPIN_LIMIT; spin++) {
        unsigned done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(pg_smem(bar)), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}
__device__ __forceinline__ void pg_tma_load(void *dst, const CUtensorMap *map, unsigned long long *bar, int col, int row) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(pg_smem(dst)),
                 "l"(reinterpret_cast<unsigned long long>(map)), "r"(pg_smem(bar)), "r"(col), "r"(row)
                 : "memory");
}

// D (16 x 8, 32 bits) += A (16 x 16) B (16 x 8), bfloat16
__device__ __forceinline__ void pg_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void pg_mma_first(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) { // D = A B
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void pg_ldmatrix(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void pg_ldmatrix_t(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ unsigned pg_transpose(unsigned v) { // an 8 x 8 matrix of 16-bit words across the warp
    unsigned r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ unsigned pg_pack(float lo, float hi) { // two words rounded to bfloat16, `lo` in the lower half
    unsigned r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// Two 32-bit words as sums of N bfloat16 pieces each: a piece is what is left rounded to 8 bits, so three hold all 24.
template <int N>
__device__ __forceinline__ void pg_split(unsigned (&piece)[N], float x, float y) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        piece[i] = pg_pack(x, y);
        if (i + 1 < N) x -= __uint_as_float(piece[i] << 16), y -= __uint_as_float(piece[i] & 0xFFFF0000u);
    }
}

// Two 32-bit words at a time.
__device__ __forceinline__ unsigned long long pg_two(float x, float y) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void pg_one(unsigned long long v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ unsigned long long pg_fma2(unsigned long long x, unsigned long long y, unsigned long long z) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ unsigned long long pg_add2(unsigned long long x, unsigned long long y) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
__device__ __forceinline__ unsigned long long pg_mul2(unsigned long long x, unsigned long long y) {
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// A kernel that joins what the one before it left: its blocks are brought in while that one ends (pg_follow_early there lets them), and go on from
// pg_follow when it has ended and what it wrote is to be seen.
__device__ __forceinline__ void pg_follow_early() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pg_follow() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename F>
inline cudaError_t launch_following(void (*kernel)(const F), dim3 grid, int threads, cudaStream_t st, const F &f) {
    cudaLaunchConfig_t c = {};
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    c.gridDim = grid, c.blockDim = dim3(threads), c.stream = st, c.attrs = &early, c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, f);
}

// A cache as a matrix of rows of head_dim, in boxes of 128 bytes by `box_rows` rows, 128-byte swizzle, zeros outside.
typedef CUresult (*PagedEncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline bool paged_map(CUtensorMap *map, const void *base, long long rows, int hd, bool f32, int box_rows) {
    static const PagedEncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<PagedEncodeFn>(p);
    }();
    if (!fn) return false;
    const int es = f32 ? 4 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)hd * es};
    const cuuint32_t box[2] = {128u / es, (cuuint32_t)box_rows}, estr[2] = {1u, 1u};
    return fn(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

} // namespace b200i

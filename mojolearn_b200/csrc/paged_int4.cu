// The kernels for caches in 4 bits: a translation unit of their own, so that it compiles beside the other.
#include "paged_int4.h"

#include "paged_append_int4.cuh"
#include "paged_few_int4.cuh"
#include "paged_fine.cuh"

namespace b200i {

int int4_few_most() { return FEW4_MOST; }
FewPlan int4_few_plan(int sms, bool f32_rows, int batch, int kv, int hdp, int rows, long long max_new, long long max_length, int window) {
    return few4_plan(sms, f32_rows, batch, kv, hdp, rows, max_new, max_length, window);
}
cudaError_t int4_few(const AttendCall &a, bool f32_rows, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches) {
    return f32_rows ? launch_few4<float>(a, p, ws, device, st, launches) : launch_few4<__nv_bfloat16>(a, p, ws, device, st, launches);
}
cudaError_t int4_many(const AttendCall &a, bool f32_rows, const ManyPlan &p, int hdp, void *ws, int device, cudaStream_t st, int *launches) {
    if (f32_rows) return hdp == 64 ? launch_fine_as<Int4, 64>(a, p, ws, device, st, launches) : launch_fine_as<Int4, 128>(a, p, ws, device, st, launches);
    return hdp == 64 ? launch_many_as<Int4, 64>(a, p, ws, device, st, launches) : launch_many_as<Int4, 128>(a, p, ws, device, st, launches);
}
cudaError_t int4_append(const AppendCall &a, bool f32_rows, double eps, int sms, cudaStream_t st) {
    return f32_rows ? launch_append4<float>(a, eps, sms, st) : launch_append4<__nv_bfloat16>(a, eps, sms, st);
}

} // namespace b200i

// The kernels for caches in 4 bits, compiled apart (paged_int4.cu), as paged.cu launches them.
#pragma once
#include "paged_append.cuh"
#include "paged_many.cuh"
#include "paged_read.cuh"

namespace b200i {

// The most rows of a sequence and key head that int4_few takes.
int int4_few_most();
FewPlan int4_few_plan(int sms, bool f32_rows, int batch, int kv, int hdp, int rows, long long max_new, long long max_length, int window);
cudaError_t int4_few(const AttendCall &a, bool f32_rows, const FewPlan &p, void *ws, int device, cudaStream_t st, int *launches);
cudaError_t int4_many(const AttendCall &a, bool f32_rows, const ManyPlan &p, int hdp, void *ws, int device, cudaStream_t st, int *launches);
cudaError_t int4_append(const AppendCall &a, bool f32_rows, double eps, int sms, cudaStream_t st);

} // namespace b200i

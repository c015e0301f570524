// What the translation units of libb200i.so share of b200i.cu: the error convention, the device, the status word.
#pragma once
#include <cstdint>

namespace b200i_library {

int64_t refuse(char *err, int64_t cap, const char *fmt, ...); // writes the message, returns 1
void accept(char *err, int64_t cap);                          // empties the message buffer
// Makes `device` current (-1: the current one stays) and hands its number out; nonzero with a message where that fails.
int64_t enter_device(int64_t device, char *err, int64_t cap, int *out);
int device_sms(int device);
// The device address of the status word that b200i_decode_status reads (the current device's); nullptr where it has none.
int *status_word(int device);
void count_launches(int n);

} // namespace b200i_library

#define LIBRARY_CUDA_TRY(expr)                                                                                               \
    do {                                                                                                                     \
        cudaError_t e_ = (expr);                                                                                             \
        if (e_ != cudaSuccess) return b200i_library::refuse(err, err_cap, "b200i: %s failed: %s", #expr, cudaGetErrorString(e_)); \
    } while (0)

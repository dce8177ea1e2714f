// op_support.h -- what the standalone ops (ops.cu, kv8.cu, logprob.cu) share on the host: the
// per-thread error text and the per-device status word behind mossgpu_op_device_status.
#pragma once

#include <cuda_runtime.h>

namespace mossgpu {

// Codes of mossgpu_op_device_status (7 and 8 are the bounded waits of k_attn_decode).
constexpr int kStatusBadPosition = 9;  // a slot or position outside the page table
constexpr int kStatusBadPage = 10;     // a page id outside the pool
constexpr int kStatusBadToken = 11;    // a token id >= vocab

// Formats the message mossgpu_op_last_error() returns on this thread; always returns 1.
#if defined(__GNUC__)
__attribute__((format(printf, 1, 2)))
#endif
int op_errorf(const char *fmt, ...) noexcept;

// The current device's ordinal and the device address of its status word; 0 or an error.
int op_device(int *dev, int **status, const char *who) noexcept;

}  // namespace mossgpu

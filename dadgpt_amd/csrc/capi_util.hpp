// What the C entry points of libdadgpt_attn.so share (capi.cpp): the thread's last error, and the
// argument checks, each of which answers a status on the host before any HIP call.
#pragma once

#include <hip/hip_runtime.h>

#include <initializer_list>

#include "kernels.hpp"

namespace dadgpt::capi {

// Records the message and returns the status.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int ok();
int from_hip(hipError_t e, const char* what);

bool supported(int d_head);
inline hipStream_t as_stream(void* s) { return static_cast<hipStream_t>(s); }

// Non-null and 16-byte aligned, by position.
int check_ptrs(const char* fn, std::initializer_list<const void*> ptrs);
int check_decode_shape(const char* fn, int n_seq, int H, int max_len, int d_head, float scale,
                       std::initializer_list<const void*> ptrs);
int check_window(const char* fn, long long S, int window, int sinks);

}  // namespace dadgpt::capi

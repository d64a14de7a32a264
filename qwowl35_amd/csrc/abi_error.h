// The C ABI's error convention, 0 + err[err_len] (Qw35FFI.m:15-22), for the entry points of every translation unit.
#pragma once

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

namespace qw35 {

inline void set_err(char* err, uintptr_t err_len, const char* fmt, ...) {
    if (!err || err_len == 0) return;
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(err, (size_t)err_len, fmt, ap);
    va_end(ap);
}

inline bool check_hip(hipError_t e, const char* what, char* err, uintptr_t err_len) {
    if (e == hipSuccess) return true;
    set_err(err, err_len, "%s: %s", what, hipGetErrorString(e));
    return false;
}

}  // namespace qw35

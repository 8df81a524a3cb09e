// What the serving operators' sources share: element types and the host-side
// checks every entry point makes.
#ifndef SERVE_COMMON_H
#define SERVE_COMMON_H

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "../../include/fa_serve.h"

namespace {

// The stream must belong to the current device: kernels and per-device state
// are looked up for the current one.
inline int check_stream_device(void* stream) {
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (!st || st == hipStreamLegacy || st == hipStreamPerThread) return FA_SERVE_OK;
  int dev = 0, sdev = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipStreamGetDevice(st, &sdev) != hipSuccess)
    return FA_SERVE_ERR_LAUNCH;
  return sdev == dev ? FA_SERVE_OK : FA_SERVE_ERR_DEVICE;
}

inline bool aligned(const void* p, uintptr_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// log2 of a page size the operators take, or -1.
inline int page_shift(int64_t size) {
  for (int s = 4; s <= 16; ++s)
    if (size == (int64_t)1 << s) return s;
  return -1;
}

// A stride in elements: a non-negative multiple of 8 (16-byte rows) within 2^40.
inline int check_strides(const int64_t* s, int n) {
  for (int i = 0; i < n; ++i) {
    if (s[i] < 0 || s[i] > (int64_t)1 << 40) return FA_SERVE_ERR_STRIDE;
    if (s[i] % 8) return FA_SERVE_ERR_ALIGN;
  }
  return FA_SERVE_OK;
}

// hipLaunchKernel returns the status of this launch alone; errors left pending
// by the caller's earlier work are neither read nor cleared.
inline int enqueue(const void* fn, dim3 grid, dim3 block, void** args, unsigned lds, void* stream) {
  return hipLaunchKernel(fn, grid, block, args, lds, reinterpret_cast<hipStream_t>(stream)) == hipSuccess
             ? FA_SERVE_OK
             : FA_SERVE_ERR_LAUNCH;
}

}  // namespace

#endif  // SERVE_COMMON_H

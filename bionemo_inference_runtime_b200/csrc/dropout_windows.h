// The windows in which a row of numbered elements is taken where rows begin off the 16-byte boundaries.  Integer code without CUDA
// calls, so that it also compiles for the host alone, where a test walks the windows of rows longer than any test's tensor.
#pragma once
#include <stdint.h>

#ifdef __CUDACC__
#define B200TA_DROPOUT_WINDOW __host__ __device__ __forceinline__
#else
#define B200TA_DROPOUT_WINDOW inline
#endif

namespace b200ta {

// A block of threads makes the bits of kDropoutBits numbered elements from a multiple of eight on; up to seven of them lie before its window.
constexpr int kDropoutBits = 2048, kDropoutWindow = kDropoutBits - 8;

struct DropoutWindow {
  int64_t outer, first;  // of which row, and the window's first element in it
  int width;
};
B200TA_DROPOUT_WINDOW int64_t dropout_windows(int64_t inner) { return (inner + kDropoutWindow - 1) / kDropoutWindow; }
// That of block `block`, with `windows` to a row of `inner` elements.
B200TA_DROPOUT_WINDOW DropoutWindow dropout_window(uint32_t block, uint32_t windows, int64_t inner) {
  const int64_t first = int64_t(block % windows) * kDropoutWindow, left = inner - first;
  return {int64_t(block / windows), first, left < kDropoutWindow ? int(left) : kDropoutWindow};
}

}  // namespace b200ta

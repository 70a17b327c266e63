// Device helpers shared by the KV-cache operators (kvattn.cu, kvcache.cu):
// which position a cache slot holds, what a node sees, the int8 query.
#pragma once

#include <climits>
#include <cstdint>
#include <cuda_runtime.h>

#include "fgm_cuda.h"

namespace fgm {
namespace kv {

// Committed tokens of sequence b, kept inside what its cache can hold, so a
// wrong length never leads outside the buffers.
__device__ __forceinline__ int committed(const fgm_cuda_kv &kv, const int32_t *lens, int b, int T) {
  const int most = kv.ring ? INT_MAX - T : kv.cap - T;
  const int n = lens[b];
  return n < 0 ? 0 : (n > most ? most : n);
}

// Slot of position t.
__device__ __forceinline__ int slot_of(const fgm_cuda_kv &kv, int t) {
  return kv.ring ? t % kv.ring : t;
}

// Position that slot x holds once positions [0, end) are written (the newest
// that maps there); negative: none.  Linear: its index (at or past end: none).
__device__ __forceinline__ int pos_of(int ring, int x, int end) {
  if (!ring) return x < end ? x : -1;
  const int last = end - 1;
  int d = (last - x) % ring;
  if (d < 0) d += ring;
  return x < ring ? last - d : -1;
}

// Lowest position a node at position p sees under `window` (0: all).
__device__ __forceinline__ int lowest(int p, int window) {
  if (!window) return INT_MIN;
  const long long v = (long long)p - window + 1;
  return v < INT_MIN ? INT_MIN : (int)v;
}

__device__ __forceinline__ float q_inv(float top) {
  return top > 0.0f ? __fdiv_rn(127.0f, top) : 0.0f;
}

// One value of the int8 query (a value that is no number gives some int8;
// its head is not-a-number by its scale).
__device__ __forceinline__ int q_int8(float v, float inv) {
  const int i = __float2int_rn(__fmul_rn(v, inv));
  return i > 127 ? 127 : (i < -127 ? -127 : i);
}

// The query scale max|q| / 127, not-a-number when a value is no finite number
// (top: the largest |q|, infinite when one of them is or is no number).
__device__ __forceinline__ float q_scale(float top) {
  return top < __int_as_float(0x7f800000) ? __fdiv_rn(top, 127.0f) : __int_as_float(0x7fffffff);
}

// |v| for the maximum, infinity for not-a-number.
__device__ __forceinline__ float q_abs(float v) {
  const float a = fabsf(v);
  return a == a ? a : __int_as_float(0x7f800000);
}

}  // namespace kv
}  // namespace fgm

// Attention of several tokens per sequence over the int8 KV cache and the
// weights it accumulates per slot.
#include "fgm_internal.h"
#include "kv_common.cuh"

namespace fgm {
namespace {

using namespace kv;

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

constexpr int kMaxHd = 512;

// Warp: int8 copy of one query head in shared memory, its scale returned.
__device__ float quant_head(const float *q, int hd, int8_t *q8, int lane) {
  float top = 0.0f;
  for (int d = lane; d < hd; d += 32) top = fmaxf(top, q_abs(q[d]));
  top = warp_max(top);
  const float inv = q_inv(top);
  for (int d = lane; d < hd; d += 32) q8[d] = (int8_t)q_int8(q[d], inv);
  __syncwarp();
  return q_scale(top);
}

__device__ __forceinline__ bool sees(const TreeParams &p, int b, int i, int len, int t, int low) {
  if (t < 0) return false;
  if (t < len) return t >= low;
  const int j = t - len;
  if (p.mask) {
    const int w = (p.T + 63) / 64;
    if (!((p.mask[((size_t)b * p.T + i) * w + (j >> 6)] >> (j & 63)) & 1)) return false;
  } else if (j > i) {
    return false;
  }
  return !p.window || (p.pos ? p.pos[b * p.T + j] : t) >= low;
}

// One CTA per (node, head): four warps walk the slots, each with its own
// running maximum, sum and output, joined at the end.
__global__ void __launch_bounds__(128) attend_kernel(const TreeParams p) {
  __shared__ __align__(16) int8_t q8[kMaxHd];
  __shared__ float s_m[4], s_l[4], s_o[4][kMaxHd];
  const int hd = p.kv.head_dim, kvd = p.kv.kv_heads * hd;
  const int r = blockIdx.x, h = blockIdx.y, b = r / p.T, i = r % p.T;
  const int kvh = h / (p.n_heads / p.kv.kv_heads);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ float s_qs;
  if (warp == 0) {
    const float s = quant_head(p.q + (size_t)r * p.q_ld + (size_t)h * hd, hd, q8, lane);
    if (lane == 0) s_qs = s;
  }
  __syncthreads();
  const float qs = s_qs;
  const int len = committed(p.kv, p.lens, b, p.T), end = len + p.T;
  const int low = lowest(p.pos ? p.pos[r] : len + i, p.window);
  const int slots = p.kv.ring ? min(p.kv.ring, end) : end;
  const int8_t *kc = p.kv.kc + (size_t)b * p.kv.kc_stride + (size_t)kvh * hd;
  const int8_t *vt = p.kv.vt + (size_t)b * p.kv.vt_stride + (size_t)kvh * hd * 4;
  const float *ks = p.kv.ks + (size_t)b * p.kv.ks_stride, *vs = p.kv.vs + (size_t)b * p.kv.vs_stride;
  float m = -INFINITY, l = 0.0f, o[16];
  for (int k = 0; k < 16; k++) o[k] = 0.0f;
  for (int x = warp; x < slots; x += 4) {
    if (!sees(p, b, i, len, pos_of(p.kv.ring, x, end), low)) continue;
    int dot = 0;
    for (int d = lane * 4; d < hd; d += 128)
      dot = __dp4a(*reinterpret_cast<const int *>(kc + (size_t)x * kvd + d),
                   *reinterpret_cast<const int *>(q8 + d), dot);
    dot = __reduce_add_sync(0xffffffffu, dot);
    const float s = __fmul_rn(__fmul_rn((float)dot, qs), ks[x]);
    const float mn = s > m ? s : m;
    const float ref = mn == -INFINITY ? 0.0f : mn;
    const float c = expf(m - ref), e = expf(s - ref);
    l = l * c + e;
    m = mn;
    for (int k = 0; k < 16; k++) {
      const int d = lane + 32 * k;
      if (d < hd)
        o[k] = o[k] * c + e * vs[x] * (float)vt[((size_t)(x >> 2) * kvd + d) * 4 + (x & 3)];
    }
  }
  if (lane == 0) s_m[warp] = m, s_l[warp] = l;
  for (int k = 0; k < 16; k++)
    if (lane + 32 * k < hd) s_o[warp][lane + 32 * k] = o[k];
  __syncthreads();
  float M = -INFINITY, L = 0.0f;
  for (int w = 0; w < 4; w++) M = s_m[w] > M ? s_m[w] : M;
  const float ref = M == -INFINITY ? 0.0f : M;
  for (int w = 0; w < 4; w++) L += s_l[w] * expf(s_m[w] - ref);
  const bool none = L == 0.0f;
  for (int d = tid; d < hd; d += 128) {
    float v = 0.0f;
    for (int w = 0; w < 4; w++) v += s_o[w][d] * expf(s_m[w] - ref);
    p.out[(size_t)r * p.out_ld + (size_t)h * hd + d] = none ? 0.0f : v / L;
  }
  if (tid == 0 && p.lse) p.lse[r * p.lse_row + h * p.lse_head] = none ? -INFINITY : M + logf(L);
}

// One warp per slot: all nodes and heads in order.
__global__ void __launch_bounds__(128) accum_kernel(const TreeParams p) {
  __shared__ __align__(16) int8_t q8[4][kMaxHd];
  const int hd = p.kv.head_dim, kvd = p.kv.kv_heads * hd, b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int x = blockIdx.x * 4 + warp;
  const int len = committed(p.kv, p.lens, b, p.T), end = len + p.T;
  const int t = pos_of(p.kv.ring, x, end);
  if (x >= p.kv.cap || t < 0) return;
  const int G = p.n_heads / p.kv.kv_heads;
  const float ks = p.kv.ks[(size_t)b * p.kv.ks_stride + x];
  float sum = 0.0f;
  for (int i = 0; i < p.T; i++) {
    const int r = b * p.T + i;
    if (p.take && !p.take[r]) continue;
    if (!sees(p, b, i, len, t, lowest(p.pos ? p.pos[r] : len + i, p.window))) continue;
    for (int h = 0; h < p.n_heads; h++) {
      const float lse = p.lse[r * p.lse_row + h * p.lse_head];
      if (lse == -INFINITY) continue;
      const float qs = quant_head(p.q + (size_t)r * p.q_ld + (size_t)h * hd, hd, q8[warp], lane);
      const int8_t *kr = p.kv.kc + (size_t)b * p.kv.kc_stride + (size_t)x * kvd + (h / G) * hd;
      int dot = 0;
      for (int d = lane * 4; d < hd; d += 128)
        dot = __dp4a(*reinterpret_cast<const int *>(kr + d),
                     *reinterpret_cast<const int *>(&q8[warp][d]), dot);
      dot = __reduce_add_sync(0xffffffffu, dot);
      __syncwarp();
      sum += expf(__fmul_rn(__fmul_rn((float)dot, qs), ks) - lse);
    }
  }
  if (lane == 0) {
    float *a = p.kv.acc + (size_t)b * p.kv.acc_stride + x;
    *a = (t < len ? p.decay * *a : 0.0f) + sum;
  }
}

}  // namespace

size_t attend_workspace(const fgm_cuda_kv &kv, int n_heads, int T) {
  return (size_t)kv.rows * T * n_heads * sizeof(float);
}

cudaError_t launch_attend_tree(const TreeParams &p, int num_sms, cudaStream_t st) {
  attend_kernel<<<dim3((unsigned)(p.kv.rows * p.T), (unsigned)p.n_heads), 128, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_attend_accum(const TreeParams &p, int num_sms, cudaStream_t st) {
  const int slots = p.kv.ring ? p.kv.ring : p.kv.cap;
  accum_kernel<<<dim3((unsigned)((slots + 3) / 4), (unsigned)p.kv.rows), 128, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_attend_acc(const TreeParams &p, int num_sms, cudaStream_t st) {
  TreeParams a = p;
  a.lse = static_cast<float *>(p.ws);
  a.lse_row = (size_t)p.n_heads;
  a.lse_head = 1;
  const cudaError_t e = launch_attend_tree(a, num_sms, st);
  return e != cudaSuccess ? e : launch_attend_accum(a, num_sms, st);
}

}  // namespace fgm

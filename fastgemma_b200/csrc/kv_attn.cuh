// What the attention kernels over the KV cache share (kvattn.cu: few query
// rows, kvtile.cu: many): visibility, the division of the work, the join of
// partial results, launch helpers.
#pragma once

#include <atomic>
#include <type_traits>

#include <cuda_fp16.h>

#include "fgm_internal.h"
#include "kv_common.cuh"

namespace fgm {
namespace kv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Four int8 as two pairs of f16, exact: 1024 + (v + 128) has v in its low
// mantissa byte, minus 1152.
__device__ __forceinline__ void i8x4_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
  w ^= 0x80808080u;
  const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
  uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  __half2 x = __hsub2(*reinterpret_cast<__half2 *>(&a), off);
  __half2 y = __hsub2(*reinterpret_cast<__half2 *>(&b), off);
  lo = *reinterpret_cast<uint32_t *>(&x);
  hi = *reinterpret_cast<uint32_t *>(&y);
}

// Whether a row's node sees position t (node: -1 for a padding row).
__device__ __forceinline__ bool sees(const TreeParams &p, int b, int node, int len, int t,
                                     int low) {
  if (t < 0 || node < 0) return false;
  if (t < len) return t >= low;
  const int j = t - len;
  if (p.mask) {
    const int w = (p.T + 63) / 64;
    if (!((p.mask[((size_t)b * p.T + node) * w + (j >> 6)] >> (j & 63)) & 1)) return false;
  } else if (j > node) {
    return false;
  }
  return !p.window || (p.pos ? p.pos[b * p.T + j] : t) >= low;
}

// Slots [first, end) of sequence b that any of its nodes can see.
struct Span {
  int len, first, end;
};
// ALL: from the first slot on, seen or not.
template <bool ALL = false>
__device__ __forceinline__ Span span_of(const TreeParams &p, int b) {
  Span s;
  s.len = committed(p.kv, p.lens, b, p.T);
  s.end = s.len + p.T;
  s.first = 0;
  if (p.kv.ring) {
    s.end = min(s.end, p.kv.ring);
  } else if (!ALL && p.window) {
    int low = INT_MAX;
    if (p.pos)
      for (int i = 0; i < p.T; i++) low = min(low, lowest(p.pos[b * p.T + i], p.window));
    else
      low = lowest(s.len, p.window);
    s.first = min(max(low, 0), s.len) & ~15;
  }
  return s;
}

// ------------------------------------------------------------- the work list
// Items (sequence, KV head, row block) of `tiles` slot tiles each, one run of
// an item's tiles per CTA.  Lengths are known on the device only, so every
// warp finds its CTA's run itself: the fewest tiles per CTA for which all runs
// fit the grid, which holds at least one CTA per item; where no item has more
// than `whole` tiles, one CTA takes each, which spares the join.  Splitting items
// instead of a flat list of tiles costs at most one tile of balance and saves a
// CTA from working on two items in turn (5 us).
constexpr int kCounters = 16384;  // grid of a launch with split items, at most

struct Work {
  int b, in_b;          // sequence, item within it
  int t0, t1;           // tiles
  int first, count;     // CTAs of the item
  Span span;
};

__device__ __forceinline__ int tiles_of(const Span &s, int tile) {
  return (s.end - s.first + tile - 1) / tile;
}

// x / d for x >= 0, d > 0: by f32 where both are exact there, which takes a
// fifth of the integer division's time at the head of every CTA.
__device__ __forceinline__ int quick_div(int x, int d) {
  if (x >= (1 << 22) || d >= (1 << 22)) return x / d;
  int q = (int)__fdividef((float)x, (float)d);
  const int r = x - q * d;
  return r < 0 ? q - 1 : (r >= d ? q + 1 : q);
}

// seq: not a CTA's own run but a sequence's first (of the launch of `grid` CTAs).
template <bool ALL = false>
__device__ __forceinline__ bool find_work(const TreeParams &p, int tile, int per_b, int whole,
                                          int lane, Work &w, int grid, int cta, int seq = -1) {
  const int rows = p.kv.rows;
  const Span mine = span_of<ALL>(p, min(lane, rows - 1));
  const int n0 = lane < rows ? tiles_of(mine, tile) : 0;  // the first 32 sequences stay here
  int total = n0, longest = n0;
  for (int b = lane + 32; b < rows; b += 32) {
    const int n = tiles_of(span_of<ALL>(p, b), tile);
    total += n;
    longest = max(longest, n);
  }
  total = __reduce_add_sync(0xffffffffu, total);
  longest = __reduce_max_sync(0xffffffffu, longest);
  // from just below the even share upwards
  int per = max(longest <= whole ? longest : 1,
                (int)(__fdividef((float)total * (float)per_b, (float)grid) * 0.9999f));
  for (;; per += 1 + per / 32) {
    int c = quick_div(n0 + per - 1, per);
    for (int b = lane + 32; b < rows; b += 32)
      c += (tiles_of(span_of<ALL>(p, b), tile) + per - 1) / per;
    if ((long long)__reduce_add_sync(0xffffffffu, c) * per_b <= grid) break;
  }
  int base = 0;
  for (int b0 = 0; b0 < rows; b0 += 32) {
    const int b = b0 + lane;
    const Span s = b0 == 0 ? mine : span_of<ALL>(p, min(b, rows - 1));
    const int tiles = b < rows ? tiles_of(s, tile) : 0, cnt = quick_div(tiles + per - 1, per);
    int inc = cnt * per_b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, seq >= 0 ? b == seq : base + inc > cta);
    if (hit) {
      const int l = __ffs(hit) - 1;
      const int t = __shfl_sync(0xffffffffu, tiles, l);
      w.span.len = __shfl_sync(0xffffffffu, s.len, l);
      w.span.first = __shfl_sync(0xffffffffu, s.first, l);
      w.span.end = __shfl_sync(0xffffffffu, s.end, l);
      w.b = b0 + l;
      w.count = __shfl_sync(0xffffffffu, cnt, l);
      const int start = base + __shfl_sync(0xffffffffu, inc - cnt * per_b, l);
      const int rel = seq >= 0 ? 0 : cta - start;
      w.in_b = quick_div(rel, w.count);
      const int k = rel - w.in_b * w.count, each = quick_div(t, w.count), more = t - each * w.count;
      w.first = start + rel - k;
      w.t0 = k * each + min(k, more);
      w.t1 = w.t0 + each + (k < more);
      return true;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  return false;
}

template <bool ALL = false>
__device__ __forceinline__ bool find_work(const TreeParams &p, int tile, int per_b, int whole,
                                          int lane, Work &w) {
  return find_work<ALL>(p, tile, per_b, whole, lane, w, gridDim.x, blockIdx.x);
}

// Four dimensions of a row from its parts (their maxima and sums `stat`), the
// first parts' values asked for together with their statistics.
struct Joined {
  float4 a;
  float M, L;
};
__device__ __forceinline__ Joined join_row4(const float2 *stat, const float4 *part, size_t stat_ld,
                                            size_t part_ld, int count) {
  Joined j{make_float4(0, 0, 0, 0), -INFINITY, 0.0f};
  constexpr int kParts = 12;
  for (int i0 = 0; i0 < count; i0 += kParts) {
    float2 s[kParts];
    float4 v[kParts];
    const int n = min(kParts, count - i0);
#pragma unroll
    for (int i = 0; i < kParts; i++) {
      s[i] = i < n ? stat[(i0 + i) * stat_ld] : make_float2(-INFINITY, 0.0f);
      v[i] = i < n ? part[(i0 + i) * part_ld] : make_float4(0, 0, 0, 0);
    }
    float N = j.M;
#pragma unroll
    for (int i = 0; i < kParts; i++) N = fmaxf(N, s[i].x);
    const float ref = N == -INFINITY ? 0.0f : N, f0 = ex2(j.M - ref);
    j.a.x *= f0, j.a.y *= f0, j.a.z *= f0, j.a.w *= f0;
    j.L *= f0;
#pragma unroll
    for (int i = 0; i < kParts; i++) {
      const float f = ex2(s[i].x - ref);
      j.L += f * s[i].y;
      j.a.x += f * v[i].x, j.a.y += f * v[i].y, j.a.z += f * v[i].z, j.a.w += f * v[i].w;
    }
    j.M = N;
  }
  const float inv = j.L == 0.0f ? 0.0f : 1.0f / j.L;
  j.a.x *= inv, j.a.y *= inv, j.a.z *= inv, j.a.w *= inv;
  return j;
}

// What the attention kernels leave behind for an item that several CTAs work
// on, and the join by the last of them to arrive.  counters are 0 before and
// after every launch.
struct Parts {
  float *part;          // [grid][rows][hd]: sums of p vs v8
  float2 *stat;         // [grid][rows]: maximum * log2(e), sum of p
  int *counters;        // [first CTA of the item]
};

__device__ __forceinline__ void store_row4(const TreeParams &p, const Work &w, int kvh, int r,
                                           int d, float4 a, float M, float L) {
  const int hd = p.kv.head_dim, G = p.n_heads / p.kv.kv_heads, node = quick_div(r, G);
  const int h = kvh * G + r - node * G;
  const size_t qr = (size_t)w.b * p.T + node;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  a.x *= inv, a.y *= inv, a.z *= inv, a.w *= inv;
  *reinterpret_cast<float4 *>(p.out + qr * p.out_ld + (size_t)h * hd + d) = a;
  if (d == 0 && p.lse)
    p.lse[qr * p.lse_row + h * p.lse_head] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
}

// Every thread of the CTA, after its partial results are written.  sm: at
// least rows * (count + 2) floats of shared memory that nothing else uses.
// The barrier orders the CTA's stores before thread 0's fence, the fence them
// before its count; whoever counts last reads what all the others wrote.
__device__ __forceinline__ void join_parts(const TreeParams &p, const Parts &q, const Work &w,
                                           int kvh, int row0, int rows, int ld, float *sm) {
  __shared__ int s_last;
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31;
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    s_last = atomicAdd(q.counters + w.first, 1) == w.count - 1;
    if (s_last) q.counters[w.first] = 0;
    __threadfence();
  }
  __syncthreads();
  if (!s_last) return;
  const int n = w.count, hd4 = p.kv.head_dim / 4, total = rows * hd4;
  float *f = sm, *tot = sm + rows * n;
  const float2 *stat = q.stat + (size_t)w.first * ld;
  for (int r = tid >> 5; r < rows; r += nt >> 5) {  // a warp per row: the parts' factors
    float M = -INFINITY, L = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const float2 v = i0 + lane < n ? __ldcg(&stat[(size_t)(i0 + lane) * ld + r])
                                     : make_float2(-INFINITY, 0.0f);
      const float N = fmaxf(M, warp_max(v.x)), ref = N == -INFINITY ? 0.0f : N;
      L = L * ex2(M - ref) + v.y * ex2(v.x - ref);
      M = N;
      if (i0 + lane < n) f[r * n + i0 + lane] = v.x;
    }
    const float ref = M == -INFINITY ? 0.0f : M;
    for (int i = lane; i < n; i += 32) f[r * n + i] = ex2(f[r * n + i] - ref);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) tot[2 * r] = M, tot[2 * r + 1] = L;
  }
  __syncthreads();
  // U outputs of a thread at a time, P parts of each on their way together
  const float4 *part = reinterpret_cast<const float4 *>(q.part) + (size_t)w.first * ld * hd4;
  auto join = [&](auto us, auto ps) {
    constexpr int U = decltype(us)::value, P = decltype(ps)::value;
    for (int i0 = tid; i0 < total; i0 += nt * U) {
      float4 a[U];
#pragma unroll
      for (int u = 0; u < U; u++) a[u] = make_float4(0, 0, 0, 0);
      for (int k = 0; k < n; k += P) {
        float4 v[U][P];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
          for (int e = 0; e < P; e++)
            v[u][e] = i0 + u * nt < total && k + e < n
                          ? __ldcg(part + (size_t)(k + e) * ld * hd4 + i0 + u * nt)
                          : make_float4(0, 0, 0, 0);
#pragma unroll
        for (int u = 0; u < U; u++) {
          const float *fr = f + quick_div(min(i0 + u * nt, total - 1), hd4) * n + k;
#pragma unroll
          for (int e = 0; e < P; e++)
            if (k + e < n) {
              const float s = fr[e];
              a[u].x += s * v[u][e].x, a[u].y += s * v[u][e].y;
              a[u].z += s * v[u][e].z, a[u].w += s * v[u][e].w;
            }
        }
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int i = i0 + u * nt;
        if (i < total) {
          const int r = quick_div(i, hd4);
          store_row4(p, w, kvh, row0 + r, (i - r * hd4) * 4, a[u], tot[2 * r], tot[2 * r + 1]);
        }
      }
    }
  };
  if (total <= nt) join(std::integral_constant<int, 1>(), std::integral_constant<int, 12>());
  else join(std::integral_constant<int, 4>(), std::integral_constant<int, 4>());
}

// ------------------------------------------------------------------ host side
inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// CTAs of a launch over `items`: the SMs, or, where the items are more, some
// more than the items, so that the longer ones split.
constexpr int kMaxSms = 256;
inline int grid_of(const fgm_cuda_kv &kv, long long items, int tile, int num_sms) {
  const long long most = items * ((kv.cap + tile - 1) / tile);
  const long long want = items <= num_sms ? num_sms : items + 2 * num_sms;
  const long long g = want <= kCounters ? want : items;
  return (int)(most < g ? most : g);
}

// What grid_of gives at most, on any device.
inline long long max_grid(const fgm_cuda_kv &kv, long long items, int tile) {
  const long long most = items * ((kv.cap + tile - 1) / tile), want = items + 2 * kMaxSms;
  return most < want ? most : want;
}

// Raises a kernel's shared-memory limit, once per device (the call is not free).
template <class K>
cudaError_t allow_smem(K kernel, int bytes, std::atomic<uint64_t> &done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e != cudaSuccess || (done.load(std::memory_order_relaxed) & bit)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

}  // namespace kv
}  // namespace fgm

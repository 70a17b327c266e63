// Trees of drafted tokens and the moves of cache rows: ancestor masks, greedy
// verification, the commit of an accepted path, eviction to a budget.
#include "fgm_internal.h"
#include "kv_common.cuh"

namespace fgm {
namespace {

using namespace kv;

constexpr int kTreeMax = FGM_CUDA_TREE_MAX;

// One CTA per tree, thread i = node i: bits of the walk to the root.  A
// parent is below its child, so the walk ends after at most T steps.
__global__ void __launch_bounds__(kTreeMax) tree_mask_kernel(uint64_t *mask, int32_t *pos,
                                                             const int32_t *parent,
                                                             const int32_t *lens, int T) {
  __shared__ int up[kTreeMax];
  const int b = blockIdx.x, i = threadIdx.x;
  if (i < T) up[i] = parent[(size_t)b * T + i];
  __syncthreads();
  if (i >= T) return;
  uint64_t w[kTreeMax / 64] = {};
  int depth = 0;
  for (int n = i;;) {
#pragma unroll
    for (int k = 0; k < kTreeMax / 64; k++)
      if (k == n >> 6) w[k] |= 1ull << (n & 63);
    const int u = up[n];
    if (u < 0 || u >= n) break;
    n = u;
    depth++;
  }
  const int words = (T + 63) / 64;
  for (int k = 0; k < words; k++) mask[((size_t)b * T + i) * words + k] = w[k];
  if (pos) pos[(size_t)b * T + i] = lens[b] + depth;
}

// One warp per tree: each step looks at all nodes at once for the lowest
// right child of the last accepted one.
__global__ void __launch_bounds__(32) tree_verify_kernel(int32_t *path, int32_t *n_acc,
                                                         int32_t *next, const int32_t *parent,
                                                         const int32_t *token,
                                                         const int32_t *target, int T) {
  constexpr int per = kTreeMax / 32;
  const int lane = threadIdx.x;
  const size_t base = (size_t)blockIdx.x * T;
  int up[per], tok[per];
#pragma unroll
  for (int k = 0; k < per; k++) {
    const int i = k * 32 + lane;
    up[k] = i < T ? parent[base + i] : -1;
    tok[k] = i < T ? token[base + i] : 0;
    if (up[k] >= i) up[k] = -1;
  }
  int cur = 0, n = 1, want = target[base];
  if (lane == 0) path[base] = 0;
  for (;;) {
    int found = T;
#pragma unroll
    for (int k = 0; k < per; k++) {
      const unsigned hit = __ballot_sync(0xffffffffu, up[k] == cur && tok[k] == want);
      if (hit && found == T) found = k * 32 + __ffs(hit) - 1;
    }
    if (found >= T) break;
    cur = found;
    want = target[base + cur];
    if (lane == 0) path[base + n] = cur;
    n++;
  }
  for (int j = n + lane; j < T; j += 32) path[base + j] = -1;
  if (lane == 0) n_acc[blockIdx.x] = n, next[blockIdx.x] = want;
}

constexpr int kLayers = 32;  // layers of one launch
struct AcceptParams {
  fgm_cuda_kv kv[kLayers];
  int T;
  const int32_t *lens, *path, *n_acc;
  int32_t *lens_new;
};

// One CTA per (sequence, layer).  A thread owns byte columns of K and words
// of V and walks the path in order, so a row is read before anything can
// overwrite it (the destination of entry j is at or before its source, and
// the sources ascend).
__global__ void __launch_bounds__(256) kv_accept_kernel(const __grid_constant__ AcceptParams p) {
  const int b = blockIdx.x, tid = threadIdx.x;
  const fgm_cuda_kv &kv = p.kv[blockIdx.y];
  const int kvd = kv.kv_heads * kv.head_dim;
  const int len = committed(kv, p.lens, b, p.T);
  const int n = min(max(p.n_acc[b], 0), p.T);
  int8_t *kc = kv.kc + (size_t)b * kv.kc_stride, *vt = kv.vt + (size_t)b * kv.vt_stride;
  float *f[3] = {kv.ks + (size_t)b * kv.ks_stride, kv.vs + (size_t)b * kv.vs_stride,
                 kv.acc ? kv.acc + (size_t)b * kv.acc_stride : nullptr};
  int32_t *tp = kv.tpos ? kv.tpos + (size_t)b * kv.tpos_stride : nullptr;
  for (int j = 0; j < n; j++) {
    const int s = p.path[(size_t)b * p.T + j];
    if (s <= j || s >= p.T) continue;
    const int from = slot_of(kv, len + s), to = slot_of(kv, len + j);
    for (int c = tid; c < kvd / 4; c += 256)
      reinterpret_cast<uint32_t *>(kc + (size_t)to * kvd)[c] =
          reinterpret_cast<const uint32_t *>(kc + (size_t)from * kvd)[c];
    for (int c = tid; c < kvd; c += 256)
      vt[((size_t)(to >> 2) * kvd + c) * 4 + (to & 3)] =
          vt[((size_t)(from >> 2) * kvd + c) * 4 + (from & 3)];
    if (tid < 3 && f[tid]) f[tid][to] = f[tid][from];
    if (tid == 3 && tp) tp[to] = tp[from];
  }
  if (p.lens_new && blockIdx.y == 0 && tid == 0) p.lens_new[b] = len + n;
}

struct EvictParams {
  fgm_cuda_kv kv;
  const int32_t *lens;
  int budget, sink, recent;
  int32_t *map, *lens_out;
  float *acc_out;
  int32_t *tpos_out;
  size_t acc_stride, tpos_stride;  // of the outputs
};

constexpr int kPlanThreads = 1024;
constexpr int kEvictMax = 524288;

// Order of acc as unsigned: not-a-number 0, then ascending, -0 equal to 0.
__device__ __forceinline__ uint32_t rank_key(float v) {
  if (v != v) return 0;
  const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ int block_sum(int v, int *red) {
  v = __reduce_add_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int s = 0;
  for (int w = 0; w < kPlanThreads / 32; w++) s += red[w];
  return s;
}

// One CTA per sequence: the budget-th largest key by four passes over its
// bytes, then the kept slots as a bitmask in shared memory (with the number
// of kept slots before each word), from which every slot finds its source.
__global__ void __launch_bounds__(kPlanThreads) evict_plan_kernel(const EvictParams p) {
  extern __shared__ uint32_t bits[];  // [words] kept slots, then [words] kept before the word
  __shared__ unsigned hist[256];
  __shared__ int red[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left, s_newest;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = committed(p.kv, p.lens, b, 0), budget = p.budget;
  const float *acc = p.kv.acc + (size_t)b * p.kv.acc_stride;
  const int32_t *tp = p.kv.tpos ? p.kv.tpos + (size_t)b * p.kv.tpos_stride : nullptr;
  int32_t *map = p.map + (size_t)b * budget;
  const int words = (n + 31) / 32;
  uint32_t *before = bits + words;
  if (n > budget) {
    if (tid == 0) s_newest = INT_MIN;
    __syncthreads();
    int newest = INT_MIN;
    for (int x = tid; x < n; x += kPlanThreads) newest = max(newest, tp ? tp[x] : x);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) atomicMax(&s_newest, newest);
    __syncthreads();
    const long long old = (long long)s_newest - p.recent;
    auto key = [&](int x) -> uint32_t {
      const int t = tp ? tp[x] : x;
      return t < p.sink || t > old ? 0xFFFFFFFFu : rank_key(acc[x]);
    };
    uint32_t prefix = 0;
    int left = budget;  // keys still to take among those that share the prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist[tid] = 0;
      __syncthreads();
      for (int x = tid; x < n; x += kPlanThreads) {
        const uint32_t k = key(x);
        if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(k >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        int v = 255, sum = 0;
        while (sum + (int)hist[v] < left) sum += (int)hist[v--];
        s_prefix = prefix | ((uint32_t)v << shift);
        s_left = left - sum;
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
      __syncthreads();
    }
    // keys above the threshold, and of the equal ones the first `left`
    int eq_seen = 0;
    for (int x0 = 0; x0 < n; x0 += kPlanThreads) {
      const int x = x0 + tid;
      const uint32_t k = x < n ? key(x) : 0;
      const unsigned eq = __ballot_sync(0xffffffffu, x < n && k == prefix);
      __syncthreads();
      if (lane == 0) red[warp] = __popc(eq);
      __syncthreads();
      int r = eq_seen;
      for (int w = 0; w < 32; w++) {
        if (w < warp) r += red[w];
        eq_seen += red[w];
      }
      r += __popc(eq & ((1u << lane) - 1));
      const bool keep = x < n && (k > prefix || (k == prefix && r < left));
      const unsigned word = __ballot_sync(0xffffffffu, keep);
      if (lane == 0 && (x >> 5) < words) bits[x >> 5] = word;
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t s = 0;
      for (int w = 0; w < words; w++) {
        before[w] = s;
        s += __popc(bits[w]);
      }
    }
    __syncthreads();
    auto kept_before = [&](int x) -> int {
      return x >= words * 32 ? budget
                             : (int)before[x >> 5] + __popc(bits[x >> 5] & ((1u << (x & 31)) - 1));
    };
    const int low = kept_before(budget);  // kept slots below the budget
    for (int x = tid; x < budget; x += kPlanThreads) {
      if ((bits[x >> 5] >> (x & 31)) & 1) {
        map[x] = x;
        continue;
      }
      const int want = low + (x - kept_before(x));  // kept slots before the one that moves here
      int lo = budget >> 5, hi = words;             // last word with before <= want
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int)before[mid] <= want) lo = mid;
        else hi = mid;
      }
      uint32_t w = bits[lo];
      for (int k = want - (int)before[lo]; k > 0; k--) w &= w - 1;
      map[x] = lo * 32 + __ffs(w) - 1;
    }
  } else {
    for (int x = tid; x < budget; x += kPlanThreads) map[x] = x < n ? x : -1;
  }
  __syncthreads();
  // the slots' own words; in place, the sources lie past the budget
  float *ao = p.acc_out + (size_t)b * p.acc_stride;
  int32_t *to = p.tpos_out ? p.tpos_out + (size_t)b * p.tpos_stride : nullptr;
  for (int x = tid; x < budget; x += kPlanThreads) {
    const int s = map[x];
    if (s < 0) continue;
    if (s != x || ao != acc) ao[x] = acc[s];
    if (to && (s != x || to != tp)) to[x] = tp ? tp[s] : s;
  }
  if (tid == 0) p.lens_out[b] = min(n, budget);
}

// A warp per 32 slots of a sequence: the rows that move, one after the other.
__global__ void __launch_bounds__(256) evict_move_kernel(const EvictParams p) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int x = (blockIdx.x * 8 + (threadIdx.x >> 5)) * 32 + lane;
  const int kvd = p.kv.kv_heads * p.kv.head_dim;
  const int s = x < p.budget ? p.map[(size_t)b * p.budget + x] : -1;
  unsigned todo = __ballot_sync(0xffffffffu, s >= 0 && s != x);
  int8_t *kc = p.kv.kc + (size_t)b * p.kv.kc_stride, *vt = p.kv.vt + (size_t)b * p.kv.vt_stride;
  float *ks = p.kv.ks + (size_t)b * p.kv.ks_stride, *vs = p.kv.vs + (size_t)b * p.kv.vs_stride;
  for (; todo; todo &= todo - 1) {
    const int l = __ffs(todo) - 1, from = __shfl_sync(0xffffffffu, s, l), to = x - lane + l;
    for (int c = lane; c < kvd / 16; c += 32)
      reinterpret_cast<uint4 *>(kc + (size_t)to * kvd)[c] =
          reinterpret_cast<const uint4 *>(kc + (size_t)from * kvd)[c];
    for (int c = lane; c < kvd; c += 32)
      vt[((size_t)(to >> 2) * kvd + c) * 4 + (to & 3)] =
          vt[((size_t)(from >> 2) * kvd + c) * 4 + (from & 3)];
    if (lane == 0) ks[to] = ks[from], vs[to] = vs[from];
  }
}

}  // namespace

cudaError_t launch_tree_mask(uint64_t *mask, int32_t *pos, const int32_t *parent,
                             const int32_t *lens, int rows, int T, cudaStream_t st) {
  tree_mask_kernel<<<rows, (T + 31) / 32 * 32, 0, st>>>(mask, pos, parent, lens, T);
  return cudaGetLastError();
}

cudaError_t launch_tree_verify(int32_t *path, int32_t *n_acc, int32_t *next, const int32_t *parent,
                               const int32_t *token, const int32_t *target, int rows, int T,
                               cudaStream_t st) {
  tree_verify_kernel<<<rows, 32, 0, st>>>(path, n_acc, next, parent, token, target, T);
  return cudaGetLastError();
}

cudaError_t launch_kv_accept(const fgm_cuda_kv *kv, int layers, int T, const int32_t *lens,
                             const int32_t *path, const int32_t *n_acc, int32_t *lens_new,
                             int *launches, cudaStream_t st) {
  AcceptParams p;
  p.T = T;
  p.lens = lens;
  p.path = path;
  p.n_acc = n_acc;
  *launches = 0;
  for (int l0 = 0; l0 < layers; l0 += kLayers) {
    const int n = layers - l0 < kLayers ? layers - l0 : kLayers;
    for (int l = 0; l < n; l++) p.kv[l] = kv[l0 + l];
    p.lens_new = l0 == 0 ? lens_new : nullptr;
    kv_accept_kernel<<<dim3((unsigned)kv->rows, (unsigned)n), 256, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    ++*launches;
  }
  return cudaSuccess;
}

cudaError_t launch_kv_evict(const fgm_cuda_kv &kv, const int32_t *lens, int budget, int sink,
                            int recent, int32_t *map, int32_t *lens_out, float *acc_out,
                            int32_t *tpos_out, size_t out_stride, cudaStream_t st) {
  EvictParams p{kv, lens, budget, sink, recent, map, lens_out, acc_out, tpos_out, out_stride,
                out_stride};
  if (!acc_out) p.acc_out = kv.acc, p.acc_stride = kv.acc_stride;
  if (!tpos_out) p.tpos_out = kv.tpos, p.tpos_stride = kv.tpos_stride;
  const size_t smem = (size_t)((kv.cap + 31) / 32) * 8;
  cudaError_t e = cudaFuncSetAttribute(evict_plan_kernel,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kEvictMax / 32 * 8);
  if (e != cudaSuccess) return e;
  evict_plan_kernel<<<kv.rows, kPlanThreads, smem, st>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  evict_move_kernel<<<dim3((unsigned)((budget + 255) / 256), (unsigned)kv.rows), 256, 0, st>>>(p);
  return cudaGetLastError();
}

}  // namespace fgm

// Trees of drafted tokens and the moves of cache rows: ancestor masks, greedy
// verification, the commit of an accepted path, eviction to a budget.
#include "fgm_internal.h"
#include "kv_attn.cuh"

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

// One CTA per (sequence, layer).  Warp 0 moves K rows, 16 bytes a lane, the
// others V, a dimension's word a lane, eight path entries at a time: their
// loads all go out before the first store.  That keeps the order right too:
// the destination of entry j lies at or before its source and the sources
// ascend, so no store of a batch lands on a row that a later entry still reads.
constexpr int kAcceptBatch = 8;
__global__ void __launch_bounds__(256) kv_accept_kernel(const __grid_constant__ AcceptParams p) {
  __shared__ int s_from[kTreeMax], s_to[kTreeMax], s_n;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const fgm_cuda_kv &kv = p.kv[blockIdx.y];
  const int kvd = kv.kv_heads * kv.head_dim;
  const int len = committed(kv, p.lens, b, p.T);
  const int n = min(max(p.n_acc[b], 0), p.T);
  if (warp == 0) {  // the entries that move, in order
    int count = 0;
    for (int j0 = 0; j0 < n; j0 += 32) {
      const int j = j0 + lane, s = j < n ? p.path[(size_t)b * p.T + j] : -1;
      const bool moves = s > j && s < p.T;
      const unsigned m = __ballot_sync(0xffffffffu, moves);
      const int at = count + __popc(m & ((1u << lane) - 1));
      if (moves) s_from[at] = slot_of(kv, len + s), s_to[at] = slot_of(kv, len + j);
      count += __popc(m);
    }
    if (lane == 0) s_n = count;
  }
  __syncthreads();
  if (p.lens_new && blockIdx.y == 0 && tid == 0) p.lens_new[b] = len + n;
  const int moves = s_n;
  int8_t *kc = kv.kc + (size_t)b * kv.kc_stride, *vt = kv.vt + (size_t)b * kv.vt_stride;
  for (int m0 = 0; m0 < moves; m0 += kAcceptBatch) {
    const int m = min(kAcceptBatch, moves - m0);
    if (warp == 0) {
      for (int c = lane * 16; c < kvd; c += 512) {
        uint4 v[kAcceptBatch];
#pragma unroll
        for (int i = 0; i < kAcceptBatch; i++)
          if (i < m) v[i] = *reinterpret_cast<const uint4 *>(kc + (size_t)s_from[m0 + i] * kvd + c);
#pragma unroll
        for (int i = 0; i < kAcceptBatch; i++)
          if (i < m) *reinterpret_cast<uint4 *>(kc + (size_t)s_to[m0 + i] * kvd + c) = v[i];
      }
      if (lane < 4) {  // the rows' own words: a lane each, in order
        float *f = lane == 0   ? kv.ks + (size_t)b * kv.ks_stride
                   : lane == 1 ? kv.vs + (size_t)b * kv.vs_stride
                   : lane == 2 ? (kv.acc ? kv.acc + (size_t)b * kv.acc_stride : nullptr)
                               : reinterpret_cast<float *>(
                                     kv.tpos ? kv.tpos + (size_t)b * kv.tpos_stride : nullptr);
        if (f) {
          uint32_t v[kAcceptBatch], *u = reinterpret_cast<uint32_t *>(f);
#pragma unroll
          for (int i = 0; i < kAcceptBatch; i++)
            if (i < m) v[i] = u[s_from[m0 + i]];
#pragma unroll
          for (int i = 0; i < kAcceptBatch; i++)
            if (i < m) u[s_to[m0 + i]] = v[i];
        }
      }
    } else {
      for (int c = tid - 32; c < kvd; c += 224) {
        uint32_t v[kAcceptBatch];
#pragma unroll
        for (int i = 0; i < kAcceptBatch; i++)
          if (i < m) {
            const int s = s_from[m0 + i];
            v[i] = reinterpret_cast<const uint32_t *>(vt)[(size_t)(s >> 2) * kvd + c] >> ((s & 3) * 8);
          }
#pragma unroll
        for (int i = 0; i < kAcceptBatch; i++)
          if (i < m) {
            const int d = s_to[m0 + i];
            vt[((size_t)(d >> 2) * kvd + c) * 4 + (d & 3)] = (int8_t)v[i];
          }
      }
    }
  }
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

// One CTA per sequence.  The budget-th largest key comes from four passes of
// 256 counters over its bytes; then every warp walks its own run of slots,
// 32 at a time, and leaves the kept ones as a bitmask in shared memory with
// the number kept before each word, from which every slot below the budget
// finds its source.  Bound by latency: a handful of passes over keys that lie
// in shared memory (CACHED: up to kCachedKeys slots; longer caches read acc
// and tpos again in each pass).
constexpr int kCachedKeys = 40960;

template <bool CACHED>
__global__ void __launch_bounds__(kPlanThreads) evict_plan_kernel(const EvictParams p) {
  extern __shared__ uint32_t smem[];  // bits [words], kept before each word [words], keys
  __shared__ unsigned hist[256];
  __shared__ int s_warp[kPlanThreads / 32], s_base[kPlanThreads / 32 + 1];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left, s_newest;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = committed(p.kv, p.lens, b, 0), budget = p.budget;
  const float *acc = p.kv.acc + (size_t)b * p.kv.acc_stride;
  const int32_t *tp = p.kv.tpos ? p.kv.tpos + (size_t)b * p.kv.tpos_stride : nullptr;
  int32_t *map = p.map + (size_t)b * budget;
  float *ao = p.acc_out + (size_t)b * p.acc_stride;
  int32_t *to = p.tpos_out ? p.tpos_out + (size_t)b * p.tpos_stride : nullptr;
  if (tid == 0) p.lens_out[b] = min(n, budget);
  // a slot's own words to where they go; in place the sources lie past the budget
  auto place = [&](int x, int s) {
    if (s != x || ao != acc) ao[x] = acc[s];
    if (to && (s != x || to != tp)) to[x] = tp ? tp[s] : s;
  };
  if (n <= budget) {
    for (int x = tid; x < budget; x += kPlanThreads) {
      map[x] = x < n ? x : -1;
      if (x < n) place(x, x);
    }
    return;
  }
  const int words = (n + 31) / 32, per_warp = (words + kPlanThreads / 32 - 1) / (kPlanThreads / 32);
  uint32_t *bits = smem, *before = smem + words, *keys = before + words;

  // the newest position (the slot's index where no positions are kept)
  if (tid == 0) s_newest = tp ? INT_MIN : n - 1;
  if (tid < 256) hist[tid] = 0;
  __syncthreads();
  if (tp) {
    int newest = INT_MIN;
#pragma unroll 8
    for (int x = tid; x < n; x += kPlanThreads) newest = max(newest, tp[x]);
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) atomicMax(&s_newest, newest);
    __syncthreads();
  }
  const long long old = (long long)s_newest - p.recent;
  auto make_key = [&](int x) -> uint32_t {
    const int t = tp ? tp[x] : x;
    return t < p.sink || t > old ? 0xFFFFFFFFu : rank_key(acc[x]);
  };
  if (CACHED) {
#pragma unroll 4
    for (int x = tid; x < n; x += kPlanThreads) {
      const uint32_t k = make_key(x);
      keys[x] = k;
      atomicAdd(&hist[k >> 24], 1u);
    }
  }
  auto key = [&](int x) -> uint32_t { return CACHED ? keys[x] : make_key(x); };

  uint32_t prefix = 0;
  int left = budget;  // keys still to take among those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (!CACHED || shift < 24) {
#pragma unroll 4
      for (int x = tid; x < n; x += kPlanThreads) {
        const uint32_t k = key(x);
        if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
          atomicAdd(&hist[(k >> shift) & 255], 1u);
      }
    }
    __syncthreads();
    if (warp == 0) {  // the digit, from the largest down: 8 counters a lane
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        c[i] = (int)hist[255 - 8 * lane - i];
        sum += c[i];
      }
      int inc = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const int l = __ffs(__ballot_sync(0xffffffffu, inc >= left)) - 1;
      if (lane == l) {
        int taken = inc - sum;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          if (taken + c[i] >= left) {
            s_prefix = prefix | ((uint32_t)(255 - 8 * lane - i) << shift);
            s_left = left - taken;
            break;
          }
          taken += c[i];
        }
      }
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
  }

  // keys above the threshold stay, and of the equal ones the first `left`
  const int w0 = min(words, warp * per_warp), w1 = min(words, w0 + per_warp);
  int count = 0;
#pragma unroll 4
  for (int w = w0; w < w1; w++) {
    const int x = w * 32 + lane;
    count += __popc(__ballot_sync(0xffffffffu, x < n && key(x) == prefix));
  }
  if (lane == 0) s_warp[warp] = count;
  __syncthreads();
  int rank = 0;
  for (int w = lane; w < warp; w += 32) rank += s_warp[w];
  rank = __reduce_add_sync(0xffffffffu, rank);
  count = 0;
#pragma unroll 4
  for (int w = w0; w < w1; w++) {
    const int x = w * 32 + lane;
    const uint32_t k = x < n ? key(x) : 0;
    const unsigned eq = __ballot_sync(0xffffffffu, x < n && k == prefix);
    const bool keep =
        x < n && (k > prefix || (k == prefix && rank + __popc(eq & ((1u << lane) - 1)) < left));
    const unsigned kept = __ballot_sync(0xffffffffu, keep);
    rank += __popc(eq);
    if (lane == 0) {
      bits[w] = kept;
      before[w] = count;
    }
    count += __popc(kept);
  }
  __syncthreads();
  if (lane == 0) s_warp[warp] = count;
  __syncthreads();
  if (warp == 0) {
    const int c = s_warp[lane];
    int inc = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    s_base[lane + 1] = inc;
    if (lane == 0) s_base[0] = 0;
  }
  __syncthreads();
  {
    const int base = s_base[warp];
    for (int w = w0 + lane; w < w1; w += 32) before[w] += base;
  }
  __syncthreads();
  auto kept_before = [&](int x) -> int {
    return (int)before[x >> 5] + __popc(bits[x >> 5] & ((1u << (x & 31)) - 1));
  };
  const int low = kept_before(budget);  // kept slots below the budget (budget < n)
#pragma unroll 2
  for (int x = tid; x < budget; x += kPlanThreads) {
    int s = x;
    if (!((bits[x >> 5] >> (x & 31)) & 1)) {
      const int want = low + (x - kept_before(x));  // kept slots before the one that moves here
      int lo = budget >> 5, hi = words;             // last word with before <= want
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int)before[mid] <= want) lo = mid;
        else hi = mid;
      }
      uint32_t w = bits[lo];
      for (int k = want - (int)before[lo]; k > 0; k--) w &= w - 1;
      s = lo * 32 + __ffs(w) - 1;
    }
    map[x] = s;
    place(x, s);
  }
}

// A warp per kMoveSlots slots of a sequence: the rows that move, their loads
// all on the way before the first store.  Rows move from past the budget to
// below it, so no order matters.
constexpr int kMoveSlots = 8, kMoveWarps = 8;
__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const EvictParams p,
                                                                     int groups) {
  const int item = blockIdx.x * kMoveWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int b = item / groups, x0 = (item - b * groups) * kMoveSlots;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (b >= p.kv.rows) return;
  const int x = x0 + lane, kvd = p.kv.kv_heads * p.kv.head_dim;
  const int s = lane < kMoveSlots && x < p.budget ? p.map[(size_t)b * p.budget + x] : -1;
  unsigned todo = __ballot_sync(0xffffffffu, s >= 0 && s != x);
  int8_t *kc = p.kv.kc + (size_t)b * p.kv.kc_stride, *vt = p.kv.vt + (size_t)b * p.kv.vt_stride;
  float *ks = p.kv.ks + (size_t)b * p.kv.ks_stride, *vs = p.kv.vs + (size_t)b * p.kv.vs_stride;
  for (; todo; todo &= todo - 1) {
    const int l = __ffs(todo) - 1, from = __shfl_sync(0xffffffffu, s, l), to = x0 + l;
    float scale = 0.0f;
    if (lane == 0) scale = ks[from];
    if (lane == 1) scale = vs[from];
    for (int c0 = 0; c0 < kvd; c0 += 512) {
      const int c = c0 + lane * 16;
      uint4 k = make_uint4(0, 0, 0, 0);
      if (c < kvd) k = *reinterpret_cast<const uint4 *>(kc + (size_t)from * kvd + c);
      // of V the words of 512 dimensions, of which one byte each moves
      uint32_t v[16];
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (c0 + i * 32 + lane < kvd)
          v[i] = reinterpret_cast<const uint32_t *>(vt)[(size_t)(from >> 2) * kvd + c0 + i * 32 + lane];
      if (c < kvd) *reinterpret_cast<uint4 *>(kc + (size_t)to * kvd + c) = k;
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (c0 + i * 32 + lane < kvd)
          vt[((size_t)(to >> 2) * kvd + c0 + i * 32 + lane) * 4 + (to & 3)] =
              (int8_t)(v[i] >> ((from & 3) * 8));
    }
    if (lane == 0) ks[to] = scale;
    if (lane == 1) vs[to] = scale;
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
  // the bitmask, its counts and, where they fit, the keys of a whole cache
  const bool cached = kv.cap <= kCachedKeys;
  const size_t words = (size_t)(kv.cap + 31) / 32, smem = words * 8 + (cached ? words * 128 : 0);
  auto plan = cached ? evict_plan_kernel<true> : evict_plan_kernel<false>;
  static std::atomic<uint64_t> done[2];
  cudaError_t e = allow_smem(plan, cached ? kCachedKeys / 32 * 136 : kEvictMax / 32 * 8, done[cached]);
  if (e != cudaSuccess) return e;
  plan<<<kv.rows, kPlanThreads, smem, st>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  const int groups = (budget + kMoveSlots - 1) / kMoveSlots;
  const long long items = (long long)kv.rows * groups;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)((items + kMoveWarps - 1) / kMoveWarps));
  cfg.blockDim = dim3(kMoveWarps * 32);
  return cudaLaunchKernelEx(&cfg, evict_move_kernel, p, groups);
}

}  // namespace fgm

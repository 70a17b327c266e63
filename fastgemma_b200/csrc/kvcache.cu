// Trees of drafted tokens and the moves of cache rows: ancestor masks, greedy
// verification, the commit of an accepted path, eviction to a budget.
#include <cooperative_groups.h>

#include "fgm_internal.h"
#include "kv_attn.cuh"

namespace cg = cooperative_groups;

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
// right child of the last accepted one, so the path's length, not the tree's
// size, is what it takes.
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

// One CTA per (sequence, layer); bound by the latency of lens, path, rows (4.2
// us with the verification for one sequence and 4 layers, 7.1 for 8 sequences of
// 61 nodes and 30 layers, in a graph; as two ordinary calls the host needs 14).
// Warp 0 moves K rows, 16 bytes a lane, the others V, a dimension's word a lane,
// eight path entries at a time: their loads all go out before the first store.
// That keeps the order right too: the destination of entry j lies at or before
// its source and the sources ascend, so no store of a batch lands on a row that
// a later entry still reads.
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
constexpr int kMaxPlanSmem = 200 * 1024;

// Order of acc as unsigned: not-a-number 0, then ascending, -0 equal to 0.
__device__ __forceinline__ uint32_t rank_key(float v) {
  if (v != v) return 0;
  const uint32_t u = __float_as_uint(v == 0.0f ? 0.0f : v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// One CTA per sequence over caches of up to kOneCta slots, else a cluster of
// kCluster, a run of slots each.  The budget-th largest
// key comes from passes of 256 counters over its bytes, summed over the cluster
// through distributed shared memory, until the keys that share the bytes so far
// all stay (`exact`) or the four bytes are known; then every warp walks its
// share of the run, 32 slots at a time, and leaves the kept ones as a bitmask
// with the number kept before each word.  Each CTA lists its kept slots past
// the budget (where the keys were); the evicted slots below it find their
// sources there, by rank over the lists.  Bound by latency: a barrier and a pass
// or two over the slots for each of six to nine steps, which is why the keys stay
// in shared memory (CACHED; longer runs read acc and tpos again in every pass).
// 8 sequences of 16K slots: 15.8 us (with one CTA each about 20 more), of which
// 2.3 until the keys are there, 1.5 for each barrier with its counters, 3.2 for
// the map; 600 slots in one CTA: 6.  With the moves, one CTA against clusters of
// two, four and eight: 10.3, 14.2, 12.7 and 12.9 us at 4096 slots; 14.6 against
// 16.9, 14.6 and 13.9 at 8000.
constexpr int kOneCta = 6144, kCluster = 8, kCachedKeys = 40960;

template <bool CACHED, bool CLUSTER>
__global__ void __launch_bounds__(kPlanThreads) evict_plan_kernel(const EvictParams p) {
  extern __shared__ uint32_t smem[];  // bits [words], kept before each word [words], keys / list
  __shared__ unsigned hist[4][256], total[256];
  __shared__ int s_warp[kPlanThreads / 32], s_newest, s_eq, s_kept, s_kept_low;
  __shared__ uint32_t s_prefix;
  __shared__ int s_left, s_exact;
  cg::cluster_group cluster = cg::this_cluster();
  constexpr int C = CLUSTER ? kCluster : 1;
  const int rank = CLUSTER ? (int)cluster.block_rank() : 0;
  auto sync = [&] {
    if (CLUSTER) cluster.sync();
    else __syncthreads();
  };
  const int b = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = committed(p.kv, p.lens, b, 0), budget = p.budget;
  const float *acc = p.kv.acc + (size_t)b * p.kv.acc_stride;
  const int32_t *tp = p.kv.tpos ? p.kv.tpos + (size_t)b * p.kv.tpos_stride : nullptr;
  int32_t *map = p.map + (size_t)b * budget;
  float *ao = p.acc_out + (size_t)b * p.acc_stride;
  int32_t *to = p.tpos_out ? p.tpos_out + (size_t)b * p.tpos_stride : nullptr;
  // a slot's own words to where they go; in place the sources lie past the budget
  auto place = [&](int x, int s) {
    if (s != x || ao != acc) ao[x] = acc[s];
    if (to && (s != x || to != tp)) to[x] = tp ? tp[s] : s;
  };
  if (n <= budget) {
    for (int x = rank * kPlanThreads + tid; x < budget; x += C * kPlanThreads) {
      map[x] = x < n ? x : -1;
      if (x < n) place(x, x);
    }
    if (rank == 0 && tid == 0) p.lens_out[b] = n;
    return;
  }
  const int words = ((n + C - 1) / C + 31) / 32, run = words * 32;  // of one CTA
  const int first = min(n, rank * run), last = min(n, first + run);
  const int per_warp = (words + kPlanThreads / 32 - 1) / (kPlanThreads / 32);
  uint32_t *bits = smem, *before = smem + words, *keys = before + words;
  // kept slots past the budget, from the run's first; a run has at most 65536
  uint16_t *list = reinterpret_cast<uint16_t *>(keys);
  // a word of every CTA of the cluster, all asked for at once
  auto all = [&](int *w, int (&v)[C]) {
#pragma unroll
    for (int r = 0; r < C; r++) v[r] = CLUSTER ? *cluster.map_shared_rank(w, r) : *w;
  };

  // the newest position (the slot's index where no positions are kept)
  if (tid == 0) {
    s_newest = INT_MIN;
    s_kept_low = 0;
  }
  for (int i = tid; i < 4 * 256; i += kPlanThreads) (&hist[0][0])[i] = 0;
  __syncthreads();
  int newest = n - 1;
  if (tp) {
    newest = INT_MIN;
#pragma unroll 4
    for (int x = first + tid; x < last; x += kPlanThreads) {
      if (CACHED) keys[x - first] = rank_key(acc[x]);
      newest = max(newest, tp[x]);
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) atomicMax(&s_newest, newest);
    sync();
    int v[C];
    all(&s_newest, v);
#pragma unroll
    for (int r = 0; r < C; r++) newest = max(newest, v[r]);
  }
  const long long old = (long long)newest - p.recent;
  auto make_key = [&](int x) -> uint32_t {
    const int t = tp ? tp[x] : x;
    if (t < p.sink || t > old) return 0xFFFFFFFFu;
    return CACHED && tp ? keys[x - first] : rank_key(acc[x]);
  };
  auto key = [&](int x) -> uint32_t { return CACHED ? keys[x - first] : make_key(x); };

  uint32_t prefix = 0;
  int left = budget;   // keys still to take among those that share the prefix
  bool exact = false;  // all of them are
  for (int pass = 0; pass < 4 && !exact; pass++) {
    const int shift = 24 - 8 * pass;
#pragma unroll 4
    for (int x = first + tid; x < last; x += kPlanThreads) {
      const uint32_t k = pass == 0 ? make_key(x) : key(x);
      if (CACHED && pass == 0) keys[x - first] = k;
      if (pass == 0 || (k >> (shift + 8)) == (prefix >> (shift + 8)))
        atomicAdd(&hist[pass][(k >> shift) & 255], 1u);
    }
    sync();
    if (tid < 256) {
      int v[C];
      all(reinterpret_cast<int *>(&hist[pass][tid]), v);
      unsigned sum = 0;
#pragma unroll
      for (int r = 0; r < C; r++) sum += (unsigned)v[r];
      total[tid] = sum;
    }
    __syncthreads();
    if (warp == 0) {  // the digit, from the largest down: 8 counters a lane
      int c[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        c[i] = (int)total[255 - 8 * lane - i];
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
            s_exact = taken + c[i] == left;
            break;
          }
          taken += c[i];
        }
      }
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    exact = s_exact;
  }

  // keys above the threshold stay, and of the equal ones the first `left`
  const int w0 = min(words, warp * per_warp), w1 = min(words, w0 + per_warp);
  // of the warps' numbers: their sum and, in s_warp, what lies before each warp
  auto scan_warps = [&](int count) {
    if (lane == 0) s_warp[warp] = count;
    __syncthreads();
    int sum = 0;
    if (warp == 0) {
      const int c = s_warp[lane];
      int inc = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      s_warp[lane] = inc - c;
      sum = __shfl_sync(0xffffffffu, inc, 31);
    }
    return sum;  // of thread 0
  };
  int v[C], lows[C];
  int seen = 0;  // equal keys before this warp's
  if (!exact) {
    int count = 0;
    for (int w = w0; w < w1; w++) {
      const int x = first + w * 32 + lane;
      count += __popc(__ballot_sync(0xffffffffu, x < last && key(x) == prefix));
    }
    const int sum = scan_warps(count);
    if (tid == 0) s_eq = sum;
    sync();
    seen = s_warp[warp];
    all(&s_eq, v);
#pragma unroll
    for (int r = 0; r < C; r++)
      if (r < rank) seen += v[r];
    __syncthreads();
  }
  int count = 0, count_low = 0;
  for (int w = w0; w < w1; w++) {
    const int x = first + w * 32 + lane;
    const uint32_t k = x < last ? key(x) : 0;
    const unsigned eq = __ballot_sync(0xffffffffu, x < last && k == prefix);
    const bool tie = k == prefix && seen + __popc(eq & ((1u << lane) - 1)) < left;
    const bool keep = x < last && (exact ? k >= prefix : k > prefix || tie);
    const unsigned kept = __ballot_sync(0xffffffffu, keep);
    count_low += __popc(__ballot_sync(0xffffffffu, keep && x < budget));
    seen += __popc(eq);
    if (lane == 0) {
      bits[w] = kept;
      before[w] = count;
    }
    count += __popc(kept);
  }
  if (lane == 0 && count_low) atomicAdd(&s_kept_low, count_low);
  const int sum = scan_warps(count);
  if (tid == 0) s_kept = sum;
  __syncthreads();
  // kept slots past the budget into the CTA's list, which takes the keys' place
  const int mine = s_warp[warp], low = s_kept_low;
  for (int w = w0; w < w1; w++) {
    const uint32_t word = bits[w];
    const int at = mine + (int)before[w] + __popc(word & ((1u << lane) - 1));
    __syncwarp();
    if (lane == 0) before[w] = mine + (int)before[w];
    if (first + w * 32 + lane >= budget && ((word >> lane) & 1))
      list[at - low] = (uint16_t)(w * 32 + lane);
  }
  sync();
  // kept slots of the runs before this one; entries of every list
  int base = 0;
  all(&s_kept, v);
  all(&s_kept_low, lows);
#pragma unroll
  for (int r = 0; r < C; r++)
    if (r < rank) base += v[r];
  for (int x = first + tid; x < min(last, budget); x += kPlanThreads) {
    const int w = (x - first) >> 5;
    const uint32_t word = bits[w], bit = 1u << (x & 31);
    int s = x;
    if (!(word & bit)) {  // as many evicted slots lie before it as kept ones before its source
      int i = x - (base + (int)before[w] + __popc(word & (bit - 1))), from = 0;
#pragma unroll
      for (int r = 0; r < C - 1; r++)
        if (from == r && i >= v[r] - lows[r]) {
          i -= v[r] - lows[r];
          from++;
        }
      s = from * run + (CLUSTER ? *cluster.map_shared_rank(list + i, from) : list[i]);
    }
    map[x] = s;
    place(x, s);
  }
  sync();  // no CTA leaves while another may read its part of the list
  if (rank == 0 && tid == 0) p.lens_out[b] = budget;
}

// A warp per `per` slots of a sequence: the rows that move, their loads
// all on the way before the first store.  Rows move from past the budget to
// below it, so no order matters.  Bound by memory latency and by sectors that
// are read and written for one byte in four of V: 14336 rows of 512 dimensions
// in 16 us.  Rows listed per CTA of 64 slots before they move took 18.7, whole
// words of V, merged and stored, 19.7, the rows past the budget asked for in L2
// during the plan 16.6.
constexpr int kMoveWarps = 4;
__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const EvictParams p,
                                                                     int groups, int per) {
  const int item = blockIdx.x * kMoveWarps + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int b = item / groups, x0 = (item - b * groups) * per;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (b >= p.kv.rows) return;
  const int x = x0 + lane, kvd = p.kv.kv_heads * p.kv.head_dim;
  const int s = lane < per && x < p.budget ? p.map[(size_t)b * p.budget + x] : -1;
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
  const int c = kv.cap <= kOneCta ? 1 : kCluster;
  const int words = ((kv.cap + c - 1) / c + 31) / 32;
  // the keys' room also takes the list of kept slots past the budget, which
  // has no more entries than there are evicted ones
  const bool cached = words * 32 <= kCachedKeys;
  auto plan = c == 1 ? evict_plan_kernel<true, false>
              : cached ? evict_plan_kernel<true, true> : evict_plan_kernel<false, true>;
  static std::atomic<uint64_t> done[3];
  cudaError_t e = allow_smem(plan, kMaxPlanSmem, done[c == 1 ? 0 : cached ? 1 : 2]);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = c > 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)(kv.rows * c));
  cfg.blockDim = dim3(kPlanThreads);
  cfg.dynamicSmemBytes = (size_t)words * 8 + (size_t)(cached ? words : (words + 1) / 2) * 128;
  if ((e = cudaLaunchKernelEx(&cfg, plan, p)) != cudaSuccess) return e;
  // Slots of a warp that moves rows: one while about all warps fit the SMs at
  // once, more to spare launches of CTAs that find nothing.  One, two, four: 6.4,
  // 7.0, 7.5 us at 512 slots in all, 7.1, 7.5, 8.2 at 4096, 16.0, 15.7, 16.2 at
  // 14400, 18.6, 17.5, 17.5 at 28800, 35.5, 30.9, 29.9 at 114688.
  const long long slots = (long long)kv.rows * budget;
  const int per = slots <= 8192 ? 1 : slots <= 32768 ? 2 : 4;
  const int groups = (budget + per - 1) / per;
  const long long items = (long long)kv.rows * groups;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  cfg.dynamicSmemBytes = 0;
  cfg.gridDim = dim3((unsigned)((items + kMoveWarps - 1) / kMoveWarps));
  cfg.blockDim = dim3(kMoveWarps * 32);
  return cudaLaunchKernelEx(&cfg, evict_move_kernel, p, groups, per);
}

}  // namespace fgm

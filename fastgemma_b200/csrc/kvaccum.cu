// The attention weights that the slots of a KV cache received, added up per
// slot, on the tcgen05 tensor cores: acc = decay * acc + the sum over query rows
// of exp(score - lse).
//
// A tile is 128 slots: the A operand is their K rows, the B operand blocks of up
// to 128 int8 query rows, so a lane of TMEM is a slot and a thread adds up its
// own slot's weights in a register, block after block, KV head after KV head,
// in a fixed order and without a reduction across threads until the four
// warps that share a lane quadrant put their quarters together.  Four score
// buffers keep the tensor cores ahead of the exponentials: one per (query row,
// slot) pair at 16 a cycle per SM.
//
// 256 nodes, 8 heads over 2, over 16K slots of head_dim 256: 25.5 us, 34 M
// exponentials (the exponential unit 42 % busy, 8.2 us alone; without any
// arithmetic on the scores 20.6, without masks 22.8).  A launch is one tile of
// slots per CTA, so what is left is the start of each: the quantisation before
// it 4 us, K and the first queries 3, and 32 KB of queries per block and KV head
// from L2.  16 nodes of 8 sequences over 4K slots: 11.9 us, latency alone.
#include <type_traits>

#include "kv_tc.cuh"

namespace fgm {
namespace {

using namespace kv;

constexpr int kAddWarps = 16;
constexpr int kThreads = 128 + kAddWarps * 32;
constexpr int kQuarter = 32;     // query rows of a thread per block
constexpr int kBufs = 4;         // score buffers of 128 TMEM columns
constexpr int kQStages = 6;      // ring of 16 KB query chunks

struct AccumParams {
  TreeParams t;
  int blocks, nkb, kbufs;
  const int8_t *q8;              // [rows * kv_heads * blocks][nkb][128][128]
  const float *cst;              // [..][2][128]: query scales, -lse
  int *err;
};

struct Bars {
  uint64_t k_full[2], k_empty[2], q_full[kQStages], q_empty[kQStages], c_full[kBufs], d_full[kBufs],
      d_empty[kBufs];
};

template <bool SMALL>  // head_dim <= 256: |q8 . k8| < 2^22
__global__ void __launch_bounds__(kThreads, 1)
    accum_kernel(const __grid_constant__ AccumParams ap, const __grid_constant__ CUtensorMap kmap) {
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) Bars bar;
  __shared__ __align__(16) float s_cst[kBufs][2][kTM];
  __shared__ float s_sum[2][4][kTN];
  __shared__ int s_low[FGM_CUDA_TREE_MAX];
  __shared__ uint64_t s_see[FGM_CUDA_TREE_MAX][4];  // nodes that each node sees
  __shared__ uint64_t s_by[kTN][4];                 // nodes that see each slot of a tile
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_high[kThreads / 32];
  const TreeParams &p = ap.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = p.kv.head_dim, G = p.n_heads / p.kv.kv_heads, R = p.T * G, kvh_n = p.kv.kv_heads;
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *ksm = sm, *qsm = sm + ap.kbufs * ap.nkb * kChunk;
  stream::pdl_launch_dependents();

  Work wk;
  if (!find_work<true>(p, kTN, 1, 1, lane, wk)) return;
  const int b = wk.b, len = wk.span.len, ring = p.kv.ring, end = len + p.T;
  const int t0 = wk.t0, t1 = wk.t1, x1 = wk.span.end;
  // tiles below this hold no slot that a node sees: they only decay
  const int live = ring ? 0 : span_of(p, b).first / kTN;

  const int first = max(t0, live);               // first tile with products
  const int kloads = max(0, t1 - first) * kvh_n; // K tiles, one per KV head
  auto load_k = [&](int i) {
    const int buf = i % ap.kbufs, t = first + i / kvh_n, kvh = i % kvh_n;
    tc::mbar_expect_tx(&bar.k_full[buf], (uint32_t)ap.nkb * kChunk);
    for (int kb = 0; kb < ap.nkb; kb++)
      tc::tma_load_3d(ksm + (buf * ap.nkb + kb) * kChunk, &kmap, &bar.k_full[buf],
                      kvh * hd + kb * 128, t * kTN, b);
  };
  auto wait = [&](uint64_t *w, uint32_t parity) { wait_phase(w, parity, &s_abort); };
  if (tid == 0) {
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&bar.k_full[i], 1);
      tc::mbar_init(&bar.k_empty[i], 1);
    }
    for (int i = 0; i < kQStages; i++) {
      tc::mbar_init(&bar.q_full[i], 1);
      tc::mbar_init(&bar.q_empty[i], 1);
    }
    for (int i = 0; i < kBufs; i++) {
      tc::mbar_init(&bar.c_full[i], 1);
      tc::mbar_init(&bar.d_full[i], 1);
      tc::mbar_init(&bar.d_empty[i], kAddWarps);
    }
    tc::fence_mbar_init();
    s_abort = 0;
    for (int i = 0; i < min(kloads, ap.kbufs); i++) load_k(i);
  }
  if (warp == 1) {
    tc::tmem_alloc(&s_tmem, 512);
    tc::tmem_relinquish();
  }
  // what each node sees of the nodes, and its lowest position
  int high = INT_MIN;
  for (int i = tid; i < p.T * 4; i += kThreads) {
    const int node = i >> 2, w = i & 3;
    const int low = lowest(p.pos ? p.pos[b * p.T + node] : len + node, p.window);
    uint64_t v = 0;
    if (w * 64 < p.T) {
      v = p.mask ? p.mask[((size_t)b * p.T + node) * ((p.T + 63) / 64) + w]
                 : bit_range(0, node + 1 - w * 64);
      v &= bit_range(0, p.T - w * 64);
      if (p.window)
        for (int k = 0; k < min(64, p.T - w * 64); k++)
          if ((p.pos ? p.pos[b * p.T + w * 64 + k] : len + w * 64 + k) < low) v &= ~(1ull << k);
    }
    s_see[node][w] = v;
    if (w == 0) s_low[node] = low;
    high = max(high, low);
  }
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) s_high[warp] = high;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem;
  high = __reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? s_high[lane] : INT_MIN);
  const int units = kloads * ap.blocks;  // score blocks

  if (warp == 0) {  // ---- K tiles
    if (lane == 0)
      for (int i = ap.kbufs; i < kloads; i++) {
        wait(&bar.k_empty[i % ap.kbufs], (i / ap.kbufs - 1) & 1);
        load_k(i);
      }
  } else if (warp == 3) {  // ---- query blocks and their constants
    if (lane == 0) {
      stream::pdl_wait();  // for the kernel that quantised the queries
      int st = 0;
      uint32_t ph = 1;
      for (int u = 0, kvh = 0, blk = 0; u < units; u++) {
        const size_t qb = ((size_t)b * kvh_n + kvh) * ap.blocks + blk;
        for (int kb = 0; kb < ap.nkb; kb++) {
          if (u * ap.nkb + kb >= kQStages) wait(&bar.q_empty[st], ph);
          tc::mbar_expect_tx(&bar.q_full[st], kChunk);
          stream::bulk_g2s(tc::smem_u32(qsm + st * kChunk), ap.q8 + (qb * ap.nkb + kb) * kChunk,
                           kChunk, &bar.q_full[st]);
          if (++st == kQStages) st = 0, ph ^= 1;
        }
        const int buf = u % kBufs;
        if (u >= kBufs) wait(&bar.d_empty[buf], (u / kBufs - 1) & 1);
        tc::mbar_expect_tx(&bar.c_full[buf], 2 * kTM * 4);
        stream::bulk_g2s(tc::smem_u32(s_cst[buf]), ap.cst + qb * 2 * kTM, 2 * kTM * 4,
                         &bar.c_full[buf]);
        if (++blk == ap.blocks) {
          blk = 0;
          if (++kvh == kvh_n) kvh = 0;
        }
      }
    }
  } else if (warp == 1) {  // ---- MMAs
    if (lane == 0) {
      const uint64_t kd = desc128(tc::smem_u32(ksm)), qd = desc128(tc::smem_u32(qsm));
      // whole blocks, padding rows too: their columns hold finite sums, which
      // their constants (0, -infinity) turn into no weight
      const uint32_t id = tc::idesc_i8(kTN, kTM);
      int st = 0, u = 0;
      uint32_t ph = 0;
      for (int i = 0; i < kloads; i++) {
        const int kbuf = i % ap.kbufs;
        wait(&bar.k_full[kbuf], (i / ap.kbufs) & 1);
        for (int blk = 0; blk < ap.blocks; blk++, u++) {
          const int buf = u % kBufs;
          if (u >= kBufs) wait(&bar.d_empty[buf], (u / kBufs - 1) & 1);
          const uint32_t d = tmem + buf * kTM;
          for (int kb = 0; kb < ap.nkb; kb++) {
            wait(&bar.q_full[st], ph);
            tc::fence_after_sync();
            const uint64_t a = kd + (kbuf * ap.nkb + kb) * (kChunk >> 4);
            const uint64_t c = qd + st * (kChunk >> 4);
            tc::mma_i8(d, a, c, id, kb > 0);
            tc::mma_i8(d, a + 2, c + 2, id, 1);
            if (hd - kb * 128 >= 128) {
              tc::mma_i8(d, a + 4, c + 4, id, 1);
              tc::mma_i8(d, a + 6, c + 6, id, 1);
            }
            tc::mma_commit(&bar.q_empty[st]);
            if (++st == kQStages) st = 0, ph ^= 1;
          }
          tc::mma_commit(&bar.d_full[buf]);
        }
        tc::mma_commit(&bar.k_empty[kbuf]);
      }
    }
  } else if (warp >= 4) {  // ---- weights: slot (warp % 4) * 32 + lane, rows 32 * quarter ...
    const int quarter = (warp - 4) >> 2, in_tile = (warp & 3) * 32 + lane;
    const uint32_t quad = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const float *ks = p.kv.ks + (size_t)b * p.kv.ks_stride;
    float *acc = p.kv.acc + (size_t)b * p.kv.acc_stride;
    // the four warps that share the quadrant's slots
    auto meet = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + (warp & 3)) : "memory"); };
    int u = 0;
    for (int t = t0; t < t1; t++) {
      const int x = t * kTN + in_tile, pos = x < x1 ? pos_of(ring, x, end) : -1;
      const float scale = pos >= 0 ? ks[x] : 0.0f;
      float old = 0.0f;
      if (quarter == 0 && pos >= 0 && pos < len) old = p.decay * acc[x];
      float sum = 0.0f;
      // seen: the block's rows that see the slot, where not all of them do
      auto block = [&](uint32_t seen, auto is_masked) {
        constexpr bool masked = decltype(is_masked)::value;
        const int buf = u % kBufs, c0 = quarter * kQuarter;
        uint32_t s[kQuarter];
        tc::tmem_ld_x32(quad + buf * kTM + c0, s);
        const float *ca = &s_cst[buf][0][c0], *cz = &s_cst[buf][1][c0];
        const uint64_t k2 = pair2(scale, scale), l2 = pair2(kLog2e, kLog2e);
        uint64_t add = 0;
        tc::tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < kQuarter; c += 4) {
          const ulonglong2 a4 = *reinterpret_cast<const ulonglong2 *>(ca + c);
          const ulonglong2 z4 = *reinterpret_cast<const ulonglong2 *>(cz + c);
          const uint64_t aa[2] = {a4.x, a4.y}, zz[2] = {z4.x, z4.y};
#pragma unroll
          for (int k = 0; k < 4; k += 2) {
            // small int32 to f32 through the mantissa of 1.5 * 2^23, which
            // spares the unit that also takes the exponentials
            const uint64_t d =
                SMALL ? add2(pair2(__uint_as_float(s[c + k] + 0x4B400000u),
                                   __uint_as_float(s[c + k + 1] + 0x4B400000u)),
                             pair2(-12582912.0f, -12582912.0f))
                      : pair2((float)(int)s[c + k], (float)(int)s[c + k + 1]);
            float e0, e1;
            split2(mul2(fma2(mul2(d, k2), aa[k >> 1], zz[k >> 1]), l2), e0, e1);
            e0 = ex2(e0);
            e1 = ex2(e1);
            if (masked) {
              if (!((seen >> (c + k)) & 1)) e0 = 0.0f;
              if (!((seen >> (c + k + 1)) & 1)) e1 = 0.0f;
            }
            add = add2(add, pair2(e0, e1));
          }
        }
        float a0, a1;
        split2(add, a0, a1);
        sum += a0 + a1;
      };
      if (t >= first) {
        const bool masked = ring || (t + 1) * kTN > len || t * kTN < high;
        if (masked) {  // which nodes see this slot, 64 of them per quarter
          uint64_t v = 0;
          const int w0 = quarter * 64, n = min(64, p.T - w0), j = pos - len;
          if (pos >= 0 && n > 0) {
            if (pos < len && !p.window) {
              v = ~0ull;
            } else if (pos < len) {
              for (int i = 0; i < n; i++) v |= (uint64_t)(pos >= s_low[w0 + i]) << i;
            } else if (!p.mask && !p.window) {
              v = bit_range(j - w0, n);
            } else {
              const uint64_t *see = &s_see[w0][j >> 6];
#pragma unroll 8
              for (int i = 0; i < n; i++) v |= ((see[i * 4] >> (j & 63)) & 1) << i;
            }
          }
          s_by[in_tile][quarter] = v;
          meet();
        }
        for (int kvh = 0; kvh < kvh_n; kvh++)
          for (int blk = 0; blk < ap.blocks; blk++, u++) {
            const int buf = u % kBufs;
            wait(&bar.c_full[buf], (u / kBufs) & 1);
            wait(&bar.d_full[buf], (u / kBufs) & 1);
            tc::fence_after_sync();
            const int row = blk * kTM + quarter * kQuarter;  // the thread's first
            if (row < R && !masked) {
              block(~0u, std::false_type());
            } else if (row < R) {
              // bits of these rows' nodes: often none, or all, of a warp's slots are seen
              const int n = quick_div(row, G), last = quick_div(min(row + kQuarter, R) - 1, G);
              const int w = n >> 6, sh = n & 63;
              uint64_t by = s_by[in_tile][w] >> sh;
              if (w < 3 && sh) by |= s_by[in_tile][w + 1] << (64 - sh);
              const uint64_t nodes = (2ull << (last - n)) - 1;
              by &= nodes;
              if (__all_sync(0xffffffffu, by == nodes)) {
                block(~0u, std::false_type());
              } else if (__any_sync(0xffffffffu, by != 0)) {
                // each node's bit once per head
                const uint32_t heads = (1u << G) - 1;
                uint32_t seen = 0, bits = (uint32_t)by;
                for (int c = n * G - row; c < kQuarter; c += G, bits >>= 1)
                  if (bits & 1) seen |= c < 0 ? heads >> -c : heads << c;
                block(seen, std::true_type());
              }
            }
            tc::fence_before_sync();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&bar.d_empty[buf]);
          }
      }
      s_sum[t & 1][quarter][in_tile] = sum;
      meet();
      if (quarter == 0 && pos >= 0)
        acc[x] = old + ((sum + s_sum[t & 1][1][in_tile]) +
                        (s_sum[t & 1][2][in_tile] + s_sum[t & 1][3][in_tile]));
    }
  }
  __syncthreads();
  if (s_abort) {  // copies that nobody waited for still land in shared memory
    if (tid == 0 && ap.err) atomicExch(ap.err, 1);
    if (warp == 0 && lane == 0)
      for (int i = max(0, kloads - ap.kbufs); i < kloads; i++)
        tc::mbar_wait(&bar.k_full[i % ap.kbufs], (i / ap.kbufs) & 1);
    if (warp == 3 && lane == 0) {
      const int n = units * ap.nkb;
      for (int c = max(0, n - kQStages); c < n; c++)
        tc::mbar_wait(&bar.q_full[c % kQStages], (c / kQStages) & 1);
      for (int c = max(0, units - kBufs); c < units; c++)
        tc::mbar_wait(&bar.c_full[c % kBufs], (c / kBufs) & 1);
    }
    __syncthreads();
  }
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// A warp per query row of a block of 128: its int8 copy in the block's
// swizzled place and its scale; 4 us for any size in use, of which the kernel
// after it, launched early, spends 3 on its own setup.  For the attention the scale times log2(e);
// for the accumulation (p.decay in use, cst set) the scale itself and -lse, 0
// and -infinity where a row adds nothing.
constexpr int kQuantRows = 8;
__global__ void __launch_bounds__(kQuantRows * 32)
    quant_rows_kernel(const __grid_constant__ TreeParams p, int blocks, int nkb, int8_t *q8,
                      float *qs, float *cst) {
  const int lane = threadIdx.x & 31;
  const unsigned row = blockIdx.x * kQuantRows + (threadIdx.x >> 5);
  const int hd = p.kv.head_dim, G = p.n_heads / p.kv.kv_heads, R = p.T * G;
  stream::pdl_launch_dependents();
  const int block = (int)(row / kTM), j = (int)(row % kTM);
  const int bk = quick_div(block, blocks), r = (block - bk * blocks) * kTM + j;
  const int b = quick_div(bk, p.kv.kv_heads), kvh = bk - b * p.kv.kv_heads;
  if (r >= R) {
    if (cst && lane == 0) {
      cst[(size_t)block * 2 * kTM + j] = 0.0f;
      cst[(size_t)block * 2 * kTM + kTM + j] = -INFINITY;
    }
    return;
  }
  const int node = quick_div(r, G), h = kvh * G + r - node * G;
  const size_t qr = (size_t)b * p.T + node;
  const float4 *src = reinterpret_cast<const float4 *>(p.q + qr * p.q_ld + (size_t)h * hd);
  float4 v[4];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[i] = lane + 32 * i < hd / 4 ? src[lane + 32 * i] : make_float4(0, 0, 0, 0);
    top = fmaxf(fmaxf(top, fmaxf(q_abs(v[i].x), q_abs(v[i].y))),
                fmaxf(q_abs(v[i].z), q_abs(v[i].w)));
  }
  top = warp_max(top);
  const float inv = q_inv(top);
  int8_t *dst = q8 + (size_t)block * nkb * kChunk + j * 128 + (((lane >> 2) ^ (j & 7)) << 4) +
                (lane & 3) * 4;
#pragma unroll
  for (int i = 0; i < 4; i++)
    if (lane + 32 * i < hd / 4)
      *reinterpret_cast<uint32_t *>(dst + i * kChunk) =
          (q_int8(v[i].x, inv) & 255) | (q_int8(v[i].y, inv) & 255) << 8 |
          (q_int8(v[i].z, inv) & 255) << 16 | q_int8(v[i].w, inv) << 24;
  if (lane != 0) return;
  if (cst) {
    const float lse = p.lse[qr * p.lse_row + h * p.lse_head];
    const bool adds = lse != -INFINITY && (!p.take || p.take[qr]);
    // no scale either where it adds nothing: one that is no number would make
    // the constant -infinity no number
    cst[(size_t)block * 2 * kTM + j] = adds ? q_scale(top) : 0.0f;
    cst[(size_t)block * 2 * kTM + kTM + j] = adds ? -lse : -INFINITY;
  } else {
    // never 0, so that a masked score stays -inf (a zero query's dots are 0)
    qs[(size_t)block * kTM + j] =
        fmaxf(q_scale(top) * kLog2e, 1e-37f) + (top < INFINITY ? 0.0f : q_scale(top));
  }
}

struct AccumPlan {
  int blocks, nkb, kbufs;
  size_t smem, q8, cst, total;
};
AccumPlan accum_plan(const fgm_cuda_kv &kv, int n_heads, int T) {
  AccumPlan q;
  const int R = T * (n_heads / kv.kv_heads);
  q.blocks = (R + kTM - 1) / kTM;
  q.nkb = (kv.head_dim + 127) / 128;
  q.kbufs = q.nkb > 2 ? 1 : 2;
  q.smem = 1024 + (size_t)(q.kbufs * q.nkb + kQStages) * kChunk;
  const size_t qb = (size_t)kv.rows * kv.kv_heads * q.blocks;
  q.q8 = kCounters * sizeof(int);
  q.cst = q.q8 + qb * q.nkb * kChunk;
  q.total = q.cst + qb * 2 * kTM * sizeof(float);
  return q;
}
constexpr int kMaxSmem = 1024 + 10 * kChunk;

}  // namespace

cudaError_t launch_quant_rows(const TreeParams &p, int blocks, int nkb, int8_t *q8, float *qs,
                              float *cst, cudaStream_t st) {
  const long long rows = (long long)p.kv.rows * p.kv.kv_heads * blocks * kTM;
  quant_rows_kernel<<<(unsigned)(rows / kQuantRows), kQuantRows * 32, 0, st>>>(p, blocks, nkb, q8,
                                                                              qs, cst);
  return cudaGetLastError();
}

size_t accum_workspace(const fgm_cuda_kv &kv, int n_heads, int T) {
  return accum_plan(kv, n_heads, T).total;
}

cudaError_t launch_attend_accum(const TreeParams &p, int num_sms, int *err, cudaStream_t st) {
  const AccumPlan q = accum_plan(p.kv, p.n_heads, p.T);
  uint8_t *ws = static_cast<uint8_t *>(p.ws);
  AccumParams ap;
  ap.t = p;
  ap.blocks = q.blocks;
  ap.nkb = q.nkb;
  ap.kbufs = q.kbufs;
  ap.q8 = reinterpret_cast<const int8_t *>(ws + q.q8);
  ap.cst = reinterpret_cast<const float *>(ws + q.cst);
  ap.err = err;
  CUtensorMap kmap;
  if (!encode_cache_map(&kmap, p.kv)) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> done[2];
  const bool small = p.kv.head_dim <= 256;
  cudaError_t e = small ? allow_smem(accum_kernel<true>, kMaxSmem, done[0])
                        : allow_smem(accum_kernel<false>, kMaxSmem, done[1]);
  if (e != cudaSuccess) return e;
  e = launch_quant_rows(p, q.blocks, q.nkb, reinterpret_cast<int8_t *>(ws + q.q8), nullptr,
                        reinterpret_cast<float *>(ws + q.cst), st);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)grid_of(p.kv, p.kv.rows, kTN, num_sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = q.smem;
  return cudaLaunchKernelEx(&cfg, small ? accum_kernel<true> : accum_kernel<false>, ap, kmap);
}

}  // namespace fgm

// Attention of many query rows per KV head over the int8 KV cache, on the
// tcgen05 tensor cores: tiles of 128 query rows (T nodes x G heads of one KV
// head) by 128 slots.
//
// Per tile: the int32 scores Q8 . K8^T (kind::i8, exact) go to TMEM; sixteen
// softmax warps read them (a lane a row, a quarter of the tile's slots each),
// which frees the columns for the next tile's, scale, mask and exponentiate,
// and write the weights p * vs to TMEM as two f16 parts (22 bits together, as
// in the streaming kernel), 64 slots a buffer; those are the A operand of two
// products with V (kind::f16) that add into the f32 output in TMEM.  So no
// MMA is waited for before the next is issued, only their inputs are.  V comes
// from the cache as int8, four slots of a dimension per word; four warps load
// it and write the f16 B operand (exact), 64 slots at a time.  The output is
// rescaled only when a row's maximum has grown by more than 2^8: until then the
// weights just grow, for which the f16 scale leaves room.
//
// The queries are quantised once, by a kernel before, into the swizzled blocks
// that the tiles copy (each CTA for itself took 6 us more at 256 nodes over 16K
// slots: nine CTAs then read the same 128 KB); partial results of items split
// over CTAs are joined by a kernel after.
//
// A tile costs 128 * 128 * hd MACs at the int8 rate and twice that at the f16
// rate, 1.45 us at head_dim 256, and takes 3.0 (3.45 with the drains below):
// the MMAs, in the order of their issue, the softmax (2.5 us) and the
// conversion (2.6 us, half of it waiting for loads and stores to land) each wait
// for the others once per tile.  Left out one at a time they gained 3 us
// (conversion) and 7 us (softmax) of 65, both together 18, before there were
// drains.  Beside the tiles a call costs 23 us: the quantisation 4, setup 3
// (under it), the way to the first weights 4, the last product and 128 KB of
// partial results a CTA 5, the join 4, the rest launches.  256 nodes, 8 heads
// over 2, head_dim 256: 74.5 us over 16K slots, 218 over 64K (630 TFLOP/s of
// the two products; each counted once).
//
// Accuracy: the tensor cores cut an f32 sum off instead of rounding it, sixteen
// times per tile, for each term that is added; over a run of 512 tiles of equal
// weights and positive values that came to 4e-4 of the output (1.2e-6 now), over 57
// tiles of random ones to 1e-5 of its norm.  So the output is drained every kDrain tiles
// into memory (L2 holds it), where the parts are added with rounding to nearest,
// and the products start anew.  Error of random values at any length, and 256
// nodes over 64K slots: without drains 1e-5 and 183 us; every 8 tiles 1.7e-6 and
// 201; 6: 1.4e-6, 206; 4: 1.0e-6, 217, which is what rounding every f32 step leaves;
// 3: 0.8e-6, 231.  A drain costs 2.2 us, 1.4 of them the stores, the first 2
// more for the join at the end.
#include <type_traits>

#include "kv_tc.cuh"

namespace fgm {
namespace {

using namespace kv;

constexpr int kHalf = 64;         // slots per V stage
constexpr int kVStages = 3;
constexpr int kSoftWarps = 16, kSoft = kSoftWarps * 32;
constexpr int kThreads = 128 + kSoft + 128;  // loads and MMAs, softmax, V conversion
constexpr int kQuarter = kTN / 4;  // slots of a softmax thread
constexpr int kGrow = 8;          // log2 by which a row's maximum may grow unnoticed
constexpr int kDrain = 4;         // tiles between two drains of the output, at most
constexpr int kUnit = 7;          // f16 weights: p * vs * 2^(kUnit - ve), below 2^(kUnit + kGrow)
// TMEM columns: output [0, 256), scores 128, weights of 64 slots 2 x (32 high, 32 low parts)
constexpr uint32_t kColS = 256, kColP = 384;

struct TileParams {
  TreeParams t;
  int blocks, dsplit, dv;  // row blocks; CTAs that share an item's head_dim, dims of each
  int nkb;                 // 128-byte chunks of a K row
  int kstages;
  const int8_t *q8;        // [rows * kv_heads * blocks][nkb][128][128]: swizzled blocks
  const float *qs;         // their scales [..][128]
  float *part;             // [grid][128][dv]
  float2 *stat;            // [grid][128]
  int2 *desc;              // [items]: first CTA, CTAs
  int *err;
};

struct Bars {
  uint64_t q_full, k_full[4], k_empty[4], v_full[kVStages], v_empty[kVStages], s_full, s_empty,
      p_full[2], p_empty[2], sc_full[2], sc_empty[2];
};

// SMALL: head_dim <= 256, so that |q8 . k8| < 2^22.
template <bool SMALL>
__global__ void __launch_bounds__(kThreads, 1)
    tile_kernel(const __grid_constant__ TileParams tp, const __grid_constant__ CUtensorMap kmap) {
  extern __shared__ uint8_t raw[];
  __shared__ __align__(8) Bars bar;
  __shared__ __align__(16) float s_ks[2][kTN], s_vs[2][kTN];
  __shared__ float s_max[2][4][kTM], s_l[4][kTM];
  __shared__ int s_pos[FGM_CUDA_TREE_MAX], s_low[kTM];
  __shared__ uint64_t s_see[kTM][4];  // nodes each row sees
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_top[kThreads / 32];
  const TreeParams &p = tp.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = p.kv.head_dim, kvd = p.kv.kv_heads * hd, G = p.n_heads / p.kv.kv_heads;
  const int R = p.T * G, dv = tp.dv;
  uint8_t *sm = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
  uint8_t *q8 = sm, *ksm = q8 + tp.nkb * kChunk, *vf = ksm + tp.kstages * kChunk;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  Work wk;
  if (!find_work(p, kTN, p.kv.kv_heads * tp.blocks * tp.dsplit, 2, lane, wk)) return;
  const int b = wk.b, ds = wk.in_b % tp.dsplit, blk = wk.in_b / tp.dsplit % tp.blocks;
  const int kvh = wk.in_b / (tp.dsplit * tp.blocks), row0 = blk * kTM, rows = min(kTM, R - row0);
  const int len = wk.span.len, ring = p.kv.ring, end = len + p.T;
  const int x0 = wk.span.first + wk.t0 * kTN, x1 = min(wk.span.end, wk.span.first + wk.t1 * kTN);
  const int tiles = wk.t1 - wk.t0;
  const float *ks = p.kv.ks + (size_t)b * p.kv.ks_stride;
  const float *vs = p.kv.vs + (size_t)b * p.kv.vs_stride;

  const int chunks = tiles * tp.nkb, halves = tiles * 2;
  // The run in segments of kDrain tiles, with a drain between; what is short of
  // whole ones is missing in the first or the last, by CTA, so that not all CTAs
  // drain at once (16 sequences, 8 KV heads, 16K slots: 642 us against 658).
  const int spare = (tiles + kDrain - 1) / kDrain * kDrain - tiles;
  const int first = kDrain - (int)blockIdx.x % (spare + 1);
  auto load_k = [&](int c) {  // chunk c: tile c / nkb, bytes 128 * (c % nkb) of the rows
    const int st = c % tp.kstages, t = c / tp.nkb;
    tc::mbar_expect_tx(&bar.k_full[st], kChunk);
    tc::tma_load_3d(ksm + st * kChunk, &kmap, &bar.k_full[st],
                    kvh * hd + (c - t * tp.nkb) * 128, x0 + t * kTN, b);
  };
  auto wait = [&](uint64_t *w, uint32_t parity) { wait_phase(w, parity, &s_abort); };

  // the largest |vs| of the run: the unit of the f16 weights
  auto exponent = [&](int x) {
    if (x >= x1 || pos_of(ring, x, end) < 0) return -100;
    const float v = fabsf(vs[x]);
    if (!(v > 0.0f && v < INFINITY)) return -100;
    return max(-100, min((int)((__float_as_uint(v) >> 23) & 255) - 126, 126));
  };
  int top_e = -100;
#pragma unroll 2
  for (int x = x0 + tid; x < x1; x += kThreads) top_e = max(top_e, exponent(x));
  int low_pos = 0;
  if (tid < kTM) {
    const int node = min(row0 + tid, R - 1) / G;
    low_pos = p.pos ? p.pos[b * p.T + node] : len + node;
  }
  if (tid == 0) {
    for (int i = 0; i < 4; i++) {
      tc::mbar_init(&bar.k_full[i], 1);
      tc::mbar_init(&bar.k_empty[i], 1);
    }
    for (int i = 0; i < kVStages; i++) {
      tc::mbar_init(&bar.v_full[i], 4);
      tc::mbar_init(&bar.v_empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      tc::mbar_init(&bar.p_full[i], kSoftWarps / 2);
      tc::mbar_init(&bar.p_empty[i], 1);
      tc::mbar_init(&bar.sc_full[i], 1);
      tc::mbar_init(&bar.sc_empty[i], kSoftWarps);
    }
    tc::mbar_init(&bar.q_full, 1);
    tc::mbar_init(&bar.s_full, 1);
    tc::mbar_init(&bar.s_empty, kSoftWarps);
    tc::fence_mbar_init();
    s_abort = 0;
    for (int c = 0; c < min(chunks, tp.kstages); c++) load_k(c);
    if (wk.t0 == 0) tp.desc[b * p.kv.kv_heads * tp.blocks * tp.dsplit + wk.in_b] =
        make_int2(wk.first, wk.count);
  }
  if (warp == 1) {
    tc::tmem_alloc(&s_tmem, 512);
    tc::tmem_relinquish();
  }
  top_e = __reduce_max_sync(0xffffffffu, top_e);
  if (lane == 0) s_top[warp] = top_e;
  if (tid < kTM) s_low[tid] = tid < rows ? lowest(low_pos, p.window) : INT_MIN;
  if (p.window)
    for (int i = tid; i < p.T; i += kThreads) s_pos[i] = p.pos ? p.pos[b * p.T + i] : len + i;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = s_tmem;
  const int ve = __reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? s_top[lane] : -100);
  const size_t qblock = ((size_t)b * p.kv.kv_heads + kvh) * tp.blocks + blk;

  if (warp == 0) {  // ---- the queries, K chunks
    if (lane == 0) {
      stream::pdl_wait();  // for the kernel that quantised the queries
      tc::mbar_expect_tx(&bar.q_full, (uint32_t)tp.nkb * kChunk);
      stream::bulk_g2s(tc::smem_u32(q8), tp.q8 + qblock * tp.nkb * kChunk,
                       (uint32_t)tp.nkb * kChunk, &bar.q_full);
      for (int c = tp.kstages; c < chunks; c++) {
        const int st = c % tp.kstages;
        wait(&bar.k_empty[st], (c / tp.kstages - 1) & 1);
        load_k(c);
      }
    }
  } else if (warp == 2) {  // ---- scales of the slots, two tiles ahead
    const float unit = pow2(kUnit - ve);
    for (int j = 0; j < tiles; j++) {
      float a[4], c[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int x = x0 + j * kTN + lane + 32 * k;
        a[k] = x < x1 ? ks[x] : 0.0f;
        c[k] = x < x1 ? vs[x] * unit : 0.0f;
      }
      if (j >= 2) wait(&bar.sc_empty[j & 1], ((j - 2) >> 1) & 1);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        s_ks[j & 1][lane + 32 * k] = a[k];
        s_vs[j & 1][lane + 32 * k] = c[k];
      }
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.sc_full[j & 1]);
    }
  } else if (warp == 1) {  // ---- MMAs
    // descriptors differ from these in their address field, 16 bytes a unit
    const uint64_t qd = desc128(tc::smem_u32(q8)), kd = desc128(tc::smem_u32(ksm));
    const uint64_t vd = desc128(tc::smem_u32(vf));
    const uint32_t id_s = tc::idesc_i8(kTM, kTN), id_o = idesc_f16(kTM, dv);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
    const int n = __shfl_sync(0xffffffffu, tiles, 0);
    int kst = 0, vst = 0, left = __shfl_sync(0xffffffffu, first, 0);
    uint32_t kph = 0, vph = 0;
    auto scores = [&] {
      const uint32_t d = tm + kColS;
      for (int kb = 0; kb < tp.nkb; kb++) {
        wait(&bar.k_full[kst], kph);
        tc::fence_after_sync();
        const uint64_t a = qd + kb * (kChunk >> 4), c = kd + kst * (kChunk >> 4);
        if (elected()) {
          tc::mma_i8(d, a, c, id_s, kb > 0);
          tc::mma_i8(d, a + 2, c + 2, id_s, 1);
          if (hd - kb * 128 >= 128) {
            tc::mma_i8(d, a + 4, c + 4, id_s, 1);
            tc::mma_i8(d, a + 6, c + 6, id_s, 1);
          }
          tc::mma_commit(&bar.k_empty[kst]);
          if (kb == tp.nkb - 1) tc::mma_commit(&bar.s_full);
        }
        __syncwarp();
        if (++kst == tp.kstages) kst = 0, kph ^= 1;
      }
    };
    wait(&bar.q_full, 0);
    scores();
    for (int j = 0; j < n; j++) {
      if (j + 1 < n) {  // the next scores once these are in registers
        wait(&bar.s_empty, j & 1);
        scores();
      }
      const bool fresh = j == 0 || left == kDrain;  // the output starts anew
      left = left == 1 ? kDrain : left - 1;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        wait(&bar.p_full[h], j & 1);
        wait(&bar.v_full[vst], vph);
        tc::fence_after_sync();
        const uint64_t v = vd + vst * (dv * 8);
        const uint32_t a = tm + kColP + h * 64;
        if (elected()) {
#pragma unroll
          for (int k = 0; k < 4; k++) {
            mma_f16_ts(tm, a + k * 8, v + k * 2, id_o, !fresh || h + k > 0);
            mma_f16_ts(tm, a + 32 + k * 8, v + k * 2, id_o, 1);
          }
          tc::mma_commit(&bar.v_empty[vst]);
          tc::mma_commit(&bar.p_empty[h]);
        }
        __syncwarp();
        if (++vst == kVStages) vst = 0, vph ^= 1;
      }
    }
  } else if (warp >= 4 + kSoftWarps) {  // ---- V to f16, K-major: a row per dimension, 64 slots
    // A thread takes four dimensions of two slot groups at a time: dimension
    // 4 i + e becomes row e * dv / 4 + i, so that a warp's rows follow one
    // another and its stores meet no bank twice.  Loads run half a tile ahead.
    const int t = tid - (4 + kSoftWarps) * 32, quads = dv / 4;
    const uint8_t *src = reinterpret_cast<const uint8_t *>(p.kv.vt) + (size_t)b * p.kv.vt_stride +
                         (size_t)(kvh * hd + ds * dv) * 4;
    const int gend = (x1 + 3) >> 2;
    uint4 w[4][2];
    uint32_t to[4];  // where a unit's first row goes; rows are quads apart
    int pairs[4], from[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int i = t + 128 * k, q = i % quads;
      pairs[k] = i / quads;
      from[k] = 2 * pairs[k] * kvd * 4 + q * 16;
      to[k] = q * 128 + ((pairs[k] ^ (q & 7)) << 4);  // quads is a multiple of 8
    }
    auto load = [&](int h) {
      const int g0 = (x0 + h * kHalf) >> 2;
      const uint8_t *base = src + (size_t)g0 * kvd * 4;
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          w[k][e] = pairs[k] < 8 && g0 + 2 * pairs[k] + e < gend
                        ? __ldg(reinterpret_cast<const uint4 *>(base + from[k] + e * kvd * 4))
                        : make_uint4(0, 0, 0, 0);
    };
    load(0);
    int st = 0;
    uint32_t ph = 1;  // the parity of the stage's last release; fresh stages are free
    for (int h = 0; h < halves; h++) {
      if (h >= kVStages) wait(&bar.v_empty[st], ph);
      uint8_t *dst = vf + st * (dv * 128);
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const uint32_t a[4] = {w[k][0].x, w[k][0].y, w[k][0].z, w[k][0].w};
        const uint32_t c[4] = {w[k][1].x, w[k][1].y, w[k][1].z, w[k][1].w};
        if (pairs[k] < 8)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            uint4 o;
            i8x4_to_f16(a[e], o.x, o.y);
            i8x4_to_f16(c[e], o.z, o.w);
            *reinterpret_cast<uint4 *>(dst + to[k] + e * quads * 128) = o;
          }
      }
      if (h + 1 < halves) load(h + 1);
      stream::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.v_full[st]);
      if (++st == kVStages) st = 0, ph ^= 1;
    }
  } else if (warp >= 4) {  // ---- softmax: row (warp % 4) * 32 + lane, slots 32 * quarter ...
    const int quarter = (warp - 4) >> 2, row = (warp & 3) * 32 + lane;
    const uint32_t quad = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool idle = (warp & 3) * 32 >= rows;  // only padding rows: nothing to compute
    stream::pdl_wait();
    const float qs = row < rows ? tp.qs[qblock * kTM + row] : 1e-37f;
    const int high = __reduce_max_sync(
        0xffffffffu, max(max(s_low[lane], s_low[lane + 32]), max(s_low[lane + 64], s_low[lane + 96])));
    {  // the nodes this row sees, a word per quarter
      uint64_t v = 0;
      const int w = quarter, low = s_low[row], node = row < rows ? (row0 + row) / G : -1;
      if (node >= 0 && w * 64 < p.T) {
        v = p.mask ? p.mask[((size_t)b * p.T + node) * ((p.T + 63) / 64) + w]
                   : bit_range(0, node + 1 - w * 64);
        v &= bit_range(0, p.T - w * 64);
        if (p.window)
          for (int i = 0; i < min(64, p.T - w * 64); i++)
            if (s_pos[w * 64 + i] < low) v &= ~(1ull << i);
      }
      s_see[row][w] = v;
    }
    // the four warps that share the quadrant's rows
    auto meet = [&] { asm volatile("bar.sync %0, 128;" ::"r"(1 + (warp & 3)) : "memory"); };
    meet();
    float m = -INFINITY, l = 0.0f;

    // The output after a segment added to what was drained before, under the
    // maximum `ref` of the row's first segment until it has grown by 2^60.  Four
    // dimensions of the quadrant's 32 rows follow one another, so that a warp's
    // stores are whole lines; the place is that of the CTA's partial results of
    // these rows.  It comes after the next tile's weights are stored, by when
    // the segment's last product is done and the scores' registers are free, and
    // before they are handed over.  64K slots: 217 us; ahead of the next tile's
    // softmax 230; by the conversion's warps 293, by warps 0 to 3 241 (registers
    // pushed out to memory).
    float4 *drained = reinterpret_cast<float4 *>(
        tp.part + ((size_t)blockIdx.x * kTM + (warp & 3) * 32) * dv) + lane;
    float ref = -INFINITY;
    bool some = false;
    auto drain = [&](int j, float top) {
      wait(&bar.p_empty[0], j & 1);
      wait(&bar.p_empty[1], j & 1);
      tc::fence_after_sync();
      if (ref == -INFINITY) ref = top;  // only zeros so far
      float scale = ref == -INFINITY ? 1.0f : ex2(top - ref), g = 1.0f;
      const bool far = some && __any_sync(0xffffffffu, scale > pow2(60));
      if (far) {
        g = ref == -INFINITY ? 1.0f : ex2(ref - top);
        ref = top;
        scale = 1.0f;
      }
      for (int c = quarter * (dv / 4); c < (quarter + 1) * (dv / 4); c += 8) {
        uint32_t o[8];
        tmem_ld_x8(quad + c, o);
        tc::tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 8; k += 4) {
          float4 *to = drained + (c + k) * 8;  // (c + k) / 4 groups of 32 rows
          const float4 v = make_float4(
              __uint_as_float(o[k]) * scale, __uint_as_float(o[k + 1]) * scale,
              __uint_as_float(o[k + 2]) * scale, __uint_as_float(o[k + 3]) * scale);
          if (!some) {
            __stcg(to, v);
          } else if (!far) {
            red_add4(to, v);
          } else {
            const float4 a = __ldcg(to);
            __stcg(to, make_float4(__fmaf_rn(a.x, g, v.x), __fmaf_rn(a.y, g, v.y),
                                   __fmaf_rn(a.z, g, v.z), __fmaf_rn(a.w, g, v.w)));
          }
        }
      }
      tc::fence_before_sync();
      meet();
      some = true;
    };

    auto tile = [&](int j, bool fresh, auto is_masked) {
      constexpr bool masked = decltype(is_masked)::value;
      const int buf = j & 1;
      const float *ksq = s_ks[buf] + quarter * kQuarter, *vsq = s_vs[buf] + quarter * kQuarter;
      uint32_t s[kQuarter];
      tc::tmem_ld_x32(quad + kColS + quarter * kQuarter, s);
      uint32_t seen = 0;
      if (masked) {
        // position of slot x: x + (x <= turn ? lo_off : hi_off)
        const int turn = ring ? (end - 1) % ring : INT_MAX, low = s_low[row];
        const int lo_off = ring ? end - 1 - turn : 0, hi_off = lo_off - ring;
        const int x = x0 + j * kTN + quarter * kQuarter, cut = turn - x;
        seen = seen_from(x + (cut >= 0 ? lo_off : hi_off), len, low, s_see[row]);
        if (cut >= 0 && cut < kQuarter - 1) {  // the ring turns inside these slots
          const uint32_t before = (2u << cut) - 1;
          seen = (seen & before) | (seen_from(x + hi_off, len, low, s_see[row]) & ~before);
        }
        seen &= (uint32_t)bit_range(0, x1 - x);
      }
      tc::tmem_wait_ld();
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.s_empty);
      float top = -INFINITY;
#pragma unroll
      for (int c = 0; c < kQuarter; c += 4) {
        const ulonglong2 k4 = *reinterpret_cast<const ulonglong2 *>(ksq + c);
        const uint64_t kk[2] = {k4.x, k4.y};
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          // int32 to f32: small ones through the mantissa of 1.5 * 2^23, which
          // spares the unit that also takes the exponentials
          const uint64_t d =
              SMALL ? add2(pair2(__uint_as_float(s[c + k] + 0x4B400000u),
                                 __uint_as_float(s[c + k + 1] + 0x4B400000u)),
                           pair2(-12582912.0f, -12582912.0f))
                    : pair2((float)(int)s[c + k], (float)(int)s[c + k + 1]);
          float u0, u1;
          split2(mul2(d, kk[k >> 1]), u0, u1);
          if (masked && !((seen >> (c + k)) & 1)) u0 = -INFINITY;
          if (masked && !((seen >> (c + k + 1)) & 1)) u1 = -INFINITY;
          top = fmaxf(top, fmaxf(u0, u1));
          s[c + k] = __float_as_uint(u0);
          s[c + k + 1] = __float_as_uint(u1);
        }
      }
      s_max[buf][quarter][row] = top;
      meet();
      top = fmaxf(fmaxf(s_max[buf][0][row], s_max[buf][1][row]),
                  fmaxf(s_max[buf][2][row], s_max[buf][3][row])) * qs;
      // a growing maximum: the sum and, once something was added, the output
      float f = 1.0f;
      if (top > m + kGrow || m == -INFINITY) {
        f = m == -INFINITY ? 1.0f : ex2(m - top);
        m = top;
        l *= f;
      }
      if (!fresh && __any_sync(0xffffffffu, f != 1.0f)) {
        wait(&bar.p_empty[0], (j - 1) & 1);
        wait(&bar.p_empty[1], (j - 1) & 1);
        tc::fence_after_sync();
        for (int c = quarter * (dv / 4); c < (quarter + 1) * (dv / 4); c += 8) {
          uint32_t o[8];
          tmem_ld_x8(quad + c, o);
          tc::tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 8; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
          tmem_st_x8(quad + c, o);
        }
        tmem_wait_st();
        // A half's product adds into all of the output's columns, but waits for
        // the weights of two quarters alone, so nobody hands over weights before
        // all four have stored.  (They see the same maxima and get here
        // together.)  It also keeps every quarter within one phase of p_empty
        // of both halves, which a wait by parity needs.
        tc::fence_before_sync();
        meet();
        tc::fence_after_sync();
      }
      const float ref = m == -INFINITY ? 0.0f : m;
      const uint64_t qs2 = pair2(qs, qs), ref2 = pair2(-ref, -ref), minus = pair2(-1.0f, -1.0f);
      uint64_t sum = 0;
      uint32_t hi[16], lo[16];
#pragma unroll
      for (int c = 0; c < kQuarter; c += 4) {
        const ulonglong2 v4 = *reinterpret_cast<const ulonglong2 *>(vsq + c);
        const uint64_t vv[2] = {v4.x, v4.y};
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const int i = c + k;
          float e0, e1, w0, w1;
          split2(fma2(pair2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), qs2, ref2), e0, e1);
          const uint64_t e = pair2(ex2(e0), ex2(e1));
          sum = add2(sum, e);
          uint64_t w = mul2(e, vv[k >> 1]);
          split2(w, w0, w1);
          if (masked) {  // an unseen slot's scale may be anything
            if (!((seen >> i) & 1)) w0 = 0.0f;
            if (!((seen >> (i + 1)) & 1)) w1 = 0.0f;
            w = pair2(w0, w1);
          }
          const __half2 h2 = __floats2half2_rn(w0, w1);
          const float2 hf = __half22float2(h2);
          hi[i / 2] = *reinterpret_cast<const uint32_t *>(&h2);
          split2(fma2(pair2(hf.x, hf.y), minus, w), w0, w1);
          lo[i / 2] = pack2(w0, w1);
        }
      }
      float la, lb;
      split2(sum, la, lb);
      l += la + lb;
      // the buffer's last weights have to be multiplied
      if (j > 0) wait(&bar.p_empty[quarter >> 1], (j - 1) & 1);
      tc::fence_after_sync();
      const uint32_t to = quad + kColP + (quarter >> 1) * 64 + (quarter & 1) * 16;
      tmem_st_x16(to, hi);
      tmem_st_x16(to + 32, lo);
      tmem_wait_st();
    };
    for (int j = 0, left = first; j < tiles; j++) {
      const bool fresh = j == 0 || left == kDrain;  // its products add to nothing
      left = left == 1 ? kDrain : left - 1;
      wait(&bar.sc_full[j & 1], (j >> 1) & 1);
      wait(&bar.s_full, j & 1);
      tc::fence_after_sync();
      if (idle) {
        if (lane == 0) tc::mbar_arrive(&bar.s_empty);
        if (j > 0) wait(&bar.p_empty[quarter >> 1], (j - 1) & 1);
      } else {
        const float was = m;
        if (ring || x0 + (j + 1) * kTN > len || x0 + j * kTN < high)
          tile(j, fresh, std::true_type());
        else
          tile(j, fresh, std::false_type());
        if (fresh && j > 0) drain(j - 1, was);
      }
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive(&bar.p_full[quarter >> 1]);
        tc::mbar_arrive(&bar.sc_empty[j & 1]);
      }
    }
    // ---- results: the quarters' sums joined, each quarter's dimensions to
    // shared memory, whole rows from there (what the loads filled is free now)
    s_l[quarter][row] = l;
    meet();
    const float L = (s_l[0][row] + s_l[1][row]) + (s_l[2][row] + s_l[3][row]);
    wait(&bar.p_empty[0], (tiles - 1) & 1);
    wait(&bar.p_empty[1], (tiles - 1) & 1);
    tc::fence_after_sync();
    const bool whole = wk.count == 1;
    const float g = ref == -INFINITY ? 0.0f : ex2(ref - m);
    float back = pow2(ve) * 0.0078125f;  // 2^-kUnit
    if (whole) back = L == 0.0f ? 0.0f : back / L;
    float *stage = reinterpret_cast<float *>(sm + (size_t)row * (dv * 4 + 16));
    // column e * dv / 4 + i of the output is dimension 4 i + e
    auto put = [&](auto step) {
      constexpr int N = decltype(step)::value;
      for (int i = quarter * (dv / 16); i < (quarter + 1) * (dv / 16); i += N) {
        uint32_t o[4][N];
#pragma unroll
        for (int e = 0; e < 4; e++) tmem_ld<N>(quad + e * (dv / 4) + i, o[e]);
        tc::tmem_wait_ld();
        if (some) {
#pragma unroll
          for (int e = 0; e < 4; e++)
#pragma unroll
            for (int k = 0; k < N; k += 2) {
              const int c = e * (dv / 4) + i + k;
              const float2 a =
                  __ldcg(reinterpret_cast<const float2 *>(drained + c / 4 * 32) + (c / 2 & 1));
              o[e][k] = __float_as_uint(__fmaf_rn(a.x, g, __uint_as_float(o[e][k])));
              o[e][k + 1] = __float_as_uint(__fmaf_rn(a.y, g, __uint_as_float(o[e][k + 1])));
            }
        }
#pragma unroll
        for (int k = 0; k < N; k++)
          *reinterpret_cast<float4 *>(stage + 4 * (i + k)) =
              make_float4(__uint_as_float(o[0][k]) * back, __uint_as_float(o[1][k]) * back,
                          __uint_as_float(o[2][k]) * back, __uint_as_float(o[3][k]) * back);
      }
    };
    if (idle) {
    } else if (dv % 128 == 0) {
      put(std::integral_constant<int, 8>());
    } else {
      put(std::integral_constant<int, 2>());
    }
    tc::fence_before_sync();
    if (some) fence_proxy_async_global();  // the copy below goes where the drained rows lie
    stream::fence_proxy_async_smem();
    meet();
    if (quarter == 0 && row < rows) {
      const int r = row0 + row, node = r / G, h = kvh * G + r - node * G;
      const size_t qr = (size_t)b * p.T + node;
      bulk_s2g(whole ? p.out + qr * p.out_ld + (size_t)h * hd + ds * dv
                     : tp.part + ((size_t)blockIdx.x * kTM + row) * dv, stage, (uint32_t)dv * 4);
      tc::bulk_commit();
      if (!whole) tp.stat[(size_t)blockIdx.x * kTM + row] = make_float2(m, L);
      else if (ds == 0 && p.lse)
        p.lse[qr * p.lse_row + h * p.lse_head] = L == 0.0f ? -INFINITY : (m + log2f(L)) * kLn2;
      tc::bulk_wait_all();
    }
  }
  __syncthreads();
  if (s_abort) {  // copies that nobody waited for still land in shared memory
    if (tid == 0 && tp.err) atomicExch(tp.err, 1);
    if (warp == 0 && lane == 0)
      for (int c = max(0, chunks - tp.kstages); c < chunks; c++)
        tc::mbar_wait(&bar.k_full[c % tp.kstages], (c / tp.kstages) & 1);
    if (warp == 0 && lane == 0) tc::mbar_wait(&bar.q_full, 0);
    __syncthreads();
  }
  if (warp == 1) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, 512);
  }
}

// Joins an item's partial results: a CTA takes a few rows, a thread four
// dimensions of one.
constexpr int kJoin = 256;
__global__ void __launch_bounds__(kJoin) tile_join_kernel(const __grid_constant__ TileParams tp,
                                                          int groups) {
  const TreeParams &p = tp.t;
  const int hd = p.kv.head_dim, G = p.n_heads / p.kv.kv_heads, R = p.T * G, dv = tp.dv, dv4 = dv / 4;
  const int item = blockIdx.x / groups, per_row = kJoin / dv4;
  const int in_row = threadIdx.x / dv4, d = threadIdx.x - in_row * dv4;
  const int row = (blockIdx.x - item * groups) * per_row + in_row;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int per_b = p.kv.kv_heads * tp.blocks * tp.dsplit;
  const int b = item / per_b, in_b = item - b * per_b;
  const int ds = in_b % tp.dsplit, blk = in_b / tp.dsplit % tp.blocks;
  const int kvh = in_b / (tp.dsplit * tp.blocks), r = blk * kTM + row;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (in_row >= per_row || row >= kTM || r >= R) return;
  const int2 de = tp.desc[item];
  if (de.y == 1) return;
  const float2 *stat = tp.stat + (size_t)de.x * kTM + row;
  const float4 *part = reinterpret_cast<const float4 *>(tp.part) + ((size_t)de.x * kTM + row) * dv4 + d;
  const Joined j = join_row4(stat, part, kTM, (size_t)kTM * dv4, de.y);
  const int node = r / G, h = kvh * G + r - node * G;
  const size_t qr = (size_t)b * p.T + node;
  reinterpret_cast<float4 *>(p.out + qr * p.out_ld + (size_t)h * hd + ds * dv)[d] = j.a;
  if (d == 0 && ds == 0 && p.lse)
    p.lse[qr * p.lse_row + h * p.lse_head] =
        j.L == 0.0f ? -INFINITY : (j.M + log2f(j.L)) * kLn2;
}

constexpr int kMaxSmem = 210 * 1024;  // of any head_dim

struct TilePlan {
  int blocks, dsplit, dv, nkb, kstages;
  long long items;
  size_t smem, part, stat, desc, q8, qs, total;
};

TilePlan tile_plan(const fgm_cuda_kv &kv, int n_heads, int T) {
  TilePlan q;
  const int hd = kv.head_dim, R = T * (n_heads / kv.kv_heads);
  q.blocks = (R + kTM - 1) / kTM;
  q.dsplit = hd > 256 ? 2 : 1;
  q.dv = hd / q.dsplit;
  q.nkb = (hd + 127) / 128;
  q.kstages = q.nkb > 2 ? 3 : 4;
  q.items = (long long)kv.rows * kv.kv_heads * q.blocks * q.dsplit;
  q.smem = 1024 + (size_t)(q.nkb + q.kstages) * kChunk + (size_t)kVStages * q.dv * 128;
  const size_t grid = (size_t)max_grid(kv, q.items, kTN);
  q.part = kCounters * sizeof(int);
  q.stat = q.part + align256(grid * kTM * q.dv * sizeof(float));
  q.desc = q.stat + align256(grid * kTM * sizeof(float2));
  q.q8 = q.desc + align256((size_t)q.items * sizeof(int2));
  const size_t qblocks = (size_t)kv.rows * kv.kv_heads * q.blocks;
  q.qs = q.q8 + qblocks * q.nkb * kChunk;
  q.total = q.qs + align256(qblocks * kTM * sizeof(float));
  return q;
}

}  // namespace

size_t attend_tile_workspace(const fgm_cuda_kv &kv, int n_heads, int T) {
  return tile_plan(kv, n_heads, T).total;
}

cudaError_t launch_attend_tile(const TreeParams &p, int num_sms, int *err, cudaStream_t st) {
  const TilePlan q = tile_plan(p.kv, p.n_heads, p.T);
  uint8_t *ws = static_cast<uint8_t *>(p.ws);
  TileParams tp;
  tp.t = p;
  tp.blocks = q.blocks;
  tp.dsplit = q.dsplit;
  tp.dv = q.dv;
  tp.nkb = q.nkb;
  tp.kstages = q.kstages;
  tp.q8 = reinterpret_cast<const int8_t *>(ws + q.q8);
  tp.qs = reinterpret_cast<const float *>(ws + q.qs);
  tp.part = reinterpret_cast<float *>(ws + q.part);
  tp.stat = reinterpret_cast<float2 *>(ws + q.stat);
  tp.desc = reinterpret_cast<int2 *>(ws + q.desc);
  tp.err = err;
  CUtensorMap kmap;
  if (!encode_cache_map(&kmap, p.kv)) return cudaErrorInvalidValue;
  static std::atomic<uint64_t> done[2];
  const bool small = p.kv.head_dim <= 256;
  cudaError_t e = small ? allow_smem(tile_kernel<true>, kMaxSmem, done[0])
                        : allow_smem(tile_kernel<false>, kMaxSmem, done[1]);
  if (e != cudaSuccess) return e;
  const int R = p.T * (p.n_heads / p.kv.kv_heads), rows = R < kTM ? R : kTM;
  e = launch_quant_rows(p, q.blocks, q.nkb, reinterpret_cast<int8_t *>(ws + q.q8),
                        reinterpret_cast<float *>(ws + q.qs), nullptr, st);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.gridDim = dim3((unsigned)grid_of(p.kv, q.items, kTN, num_sms));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = q.smem;
  e = cudaLaunchKernelEx(&cfg, small ? tile_kernel<true> : tile_kernel<false>, tp, kmap);
  if (e != cudaSuccess) return e;
  const int per = kJoin / (q.dv / 4), groups = (rows + per - 1) / per;
  cfg.gridDim = dim3((unsigned)(q.items * groups));
  cfg.blockDim = dim3(kJoin);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, tile_join_kernel, tp, groups);
}

}  // namespace fgm

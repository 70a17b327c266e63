// Attention of several tokens per sequence over the int8 KV cache and the
// weights it accumulates per slot.
//
// R = T * G query rows share one KV head's K and V (T nodes, G query heads
// per KV head).  Per row: s = (q8 . k8) * qs * ks over the visible slots,
// p = exp(s - max), out = sum p vs v8 / sum p.
#include <cuda_fp16.h>

#include "fgm_common.cuh"
#include "fgm_internal.h"
#include "kv_common.cuh"

namespace fgm {
namespace {

using namespace kv;

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

__device__ __forceinline__ uint32_t smem_addr(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t a, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a));
}

__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// D += A(16x16 f16, row) * B(16x8 f16, col), f32 accumulate.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

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

// 2^e for -126 <= e <= 127.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

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
__device__ __forceinline__ Span span_of(const TreeParams &p, int b) {
  Span s;
  s.len = committed(p.kv, p.lens, b, p.T);
  s.end = s.len + p.T;
  s.first = 0;
  if (p.kv.ring) {
    s.end = min(s.end, p.kv.ring);
  } else if (p.window) {
    int low = INT_MAX;
    if (p.pos)
      for (int i = 0; i < p.T; i++) low = min(low, lowest(p.pos[b * p.T + i], p.window));
    else
      low = lowest(s.len, p.window);
    s.first = min(max(low, 0), s.len) & ~15;
  }
  return s;
}

// ------------------------------------------------------- few rows: streaming
// Up to 8 * NT query rows against a stream of K and V: bound by reading the
// cache.  Every warp runs on its own: a private ring of 16-slot stages filled
// by 16-byte asynchronous copies, the exact int8 scores as slots x rows
// (m16n8k32, K rows as they lie), a running maximum and sum, and P.V as dims x
// rows (m16n8k16).  The slot order inside a step is chosen so that the score
// fragment, transposed 8 x 8, is the weight fragment and one 32-bit word of
// the slot-interleaved V is a lane's four slots of one dimension: V needs no
// shuffling, only its conversion to f16, which is exact.  A weight p * vs is
// split into two f16 (scaled by a running power of two above the largest
// |vs|), 22 bits in all, so the products lose less than f32 rounding does.
//
// The work is one list of 128-slot tiles over all (sequence, KV head, row
// block) items, cut into equal runs, one per CTA, whatever the lengths; an
// item that spans several CTAs leaves partial results that finish_kernel
// joins.
constexpr int kTile = 128;   // slots per unit of the work list
constexpr int kStep = 16;    // slots per warp step

__host__ __device__ constexpr int stream_warps(int hd) { return hd <= 256 ? 8 : 4; }
__host__ __device__ constexpr int stage_bytes(int hd) { return 32 * hd + 16 * 16 + 4 * 32 + 128; }
__host__ __device__ constexpr int stream_stages(int hd) {
  const int s = 212992 / (stream_warps(hd) * stage_bytes(hd));
  return s > 8 ? 8 : s;
}
__host__ __device__ constexpr int q8_bytes(int hd) { return 16 * (hd + 16); }
__host__ __device__ constexpr int stream_smem(int hd) {
  return stream_warps(hd) * stream_stages(hd) * stage_bytes(hd) + q8_bytes(hd);
}

struct Desc {
  int first, count;  // CTAs of an item
};

struct StreamParams {
  TreeParams t;
  int blocks;       // row blocks per (sequence, KV head)
  int grid;
  float *part;      // [grid + items][8 NT][hd]
  float2 *stat;     // [grid + items][8 NT]: max * log2(e), sum
  Desc *desc;       // [items]
  float *scores;    // [rows][n_heads][score_ld], or null
  int score_ld;
};

template <int HD, int NT>
__global__ void __launch_bounds__(stream_warps(HD) * 32, 1)
    stream_kernel(const __grid_constant__ StreamParams sp) {
  constexpr int W = stream_warps(HD), S = stream_stages(HD), SB = stage_bytes(HD);
  constexpr int KLD = HD + 16, VLD = HD * 4 + 32, ROWS = 8 * NT, QLD = HD + 16;
  constexpr int OFF_V = 16 * KLD, OFF_KS = OFF_V + 4 * VLD, OFF_VS = OFF_KS + 64;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ float s_qs[ROWS], s_ml[W][ROWS], s_l[W][ROWS];
  __shared__ int s_node[ROWS], s_low[ROWS], s_e[W], s_at[4], s_high;
  const TreeParams &p = sp.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  const int kvd = p.kv.kv_heads * HD, G = p.n_heads / p.kv.kv_heads, R = p.T * G;
  const int per_b = p.kv.kv_heads * sp.blocks;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint8_t *q8 = sm + W * S * SB;

  // this CTA's run of the work list: [u, u1), and the sequence it starts in
  if (warp == 0) {
    long long total = 0;
    for (int b = lane; b < p.kv.rows; b += 32) {
      const Span s = span_of(p, b);
      total += (long long)((s.end - s.first + kTile - 1) / kTile) * per_b;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const long long per = (total + sp.grid - 1) / sp.grid;
    const long long u0 = per * blockIdx.x, u1 = min(total, u0 + per);
    long long base = 0;  // units before the chunk of 32 sequences
    int found = -1;
    long long before = 0;
    for (int b0 = 0; b0 < p.kv.rows && u0 < u1; b0 += 32) {
      long long n = 0;
      if (b0 + lane < p.kv.rows) {
        const Span s = span_of(p, b0 + lane);
        n = (long long)((s.end - s.first + kTile - 1) / kTile) * per_b;
      }
      long long inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + inc > u0);
      if (hit) {
        found = b0 + __ffs(hit) - 1;
        before = base + __shfl_sync(0xffffffffu, inc - n, __ffs(hit) - 1);
        break;
      }
      base += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) {
      s_at[0] = found;
      s_at[1] = (int)(u0 - before);
      s_at[2] = (int)(u1 - u0);
      s_at[3] = (int)per;
    }
  }
  __syncthreads();
  int b = s_at[0], rel = s_at[1], left = s_at[2];
  const int per = s_at[3];
  if (b < 0) return;
  // unit index of sequence b's first tile, as this CTA's first unit minus rel
  long long ub = (long long)per * blockIdx.x - rel;

  while (left > 0) {
    const Span span = span_of(p, b);
    const int tiles = (span.end - span.first + kTile - 1) / kTile;
    if (rel >= tiles * per_b) {
      ub += (long long)tiles * per_b;
      rel = 0;
      b++;
      continue;
    }
    const int in_b = rel / tiles, t0 = rel - in_b * tiles, t1 = min(tiles, t0 + left);
    rel += t1 - t0;
    left -= t1 - t0;
    const int kvh = in_b / sp.blocks, row0 = (in_b - kvh * sp.blocks) * ROWS;
    const int item = b * per_b + in_b, len = span.len, ring = p.kv.ring, end = len + p.T;
    const int x0 = span.first + t0 * kTile, x1 = min(span.end, span.first + t1 * kTile);
    const long long ui = ub + (long long)in_b * tiles;
    const int c0 = (int)(ui / per), c1 = (int)((ui + tiles - 1) / per);
    const int8_t *kc = p.kv.kc + (size_t)b * p.kv.kc_stride + (size_t)kvh * HD;
    const int8_t *vt = p.kv.vt + (size_t)b * p.kv.vt_stride + (size_t)kvh * HD * 4;
    const float *ks = p.kv.ks + (size_t)b * p.kv.ks_stride;
    const float *vs = p.kv.vs + (size_t)b * p.kv.vs_stride;
    const uint32_t ring0 = smem_addr(sm) + warp * S * SB;

    auto fetch = [&](int x, int stage) {  // slots [x, x + 16) into a stage
      if (x < x1) {
        const uint32_t st = ring0 + stage * SB;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
          const int c = lane + 32 * i, r = c / (HD / 16), k = c % (HD / 16);
          if (x + r < x1) cp16(st + r * KLD + k * 16, kc + (size_t)(x + r) * kvd + k * 16);
        }
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
          const int c = lane + 32 * i, g = c / (HD / 4), k = c % (HD / 4);
          if (x + 4 * g < x1)
            cp16(st + OFF_V + g * VLD + k * 16, vt + ((size_t)(x >> 2) + g) * kvd * 4 + k * 16);
        }
        const int s = lane & 15;
        if (x + s < x1) cp4(st + (lane < 16 ? OFF_KS : OFF_VS) + s * 4, (lane < 16 ? ks : vs) + x + s);
      }
      cp_commit();
    };
    const int xw = x0 + warp * kStep;
    constexpr int stride = W * kStep;
#pragma unroll
    for (int s = 0; s < S - 1; s++) fetch(xw + s * stride, s);

    // the block's queries to int8, a row per warp
    if (tid == 0) s_high = INT_MIN;
    for (int j = warp; j < ROWS; j += W) {
      const int r = row0 + j, node = r < R ? r / G : -1;
      uint32_t *dst = reinterpret_cast<uint32_t *>(q8 + j * QLD);
      if (node < 0) {
        for (int d = lane; d < HD / 4; d += 32) dst[d] = 0;
        if (lane == 0) s_node[j] = -1, s_low[j] = INT_MIN, s_qs[j] = 0.0f;
        continue;
      }
      const float4 *src = reinterpret_cast<const float4 *>(
          p.q + ((size_t)b * p.T + node) * p.q_ld + (size_t)(kvh * G + r - node * G) * HD);
      float4 v[(HD + 127) / 128];
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < (HD + 127) / 128; i++) {
        v[i] = lane + 32 * i < HD / 4 ? src[lane + 32 * i] : make_float4(0, 0, 0, 0);
        top = fmaxf(fmaxf(top, fmaxf(q_abs(v[i].x), q_abs(v[i].y))),
                    fmaxf(q_abs(v[i].z), q_abs(v[i].w)));
      }
      top = warp_max(top);
      const float inv = q_inv(top);
#pragma unroll
      for (int i = 0; i < (HD + 127) / 128; i++)
        if (lane + 32 * i < HD / 4)
          dst[lane + 32 * i] = (q_int8(v[i].x, inv) & 255) | (q_int8(v[i].y, inv) & 255) << 8 |
                               (q_int8(v[i].z, inv) & 255) << 16 | q_int8(v[i].w, inv) << 24;
      if (lane == 0) {
        s_node[j] = node;
        s_low[j] = lowest(p.pos ? p.pos[b * p.T + node] : len + node, p.window);
        s_qs[j] = q_scale(top);
      }
    }
    __syncthreads();
    if (warp == 0) {
      const int v = lane < ROWS ? s_low[lane] : INT_MIN;
      const int h = __reduce_max_sync(0xffffffffu, v);
      if (lane == 0) s_high = h;
    }
    __syncthreads();
    const int high = s_high;

    uint32_t qf[NT][HD / 32][2];
    float qs[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int k = 0; k < HD / 32; k++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          qf[n][k][e] = *reinterpret_cast<const uint32_t *>(q8 + (n * 8 + gid) * QLD + k * 32 +
                                                            e * 16 + tig * 4);
      qs[n][0] = s_qs[n * 8 + 2 * tig];
      qs[n][1] = s_qs[n * 8 + 2 * tig + 1];
    }
    float o[NT][HD / 16][4], ml[NT][2], l[NT][2];
    int ve = -100;  // the weights' unit: 2^ve is at least every |vs| so far
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int m = 0; m < HD / 16; m++) o[n][m][0] = o[n][m][1] = o[n][m][2] = o[n][m][3] = 0.0f;
      ml[n][0] = ml[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
    }
    // row of the K fragment this lane addresses, as a slot of the step
    const int lr = lane & 7, ls = 4 * (lr >> 1) + (lr & 1) + ((lane & 8) ? 2 : 0);
    const int sa = 4 * (gid >> 1) + (gid & 1);  // slots of this lane's scores: sa, sa + 2

    int stage = 0;
    for (int x = xw; x < x1; x += stride) {
      fetch(x + (S - 1) * stride, stage == 0 ? S - 1 : stage - 1);
      cp_wait<S - 1>();
      __syncwarp();
      const uint8_t *st = sm + (warp * S + stage) * SB;
      const uint32_t sta = ring0 + stage * SB;
      int32_t d[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0;
#pragma unroll
      for (int k = 0; k < HD / 32; k++) {
        uint32_t a[4];
        ldsm4(sta + ls * KLD + k * 32 + (lane & 16), a);
#pragma unroll
        for (int n = 0; n < NT; n++)
          mma_s8_m16n8k32(d[n], a[0], a[1], a[2], a[3], qf[n][k][0], qf[n][k][1]);
      }
      float kq[2], vq[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        kq[e] = *reinterpret_cast<const float *>(st + OFF_KS + (sa + 2 * e) * 4);
        vq[e] = *reinterpret_cast<const float *>(st + OFF_VS + (sa + 2 * e) * 4);
      }
      float s[NT][4];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          s[n][e] = __fmul_rn(__fmul_rn((float)d[n][e], qs[n][e & 1]), kq[e >> 1]);
      if (ring || x + kStep > len || x < high) {
        bool any[2] = {false, false};
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const int t = x + sa + 2 * e < x1 ? pos_of(ring, x + sa + 2 * e, end) : -1;
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
              const int row = n * 8 + 2 * tig + c;
              const bool v = sees(p, b, s_node[row], len, t, s_low[row]);
              if (!v) s[n][2 * e + c] = -INFINITY;
              any[e] |= v;
            }
          // a slot that no row sees may hold any scale
          const unsigned m = __ballot_sync(0xffffffffu, any[e]);
          if (!((m >> (gid * 4)) & 15)) vq[e] = 0.0f;
        }
      }
      if (sp.scores) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int row = row0 + n * 8 + 2 * tig + (e & 1), xs = x + sa + 2 * (e >> 1);
            if (row < R && xs < x1)
              sp.scores[((size_t)b * p.n_heads + kvh * G + row) * sp.score_ld + xs] = s[n][e];
          }
      }
      // the weights' unit grows when a scale passes it
      const float va = fmaxf(fabsf(vq[0]), fabsf(vq[1]));
      bool grow = false;
      float shrink = 1.0f;
      if (__any_sync(0xffffffffu, va > pow2(ve))) {
        const float top = warp_max(va);
        const int e = min((int)((__float_as_uint(top) >> 23) & 255) - 126, 126);
        shrink = ve - e < -126 ? 0.0f : pow2(ve - e);
        ve = e;
        grow = true;
      }
      float corr[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
          float mx = fmaxf(s[n][c], s[n][2 + c]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float mn = fmaxf(ml[n][c], mx * kLog2e);
          corr[n][c] = mn > ml[n][c] ? ex2(ml[n][c] - mn) : 1.0f;
          grow |= mn > ml[n][c];
          ml[n][c] = mn;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          l[n][0] *= corr[n][0];
          l[n][1] *= corr[n][1];
          const float f0 = corr[n][0] * shrink, f1 = corr[n][1] * shrink;
#pragma unroll
          for (int m = 0; m < HD / 16; m++) {
            o[n][m][0] *= f0;
            o[n][m][1] *= f1;
            o[n][m][2] *= f0;
            o[n][m][3] *= f1;
          }
        }
      }
      const float unit = pow2(13 - ve);
      uint32_t bh[NT][2], bl[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          float w[2];
#pragma unroll
          for (int c = 0; c < 2; c++) {
            const float ref = ml[n][c] == -INFINITY ? 0.0f : ml[n][c];
            const float pr = ex2(__fmaf_rn(s[n][2 * e + c], kLog2e, -ref));
            l[n][c] += pr;
            w[c] = pr * (vq[e] * unit);
          }
          const __half2 h = __floats2half2_rn(w[0], w[1]);
          const float2 hf = __half22float2(h);
          const __half2 r = __floats2half2_rn(w[0] - hf.x, w[1] - hf.y);
          bh[n][e] = transpose8(*reinterpret_cast<const uint32_t *>(&h));
          bl[n][e] = transpose8(*reinterpret_cast<const uint32_t *>(&r));
        }
#pragma unroll
      for (int j = 0; j < HD / 32; j++) {
        const uint4 v = *reinterpret_cast<const uint4 *>(st + OFF_V + tig * VLD + j * 128 + gid * 16);
        const uint32_t vw[4] = {v.x, v.y, v.z, v.w};
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; i++) i8x4_to_f16(vw[i], lo[i], hi[i]);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
          for (int n = 0; n < NT; n++) {
            mma_f16(o[n][2 * j + i], lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1], bh[n][0],
                    bh[n][1]);
            mma_f16(o[n][2 * j + i], lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1], bl[n][0],
                    bl[n][1]);
          }
      }
      __syncwarp();
      stage = stage + 1 == S ? 0 : stage + 1;
    }
    cp_wait<0>();

    // ---- the warps' results joined in shared memory (the ring's, now idle)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        float v = l[n][c];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (gid == 0) {
          s_ml[warp][n * 8 + 2 * tig + c] = ml[n][c];
          s_l[warp][n * 8 + 2 * tig + c] = v;
        }
      }
    if (lane == 0) s_e[warp] = ve;
    __syncthreads();
    int e_all = -100;
#pragma unroll
    for (int w = 0; w < W; w++) e_all = max(e_all, s_e[w]);
    float *red = reinterpret_cast<float *>(sm);
    constexpr int RLD = HD + 4;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int c = 0; c < 2; c++) {
        const int row = n * 8 + 2 * tig + c;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, s_ml[w][row]);
        const float f = ex2(ml[n][c] - (M == -INFINITY ? 0.0f : M)) *
                        (ve - e_all < -126 ? 0.0f : pow2(ve - e_all));
#pragma unroll
        for (int m = 0; m < HD / 16; m++)
          *reinterpret_cast<float2 *>(red + (warp * ROWS + row) * RLD + (m >> 1) * 32 + gid * 4 +
                                      (m & 1) * 2) = make_float2(o[n][m][c] * f, o[n][m][2 + c] * f);
      }
    __syncthreads();
    const float back = pow2(e_all) * 0.0001220703125f;  // 2^-13
    const int rows = min(ROWS, R - row0), part = blockIdx.x + item;
    for (int i = tid; i < rows * (HD / 4); i += W * 32) {
      const int row = i / (HD / 4), d = (i - row * (HD / 4)) * 4;
      float4 a = make_float4(0, 0, 0, 0);
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int w = 0; w < W; w++) {
        const float4 v = *reinterpret_cast<const float4 *>(red + (w * ROWS + row) * RLD + d);
        a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
        M = fmaxf(M, s_ml[w][row]);
      }
      const float ref = M == -INFINITY ? 0.0f : M;
#pragma unroll
      for (int w = 0; w < W; w++) L += s_l[w][row] * ex2(s_ml[w][row] - ref);
      a.x *= back, a.y *= back, a.z *= back, a.w *= back;
      if (c0 == c1) {
        const int r = row0 + row, node = r / G, h = kvh * G + r - node * G;
        const size_t qr = (size_t)b * p.T + node;
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        a.x *= inv, a.y *= inv, a.z *= inv, a.w *= inv;
        *reinterpret_cast<float4 *>(p.out + qr * p.out_ld + (size_t)h * HD + d) = a;
        if (d == 0 && p.lse)
          p.lse[qr * p.lse_row + h * p.lse_head] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
      } else {
        *reinterpret_cast<float4 *>(sp.part + ((size_t)part * ROWS + row) * HD + d) = a;
      }
      if (d == 0 && (c0 != c1 || sp.scores)) sp.stat[(size_t)part * ROWS + row] = make_float2(M, L);
    }
    if (tid == 0 && t0 == 0) sp.desc[item] = Desc{c0, c1 - c0 + 1};
    __syncthreads();
  }
}

// Joins the partial results of an item's row (the first `joins` CTAs, one
// per row of every item), or adds the weights of the stored scores to 512
// slots of a sequence (the others).
constexpr int kFinish = 128, kAccSlots = 512;
constexpr int kMaxParts = 512;  // more CTAs than any grid

__global__ void __launch_bounds__(kFinish) finish_kernel(const __grid_constant__ StreamParams sp,
                                                         int rows_pb, int joins) {
  __shared__ float s_f[kMaxParts], s_red[4][512], s_w[4], s_lse[2048];
  const TreeParams &p = sp.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int hd = p.kv.head_dim, G = p.n_heads / p.kv.kv_heads, R = p.T * G;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if ((int)blockIdx.x < joins) {
    const int item = blockIdx.x / rows_pb, row = blockIdx.x - item * rows_pb;
    const int blk = item % sp.blocks, r = blk * rows_pb + row;
    if (r >= R) return;
    const Desc de = sp.desc[item];
    if (de.count == 1) return;
    const int bk = item / sp.blocks, b = bk / p.kv.kv_heads, kvh = bk - b * p.kv.kv_heads;
    const int node = r / G, h = kvh * G + r - node * G;
    const float2 *stat = sp.stat + (size_t)(de.first + item) * rows_pb + row;
    float M = -INFINITY;
    for (int i = tid; i < de.count; i += kFinish) M = fmaxf(M, stat[(size_t)i * rows_pb].x);
    M = warp_max(M);
    if (lane == 0) s_w[warp] = M;
    __syncthreads();
    M = fmaxf(fmaxf(s_w[0], s_w[1]), fmaxf(s_w[2], s_w[3]));
    __syncthreads();
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    for (int i = tid; i < de.count; i += kFinish) {
      const float2 v = stat[(size_t)i * rows_pb];
      const float f = ex2(v.x - ref);
      s_f[i] = f;
      L += f * v.y;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) s_w[warp] = L;
    __syncthreads();
    L = (s_w[0] + s_w[1]) + (s_w[2] + s_w[3]);
    // warps take parts in turn, lanes the dimensions
    const float *src = sp.part + ((size_t)(de.first + item) * rows_pb + row) * hd;
    float4 a[4];
#pragma unroll
    for (int k = 0; k < 4; k++) a[k] = make_float4(0, 0, 0, 0);
    for (int i = warp; i < de.count; i += 4) {
      const float f = s_f[i];
      const float4 *v = reinterpret_cast<const float4 *>(src + (size_t)i * rows_pb * hd);
#pragma unroll
      for (int k = 0; k < 4; k++)
        if (lane + 32 * k < hd / 4) {
          const float4 u = v[lane + 32 * k];
          a[k].x += f * u.x, a[k].y += f * u.y, a[k].z += f * u.z, a[k].w += f * u.w;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; k++)
      if (lane + 32 * k < hd / 4) reinterpret_cast<float4 *>(s_red[warp])[lane + 32 * k] = a[k];
    __syncthreads();
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    const size_t qr = (size_t)b * p.T + node;
    for (int d = tid; d < hd; d += kFinish)
      p.out[qr * p.out_ld + (size_t)h * hd + d] =
          ((s_red[0][d] + s_red[1][d]) + (s_red[2][d] + s_red[3][d])) * inv;
    if (tid == 0 && p.lse)
      p.lse[qr * p.lse_row + h * p.lse_head] = L == 0.0f ? -INFINITY : (M + log2f(L)) * kLn2;
    return;
  }
  // accumulation (T = 1): a sequence's heads' log sums, then its slots
  const int per = (p.kv.cap + kAccSlots - 1) / kAccSlots;
  const int ix = blockIdx.x - joins, b = ix / per, x0 = (ix - b * per) * kAccSlots;
  const int len = committed(p.kv, p.lens, b, 1);
  if (x0 > len) return;
  for (int h = warp; h < p.n_heads; h += 4) {
    const int kvh = h / G, g = h - kvh * G;
    const int item = (b * p.kv.kv_heads + kvh) * sp.blocks + g / rows_pb;
    const Desc de = sp.desc[item];
    const float2 *stat = sp.stat + (size_t)(de.first + item) * rows_pb + g % rows_pb;
    float M = -INFINITY, L = 0.0f;
    for (int i = lane; i < de.count; i += 32) {
      const float2 v = stat[(size_t)i * rows_pb];
      const float n = fmaxf(M, v.x), ref = n == -INFINITY ? 0.0f : n;
      L = L * ex2(M - ref) + v.y * ex2(v.x - ref);
      M = n;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, M, o), l2 = __shfl_xor_sync(0xffffffffu, L, o);
      const float n = fmaxf(M, m2), ref = n == -INFINITY ? 0.0f : n;
      L = L * ex2(M - ref) + l2 * ex2(m2 - ref);
      M = n;
    }
    if (lane == 0) s_lse[h] = L == 0.0f ? INFINITY : M + log2f(L);
  }
  __syncthreads();
  float *acc = p.kv.acc + (size_t)b * p.kv.acc_stride;
  for (int x = x0 + tid; x < min(x0 + kAccSlots, len + 1); x += kFinish) {
    float sum = 0.0f;
    for (int h = 0; h < p.n_heads; h++)
      sum += ex2(__fmaf_rn(sp.scores[((size_t)b * p.n_heads + h) * sp.score_ld + x], kLog2e,
                           -s_lse[h]));
    acc[x] = (x < len ? p.decay * acc[x] : 0.0f) + sum;
  }
}

// --------------------------------------------------------------- accumulation
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

// ------------------------------------------------------------------ launching
constexpr int kMaxGrid = 296;  // CTAs of the streaming kernel, at most

size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Row blocks of 8 * nt rows: one block of 16 where the accumulators of 16
// rows fit the registers (head_dim <= 256), else blocks of 8.
void stream_blocks(const fgm_cuda_kv &kv, int n_heads, int T, int &nt, int &blocks) {
  const int R = T * (n_heads / kv.kv_heads);
  nt = R > 8 && kv.head_dim <= 256 ? 2 : 1;
  blocks = (R + 8 * nt - 1) / (8 * nt);
}

struct StreamWs {
  size_t part, stat, desc, scores, total;
  int score_ld;
};
StreamWs stream_ws(const fgm_cuda_kv &kv, int n_heads, int T) {
  int nt, blocks;
  stream_blocks(kv, n_heads, T, nt, blocks);
  const size_t items = (size_t)kv.rows * kv.kv_heads * blocks, parts = items + kMaxGrid;
  StreamWs w;
  w.part = 0;
  w.stat = w.part + align256(parts * 8 * nt * kv.head_dim * sizeof(float));
  w.desc = w.stat + align256(parts * 8 * nt * sizeof(float2));
  w.scores = w.desc + align256(items * sizeof(Desc));
  w.score_ld = (kv.cap + 31) & ~31;
  w.total = w.scores +
            (T == 1 ? align256((size_t)kv.rows * n_heads * w.score_ld * sizeof(float)) : 0);
  return w;
}

template <int HD, int NT>
cudaError_t launch_stream_as(const StreamParams &sp, cudaStream_t st) {
  cudaError_t e = cudaFuncSetAttribute(stream_kernel<HD, NT>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       stream_smem(HD));
  if (e != cudaSuccess) return e;
  stream_kernel<HD, NT><<<sp.grid, stream_warps(HD) * 32, stream_smem(HD), st>>>(sp);
  return cudaGetLastError();
}

cudaError_t launch_stream(const TreeParams &p, bool accumulate, int num_sms, cudaStream_t st) {
  int nt, blocks;
  stream_blocks(p.kv, p.n_heads, p.T, nt, blocks);
  const StreamWs w = stream_ws(p.kv, p.n_heads, p.T);
  uint8_t *ws = static_cast<uint8_t *>(p.ws);
  StreamParams sp;
  sp.t = p;
  sp.blocks = blocks;
  const long long items = (long long)p.kv.rows * p.kv.kv_heads * blocks;
  const long long most = items * ((p.kv.cap + kTile - 1) / kTile);
  sp.grid = (int)(most < num_sms ? most : num_sms);
  if (sp.grid > kMaxGrid) sp.grid = kMaxGrid;
  sp.part = reinterpret_cast<float *>(ws + w.part);
  sp.stat = reinterpret_cast<float2 *>(ws + w.stat);
  sp.desc = reinterpret_cast<Desc *>(ws + w.desc);
  sp.scores = accumulate ? reinterpret_cast<float *>(ws + w.scores) : nullptr;
  sp.score_ld = w.score_ld;
  cudaError_t e = cudaErrorInvalidValue;
  switch (p.kv.head_dim * 2 + nt - 1) {
    case 128: e = launch_stream_as<64, 1>(sp, st); break;
    case 129: e = launch_stream_as<64, 2>(sp, st); break;
    case 256: e = launch_stream_as<128, 1>(sp, st); break;
    case 257: e = launch_stream_as<128, 2>(sp, st); break;
    case 384: e = launch_stream_as<192, 1>(sp, st); break;
    case 385: e = launch_stream_as<192, 2>(sp, st); break;
    case 512: e = launch_stream_as<256, 1>(sp, st); break;
    case 513: e = launch_stream_as<256, 2>(sp, st); break;
    case 640: e = launch_stream_as<320, 1>(sp, st); break;
    case 768: e = launch_stream_as<384, 1>(sp, st); break;
    case 896: e = launch_stream_as<448, 1>(sp, st); break;
    case 1024: e = launch_stream_as<512, 1>(sp, st); break;
  }
  if (e != cudaSuccess) return e;
  const long long joins = items * 8 * nt;
  const long long adds =
      accumulate ? (long long)p.kv.rows * ((p.kv.cap + kAccSlots - 1) / kAccSlots) : 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(joins + adds));
  cfg.blockDim = dim3(kFinish);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, finish_kernel, sp, 8 * nt, (int)joins);
}

}  // namespace

size_t attend_workspace(const fgm_cuda_kv &kv, int n_heads, int T) {
  return stream_ws(kv, n_heads, T).total;
}

cudaError_t launch_attend_tree(const TreeParams &p, int num_sms, cudaStream_t st) {
  return launch_stream(p, false, num_sms, st);
}

cudaError_t launch_attend_accum(const TreeParams &p, int num_sms, cudaStream_t st) {
  const int slots = p.kv.ring ? p.kv.ring : p.kv.cap;
  accum_kernel<<<dim3((unsigned)((slots + 3) / 4), (unsigned)p.kv.rows), 128, 0, st>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_attend_acc(const TreeParams &p, int num_sms, cudaStream_t st) {
  return launch_stream(p, true, num_sms, st);
}

}  // namespace fgm

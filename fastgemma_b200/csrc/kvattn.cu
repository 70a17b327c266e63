// Attention of several tokens per sequence over the int8 KV cache and the
// weights it accumulates per slot.
//
// R = T * G query rows share one KV head's K and V (T nodes, G query heads
// per KV head).  Per row: s = (q8 . k8) * qs * ks over the visible slots,
// p = exp(s - max), out = sum p vs v8 / sum p.
#include <algorithm>

#include <cuda_fp16.h>

#include "fgm_common.cuh"
#include "fgm_internal.h"
#include "kv_attn.cuh"

namespace fgm {
namespace {

using namespace kv;

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

// The same into fresh registers: D = A * B.
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                            uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 "
      "{%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}

// (a, b) += (c, d): the packed form of the FP32 pipe.
__device__ __forceinline__ void add_pair(float &a, float &b, float c, float d) {
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(a), "+f"(b)
      : "f"(c), "f"(d));
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
// |vs|), 22 bits in all, so the products lose less than f32 rounding does.  The
// tensor cores round a sum towards zero, which adds up over a long run (a warp's
// 512 steps over 64K slots: 1e-5 of the output's norm), so a step's product starts
// from zero, its small part first, and is added to the output by rounding to nearest
// (1.8e-6; at 16K slots of head_dim 64 0.5e-6 against 1.5e-6; with equal weights
// and positive values a mean error of 3e-8 instead of 5e-5).  That costs 1 to 2 %
// where reading bounds the call, 6 % at head_dim 512, 8 % with 16 rows of 256 and
// 19 % at 320 (8 sequences of 16K slots; 16 of 20K).
//
// 8 sequences of up to 32K slots, 8 heads over 2 of head_dim 256: 51 us for
// 212 MB (4.1 TB/s over the launch, 6 to 7 while the rings run; 36 % of the
// issue slots, 18 % of the tensor cycles): 6 us before the first stage has
// landed, up to 6 % longer runs on some CTAs, 3 to 5 for a join.  Two CTAs an
// SM with rings of half the length took 54.  Short calls are latency: 4 nodes
// over 96 slots 10.1 us.
constexpr int kTile = 128;   // slots per tile of the work list
constexpr int kStep = 16;    // slots per warp step
// Tiles of an item that one CTA takes alone: another tile there against the
// join of two CTAs, measured at two tiles 9.2 against 9.9 us (4 rows, head_dim
// 256) and 12.8 against 16.3 (16 rows), at four 11.9 against 10.0 and 16.4
// against 15.8; at four of head_dim 64 8.0 against 8.6 and 10.8 against 11.0.
__host__ __device__ constexpr int whole_tiles(int hd) { return hd <= 128 ? 4 : 2; }

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

struct StreamParams {
  TreeParams t;
  Parts parts;
  int blocks;       // row blocks per (sequence, KV head)
  float *scores;    // [rows][n_heads][score_ld], or null: no accumulation behind
  int score_ld;
};

template <int HD, int NT>
__global__ void __launch_bounds__(stream_warps(HD) * 32, 1)
    stream_kernel(const __grid_constant__ StreamParams sp) {
  constexpr int W = stream_warps(HD), S = stream_stages(HD), SB = stage_bytes(HD);
  constexpr int KLD = HD + 16, VLD = HD * 4 + 32, ROWS = 8 * NT, QLD = HD + 16;
  constexpr int OFF_V = 16 * KLD, OFF_KS = OFF_V + 4 * VLD, OFF_VS = OFF_KS + 64;
  constexpr int QV = (HD + 127) / 128, QPW = (ROWS + W - 1) / W;  // query rows per warp
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ float s_qs[ROWS], s_ml[W][ROWS], s_l[W][ROWS], s_M[ROWS], s_L[ROWS];
  __shared__ int s_node[ROWS], s_low[ROWS], s_e[W];
  const TreeParams &p = sp.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gid = lane >> 2, tig = lane & 3;
  const int kvd = p.kv.kv_heads * HD, G = p.n_heads / p.kv.kv_heads, R = p.T * G;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint8_t *q8 = sm + W * S * SB;
  Work wk;
  if (!find_work(p, kTile, p.kv.kv_heads * sp.blocks, whole_tiles(HD), lane, wk)) return;
  const int b = wk.b, kvh = wk.in_b / sp.blocks, row0 = (wk.in_b - kvh * sp.blocks) * ROWS;
  const int len = wk.span.len, ring = p.kv.ring, end = len + p.T;
  const int x0 = wk.span.first + wk.t0 * kTile, x1 = min(wk.span.end, wk.span.first + wk.t1 * kTile);

  // the block's queries on their way before the ring fills behind them
  float4 qv[QPW][QV];
  int pos[QPW];
#pragma unroll
  for (int u = 0; u < QPW; u++) {
    const int r = row0 + warp + u * W;
    const bool on = warp + u * W < ROWS && r < R;
    const int node = on ? r / G : 0;
    const float4 *src = reinterpret_cast<const float4 *>(
        p.q + ((size_t)b * p.T + node) * p.q_ld + (size_t)(kvh * G + (on ? r - node * G : 0)) * HD);
#pragma unroll
    for (int i = 0; i < QV; i++)
      qv[u][i] = on && lane + 32 * i < HD / 4 ? src[lane + 32 * i] : make_float4(0, 0, 0, 0);
    pos[u] = p.pos ? p.pos[b * p.T + node] : len + node;
  }
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

  // queries to int8, a row per warp
#pragma unroll
  for (int u = 0; u < QPW; u++) {
    const int j = warp + u * W, r = row0 + j;
    if (j >= ROWS) break;
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < QV; i++)
      top = fmaxf(fmaxf(top, fmaxf(q_abs(qv[u][i].x), q_abs(qv[u][i].y))),
                  fmaxf(q_abs(qv[u][i].z), q_abs(qv[u][i].w)));
    top = warp_max(top);
    const float inv = q_inv(top);
    uint32_t *dst = reinterpret_cast<uint32_t *>(q8 + j * QLD);
#pragma unroll
    for (int i = 0; i < QV; i++)
      if (lane + 32 * i < HD / 4)
        dst[lane + 32 * i] = (q_int8(qv[u][i].x, inv) & 255) | (q_int8(qv[u][i].y, inv) & 255) << 8 |
                             (q_int8(qv[u][i].z, inv) & 255) << 16 | q_int8(qv[u][i].w, inv) << 24;
    if (lane == 0) {
      s_node[j] = r < R ? r / G : -1;
      s_low[j] = r < R ? lowest(pos[u], p.window) : INT_MIN;
      s_qs[j] = q_scale(top);
    }
  }
  __syncthreads();
  // slots from here to the committed ones' end are seen by every row
  const int high = __reduce_max_sync(0xffffffffu, s_low[lane % ROWS]);

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
    int32_t d[NT][2][4];  // two chains, summed below
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int e = 0; e < 4; e++) d[n][0][e] = d[n][1][e] = 0;
#pragma unroll
    for (int k = 0; k < HD / 32; k++) {
      uint32_t a[4];
      ldsm4(sta + ls * KLD + k * 32 + (lane & 16), a);
#pragma unroll
      for (int n = 0; n < NT; n++)
        mma_s8_m16n8k32(d[n][k & 1], a[0], a[1], a[2], a[3], qf[n][k][0], qf[n][k][1]);
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
        s[n][e] = __fmul_rn(__fmul_rn((float)(d[n][0][e] + d[n][1][e]), qs[n][e & 1]), kq[e >> 1]);
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
      float t[2][NT][4];
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int n = 0; n < NT; n++)
          mma_f16_new(t[i][n], lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1], bl[n][0],
                      bl[n][1]);
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int n = 0; n < NT; n++)
          mma_f16(t[i][n], lo[2 * i], lo[2 * i + 1], hi[2 * i], hi[2 * i + 1], bh[n][0], bh[n][1]);
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int e = 0; e < 4; e += 2)
            add_pair(o[n][2 * j + i][e], o[n][2 * j + i][e + 1], t[i][n][e], t[i][n][e + 1]);
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
      for (int m = 0; m < HD / 16; m += 2)
        *reinterpret_cast<float4 *>(red + (warp * ROWS + row) * RLD + m * 16 + gid * 4) =
            make_float4(o[n][m][c] * f, o[n][m][2 + c] * f, o[n][m + 1][c] * f,
                        o[n][m + 1][2 + c] * f);
    }
  if (tid < ROWS) {
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < W; w++) M = fmaxf(M, s_ml[w][tid]);
#pragma unroll
    for (int w = 0; w < W; w++)
      L += s_l[w][tid] * ex2(s_ml[w][tid] - (M == -INFINITY ? 0.0f : M));
    s_M[tid] = M;
    s_L[tid] = L;
  }
  __syncthreads();
  const float back = pow2(e_all) * 0.0001220703125f;  // 2^-13
  const int rows = min(ROWS, R - row0);
  const bool whole = wk.count == 1 && !sp.scores;  // with scores the next kernel joins
  for (int i = tid; i < rows * (HD / 4); i += W * 32) {
    const int row = i / (HD / 4), d = (i - row * (HD / 4)) * 4;
    float4 a = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < W; w++) {
      const float4 v = *reinterpret_cast<const float4 *>(red + (w * ROWS + row) * RLD + d);
      a.x += v.x, a.y += v.y, a.z += v.z, a.w += v.w;
    }
    a.x *= back, a.y *= back, a.z *= back, a.w *= back;
    if (whole) {
      store_row4(p, wk, kvh, row0 + row, d, a, s_M[row], s_L[row]);
    } else {
      *reinterpret_cast<float4 *>(sp.parts.part + ((size_t)blockIdx.x * ROWS + row) * HD + d) = a;
      if (d == 0) sp.parts.stat[(size_t)blockIdx.x * ROWS + row] = make_float2(s_M[row], s_L[row]);
    }
  }
  if (wk.count > 1 && !sp.scores) join_parts(p, sp.parts, wk, kvh, row0, rows, ROWS, red);
}

// The second half of a decode step (T = 1), launched under the attention: a
// sequence's first CTAs add the weights of the stored scores to its slots, four
// slots a thread, the others join the outputs of its items.  The
// weights need every head's log-sum, which no CTA of the attention has before
// its end, so each CTA takes it from the parts' statistics: the attention ends
// without a join of its own (51.0 us for 8 sequences of up to 32K slots, 9.0 for
// one of 1000; with that join 52.8 and 12.0).  Reads back 4 bytes a head and slot, from L2.
constexpr int kAdd = 256;
__global__ void __launch_bounds__(kAdd) finish_decode_kernel(const __grid_constant__ StreamParams sp,
                                                             int grid, int rows, int adds) {
  __shared__ float s_z[128 * 16];  // log2 of the sum of exp(score), by head
  const TreeParams &p = sp.t;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.y;
  const int hd = p.kv.head_dim, G = p.n_heads / p.kv.kv_heads, H = p.n_heads;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  // lens and acc come from before the attention, which writes neither
  const int x = (blockIdx.x * kAdd + tid) * 4, len = committed(p.kv, p.lens, b, 1);
  if ((int)blockIdx.x < adds && (int)blockIdx.x * kAdd * 4 > len) return;
  Work wk;
  find_work(p, kTile, p.kv.kv_heads * sp.blocks, whole_tiles(hd), lane, wk, grid, 0, b);
  // a head's statistics: of part i at + i * rows
  auto stat_of = [&](int h) {
    const int kvh = quick_div(h, G), r = h - kvh * G, blk = quick_div(r, rows);
    return (size_t)(wk.first + (kvh * sp.blocks + blk) * wk.count) * rows + (r - blk * rows);
  };
  if ((int)blockIdx.x >= adds) {  // ---- outputs
    const int hd4 = hd / 4, per = kAdd / hd4, in = tid / hd4, d = tid - in * hd4;
    const int h = ((int)blockIdx.x - adds) * per + in;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (in >= per || h >= H) return;
    const size_t at = stat_of(h);
    const float4 *part = reinterpret_cast<const float4 *>(sp.parts.part) + at * hd4 + d;
    const Joined j = join_row4(sp.parts.stat + at, part, rows, (size_t)rows * hd4, wk.count);
    reinterpret_cast<float4 *>(p.out + (size_t)b * p.out_ld + (size_t)h * hd)[d] = j.a;
    return;
  }
  float *acc = p.kv.acc + (size_t)b * p.kv.acc_stride + x;
  float old[4];
#pragma unroll
  for (int k = 0; k < 4; k++) old[k] = x + k < len ? p.decay * acc[k] : 0.0f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const float *s = sp.scores + (size_t)b * H * sp.score_ld + x;
  constexpr int kHeads = 8;  // whose scores are on their way together
  float4 v[kHeads];
  auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kHeads; i++)
      if (x <= len && h0 + i < H)
        v[i] = *reinterpret_cast<const float4 *>(s + (size_t)(h0 + i) * sp.score_ld);
  };
  load(0);
  for (int h = warp; h < H; h += kAdd / 32) {
    const float2 *stat = sp.parts.stat + stat_of(h);
    float M = -INFINITY, L = 0.0f;
    for (int i0 = 0; i0 < wk.count; i0 += 32) {
      const float2 w = i0 + lane < wk.count ? stat[(size_t)(i0 + lane) * rows]
                                            : make_float2(-INFINITY, 0.0f);
      const float N = fmaxf(M, warp_max(w.x)), ref = N == -INFINITY ? 0.0f : N;
      L = L * ex2(M - ref) + w.y * ex2(w.x - ref);
      M = N;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    if (lane == 0) s_z[h] = M + log2f(L);  // never empty: a token sees itself
  }
  __syncthreads();
  float sum[4] = {};
  for (int h0 = 0; h0 < H; h0 += kHeads) {
    if (h0 > 0) load(h0);
#pragma unroll
    for (int i = 0; i < kHeads; i++)
      if (h0 + i < H) {
        const float z = s_z[h0 + i];
        sum[0] += ex2(__fmaf_rn(v[i].x, kLog2e, -z));
        sum[1] += ex2(__fmaf_rn(v[i].y, kLog2e, -z));
        sum[2] += ex2(__fmaf_rn(v[i].z, kLog2e, -z));
        sum[3] += ex2(__fmaf_rn(v[i].w, kLog2e, -z));
      }
  }
#pragma unroll
  for (int k = 0; k < 4; k++)
    if (x + k <= len) acc[k] = old[k] + sum[k];
}

// ------------------------------------------------------------------ launching
// Row blocks of 8 * nt rows: one block of 16 where the accumulators of 16
// rows fit the registers (head_dim <= 256), else blocks of 8.
void stream_blocks(const fgm_cuda_kv &kv, int n_heads, int T, int &nt, int &blocks) {
  const int R = T * (n_heads / kv.kv_heads);
  nt = R > 8 && kv.head_dim <= 256 ? 2 : 1;
  blocks = (R + 8 * nt - 1) / (8 * nt);
}

struct Ws {
  size_t counters, part, stat, scores, total;
  int score_ld;
};
Ws ws_of(const fgm_cuda_kv &kv, int n_heads, int T) {
  int nt, blocks;
  stream_blocks(kv, n_heads, T, nt, blocks);
  const long long items = (long long)kv.rows * kv.kv_heads * blocks;
  const size_t grid = (size_t)max_grid(kv, items, kTile);
  Ws w;
  w.counters = 0;
  w.part = kCounters * sizeof(int);
  w.stat = w.part + align256(grid * 8 * nt * kv.head_dim * sizeof(float));
  w.scores = w.stat + align256(grid * 8 * nt * sizeof(float2));
  w.score_ld = (kv.cap + 31) & ~31;
  w.total = w.scores +
            (T == 1 ? align256((size_t)kv.rows * n_heads * w.score_ld * sizeof(float)) : 0);
  return w;
}

template <int HD, int NT>
cudaError_t launch_stream_as(const StreamParams &sp, int grid, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(stream_kernel<HD, NT>, stream_smem(HD), done);
  if (e != cudaSuccess) return e;
  stream_kernel<HD, NT><<<grid, stream_warps(HD) * 32, stream_smem(HD), st>>>(sp);
  return cudaGetLastError();
}

cudaError_t launch_stream(const TreeParams &p, bool accumulate, int num_sms, cudaStream_t st) {
  int nt, blocks;
  stream_blocks(p.kv, p.n_heads, p.T, nt, blocks);
  const Ws w = ws_of(p.kv, p.n_heads, p.T);
  uint8_t *ws = static_cast<uint8_t *>(p.ws);
  StreamParams sp;
  sp.t = p;
  sp.blocks = blocks;
  const int grid = grid_of(p.kv, (long long)p.kv.rows * p.kv.kv_heads * blocks, kTile,
                           num_sms < kMaxSms ? num_sms : kMaxSms);
  sp.parts.part = reinterpret_cast<float *>(ws + w.part);
  sp.parts.stat = reinterpret_cast<float2 *>(ws + w.stat);
  sp.parts.counters = reinterpret_cast<int *>(ws + w.counters);
  sp.scores = accumulate ? reinterpret_cast<float *>(ws + w.scores) : nullptr;
  sp.score_ld = w.score_ld;
  cudaError_t e = cudaErrorInvalidValue;
  switch (p.kv.head_dim * 2 + nt - 1) {
    case 128: e = launch_stream_as<64, 1>(sp, grid, st); break;
    case 129: e = launch_stream_as<64, 2>(sp, grid, st); break;
    case 256: e = launch_stream_as<128, 1>(sp, grid, st); break;
    case 257: e = launch_stream_as<128, 2>(sp, grid, st); break;
    case 384: e = launch_stream_as<192, 1>(sp, grid, st); break;
    case 385: e = launch_stream_as<192, 2>(sp, grid, st); break;
    case 512: e = launch_stream_as<256, 1>(sp, grid, st); break;
    case 513: e = launch_stream_as<256, 2>(sp, grid, st); break;
    case 640: e = launch_stream_as<320, 1>(sp, grid, st); break;
    case 768: e = launch_stream_as<384, 1>(sp, grid, st); break;
    case 896: e = launch_stream_as<448, 1>(sp, grid, st); break;
    case 1024: e = launch_stream_as<512, 1>(sp, grid, st); break;
  }
  if (e != cudaSuccess || !accumulate) return e;
  const int adds = (p.kv.cap + 4 * kAdd - 1) / (4 * kAdd), per = kAdd / (p.kv.head_dim / 4);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(adds + (p.n_heads + per - 1) / per), (unsigned)p.kv.rows);
  cfg.blockDim = dim3(kAdd);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, finish_decode_kernel, sp, grid, 8 * nt, adds);
}

}  // namespace

// The streaming kernel up to 16 query rows per KV head; beyond, the tensor
// tiles, except over caches so short that the row blocks of 16 fit the SMs at
// once and run their few slots through before a tile kernel's three launches
// would be done: at 230 slots of head_dim 256 and 64 rows for each of 8 sequences
// 13.1 against 17.9 us, at 990 slots 23.9 against 19.4; at 990 of head_dim 64 14.5
// against 17.4, at 4000 24.9 against 23.7.
//
// Up to 16 rows, streaming against tiles, two KV heads, 16K slots: 4 rows of
// head_dim 256 17.1 against 26.6 us for one sequence, 34.3 against 63.1 for
// eight; 16 rows of 64 17.2 against 25.4 and 24.8 against 47.1.  The number of rows
// alone is a coarse rule: at 16 rows of 256 the tiles are ahead for one sequence
// (27.3 against 31.7) and behind for eight (63.8 against 55.7), and from 1000 slots
// on they are ahead for one sequence of head_dim 320 and more from 8 rows on (512:
// 30.3 against 47.4) and for eight of 512 with 16 rows (118.8 against 141.1),
// where the stream runs four warps and reads the cache once per 8 rows.
bool streams(const TreeParams &p) {
  const int R = p.T * (p.n_heads / p.kv.kv_heads);
  if (R <= 16) return true;
  long long slots = p.kv.ring ? p.kv.ring : p.kv.cap;
  if (p.window) slots = std::min(slots, (long long)p.window + p.T + 16);
  int nt, blocks;
  stream_blocks(p.kv, p.n_heads, p.T, nt, blocks);
  return slots <= (p.kv.head_dim <= 128 ? 1024 : 256) &&
         (long long)p.kv.rows * p.kv.kv_heads * blocks <= 144;
}

size_t attend_workspace(const fgm_cuda_kv &kv, int n_heads, int T) {
  const size_t n = std::max(ws_of(kv, n_heads, T).total, attend_tile_workspace(kv, n_heads, T));
  return std::max(n, accum_workspace(kv, n_heads, T));
}

cudaError_t launch_attend_tree(const TreeParams &p, int num_sms, int *err, int *launches,
                               cudaStream_t st) {
  const bool tiles = !streams(p);
  const cudaError_t e = tiles ? launch_attend_tile(p, num_sms, err, st)
                              : launch_stream(p, false, num_sms, st);
  if (e == cudaSuccess) *launches = tiles ? 3 : 1;
  return e;
}

cudaError_t launch_attend_acc(const TreeParams &p, int num_sms, cudaStream_t st) {
  return launch_stream(p, true, num_sms, st);
}

}  // namespace fgm

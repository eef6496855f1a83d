// Attention of the newest tokens of every sequence over the paged KV cache:
// one token (plain decoding), a chain, or a tree of drafted tokens.
//
// Sequence b has seq_lens[b] keys; the last n_b = row_start[b+1] - row_start[b]
// of them are its query rows' own ("nodes", node i at key len - n + i).  Every
// node sees all earlier keys (the context) and, among the nodes, those its
// 64-bit mask names (no masks: itself and the nodes before it).
//
// Cache: [L, NB, Hkv, 16, D] bf16, or e4m3 codes with one fp32 scale for each
// (token, kv head) of K and of V, [L, NB, Hkv, 16].  With scales
//
//   t_j = (q . kc_j) ks_j scale log2(e) + log2 vs_j,     M = max_j t_j
//   w_j = 2^(t_j - M),   out = sum_j w_j vc_j / sum_j (w_j / vs_j)
//
// so that the weights of the value codes stay in [0, 1] whatever the scales
// are, for one exponential a score.  Scores are 8-bit products: the codes of K as
// they are and q as two e4m3 numbers, q = hi + lo, scaled by a power of two of its
// own for every row: exact down to 2^-9 of the row's largest value, and to 2^-18 of
// it below that.  The codes of V are exact in fp16, and the weights are held as
// 2^8 w in fp16 (11 bits; w / vs summed over 2^19 keys stays finite down to the
// smallest scale, 2^-100).  With the bf16 cache the weights are
// rounded to bf16, as its values are.  Sums and statistics are fp32.
//
// Work split: the keys of all (sequence, kv head, row tile) jobs form one line
// of 16-token blocks that is cut into equal pieces, one for each CTA, so a
// batch of uneven contexts keeps every SM busy to the end.  Lengths are read
// on the device: a captured graph stays right when they change.  A job cut by
// piece ends is joined by the last CTA that finishes a part of it, in the order
// of the parts (the result does not depend on which CTA that is).
//
// Up to 16 query rows of a kv head and sequence run here, on warp-level products
// fed from registers; more run on the tile kernel (attn_tree_tiles.cu).
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>

#include "attn_tree.cuh"
#include "common.cuh"
#include "host_utils.h"

namespace cb {
namespace tree {

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr float kUp = 8.f;  // fp16 weights are held as 2^kUp w

// Transpose of an 8 x 8 matrix of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// One warp's view of one 16-token block: K and V as loaded, and the scales.
template <int D, bool FP8>
struct Block {
  static constexpr int KC = FP8 ? D / 64 : D / 32;  // 16-byte K chunks of a lane and token
  static constexpr int VW = FP8 ? D / 32 : D / 16;  // V words of a lane and token
  uint4 k[2][KC];
  uint32_t v[4][VW];
  float ks[2], vs[2];

  // Tokens of lane (g, t4): K rows g and 8 + g (their scales too); V rows
  // 2 t4, 2 t4 + 1 and those plus 8.  A lane's K chunk c holds the head dims of
  // its k-steps (any order of the summed dims will do, if q has the same), its
  // V words the D / 8 dims from g D / 8 on.
  __device__ __forceinline__ void load(const Args& a, int page, int h, int g, int t4) {
    const int64_t row = ((a.layer_blocks + page) * a.Hkv + h) * 16;
    constexpr int RB = FP8 ? D : 2 * D;  // bytes of a row
    const uint8_t* kp = a.k + row * RB;
    const uint8_t* vp = a.v + row * RB;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < KC; ++c) k[i][c] = ldg_stream16(kp + (8 * i + g) * RB + c * 64 + t4 * 16);
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = __ldg(a.ks + row + 8 * i + g);
        vs[i] = __ldg(a.vs + row + 8 * i + g);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* p = vp + (8 * (i >> 1) + 2 * t4 + (i & 1)) * RB + g * (RB / 8);
      if constexpr (VW == 2) {
        const uint2 u = ldg_stream8(p);
        v[i][0] = u.x;
        v[i][1] = u.y;
      } else {
#pragma unroll
        for (int w = 0; w < VW / 4; ++w) {
          const uint4 u = ldg_stream16(p + 16 * w);
          v[i][4 * w] = u.x;
          v[i][4 * w + 1] = u.y;
          v[i][4 * w + 2] = u.z;
          v[i][4 * w + 3] = u.w;
        }
      }
    }
  }
};

// What a warp carries through a job's keys for NR x 8 query rows.  Products are
// taken transposed, S^T = K q^T and O^T = V^T P^T, so that the keys fill the 16
// rows of the warp-level product and the query rows its 8 columns: a single
// token's group of up to 8 heads wastes nothing.
template <int D, bool FP8, int NR>
struct Warp {
  static constexpr int NKS = D / 16;
  static constexpr int NT = D / 8;
  uint32_t q[NR][NKS][2];
  float row_scale[NR][2];
  int node[NR][2];  // of score columns 2 t4, 2 t4 + 1
  float o[NR][NT / 2][4];
  float m[NR][2], l[NR][2];

  __device__ __forceinline__ bool sees(const Args& a, int n, int e, int j, int q_row0) const {
    if (a.masks == nullptr) return j <= node[n][e];
    return j < 64 && (__ldg(a.masks + q_row0 + node[n][e]) >> (j & 63) & 1);
  }

  __device__ __forceinline__ void step(const Args& a, Block<D, FP8>& x, int blk, int page, int h,
                                       int len, int ctx, int q_row0, int g, int t4) {
    const int pos0 = blk * 16;
    float sc[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < Block<D, FP8>::KC; ++c) {
      const uint32_t w0[4] = {x.k[0][c].x, x.k[0][c].y, x.k[0][c].z, x.k[0][c].w};
      const uint32_t w1[4] = {x.k[1][c].x, x.k[1][c].y, x.k[1][c].z, x.k[1][c].w};
      if constexpr (FP8) {
        // The codes as they are, times the high and the low parts of q.
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t kf[4] = {w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1]};
#pragma unroll
          for (int n = 0; n < NR; ++n) {
            mma_e4m3(sc[n], kf, q[n][4 * c + 2 * i][0], q[n][4 * c + 2 * i + 1][0]);
            mma_e4m3(sc[n], kf, q[n][4 * c + 2 * i][1], q[n][4 * c + 2 * i + 1][1]);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t kf[4] = {w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1]};
#pragma unroll
          for (int n = 0; n < NR; ++n) mma_16816(sc[n], kf, q[n][2 * c + i][0], q[n][2 * c + i][1]);
        }
      }
    }
    // Scores in base 2 (tokens g and g + 8 x rows 2 t4 and 2 t4 + 1).
    float inv_vs[2] = {1.f, 1.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float kk = 1.f, lv = 0.f;
      if constexpr (FP8) {
        kk = x.ks[i];
        lv = __log2f(x.vs[i]);
        inv_vs[i] = ex2(-lv);
      }
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sc[n][2 * i + e] = FP8 ? fmaf(sc[n][2 * i + e], kk * row_scale[n][e], lv)
                                 : sc[n][2 * i + e] * row_scale[n][e];
    }
    const bool tail = pos0 + 16 > ctx;
    if (tail) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int pos = pos0 + 8 * i + g;
        // A NaN scale of a key that some rows do not see stays out of their sums.
        if (pos >= len) inv_vs[i] = 0.f;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (pos >= len || (pos >= ctx && !sees(a, n, e, pos - ctx, q_row0)))
              sc[n][2 * i + e] = -INFINITY;
      }
      // Value rows past the end may hold anything: a weight of zero does not
      // remove a NaN from a product.
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (pos0 + 8 * (i >> 1) + 2 * t4 + (i & 1) >= len) {
#pragma unroll
          for (int w = 0; w < Block<D, FP8>::VW; ++w) x.v[i][w] = 0u;
        }
      if constexpr (!FP8) take_out_infinities(a, x, pos0, page, h, len, ctx, q_row0, g, t4);
    }
    uint32_t pf[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float p[4];
      float alpha[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(sc[n][e], sc[n][2 + e]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float m_new = fmaxf(m[n][e], mx);
        alpha[e] = ex2(m[n][e] - m_new);
        const float base = FP8 ? m_new - kUp : m_new;
        m[n][e] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float w = ex2(sc[n][2 * i + e] - base);
          p[2 * i + e] = w;
          // (a hidden key's weight is 0: its scale, which may be a NaN, must
          // not turn that into one)
          if constexpr (FP8) sum += tail && w == 0.f ? 0.f : w * inv_vs[i];
          else sum += w;
        }
        l[n][e] = fmaf(l[n][e], alpha[e], sum);
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) {
          o[n][i][0] *= alpha[0];
          o[n][i][1] *= alpha[1];
          o[n][i][2] *= alpha[0];
          o[n][i][3] *= alpha[1];
        }
      }
      // Weights as the second operand: token pairs of one row a register.
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pf[n][i] = transpose8(FP8 ? pack_f16(p[2 * i], p[2 * i + 1])
                                  : pack_bf16(p[2 * i], p[2 * i + 1]));
    }
#pragma unroll
    for (int w = 0; w < Block<D, FP8>::VW; ++w) {
      if constexpr (FP8) {
        // Bytes of two tokens side by side, two dims a word.
        uint32_t v0[4], v1[4];
        e4m3_to_f16(__byte_perm(x.v[0][w], x.v[1][w], 0x5410), v0[0], v0[1]);
        e4m3_to_f16(__byte_perm(x.v[2][w], x.v[3][w], 0x5410), v0[2], v0[3]);
        e4m3_to_f16(__byte_perm(x.v[0][w], x.v[1][w], 0x7632), v1[0], v1[1]);
        e4m3_to_f16(__byte_perm(x.v[2][w], x.v[3][w], 0x7632), v1[2], v1[3]);
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          mma_f16(o[n][2 * w], v0, pf[n][0], pf[n][1]);
          mma_f16(o[n][2 * w + 1], v1, pf[n][0], pf[n][1]);
        }
      } else {
        const uint32_t vf[4] = {__byte_perm(x.v[0][w], x.v[1][w], 0x5410),
                                __byte_perm(x.v[0][w], x.v[1][w], 0x7632),
                                __byte_perm(x.v[2][w], x.v[3][w], 0x5410),
                                __byte_perm(x.v[2][w], x.v[3][w], 0x7632)};
#pragma unroll
        for (int n = 0; n < NR; ++n) mma_16816(o[n][w], vf, pf[n][0], pf[n][1]);
      }
    }
  }

  // A node may hold an infinity or a NaN that its siblings do not see: such
  // values leave the product and are added to the rows that do.
  __device__ __forceinline__ void take_out_infinities(const Args& a, Block<D, FP8>& x, int pos0,
                                                      int page, int h, int len, int ctx,
                                                      int q_row0, int g, int t4) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < Block<D, FP8>::VW; ++w) {
        uint32_t y = x.v[i][w];
        if ((y & 0x7f80u) == 0x7f80u) { y &= 0xffff0000u; bad = true; }
        if ((y & 0x7f800000u) == 0x7f800000u) { y &= 0xffffu; bad = true; }
        x.v[i][w] = y;
      }
    if (!__any_sync(0xffffffffu, bad)) return;
    const int64_t row = ((a.layer_blocks + page) * a.Hkv + h) * 16;
    const __nv_bfloat16* vp = reinterpret_cast<const __nv_bfloat16*>(a.v) + row * D;
    for (int tok = 0; tok < 16 && pos0 + tok < len; ++tok) {
      const int j = pos0 + tok - ctx;
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (j >= 0 && !sees(a, n, e, j, q_row0)) continue;
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const float val = __bfloat162float(vp[tok * D + g * NT + i]);
            if (!(fabsf(val) <= 3.4e38f)) o[n][i / 2][2 * (i & 1) + e] += val;
          }
        }
    }
  }
};

// 4 warps; each takes every fourth block of a job's keys for all rows of the
// job's tile and streams K and V from global memory straight into the operand
// registers of its warp-level products (a row of 128 B is one whole line, and
// no byte is used by two warps, so shared memory would only add a copy).  The
// next block is in flight while one is worked on.
template <int D, bool FP8, int NR>
__global__ void __launch_bounds__(128, NR == 1 && FP8 ? 3 : 2) attn_rows_kernel(const Args a) {
  constexpr int ROWS = 8 * NR;
  constexpr int NKS = D / 16;
  constexpr int NT = D / 8;
  constexpr int LD = D + 4;  // row pitch of the joined sums in shared memory
  extern __shared__ __align__(16) uint8_t smem_raw[];
  int64_t* pre = reinterpret_cast<int64_t*>(smem_raw);
  float* sm_o = reinterpret_cast<float*>(smem_raw + ((a.B + 2) / 2 * 2) * 8);  // [4][ROWS][LD]
  float* sm_ml = sm_o + 4 * ROWS * LD;                                        // [4][ROWS][2]
  __shared__ int64_t s_sum[4];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  grid_dep_launch();
  grid_dep_wait();

  scan_work<16, 128>(a, ROWS, pre, s_sum);
  const int64_t total = pre[a.B];
  // At least 8 blocks a piece: two for each warp.
  const int64_t piece = max((int64_t)8, (total + gridDim.x - 1) / gridDim.x);
  int64_t u = (int64_t)blockIdx.x * piece;
  const int64_t u_end = min(total, u + piece);

  while (u < u_end) {
    const int b = find_seq(pre, a.B, u);
    const SeqShape s = seq_shape<16>(a, b, ROWS);
    const int64_t local = u - pre[b];
    const int job = (int)(local / s.nb);
    const int k0 = (int)(local - (int64_t)job * s.nb);
    const int k1 = (int)min((int64_t)s.nb, k0 + (u_end - u));
    const int h = job / s.tiles, tile = job - h * s.tiles;
    const int ctx = s.len - s.n;
    const int* table = a.table + (int64_t)b * a.table_stride;
    const int q_row0 = a.row_start[b];
    const int rows_left = s.n * a.G - tile * ROWS;

    const int blk_end = min(k1, (s.len + 15) >> 4);
    const int first = k0 + warp;
    // Pages of this warp's blocks, 32 at a time, one in each lane.
    int pages = first + 4 * lane < blk_end ? __ldg(table + first + 4 * lane) : 0;
    Block<D, FP8> x[2];
    if (first < blk_end) x[0].load(a, __shfl_sync(0xffffffffu, pages, 0), h, g, t4);

    Warp<D, FP8, NR> w;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      // Row 8 n + g as the second operand: dims in the K chunks' order (8-bit: the
      // four of a k-step's first 16-bit pair and second in one word).
      const int r = 8 * n + g;
      const bool live = r < rows_left;
      const int rr = tile * ROWS + (live ? r : 0);
      const __nv_bfloat16* qp = a.q + (int64_t)(q_row0 + rr / a.G) * a.q_stride +
                                (int64_t)(h * a.G + rr % a.G) * D;
      uint32_t top = 0;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const int d = FP8 ? (ks >> 2) * 64 + t4 * 16 + (ks & 3) * 4
                          : (ks >> 1) * 32 + t4 * 8 + (ks & 1) * 4;
        const uint2 y = live ? *reinterpret_cast<const uint2*>(qp + d) : make_uint2(0u, 0u);
        w.q[n][ks][0] = y.x;
        w.q[n][ks][1] = y.y;
        if constexpr (FP8) {
          top = max(top, max(y.x & 0x7fffu, (y.x >> 16) & 0x7fffu));
          top = max(top, max(y.y & 0x7fffu, (y.y >> 16) & 0x7fffu));
        }
      }
      float back = a.scale_log2;
      if constexpr (FP8) {
        // Four dims as e4m3, a high and a low part.
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const QScale qs = q_scale(top);
        back *= qs.down;
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks)
          split_e4m3(w.q[n][ks][0], w.q[n][ks][1], qs.up, w.q[n][ks][0], w.q[n][ks][1]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        w.row_scale[n][e] = __shfl_sync(0xffffffffu, back, (2 * t4 + e) * 4);
        const int c = 8 * n + 2 * t4 + e;
        w.node[n][e] = (tile * ROWS + (c < rows_left ? c : 0)) / a.G;
        w.m[n][e] = kNegBig;
        w.l[n][e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < NT / 2; ++i)
        w.o[n][i][0] = w.o[n][i][1] = w.o[n][i][2] = w.o[n][i][3] = 0.f;
    }

    int idx = 0;
    for (int blk = first; blk < blk_end; blk += 8) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int cur = blk + 4 * half;
        if (cur >= blk_end) break;
        const int page = __shfl_sync(0xffffffffu, pages, idx & 31);
        if (((idx + 1) & 31) == 0)
          pages = cur + 4 + 4 * lane < blk_end ? __ldg(table + cur + 4 + 4 * lane) : 0;
        ++idx;
        if (cur + 4 < blk_end)
          x[half ^ 1].load(a, __shfl_sync(0xffffffffu, pages, idx & 31), h, g, t4);
        w.step(a, x[half], cur, page, h, s.len, ctx, q_row0, g, t4);
      }
    }

    // Join the four warps, then the CTAs that share the job.
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1)
          w.l[n][e] += __shfl_xor_sync(0xffffffffu, w.l[n][e], o);
        const int row = 8 * n + 2 * t4 + e;
        if (row < rows_left) {
          float* dst = sm_o + (warp * ROWS + row) * LD + g * NT;
#pragma unroll
          for (int i = 0; i < NT / 2; i += 2)
            *reinterpret_cast<float4*>(dst + 2 * i) =
                make_float4(w.o[n][i][e], w.o[n][i][2 + e], w.o[n][i + 1][e], w.o[n][i + 1][2 + e]);
          if (g == 0) {
            sm_ml[(warp * ROWS + row) * 2] = w.m[n][e];
            sm_ml[(warp * ROWS + row) * 2 + 1] = w.l[n][e];
          }
        }
      }
    __syncthreads();
    const int64_t js = pre[b] + (int64_t)job * s.nb;
    const int64_t c0 = js / piece, c1 = (js + s.nb - 1) / piece;
    const int rows = min(ROWS, rows_left);
    const bool whole = c0 == c1;
    float* part = a.part + ((int64_t)blockIdx.x * 2 + (blockIdx.x == c0 ? 1 : 0)) * ROWS * (D + 2);
    for (int i = tid; i < rows * D; i += 128) {
      const int row = i / D, d = i % D;
      float M = kNegBig;
#pragma unroll
      for (int k = 0; k < 4; ++k) M = fmaxf(M, sm_ml[(k * ROWS + row) * 2]);
      float L = 0.f, O = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = ex2(sm_ml[(k * ROWS + row) * 2] - M);
        L += sm_ml[(k * ROWS + row) * 2 + 1] * f;
        O += sm_o[(k * ROWS + row) * LD + d] * f;
      }
      if (whole) {
        const int rr = tile * ROWS + row;
        a.out[(int64_t)(q_row0 + rr / a.G) * a.out_stride + (int64_t)(h * a.G + rr % a.G) * D + d] =
            __float2bfloat16(L == 0.f ? 0.f : (FP8 ? 256.f * O : O) / L);
      } else {
        part[row * (D + 2) + 2 + d] = O;
        if (d == 0) {
          part[row * (D + 2)] = M;
          part[row * (D + 2) + 1] = L;
        }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        const int parts = (int)(c1 - c0 + 1);
        s_last = atomicAdd(a.counters + c0, 1) == parts - 1;
        if (s_last) a.counters[c0] = 0;
      }
      __syncthreads();
      if (s_last) {
        __threadfence();
        for (int i = tid; i < rows * D; i += 128) {
          const int row = i / D, d = i % D;
          float M = kNegBig, L = 0.f, O = 0.f;
          for (int64_t c = c0; c <= c1; ++c) {
            const float* src =
                a.part + (c * 2 + (c == c0 ? 1 : 0)) * ROWS * (D + 2) + row * (D + 2);
            const float m_c = __ldcg(src), l_c = __ldcg(src + 1), o_c = __ldcg(src + 2 + d);
            const float m_new = fmaxf(M, m_c);
            const float f0 = ex2(M - m_new), f1 = ex2(m_c - m_new);
            L = L * f0 + l_c * f1;
            O = O * f0 + o_c * f1;
            M = m_new;
          }
          const int rr = tile * ROWS + row;
          a.out[(int64_t)(q_row0 + rr / a.G) * a.out_stride + (int64_t)(h * a.G + rr % a.G) * D +
                d] = __float2bfloat16(L == 0.f ? 0.f : (FP8 ? 256.f * O : O) / L);
        }
      }
    }
    __syncthreads();  // shared buffers are reused by the next job
    u += k1 - k0;
  }
}

template <int D, bool FP8, int NR>
void launch_rows(const Args& a, int grid, cudaStream_t stream) {
  const int smem = (a.B + 2) / 2 * 2 * 8 + 4 * 8 * NR * (D + 6) * 4;
  static int configured = 0;
  if (smem > configured) {
    CB_CUDA_CHECK(cudaFuncSetAttribute(attn_rows_kernel<D, FP8, NR>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured = smem;
  }
  launch_kernel(attn_rows_kernel<D, FP8, NR>, dim3(grid), dim3(128), smem, stream, a);
}

// By the query rows of a kv head and sequence.
template <int D, bool FP8>
void launch(const Args& a, int64_t max_rows, cudaStream_t stream) {
  if (max_rows <= 8) launch_rows<D, FP8, 1>(a, (FP8 ? 3 : 2) * num_sms(), stream);
  else if (max_rows <= 16) launch_rows<D, FP8, 2>(a, 2 * num_sms(), stream);
  else launch_tiles<D, FP8>(a, stream);
}

}  // namespace tree

// {largest grid, workspace floats, workspace counters} of attn_tree.
std::vector<int64_t> attn_tree_plan(int64_t head_dim) {
  const int64_t sms = num_sms();
  return {3 * sms, sms * 2 * 256 * (head_dim + 2), 3 * sms};
}

// q, out: [rows, Hq * D]; rows of sequence b are row_start[b] .. row_start[b+1].
void attn_tree(at::Tensor q, at::Tensor k_cache, at::Tensor v_cache,
               c10::optional<at::Tensor> k_scale, c10::optional<at::Tensor> v_scale,
               at::Tensor block_tables, at::Tensor seq_lens, at::Tensor row_start,
               c10::optional<at::Tensor> masks, at::Tensor out, int64_t layer, double scale,
               int64_t max_nodes, at::Tensor ws, at::Tensor counters,
               at::Tensor status) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 2 && q.scalar_type() == at::kBFloat16 &&
                  out.dim() == 2 && out.scalar_type() == at::kBFloat16 && q.stride(1) == 1 &&
                  out.stride(1) == 1 && out.size(0) >= q.size(0) && out.size(1) == q.size(1),
              "q / out must be bf16 [rows, Hq * D] with inner stride 1");
  TORCH_CHECK(k_cache.dim() == 5 && k_cache.size(3) == 16 && k_cache.is_contiguous() &&
                  v_cache.is_contiguous() && v_cache.sizes() == k_cache.sizes() &&
                  v_cache.scalar_type() == k_cache.scalar_type(),
              "kv cache must be [L, NB, Hkv, 16, D] contiguous");
  const bool fp8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK(fp8 || k_cache.scalar_type() == at::kBFloat16,
              "kv cache must be bf16 or float8_e4m3fn");
  TORCH_CHECK(fp8 == k_scale.has_value() && fp8 == v_scale.has_value(),
              "the 8-bit cache comes with k_scale and v_scale, the bf16 cache without");
  const int D = (int)k_cache.size(4), Hkv = (int)k_cache.size(2);
  TORCH_CHECK(D == 64 || D == 128, "head_dim must be 64 or 128");
  TORCH_CHECK(q.size(1) % D == 0 && (q.size(1) / D) % Hkv == 0, "query heads must divide");
  TORCH_CHECK(layer >= 0 && layer < k_cache.size(0), "layer outside the cache");
  const int64_t B = seq_lens.numel();
  TORCH_CHECK(B <= tree::kMaxBatch, "at most 2048 sequences");
  TORCH_CHECK(block_tables.scalar_type() == at::kInt && block_tables.dim() == 2 &&
                  block_tables.size(0) >= B && block_tables.stride(1) == 1 &&
                  seq_lens.scalar_type() == at::kInt && seq_lens.is_contiguous() &&
                  row_start.scalar_type() == at::kInt && row_start.is_contiguous() &&
                  row_start.numel() >= B + 1,
              "int32 block tables [B, W], seq lens [B] and row starts [B + 1]");
  for (const at::Tensor* t :
       {&out, &k_cache, &v_cache, &block_tables, &seq_lens, &row_start, &ws, &counters})
    TORCH_CHECK(t->device() == q.device(), "all tensors must be on one device");
  if (fp8) {
    for (const at::Tensor* t : {&*k_scale, &*v_scale})
      TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() &&
                      t->numel() == k_cache.numel() / D && t->device() == q.device(),
                  "k/v scales must be fp32 [L, NB, Hkv, 16] contiguous");
  }
  if (masks.has_value())
    TORCH_CHECK(masks->scalar_type() == at::kLong && masks->is_contiguous() &&
                    masks->numel() >= q.size(0) && masks->device() == q.device(),
                "masks must be int64, one per row");
  TORCH_CHECK(max_nodes >= 1 && (!masks.has_value() || max_nodes <= 64),
              "a tree has at most 64 nodes");
  TORCH_CHECK((q.stride(0) * 2) % 16 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "q rows must be 16-byte aligned");
  if (B == 0 || q.size(0) == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  const std::vector<int64_t> plan = attn_tree_plan(D);
  TORCH_CHECK(ws.scalar_type() == at::kFloat && ws.numel() >= plan[1] &&
                  counters.scalar_type() == at::kInt && counters.numel() >= plan[2],
              "workspace too small");
  tree::Args a;
  a.q = reinterpret_cast<const __nv_bfloat16*>(q.data_ptr());
  a.q_stride = q.stride(0);
  a.k = reinterpret_cast<const uint8_t*>(k_cache.data_ptr());
  a.v = reinterpret_cast<const uint8_t*>(v_cache.data_ptr());
  a.ks = fp8 ? k_scale->data_ptr<float>() : nullptr;
  a.vs = fp8 ? v_scale->data_ptr<float>() : nullptr;
  a.table = block_tables.data_ptr<int>();
  a.table_stride = block_tables.stride(0);
  a.table_width = (int)block_tables.size(1);
  a.seq_lens = seq_lens.data_ptr<int>();
  a.row_start = row_start.data_ptr<int>();
  a.masks = masks.has_value() ? masks->data_ptr<int64_t>() : nullptr;
  a.out = reinterpret_cast<__nv_bfloat16*>(out.data_ptr());
  a.out_stride = out.stride(0);
  a.part = ws.data_ptr<float>();
  a.counters = counters.data_ptr<int>();
  a.status = status.data_ptr<int>();
  a.out_vec = (out.stride(0) * 2) % 16 == 0 && reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0;
  a.layer_blocks = layer * k_cache.size(1);
  a.B = (int)B;
  a.Hkv = Hkv;
  a.G = (int)(q.size(1) / D / Hkv);
  a.scale_log2 = (float)scale * tree::kLog2e;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const int64_t rows = max_nodes * a.G;
  if (D == 128) {
    if (fp8) tree::launch<128, true>(a, rows, stream);
    else tree::launch<128, false>(a, rows, stream);
  } else {
    if (fp8) tree::launch<64, true>(a, rows, stream);
    else tree::launch<64, false>(a, rows, stream);
  }
}

}  // namespace cb

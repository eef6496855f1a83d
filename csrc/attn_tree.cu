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
// it below that.  The codes of V are exact in fp16, and the weights are held in fp16
// too, times a power of two (11 bits down to 2^-27, the rest of them to within 2^-37),
// and summed as 2^6 w / vs, which stays finite for 2^19 keys (w up to 4, see kLag)
// down to the smallest scale, 2^-100.  (Weights as sums of 8-bit numbers would spare V's unpacking.  Two
// e4m3 parts lose all below 2^-18 of the largest: the many small weights beside one
// large one.  Four e5m2 parts hold them, but double the products of V: 150 us against
// 132 when tried.)  With the bf16 cache the weights are rounded to bf16, as
// its values are.  Sums and statistics are fp32.
//
// Work split: the keys of all (sequence, kv head, row tile) jobs form one line
// of 16-token blocks that is cut into equal pieces, one for each CTA, so a
// batch of uneven contexts keeps every SM busy to the end.  Lengths are read
// on the device: a captured graph stays right when they change.  A job cut by
// piece ends is joined by the last CTA that finishes a part of it, in the order
// of the parts (the result does not depend on which CTA that is).
//
// Up to 16 query rows of a kv head and sequence run here, on warp-level products;
// more run on the tile kernel (attn_tree_tiles.cu).
//
// Bound: memory, for long contexts.  64 sequences of 517 to 8191 keys, 8 kv heads of
// 128, 4 query heads each, 8-bit cache: 591 MB in 111 us, 5.3 TB/s.  (The products and
// the softmax alone take 84 us, the loads alone 89.)  One sequence of 1151 keys: 10 us,
// of which launch, scan of the lengths and joins of the pieces are most.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>

#include "attn_tree.cuh"
#include "common.cuh"
#include "host_utils.h"

namespace cb {
namespace tree {

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

constexpr float kLag = 2.f;   // scores may pass the maximum in use by a factor 2^kLag
constexpr float kUp = 13.f;   // fp16 weights are held as 2^kUp w: at most 2^(kUp + kLag)
constexpr float kSum = 6.f;   // and summed as 2^kSum w / vs
constexpr float kBack = 1.f / 128;  // 2^(kSum - kUp)

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Transpose of an 8 x 8 matrix of 16-bit values held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ float lds32(uint32_t p) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t p) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(p) : "memory");
  return v;
}
// One warp's view of one 16-token block: K and V words and the scales.
//
// Tokens of lane (g, t4): K rows g and 8 + g (their scales too); V rows 2 t4, 2 t4 + 1
// and those plus 8.  A lane's K chunk c holds the head dims of its k-steps (any
// order of the summed dims will do, if q has the same), its V words the D / 8 dims
// from g D / 8 on.
//
// Blocks pass through a ring of stages in shared memory, as they lie in the cache (a
// kv head's 16 rows of a page are one run of bytes, copied whole lines at a time)
// but for the order of the 16-byte pieces within a line, which spares the reads bank
// conflicts.  (Copies of just the bytes that each lane would use, 4 to 8 lines an
// instruction, took 134 us for the 591 MB of 64 contexts of up to 8191 keys, whole
// lines 89 us.)
template <int D, bool FP8>
struct Block {
  static constexpr int KC = FP8 ? D / 64 : D / 32;  // 16-byte K chunks of a lane and token
  static constexpr int VW = FP8 ? D / 32 : D / 16;  // V words of a lane and token
  static constexpr int RB = FP8 ? D : 2 * D;        // bytes of a row
  static constexpr int kStage = 32 * RB + (FP8 ? 128 : 0);
  uint4 k[2][KC];
  uint32_t v[4][VW];
  float ks[2], vs[2];

  // Where a 16-byte piece of a row lies among the eight of its 128-byte line, as an
  // exclusive or.  K is read by rows (g) and quarters (t4), V by row pairs (t4) and
  // eighths (g).
  __device__ static constexpr __forceinline__ int k_turn(int row) {
    return RB == 64 ? 0 : (row & 1) << 2;
  }
  __device__ static constexpr __forceinline__ int v_turn(int row) {
    return RB == 256 ? ((row >> 1) & 1) | (row & 4) : row & 6;
  }

  __device__ static __forceinline__ void copy(const Args& a, int page, int h, int lane,
                                              uint32_t stage) {
    const int64_t row = ((a.layer_blocks + page) * a.Hkv + h) * 16;
    const uint8_t* kp = a.k + row * RB + lane * 16;
    const uint8_t* vp = a.v + row * RB + lane * 16;
#pragma unroll
    for (int c = 0; c < RB / 32; ++c) {
      const int piece = c * 32 + lane, r = piece / (RB / 16);
      copy16(stage + (piece ^ k_turn(r)) * 16, kp + c * 512);
      copy16(stage + 16 * RB + (piece ^ v_turn(r)) * 16, vp + c * 512);
    }
    if constexpr (FP8) {
      if (lane < 8)
        copy16(stage + 32 * RB + lane * 16, (lane < 4 ? a.ks : a.vs - 16) + row + lane * 4);
    }
  }

  __device__ __forceinline__ void fetch_keys(int lane, uint32_t stage) {
    const int g = lane >> 2, t4 = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < KC; ++c)
        k[i][c] = lds128(stage + 8 * i * RB + ((g * (RB / 16) + 4 * c + t4) ^ k_turn(g)) * 16);
    if constexpr (FP8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ks[i] = lds32(stage + 32 * RB + (8 * i + g) * 4);
        vs[i] = lds32(stage + 32 * RB + 64 + (8 * i + g) * 4);
      }
    }
  }
  __device__ __forceinline__ void fetch_values(int lane, uint32_t stage) {
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t at = stage + 16 * RB;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 2 * t4 + (i & 1) + 8 * (i >> 1);
      if constexpr (VW == 2) {
        const uint2 u = lds64(at + ((r * 4 + (g >> 1)) ^ v_turn(r)) * 16 + (g & 1) * 8);
        v[i][0] = u.x;
        v[i][1] = u.y;
      } else {
#pragma unroll
        for (int w = 0; w < VW / 4; ++w) {
          const uint4 u = lds128(at + ((r * (RB / 16) + g * (VW / 4) + w) ^ v_turn(r)) * 16);
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

  // One block of keys, from its stage of the ring.
  __device__ __forceinline__ void step(const Args& a, uint32_t stage, int blk, const int* table,
                                       int h, int len, int ctx, int q_row0, int lane) {
    const int g = lane >> 2, t4 = lane & 3;
    Block<D, FP8> x;
    x.fetch_keys(lane, stage);
    float sc[NR][4];
#pragma unroll
    for (int n = 0; n < NR; ++n) sc[n][0] = sc[n][1] = sc[n][2] = sc[n][3] = 0.f;
    float sl[NR][4];  // a second chain, for the low parts
#pragma unroll
    for (int n = 0; n < NR; ++n) sl[n][0] = sl[n][1] = sl[n][2] = sl[n][3] = 0.f;
#pragma unroll
    for (int c = 0; c < Block<D, FP8>::KC; ++c) {
      const uint32_t w0[4] = {x.k[0][c].x, x.k[0][c].y, x.k[0][c].z, x.k[0][c].w};
      const uint32_t w1[4] = {x.k[1][c].x, x.k[1][c].y, x.k[1][c].z, x.k[1][c].w};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t kf[4] = {w0[2 * i], w1[2 * i], w0[2 * i + 1], w1[2 * i + 1]};
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          if constexpr (FP8) {
            // The codes as they are, times the high and the low parts of q.
            mma_e4m3(sc[n], kf, q[n][4 * c + 2 * i][0], q[n][4 * c + 2 * i + 1][0]);
            mma_e4m3(sl[n], kf, q[n][4 * c + 2 * i][1], q[n][4 * c + 2 * i + 1][1]);
          } else {
            mma_16816(sc[n], kf, q[n][2 * c + i][0], q[n][2 * c + i][1]);
          }
        }
      }
    }
    // Scores in base 2 (tokens g and g + 8 x rows 2 t4 and 2 t4 + 1).
    const int pos0 = blk * 16;
    float inv_vs[2] = {1.f, 1.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float kk = 1.f, lv = 0.f;
      if constexpr (FP8) {
        kk = x.ks[i];
        lv = lg2(x.vs[i]);
        if (lv < -126.f) lv = -126.f;  // a row never written, scale 0
        inv_vs[i] = ex2(kSum - kUp - lv);
      }
#pragma unroll
      for (int n = 0; n < NR; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          sc[n][2 * i + e] = FP8 ? fmaf(sc[n][2 * i + e] + sl[n][2 * i + e], kk * row_scale[n][e], lv)
                                 : sc[n][2 * i + e] * row_scale[n][e];
    }
    const bool tail = pos0 + 16 > ctx;
    if (tail) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int pos = pos0 + 8 * i + g;
        // A NaN scale stays out of the sums of rows that do not see the key; those
        // that do have it in their scores.
        if (!(inv_vs[i] < INFINITY)) inv_vs[i] = 0.f;
#pragma unroll
        for (int n = 0; n < NR; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (pos >= len || (pos >= ctx && !sees(a, n, e, pos - ctx, q_row0)))
              sc[n][2 * i + e] = -INFINITY;
      }
    }
    // The maximum in use lags: it moves only when a score passes it by 2^kLag.
    bool passed = false;
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) passed |= fmaxf(sc[n][e], sc[n][2 + e]) > m[n][e] + kLag;
    if (__any_sync(0xffffffffu, passed)) {
#pragma unroll
      for (int n = 0; n < NR; ++n) {
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float mx = fmaxf(sc[n][e], sc[n][2 + e]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          mx = fmaxf(m[n][e], mx);
          alpha[e] = ex2(m[n][e] - mx);
          m[n][e] = mx;
          l[n][e] *= alpha[e];
        }
#pragma unroll
        for (int i = 0; i < NT / 2; ++i) {
          o[n][i][0] *= alpha[0];
          o[n][i][1] *= alpha[1];
          o[n][i][2] *= alpha[0];
          o[n][i][3] *= alpha[1];
        }
      }
    }
    // Weights as the second operand: the tokens of a row side by side.
    uint32_t pf[NR][2];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float base = FP8 ? m[n][e] - kUp : m[n][e];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          p[2 * i + e] = ex2(sc[n][2 * i + e] - base);
          l[n][e] = FP8 ? fmaf(p[2 * i + e], inv_vs[i], l[n][e]) : l[n][e] + p[2 * i + e];
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pf[n][i] = transpose8(FP8 ? pack_f16(p[2 * i], p[2 * i + 1])
                                  : pack_bf16(p[2 * i], p[2 * i + 1]));
    }
    x.fetch_values(lane, stage);
    if (tail) {
      // Value rows past the end may hold anything: a weight of zero does not
      // remove a NaN from a product.
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (pos0 + 8 * (i >> 1) + 2 * t4 + (i & 1) >= len) {
#pragma unroll
          for (int w = 0; w < Block<D, FP8>::VW; ++w) x.v[i][w] = 0u;
        }
      if constexpr (!FP8) take_out_infinities(a, x, pos0, table, h, len, ctx, q_row0, g, t4);
    }
#pragma unroll
    for (int w = 0; w < Block<D, FP8>::VW; ++w) {
      if constexpr (FP8) {
        // Bytes of two tokens side by side, two dims a word.
        uint32_t v0[4], v1[4];
        codes_to_f16(__byte_perm(x.v[0][w], x.v[1][w], 0x5140), v0[0], v0[1]);
        codes_to_f16(__byte_perm(x.v[2][w], x.v[3][w], 0x5140), v0[2], v0[3]);
        codes_to_f16(__byte_perm(x.v[0][w], x.v[1][w], 0x7362), v1[0], v1[1]);
        codes_to_f16(__byte_perm(x.v[2][w], x.v[3][w], 0x7362), v1[2], v1[3]);
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
                                                      const int* table, int h, int len, int ctx,
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
    const int64_t row = ((a.layer_blocks + table[pos0 >> 4]) * a.Hkv + h) * 16;
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

// Four dims of a finished row.
template <int D, bool FP8>
__device__ __forceinline__ void put(const Args& a, int row0, int r, int h, int d,
                                    const float (&O)[4], float L) {
  __nv_bfloat16* dst =
      a.out + (int64_t)(row0 + r / a.G) * a.out_stride + (int64_t)(h * a.G + r % a.G) * D + d;
  float y[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) y[x] = L == 0.f ? 0.f : (FP8 ? kBack * O[x] : O[x]) / L;
  if (a.out_vec) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(y[0], y[1]), pack_bf16(y[2], y[3]));
  } else {
#pragma unroll
    for (int x = 0; x < 4; ++x) dst[x] = __float2bfloat16(y[x]);
  }
}

// Stages of a warp's ring, and CTAs of an SM: 64 KB and more of an SM's loads in
// flight, and registers for a block without spilling.
template <int D, bool FP8>
__host__ __device__ constexpr int ring_stages() {
  return D == 128 && !FP8 ? 2 : 3;
}
template <int D, bool FP8, int NR>
constexpr int rows_ctas() {
  return NR == 1 && (FP8 || D == 64) ? 3 : 2;
}

// Shared memory: the warps' rings, their sums at the end of a job, query rows of this
// job and the next, the sequences.
template <int D, bool FP8, int NR>
struct Smem {
  static constexpr int ROWS = 8 * NR;
  static constexpr int LD = D + 4;       // floats of a row of sums
  static constexpr int LQ = 2 * D + 16;  // bytes of a query row
  static constexpr int kSums = 4 * ring_stages<D, FP8>() * Block<D, FP8>::kStage;
  static constexpr int kStats = kSums + 4 * ROWS * LD * 4;  // maximum and sum of weights
  static constexpr int kQ = kStats + 4 * ROWS * 2 * 4;
  static constexpr int kSeqs = kQ + 2 * ROWS * LQ;
  static int bytes(int B) { return kSeqs + 2 * (B + 1) * 8; }
};

// Rows of a sequence and a run of its blocks.
struct Job {
  int b, tile, k0, k1, len, ctx, row0, rows;  // rows: of this tile and those after it
  int64_t start;                              // its first block's place in the line
  int blocks;
};

// 4 warps; each takes every fourth block of a job's keys for all rows of the job's
// tile.  While a job is computed, the next one's query rows and, at its end, first
// blocks are on their way; results of jobs that other CTAs share are joined at the
// very end: nothing but the first job waits for memory.
template <int D, bool FP8, int NR>
__global__ void __launch_bounds__(128, rows_ctas<D, FP8, NR>()) attn_rows_kernel(const Args a) {
  constexpr int ROWS = 8 * NR;
  constexpr int NKS = D / 16;
  constexpr int NT = D / 8;
  constexpr int ST = ring_stages<D, FP8>();
  using Blk = Block<D, FP8>;
  using Sm = Smem<D, FP8, NR>;
  constexpr int LD = Sm::LD;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  float* sm_o = reinterpret_cast<float*>(smem_raw + Sm::kSums);    // [4][ROWS][LD]
  float* sm_ml = reinterpret_cast<float*>(smem_raw + Sm::kStats);  // [4][ROWS][2]
  int64_t* pre = reinterpret_cast<int64_t*>(smem_raw + Sm::kSeqs);
  int2* seqs = reinterpret_cast<int2*>(pre + a.B + 1);
  __shared__ int64_t s_sum[4];
  __shared__ Job s_open[2];  // jobs shared with the pieces before and after
  __shared__ int s_parts[2], s_last[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;
  grid_dep_launch();
  grid_dep_wait();

  // A line of work for each kv head; CTAs side by side take the same piece of it for
  // all heads, so that the heads' rows of a block, which lie together, are read at
  // about the same time.
  if (tid < 2) s_parts[tid] = 0;
  scan_work<16, 128>(a, ROWS, 1, pre, s_sum, seqs);
  const int64_t total = pre[a.B];
  const int h = blockIdx.x % a.Hkv, cta = blockIdx.x / a.Hkv, ctas = gridDim.x / a.Hkv;
  // At least 8 blocks a piece: two for each warp.
  const int64_t piece = max((int64_t)8, divide(total + ctas - 1, ctas));
  int64_t u = (int64_t)cta * piece;
  const int64_t u_end = min(total, u + piece);
  if (u >= u_end) return;

  auto job_at = [&](int64_t at) {
    Job j;
    j.b = find_seq(pre, a.B, at);
    const int2 sq = seqs[j.b];
    const int n = max(0, seqs[j.b + 1].y - sq.y);
    j.len = sq.x;
    j.ctx = j.len - n;
    j.row0 = sq.y;
    j.blocks = max(1, (j.len + 15) >> 4);
    const int64_t local = at - pre[j.b];
    j.tile = (int)divide(local, j.blocks);
    j.start = pre[j.b] + (int64_t)j.tile * j.blocks;
    j.k0 = (int)(at - j.start);
    j.k1 = (int)min((int64_t)j.blocks, j.k0 + (u_end - at));
    j.rows = n * a.G - j.tile * ROWS;
    return j;
  };
  auto q_row = [&](const Job& j, int r) {
    const int rr = j.tile * ROWS + r;
    return (int64_t)(j.row0 + rr / a.G) * a.q_stride + (int64_t)(h * a.G + rr % a.G) * D;
  };
  const uint32_t sm_q = smem_u32(smem_raw) + Sm::kQ;
  auto copy_q = [&](const Job& j, int turn) {
    for (int i = tid; i < ROWS * (D / 8); i += 128) {
      const int r = i / (D / 8), c = i % (D / 8);
      if (r < j.rows) copy16(sm_q + (turn * ROWS + r) * Sm::LQ + c * 16, a.q + q_row(j, r) + c * 8);
    }
  };
  // This warp's blocks of a job are first + 4 i, i < count; their pages 32 at a time,
  // one in each lane.
  auto count_of = [&](const Job& j) {
    const int left = min(j.k1, (j.len + 15) >> 4) - j.k0 - warp;
    return left > 0 ? (left + 3) >> 2 : 0;
  };
  auto pages_of = [&](const Job& j, int i, int count) {
    return i + lane < count
               ? __ldg(a.table + (int64_t)j.b * a.table_stride + j.k0 + warp + 4 * (i + lane))
               : 0;
  };
  const uint32_t ring = smem_u32(smem_raw) + warp * ST * Blk::kStage;
  uint32_t fill = ring, use = ring;  // stages

  Job j = job_at(u);
  int count = count_of(j), pages = pages_of(j, 0, count), ahead = 0;
  copy_q(j, 0);
  copies_commit();
  copies_wait<0>();
  __syncthreads();
  for (int turn = 0;; turn ^= 1) {
    const int64_t u_next = u + (j.k1 - j.k0);
    const bool more = u_next < u_end;
    int next_count = 0, next_pages = 0;
    if (more) {
      const Job nj = job_at(u_next);
      next_count = count_of(nj);
      next_pages = pages_of(nj, 0, next_count);
      copy_q(nj, turn ^ 1);  // its group ends with the next block's copies
    }
    int later = pages_of(j, 32, count);
    // Block i of this job, or of the next one when this one has no more.
    auto start = [&](int i) {
      if (i > 0 && (i & 31) == 0) {
        pages = later;
        later = pages_of(j, i + 32, count);
      }
      const int from = i < count ? pages : next_pages, k = i < count ? i & 31 : i - count;
      const int page = __shfl_sync(0xffffffffu, from, k & 31);
      if (i < count || k < next_count) {
        Blk::copy(a, page, h, lane, fill);
        fill = fill == ring + (ST - 1) * Blk::kStage ? ring : fill + Blk::kStage;
      }
      copies_commit();
    };
    for (int i = ahead; i < ST - 1; ++i) start(i);

    Warp<D, FP8, NR> w;
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      // Row 8 n + g as the second operand: dims in the K chunks' order (8-bit: the
      // four of a k-step's first 16-bit pair and second in one word).
      const int r = 8 * n + g;
      const bool live = r < j.rows;
      const uint32_t qp = sm_q + (turn * ROWS + r) * Sm::LQ;
      uint32_t top = 0;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const int d = FP8 ? (ks >> 2) * 64 + t4 * 16 + (ks & 3) * 4
                          : (ks >> 1) * 32 + t4 * 8 + (ks & 1) * 4;
        const uint2 y = live ? lds64(qp + 2 * d) : make_uint2(0u, 0u);
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
        w.node[n][e] = (j.tile * ROWS + (c < j.rows ? c : 0)) / a.G;
        w.m[n][e] = kNegBig;
        w.l[n][e] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < NT / 2; ++i)
        w.o[n][i][0] = w.o[n][i][1] = w.o[n][i][2] = w.o[n][i][3] = 0.f;
    }

    const int* table = a.table + (int64_t)j.b * a.table_stride;
    for (int i = 0; i < count; ++i) {
      copies_wait<ST - 2>();
      __syncwarp();  // the other lanes' copies too; and all have read the stage before
      start(i + ST - 1);
      w.step(a, use, j.k0 + warp + 4 * i, table, h, j.len, j.ctx, j.row0, lane);
      use = use == ring + (ST - 1) * Blk::kStage ? ring : use + Blk::kStage;
    }
    if (count < ST) copies_wait<0>();  // the next query rows are there, at the latest now

    // Join the four warps.
#pragma unroll
    for (int n = 0; n < NR; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o <= 16; o <<= 1)
          w.l[n][e] += __shfl_xor_sync(0xffffffffu, w.l[n][e], o);
        const int row = 8 * n + 2 * t4 + e;
        if (row < j.rows) {
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
    const int rows = min(ROWS, j.rows);
    const int64_t c0 = divide(j.start, piece), c1 = divide(j.start + j.blocks - 1, piece);
    const bool whole = c0 == c1;
    const int side = cta == c0 ? 1 : 0;
    float* part = a.part + (((int64_t)cta * a.Hkv + h) * 2 + side) * ROWS * (D + 2);
    for (int i = tid; i < rows * (D / 4); i += 128) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      float M = kNegBig;
#pragma unroll
      for (int k = 0; k < 4; ++k) M = fmaxf(M, sm_ml[(k * ROWS + row) * 2]);
      float L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = ex2(sm_ml[(k * ROWS + row) * 2] - M);
        const float4 y = *reinterpret_cast<const float4*>(sm_o + (k * ROWS + row) * LD + d);
        L = fmaf(sm_ml[(k * ROWS + row) * 2 + 1], f, L);
        O[0] = fmaf(y.x, f, O[0]);
        O[1] = fmaf(y.y, f, O[1]);
        O[2] = fmaf(y.z, f, O[2]);
        O[3] = fmaf(y.w, f, O[3]);
      }
      if (whole) {
        put<D, FP8>(a, j.row0, j.tile * ROWS + row, h, d, O, L);
      } else {
        *reinterpret_cast<float4*>(part + row * D + d) = make_float4(O[0], O[1], O[2], O[3]);
        if (d == 0) *reinterpret_cast<float2*>(part + ROWS * D + 2 * row) = make_float2(M, L);
      }
    }
    if (!whole && tid == 0) {
      s_open[side] = j;
      s_parts[side] = (int)(c1 - c0 + 1);
    }
    if (!more) break;
    u = u_next;
    j = job_at(u);
    count = next_count;
    pages = next_pages;
    ahead = min(ST - 1, next_count);
    __syncthreads();  // the sums are read
  }

  // Join the CTAs that share a job, in the order of their pieces, in the last of them.
  __threadfence();
  __syncthreads();
  if (tid < 2 && s_parts[tid] > 0) {
    int* counter = a.counters + divide(s_open[tid].start, piece) * a.Hkv + h;
    const bool last = atomicAdd(counter, 1) == s_parts[tid] - 1;
    if (last) *counter = 0;
    s_last[tid] = last;
  }
  __syncthreads();
  for (int side = 0; side < 2; ++side) {
    if (s_parts[side] == 0 || !s_last[side]) continue;
    __threadfence();
    const Job o = s_open[side];
    const int rows = min(ROWS, o.rows);
    const int64_t c0 = divide(o.start, piece);
    for (int i = tid; i < rows * (D / 4); i += 128) {
      const int row = i / (D / 4), d = i % (D / 4) * 4;
      constexpr int P = 8;  // parts whose loads are in flight together
      float M = kNegBig, L = 0.f, O[4] = {0.f, 0.f, 0.f, 0.f};
      for (int c = 0; c < s_parts[side]; c += P) {
        float2 ml[P];
        float4 y[P];
        float m_new = M;
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const int64_t at = c0 + min(c + k, s_parts[side] - 1);
          const float* src =
              a.part + ((at * a.Hkv + h) * 2 + (at == c0 ? 1 : 0)) * ROWS * (D + 2);
          ml[k] = __ldcg(reinterpret_cast<const float2*>(src + ROWS * D + 2 * row));
          y[k] = __ldcg(reinterpret_cast<const float4*>(src + row * D + d));
        }
#pragma unroll
        for (int k = 0; k < P; ++k) {
          if (c + k >= s_parts[side]) {
            ml[k] = make_float2(kNegBig, 0.f);
            y[k] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
          m_new = fmaxf(m_new, ml[k].x);
        }
        const float keep = ex2(M - m_new);
        L *= keep;
#pragma unroll
        for (int x = 0; x < 4; ++x) O[x] *= keep;
#pragma unroll
        for (int k = 0; k < P; ++k) {
          const float f = ex2(ml[k].x - m_new);
          L = fmaf(ml[k].y, f, L);
          O[0] = fmaf(y[k].x, f, O[0]);
          O[1] = fmaf(y[k].y, f, O[1]);
          O[2] = fmaf(y[k].z, f, O[2]);
          O[3] = fmaf(y[k].w, f, O[3]);
        }
        M = m_new;
      }
      put<D, FP8>(a, o.row0, o.tile * ROWS + row, h, d, O, L);
    }
  }
}

template <int D, bool FP8, int NR>
void launch_rows(const Args& a, cudaStream_t stream) {
  const int smem = Smem<D, FP8, NR>::bytes(a.B);
  static PerDevice allowed;
  allow_smem(attn_rows_kernel<D, FP8, NR>, Smem<D, FP8, NR>::bytes(kMaxBatch), allowed);
  // A whole number of CTAs for each kv head.
  const int per_head = std::max(1, rows_ctas<D, FP8, NR>() * num_sms() / a.Hkv);
  launch_kernel(attn_rows_kernel<D, FP8, NR>, dim3(per_head * a.Hkv), dim3(128), smem, stream, a);
}

// By the query rows of a kv head and sequence.  64 sequences of 2048 keys, 8 kv heads
// of 128, 8-bit cache (bf16): 8 rows 59 us here and 78 with room for 16 (93 and 94); 16
// rows 100 and 85 (169 and 101), 147 on the tile kernel (124); 20 rows 147 here, where
// they read the keys twice, and 147 on the tile kernel (179 and 125), 48 rows 149 there.
template <int D, bool FP8>
void launch(const Args& a, int64_t max_rows, cudaStream_t stream) {
  if (max_rows <= 8)
    launch_rows<D, FP8, 1>(a, stream);
  else if (max_rows <= 16)
    launch_rows<D, FP8, 2>(a, stream);
  else
    launch_tiles<D, FP8>(a, stream);
}

}  // namespace tree

// {largest grid, workspace floats, workspace counters} of attn_tree.
std::vector<int64_t> attn_tree_plan(int64_t head_dim) {
  const int64_t sms = num_sms();
  return {4 * sms, sms * 2 * 256 * (head_dim + 2), 4 * sms};
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
  TORCH_CHECK(Hkv > 0 && q.size(1) > 0 && q.size(1) % D == 0 && (q.size(1) / D) % Hkv == 0,
              "query heads must divide");
  TORCH_CHECK(Hkv <= 2 * num_sms(), "too many kv heads");
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
       {&out, &k_cache, &v_cache, &block_tables, &seq_lens, &row_start, &ws, &counters, &status})
    TORCH_CHECK(t->device() == q.device(), "all tensors must be on one device");
  auto aligned16 = [](const at::Tensor& t) {
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  };
  TORCH_CHECK(aligned16(k_cache) && aligned16(v_cache), "k/v cache must be 16-byte aligned");
  if (fp8) {
    for (const at::Tensor* t : {&*k_scale, &*v_scale})
      TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() &&
                      t->numel() == k_cache.numel() / D && t->device() == q.device(),
                  "k/v scales must be fp32 [L, NB, Hkv, 16] contiguous");
    TORCH_CHECK(aligned16(*k_scale) && aligned16(*v_scale), "k/v scales must be 16-byte aligned");
  }
  if (masks.has_value())
    TORCH_CHECK(masks->scalar_type() == at::kLong && masks->is_contiguous() &&
                    masks->numel() >= q.size(0) && masks->device() == q.device(),
                "masks must be int64, one per row");
  TORCH_CHECK(max_nodes >= 1 && (!masks.has_value() || max_nodes <= 64),
              "a tree has at most 64 nodes");
  TORCH_CHECK((q.stride(0) * 2) % 16 == 0 && aligned16(q),
              "q rows must be 16-byte aligned");
  if (B == 0 || q.size(0) == 0) return;
  const c10::cuda::CUDAGuard guard(q.device());
  const std::vector<int64_t> plan = attn_tree_plan(D);
  TORCH_CHECK(ws.scalar_type() == at::kFloat && ws.numel() >= plan[1] &&
                  counters.scalar_type() == at::kInt && counters.numel() >= plan[2] &&
                  aligned16(ws) && status.scalar_type() == at::kInt && status.numel() >= 1,
              "workspace too small, or not 16-byte aligned");
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
  a.per_g = a.G == 1 ? 0u : (uint32_t)(((1ull << 32) + a.G - 1) / a.G);
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

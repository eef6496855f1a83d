// Attention over the paged cache for many new tokens: 128 query rows of a kv
// head a tile, on the tcgen05 tensor cores (formulas in attn_tree.cu).
//
// One CTA an SM, 13 warps:
//   warps 0-3, 4-7  softmax, one thread a row;
//   warps 8-11      K / V: global memory -> registers -> (e4m3 to fp16) -> shared
//                   memory in the 128-byte swizzle, two stages of 128 tokens;
//   warp 12         one thread issues the products.
// Tensor memory (512 columns): scores S0, S1 and sums O0, O1.  S = Q K^T reads
// both operands from shared memory; the weights overwrite their scores as 16-bit
// pairs and enter O += P V from there, V as it lies ([token][dim], dims contiguous).
// With more than 128 rows a job has two row tiles, one for each softmax group,
// that share every K / V tile; otherwise the groups take K / V tiles in turn and
// their sums are joined at the end.  Either way one group's products run while
// the other computes its weights.
//
// The sums are rescaled only when a row's maximum has grown by more than 2^8
// since they were last (weights then stay below 2^8: fp16 weights are held as
// 2^7 w, below 2^15).
#include <ATen/core/Tensor.h>
#include <cuda_fp8.h>

#include "attn_tree.cuh"
#include "common.cuh"
#include "host_utils.h"

namespace cb {
namespace tree {

constexpr int kTok = 128;          // tokens of a K / V tile
constexpr int kTileRows = 256;     // query rows of a job: two tiles of 128
constexpr int kTileThreads = 416;  // 13 warps
constexpr int kScaleBufs = 4;

template <int D>
struct TileSmem {
  static constexpr int kOperand = 128 * D * 2;     // one K, V or Q tile
  static constexpr int kK = 0;                     // [2]
  static constexpr int kV = 2 * kOperand;          // [2]
  static constexpr int kQ = 4 * kOperand;          // [2]
  static constexpr int kScales = 6 * kOperand;     // [kScaleBufs][3][128] fp32
  static constexpr int kMl = kScales + kScaleBufs * 3 * kTok * 4;  // [2][128][2]
  static constexpr int kBars = kMl + 2 * 128 * 2 * 4;
  static constexpr int kPre = kBars + 256;
  static int bytes(int B) { return kPre + (B + 2) / 2 * 2 * 8 + 1024; }
};

// Shared-memory matrix descriptors, 128-byte swizzle.  K-major (Q, K): rows of
// 64 summed values, groups of 8 rows 1024 bytes apart.  MN-major (V): rows are
// tokens, 64 dims each; `slab` is the distance of the next 64 dims.
__device__ __forceinline__ uint64_t desc_v(uint32_t addr, uint32_t slab) {
  uint64_t d = 0;
  d |= (uint64_t)((addr >> 4) & 0x3FFFu);
  d |= (uint64_t)(slab >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// 128 x n products of 16-bit values with fp32 sums.
template <bool F16>
__device__ constexpr uint32_t idesc(int n, bool b_mn_major) {
  return (1u << 4) | (F16 ? 0u : (1u << 7) | (1u << 10)) | (b_mn_major ? 1u << 16 : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Which of the 32 keys from position p0 on a row sees.
struct RowSight {
  int len, ctx, node;
  uint64_t mask;  // nodes it sees (with masks)
  bool masked;
  __device__ __forceinline__ uint32_t low_bits(int n) const {
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
  }
  __device__ __forceinline__ uint32_t at(int p0) const {
    uint32_t v;
    if (!masked) {
      v = low_bits(ctx + node + 1 - p0);
    } else {
      const int sh = p0 - ctx;
      if (sh >= 64) v = 0u;
      else if (sh >= 0) v = (uint32_t)(mask >> sh);
      else if (sh > -32) v = low_bits(-sh) | (uint32_t)(mask << -sh);
      else v = 0xffffffffu;
    }
    return v & low_bits(len - p0);
  }
};

// A wait of a whole warp: the warp stays together, and gives up together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* status,
                                          volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, kStatusAttnTimeout, abort_flag));
}

template <int D, bool FP8>
__global__ void __launch_bounds__(kTileThreads, 1) attn_tiles_kernel(const Args a) {
  using S = TileSmem<D>;
  constexpr int RB = FP8 ? D : 2 * D;       // bytes of a cache row
  constexpr int LPT = RB / 16;              // lanes that share a row, 16 bytes each
  constexpr int NI = LPT;                   // 16-byte loads of a lane for one tile
  constexpr int TPW = 32 / LPT;             // rows of one warp-wide load
  constexpr uint32_t kSlab = 128 * 128;     // 64 values of 128 rows
  constexpr float kUp = FP8 ? 7.f : 0.f;    // weights are held as 2^kUp w
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* scales = reinterpret_cast<float*>(smem + S::kScales);
  float* sm_ml = reinterpret_cast<float*>(smem + S::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* k_full = bars;        // [2]
  uint64_t* v_full = bars + 2;    // [2]
  uint64_t* k_free = bars + 4;    // [2]
  uint64_t* v_free = bars + 6;    // [2]
  uint64_t* s_full = bars + 8;    // [2]
  uint64_t* p_full = bars + 10;   // [2]
  uint64_t* pv_done = bars + 12;  // [2]
  uint64_t* sc_full = bars + 14;  // [kScaleBufs]
  int64_t* pre = reinterpret_cast<int64_t*>(smem + S::kPre);
  __shared__ int64_t s_sum[kTileThreads / 32];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_last, s_nonfinite;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 128);
      mbar_init(v_full + i, 128);
      mbar_init(k_free + i, 1);
      mbar_init(v_free + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
      mbar_init(pv_done + i, 1);
    }
    for (int i = 0; i < kScaleBufs; ++i) mbar_init(sc_full + i, 128);
    fence_mbar_init();
    s_abort = 0;
  }
  // Tensor memory is taken only once the kernels before are done, and the next
  // one is let in only then: neither ever waits for columns the other holds.
  grid_dep_wait();
  if (warp == 12) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  grid_dep_launch();

  scan_work<kTok, kTileThreads>(a, kTileRows, pre, s_sum);
  const int64_t total = pre[a.B];
  const int64_t piece = max((int64_t)1, (total + gridDim.x - 1) / gridDim.x);
  int64_t u = (int64_t)blockIdx.x * piece;
  const int64_t u_end = min(total, u + piece);
  volatile int* abort_flag = &s_abort;

  int kc0 = 0;              // K / V tiles of earlier segments
  int done[2] = {0, 0};     // products O += P V of each group so far

  while (u < u_end) {
    const int b = find_seq(pre, a.B, u);
    const SeqShape s = seq_shape<kTok>(a, b, kTileRows);
    const int64_t local = u - pre[b];
    const int job = (int)(local / s.nb);
    const int k0 = (int)(local - (int64_t)job * s.nb);
    const int k1 = (int)min((int64_t)s.nb, k0 + (u_end - u));
    const int h = job / s.tiles, tile = job - h * s.tiles;
    const int ctx = s.len - s.n;
    const int* table = a.table + (int64_t)b * a.table_stride;
    const int q_row0 = a.row_start[b];
    const int rows = min(kTileRows, s.n * a.G - tile * kTileRows);
    const int mt = rows > 128 ? 2 : 1;
    const int blocks = (s.len + 15) >> 4;
    int nt = max(0, min(k1, (s.len + kTok - 1) / kTok) - k0);
    if (*abort_flag) nt = 0;
    const int ns = nt * mt;

    // This softmax thread's row, and its query row in shared memory.
    const int wg = warp >> 2;
    const int row = mt == 2 ? tid : tid & 127;
    const bool live_row = warp < 8 && row < rows;
    const int rr = tile * kTileRows + (live_row ? row : 0);
    const int node = rr / a.G;
    const int64_t q_row = q_row0 + node;
    const int head = h * a.G + rr % a.G;
    float row_scale = a.scale_log2;
    if (warp < 8) {
      uint4 y[D / 8];
      const __nv_bfloat16* qp = a.q + q_row * a.q_stride + (int64_t)head * D;
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        y[c] = live_row ? *reinterpret_cast<const uint4*>(qp + 8 * c) : make_uint4(0u, 0u, 0u, 0u);
        if constexpr (FP8) {
          const uint32_t w[4] = {y[c].x, y[c].y, y[c].z, y[c].w};
#pragma unroll
          for (int i = 0; i < 4; ++i)
            top = max(top, max(w[i] & 0x7fffu, (w[i] >> 16) & 0x7fffu));
        }
      }
      float up = 1.f;
      if constexpr (FP8) {
        const int e = (int)(top >> 7);
        const int sh = e == 0 || e == 255 ? 0 : min(100, 127 + 14 - e);
        up = __int_as_float((127 + sh) << 23);
        row_scale *= __int_as_float((127 - sh) << 23);
      }
      if (mt == 2 || wg == 0) {
        const uint32_t dst = smem_u32(smem + S::kQ) + (mt == 2 ? wg : 0) * S::kOperand;
        const int r = tid & 127;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint32_t w[4] = {y[c].x, y[c].y, y[c].z, y[c].w};
          if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              w[i] = pack_f16(__uint_as_float(w[i] << 16) * up,
                              __uint_as_float(w[i] & 0xffff0000u) * up);
          }
          sts128(dst + (c >> 3) * kSlab + r * 128 + (((c & 7) ^ (r & 7)) << 4), w[0], w[1], w[2],
                 w[3]);
        }
      }
      fence_proxy_async_smem();
    }
    if (tid == 0) s_nonfinite = 0;
    __syncthreads();

    float m = kNegBig, l = 0.f;
    if (warp < 8) {
      // ------------------------------------------------------------ softmax
      const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t s_addr = lane_base + wg * 128;
      const uint32_t o_addr = lane_base + 256 + wg * 128;
      const bool live_warp = (mt == 2 ? warp : warp & 3) * 32 < rows;
      RowSight sight;
      sight.len = s.len;
      sight.ctx = ctx;
      sight.node = node;
      sight.masked = a.masks != nullptr;
      sight.mask = sight.masked && live_row ? (uint64_t)a.masks[q_row] : 0;
      int n = done[wg];
      for (int st = wg; st < ns; st += 2) {
        const int kt = mt == 2 ? st >> 1 : st;
        const int kc = kc0 + kt;
        const int pos0 = (k0 + kt) * kTok;
        if (!warp_wait(s_full + wg, n & 1, a.status, abort_flag)) break;
        if (!warp_wait(sc_full + (kc & (kScaleBufs - 1)), (kc / kScaleBufs) & 1, a.status,
                       abort_flag))
          break;
        tc_fence_after();
        bool ok = true;
        if (live_warp) {
          const float* sc = scales + (kc & (kScaleBufs - 1)) * 3 * kTok;
          const bool tail = pos0 + kTok > ctx;
          // Scores of columns c .. c + 3 in base 2, with log2 of the values'
          // scales added.
          auto score4 = [&](float* v, int c) {
            if constexpr (FP8) {
              const float4 k4 = *reinterpret_cast<const float4*>(sc + c);
              const float4 l4 = *reinterpret_cast<const float4*>(sc + kTok + c);
              v[0] = fmaf(v[0] * k4.x, row_scale, l4.x);
              v[1] = fmaf(v[1] * k4.y, row_scale, l4.y);
              v[2] = fmaf(v[2] * k4.z, row_scale, l4.z);
              v[3] = fmaf(v[3] * k4.w, row_scale, l4.w);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) v[i] *= row_scale;
            }
          };
          float mx = -INFINITY;
#pragma unroll
          for (int c0 = 0; c0 < kTok; c0 += 32) {
            float v[32];
            __syncwarp();
            tmem_ld32(s_addr + c0, v);
            const uint32_t seen = tail ? sight.at(pos0 + c0) : 0xffffffffu;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              score4(v + i, c0 + i);
              if (tail) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i + e] = seen >> (i + e) & 1 ? v[i + e] : -INFINITY;
              }
              mx = fmaxf(mx, fmaxf(fmaxf(v[i], v[i + 1]), fmaxf(v[i + 2], v[i + 3])));
            }
          }
          float alpha = 1.f;
          if (mx > m + 8.f) {
            alpha = ex2(m - mx);
            m = mx;
            l *= alpha;
          }
          if (__any_sync(0xffffffffu, alpha != 1.f) && st >= 2) {
            ok = warp_wait(pv_done + wg, (n - 1) & 1, a.status, abort_flag);
            if (ok) {
              tc_fence_after();
#pragma unroll
              for (int c0 = 0; c0 < D; c0 += 32) {
                float v[32];
                tmem_ld32(o_addr + c0, v);
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * alpha);
                tmem_st16(o_addr + c0, w);
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[16 + i] * alpha);
                tmem_st16(o_addr + c0 + 16, w);
              }
              tmem_st_wait();
            }
          }
          const float base = m - kUp;
          float sum = 0.f;
#pragma unroll
          for (int c0 = 0; c0 < kTok; c0 += 32) {
            float v[32];
            __syncwarp();
            tmem_ld32(s_addr + c0, v);
            const uint32_t seen = tail ? sight.at(pos0 + c0) : 0xffffffffu;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              score4(v + i, c0 + i);
              alignas(16) float inv[4] = {1.f, 1.f, 1.f, 1.f};
              if constexpr (FP8)
                *reinterpret_cast<float4*>(inv) =
                    *reinterpret_cast<const float4*>(sc + 2 * kTok + c0 + i);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float w = ex2(v[i + e] - base);
                float part = FP8 ? w * inv[e] : w;
                // (a hidden key's scale may be a NaN)
                if (tail && !(seen >> (i + e) & 1)) w = part = 0.f;
                sum += part;
                v[i + e] = w;
              }
            }
            uint32_t p[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if constexpr (FP8) {
                p[i] = pack_f16(v[2 * i], v[2 * i + 1]);
              } else {
                const __nv_bfloat162 y = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                p[i] = *reinterpret_cast<const uint32_t*>(&y);
              }
            }
            tmem_st16(s_addr + c0 / 2, p);
          }
          l += sum;
          tmem_st_wait();
        }
        if (!ok) break;
        tc_fence_before();
        mbar_arrive(p_full + wg);
        ++n;
      }
      if (n > done[wg]) warp_wait(pv_done + wg, (n - 1) & 1, a.status, abort_flag);
      tc_fence_after();
      // The groups' statistics, for joining.
      sm_ml[(wg * 128 + (tid & 127)) * 2] = ns > wg ? m : kNegBig;
      sm_ml[(wg * 128 + (tid & 127)) * 2 + 1] = ns > wg ? l : 0.f;
    } else if (warp < 12) {
      // ------------------------------------------------------------ K and V
      const int ct = tid - 256, cw = ct >> 5;
      const int piece16 = lane % LPT;
      auto token_of = [&](int i) { return i * 4 * TPW + cw * TPW + lane / LPT; };
      uint4 kb[NI];
      uint4 vb[NI];  // (bf16 rows are twice as long: kb alone serves both)
      float ks_r = 0.f, vs_r = 1.f;
      int pages = 0;
      auto fetch_pages = [&](int kt) {
        const int blk = (k0 + kt) * 8 + lane;
        return lane < 8 && blk < blocks ? __ldg(table + blk) : -1;
      };
      auto load = [&](uint4(&buf)[NI], const uint8_t* base, int kt) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int tok = token_of(i);
          const int page = __shfl_sync(0xffffffffu, pages, tok >> 4);
          buf[i] = page >= 0 ? ldg_stream16(base + (((a.layer_blocks + page) * a.Hkv + h) * 16 +
                                                    (tok & 15)) * RB + piece16 * 16)
                             : make_uint4(0u, 0u, 0u, 0u);
        }
      };
      auto load_scales = [&](int kt) {
        if constexpr (FP8) {
          const int page = __shfl_sync(0xffffffffu, pages, ct >> 4);
          const bool there = page >= 0 && (k0 + kt) * kTok + ct < s.len;
          const int64_t r = ((a.layer_blocks + page) * a.Hkv + h) * 16 + (ct & 15);
          ks_r = there ? __ldg(a.ks + r) : 0.f;
          vs_r = there ? __ldg(a.vs + r) : 1.f;
        }
      };
      auto store = [&](const uint4(&buf)[NI], uint32_t dst) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int tok = token_of(i);
          const uint32_t w[4] = {buf[i].x, buf[i].y, buf[i].z, buf[i].w};
          if constexpr (FP8) {
            uint32_t f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              f[2 * j] = e4m3x2_to_f16x2(w[j] & 0xffffu);
              f[2 * j + 1] = e4m3x2_to_f16x2(w[j] >> 16);
            }
            // Two chunks of 8 values; the lanes of the second slab start with
            // the other one, which keeps the eight lanes of a phase on
            // different banks.
            const int c = 2 * piece16;
            const uint32_t at = dst + (c >> 3) * kSlab + tok * 128;
            const uint32_t c0 = at + (((c & 7) ^ (tok & 7)) << 4);
            const uint32_t c1 = at + ((((c & 7) + 1) ^ (tok & 7)) << 4);
            if (c >> 3) {
              sts128(c1, f[4], f[5], f[6], f[7]);
              sts128(c0, f[0], f[1], f[2], f[3]);
            } else {
              sts128(c0, f[0], f[1], f[2], f[3]);
              sts128(c1, f[4], f[5], f[6], f[7]);
            }
          } else {
            sts128(dst + (piece16 >> 3) * kSlab + tok * 128 +
                       (((piece16 & 7) ^ (tok & 7)) << 4),
                   w[0], w[1], w[2], w[3]);
          }
        }
      };
      // Value rows that a product must not meet: past the end anything may
      // lie there, and a bf16 node may hold an infinity or a NaN that its
      // siblings do not see (added to the rows that do see it at the end).
      auto clean = [&](uint4(&buf)[NI], int kt) {
        const int pos0 = (k0 + kt) * kTok;
        if (pos0 + kTok <= ctx) return;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          if (pos0 + token_of(i) >= s.len) buf[i] = make_uint4(0u, 0u, 0u, 0u);
          if constexpr (!FP8) {
            uint32_t w[4] = {buf[i].x, buf[i].y, buf[i].z, buf[i].w};
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if ((w[j] & 0x7f80u) == 0x7f80u) { w[j] &= 0xffff0000u; bad = true; }
              if ((w[j] & 0x7f800000u) == 0x7f800000u) { w[j] &= 0xffffu; bad = true; }
            }
            if (bad) s_nonfinite = 1;
            buf[i] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      };
      if (nt > 0) {
        pages = fetch_pages(0);
        load(kb, a.k, 0);
        load_scales(0);
        if constexpr (FP8) load(vb, a.v, 0);
      }
      for (int kt = 0; kt < nt; ++kt) {
        const int kc = kc0 + kt, st = kc & 1;
        const uint32_t parity = ((kc >> 1) + 1) & 1;
        if (kc >= 2 && !warp_wait(k_free + st, parity, a.status, abort_flag)) break;
        store(kb, smem_u32(smem + S::kK) + st * S::kOperand);
        float* sc = scales + (kc & (kScaleBufs - 1)) * 3 * kTok;
        if constexpr (FP8) {
          const float lv = __log2f(vs_r);
          sc[ct] = ks_r;
          sc[kTok + ct] = lv;
          sc[2 * kTok + ct] = ex2(-lv);
        }
        mbar_arrive(sc_full + (kc & (kScaleBufs - 1)));
        fence_proxy_async_smem();
        mbar_arrive(k_full + st);
        if constexpr (FP8) {
          if (kt + 1 < nt) {
            pages = fetch_pages(kt + 1);
            load(kb, a.k, kt + 1);
            load_scales(kt + 1);
          }
        } else {
          load(kb, a.v, kt);
        }
        if (kc >= 2 && !warp_wait(v_free + st, parity, a.status, abort_flag)) break;
        if constexpr (FP8) {
          clean(vb, kt);
          store(vb, smem_u32(smem + S::kV) + st * S::kOperand);
        } else {
          clean(kb, kt);
          store(kb, smem_u32(smem + S::kV) + st * S::kOperand);
        }
        fence_proxy_async_smem();
        mbar_arrive(v_full + st);
        if (kt + 1 < nt) {
          if constexpr (FP8) {
            load(vb, a.v, kt + 1);
          } else {
            pages = fetch_pages(kt + 1);
            load(kb, a.k, kt + 1);
          }
        }
      }
    } else if (lane == 0) {
      // ------------------------------------------------------------ products
      int n[2] = {done[0], done[1]};
      auto scores = [&](int st) {
        const int g = st & 1, kt = mt == 2 ? st >> 1 : st, kc = kc0 + kt, sg = kc & 1;
        if (!mbar_wait(k_full + sg, (kc >> 1) & 1, a.status, kStatusAttnTimeout, abort_flag))
          return false;
        tc_fence_after();
        const uint32_t qa = smem_u32(smem + S::kQ) + (mt == 2 ? g : 0) * S::kOperand;
        const uint32_t ka = smem_u32(smem + S::kK) + sg * S::kOperand;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks >> 2) * kSlab + (ks & 3) * 32;
          mma_bf16_ss(tmem + g * 128, umma_desc_sw128(qa + off), umma_desc_sw128(ka + off),
                      idesc<FP8>(kTok, false), ks != 0);
        }
        mma_commit(s_full + g);
        if (mt == 1 || g == 1) mma_commit(k_free + sg);
        return true;
      };
      bool ok = true;
      for (int st = 0; st < min(2, ns) && ok; ++st) ok = scores(st);
      for (int st = 0; st < ns && ok; ++st) {
        const int g = st & 1, kt = mt == 2 ? st >> 1 : st, kc = kc0 + kt, sg = kc & 1;
        ok = mbar_wait(v_full + sg, (kc >> 1) & 1, a.status, kStatusAttnTimeout, abort_flag) &&
             mbar_wait(p_full + g, n[g] & 1, a.status, kStatusAttnTimeout, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t va = smem_u32(smem + S::kV) + sg * S::kOperand;
#pragma unroll
        for (int ks = 0; ks < kTok / 16; ++ks)
          mma_bf16_ts(tmem + 256 + g * 128, tmem + g * 128 + ks * 8,
                      desc_v(va + ks * 2048, kSlab), idesc<FP8>(D, true), st >= 2 || ks != 0);
        mma_commit(pv_done + g);
        if (mt == 1 || g == 1) mma_commit(v_free + sg);
        if (st + 2 < ns) {
          // The next scores overwrite the weights this product reads.
          ok = mbar_wait(pv_done + g, n[g] & 1, a.status, kStatusAttnTimeout, abort_flag) &&
               scores(st + 2);
        }
        ++n[g];
      }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    // Join the groups (one row tile) and the CTAs that share the job.
    const int64_t js = pre[b] + (int64_t)job * s.nb;
    const int64_t c0 = js / piece, c1 = (js + s.nb - 1) / piece;
    const bool whole = c0 == c1;
    const bool ok = !*abort_flag;
    // With one row tile each group joins and stores half of the dims.
    const int d_lo = mt == 2 ? 0 : wg * (D / 2), d_hi = mt == 2 ? D : d_lo + D / 2;
    float* slot = a.part + ((int64_t)blockIdx.x * 2 + (blockIdx.x == c0 ? 1 : 0)) * kTileRows *
                               (D + 2);
    const bool live_warp = warp < 8 && (mt == 2 ? warp : warp & 3) * 32 < rows;
    auto put = [&](int d, const float (&y)[16]) {
      __nv_bfloat16* dst = a.out + q_row * a.out_stride + (int64_t)head * D + d;
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(y[2 * i], y[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p);
      }
      if (a.out_vec) {
        reinterpret_cast<uint4*>(dst)[0] = make_uint4(w[0], w[1], w[2], w[3]);
        reinterpret_cast<uint4*>(dst)[1] = make_uint4(w[4], w[5], w[6], w[7]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          reinterpret_cast<uint16_t*>(dst)[2 * i] = (uint16_t)w[i];
          reinterpret_cast<uint16_t*>(dst)[2 * i + 1] = (uint16_t)(w[i] >> 16);
        }
      }
    };
    if (live_warp && ok) {
      const int r = tid & 127;
      float f[2], M = m, L = l;
      f[0] = f[1] = 0.f;
      if (mt == 2) {
        f[wg] = 1.f;
        if (ns == 0) L = 0.f;
      } else {
        const float m0 = sm_ml[r * 2], m1 = sm_ml[(128 + r) * 2];
        M = fmaxf(m0, m1);
        f[0] = ex2(m0 - M);
        f[1] = ex2(m1 - M);
        L = sm_ml[r * 2 + 1] * f[0] + sm_ml[(128 + r) * 2 + 1] * f[1];
      }
      if (!whole && live_row && (mt == 2 || wg == 0)) {
        slot[row] = M;
        slot[kTileRows + row] = L;
      }
      const bool more = !FP8 && s_nonfinite;
#pragma unroll 1
      for (int d = d_lo; d < d_hi; d += 16) {
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = 0.f;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          if ((mt == 2 && g != wg) || ns <= g) continue;
          float v[16];
          __syncwarp();
          tmem_ld16(tmem + ((uint32_t)((warp & 3) * 32) << 16) + 256 + g * 128 + d, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = fmaf(v[i], f[g], y[i]);
        }
        if (more && live_row) {
          // The infinities and NaNs that were kept out of the products.
          const bool masked = a.masks != nullptr;
          const uint64_t mask = masked ? (uint64_t)a.masks[q_row] : 0;
          for (int pos = max(k0, ctx / kTok) * kTok; pos < min(k1 * kTok, s.len); ++pos) {
            const int j = pos - ctx;
            if (j >= 0 && !(masked ? j < 64 && (mask >> (j & 63) & 1) : j <= node)) continue;
            const int64_t vr = ((a.layer_blocks + table[pos >> 4]) * a.Hkv + h) * 16 + (pos & 15);
            const __nv_bfloat16* vp = reinterpret_cast<const __nv_bfloat16*>(a.v) + vr * D + d;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float val = __bfloat162float(vp[i]);
              if (!(fabsf(val) <= 3.4e38f)) y[i] += val;
            }
          }
        }
        if (!live_row) continue;
        if (whole) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = L == 0.f ? 0.f : y[i] * inv;
          put(d, y);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) slot[(2 + d + i) * kTileRows + row] = y[i];
        }
      }
    }
    if (!whole) {
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        s_last = atomicAdd(a.counters + c0, 1) == (int)(c1 - c0);
        if (s_last) a.counters[c0] = 0;
      }
      __syncthreads();
      if (s_last && live_row && ok) {
        __threadfence();
        auto part_of = [&](int64_t c) {
          return a.part + (c * 2 + (c == c0 ? 1 : 0)) * kTileRows * (D + 2) + row;
        };
        float M = kNegBig, L = 0.f;
        for (int64_t c = c0; c <= c1; ++c) M = fmaxf(M, __ldcg(part_of(c)));
        for (int64_t c = c0; c <= c1; ++c)
          L += __ldcg(part_of(c) + kTileRows) * ex2(__ldcg(part_of(c)) - M);
        const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll 1
        for (int d = d_lo; d < d_hi; d += 16) {
          float y[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = 0.f;
          for (int64_t c = c0; c <= c1; ++c) {
            const float* p = part_of(c);
            const float f = ex2(__ldcg(p) - M);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = fmaf(__ldcg(p + (2 + d + i) * kTileRows), f, y[i]);
          }
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = L == 0.f ? 0.f : y[i] * inv;
          put(d, y);
        }
      }
    }
    tc_fence_before();
    __syncthreads();  // shared and tensor memory are reused by the next job
    tc_fence_after();
    kc0 += nt;
    done[0] += (ns + 1) / 2;
    done[1] += ns / 2;
    u += k1 - k0;
  }
  __syncthreads();
  if (warp == 12) tmem_dealloc(tmem, 512);
}

template <int D, bool FP8>
void launch_tiles(const Args& a, cudaStream_t stream) {
  const int smem = TileSmem<D>::bytes(a.B);
  static int configured = 0;
  if (smem > configured) {
    CB_CUDA_CHECK(cudaFuncSetAttribute(attn_tiles_kernel<D, FP8>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    configured = smem;
  }
  launch_kernel(attn_tiles_kernel<D, FP8>, dim3(num_sms()), dim3(kTileThreads), smem, stream, a);
}

template void launch_tiles<64, false>(const Args&, cudaStream_t);
template void launch_tiles<64, true>(const Args&, cudaStream_t);
template void launch_tiles<128, false>(const Args&, cudaStream_t);
template void launch_tiles<128, true>(const Args&, cudaStream_t);

}  // namespace tree
}  // namespace cb

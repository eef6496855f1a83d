// Attention over the paged cache for many new tokens: 128 query rows of a kv
// head a tile, on the tcgen05 tensor cores (formulas in attn_tree.cu).
//
// One CTA an SM:
//   warps 0-3, 4-7  softmax, one thread a row;
//   warps 8-15      K and V: global memory -> shared memory in the 128-byte swizzle,
//                   two stages of 128 tokens, 64 tokens for each four warps;
//   warps 16-19     one thread of each issues the products.
// Tensor memory (512 columns): for each softmax group the scores of two steps of 64
// tokens and the sums.  S = Q K^T reads both operands from shared memory; the weights
// overwrite their scores as 16-bit pairs and enter O += P V from there, V as it lies
// ([token][dim], dims contiguous).  While a group computes the weights of one step
// the scores of its next are made: a step of 128 tokens with one score buffer left
// every group idle for its products, twice the time.
// With more than 128 rows a job has two row tiles, one for each softmax group,
// that share every K / V tile; otherwise the groups take K / V tiles in turn and
// their sums are joined at the end.
//
// 8-bit cache.  Scores: the codes of K enter an 8-bit product as they are, q as two
// e4m3 numbers (q = hi + lo to its last bit, down to 2^-9 of the row's largest value;
// below that to 2^-18 of it), at twice the rate of a 16-bit product, so that no key
// has to be unpacked; a score is then multiplied by its key's scale.  Values: code x
// scale / r in fp16, with r a power of two, the largest scale of the 128-token tile
// rounded up, so that a softmax thread needs one number a tile for them instead of
// two for each column (shared-memory bandwidth).  The price is one rounding to
// fp16's 11 bits, 2^-12 of a value against the 2^-5 of its code and the 2^-9 of the
// bf16 result; the scale itself enters as a pair of fp16 numbers, 22 bits.  Scales far
// below the reference would lose bits, and all of them beside a hidden or weightless
// key with a large one: a tile whose scales span 2^kSpan or more takes an r for each key,
// at the cost of the slower pass over its scores.
//
// Weights are computed in one pass over the scores, in the frame of the maximum
// that the row had before; only if a score is more than 2^8 over it (or keys of
// the tile are hidden) the tile is taken again in two passes and the sums are
// rescaled.  Weights thus stay below 2^8: fp16 weights are held as 2^7 w, below
// 2^15.
//
// Bound: the softmax threads' own time, 2100 cycles for a step of 64 tokens and 700
// for its waits, while the products take about 800 and the loads less.  8 trees of 64
// nodes x 4 heads over 8192 keys, 8 kv heads of 128, 8-bit cache: 163 us, 418 TFLOP/s
// (146 MB).  Some 50 us of it are not in the steps (56 for a CTA, 157 000 cycles): start,
// ends of jobs and joins.  With one row tile the loading warps, 3000 cycles for 128 tokens
// of the 8-bit cache: 64 sequences of 2048 keys, 20 rows, 147 us (bf16 cache 125 us,
// 4.3 TB/s).
#include "attn_tree.cuh"
#include "common.cuh"
#include "host_utils.h"

namespace cb {
namespace tree {

constexpr int kTok = 128;          // tokens of a K / V tile
constexpr int kStep = 64;           // tokens of a step
constexpr int kSb = 128 / kStep;    // score buffers of a softmax group
constexpr int kSpt = kTok / kStep;  // steps of a tile
constexpr int kTileRows = 256;     // query rows of a job: two tiles of 128
constexpr int kTileThreads = 640;
// Registers of a thread: at launch, and after the groups have shared them out.
constexpr int kRegsLaunch = 96, kRegsSoftmax = 128, kRegsLoad = 88, kRegsIssue = 48;
static_assert(2 * kRegsSoftmax + 2 * kRegsLoad + kRegsIssue <= 5 * kRegsLaunch,
              "more registers than the block has: the groups would wait for them for ever");
static_assert(kRegsLoad <= kRegsLaunch && kRegsIssue <= kRegsLaunch && kRegsLaunch <= kRegsSoftmax,
              "a share may only shrink below the launch's, or grow above it");
constexpr int kTileBufs = 8;       // tiles whose scale references are kept
constexpr int kSpan = 12;          // log2 of the span of scales that share one
constexpr float kEachItsOwn = 1e9f;  // in place of a tile's reference

template <int D, bool FP8>
struct TileSmem {
  static constexpr int kSlab = 128 * 128;             // 128 rows of 128 bytes
  static constexpr int kVTile = D / 64 * kSlab;       // 16-bit values
  static constexpr int kKTile = FP8 ? kSlab : kVTile;  // codes: one slab, also half filled
  static constexpr int kQTile = FP8 ? 2 * kSlab : kVTile;
  static constexpr int kK = 0;                       // [2]
  static constexpr int kV = kK + 2 * kKTile;         // [2]
  static constexpr int kQ = kV + 2 * kVTile;         // [2]
  static constexpr int kRaw = kQ + 2 * kQTile;       // V's codes as they come: [2][128][D]
  static constexpr int kScale = kRaw + (FP8 ? 2 * 128 * D : 0);  // K's: [kTileBufs][128] fp32
  static constexpr int kPairs = kScale + kTileBufs * kTok * 4;  // V's: [8 warps][128]
  static constexpr int kRefs = kPairs + 8 * kTok * 4;  // keys' own references: [kTileBufs][128]
  static constexpr int kMl = kRefs + (FP8 ? kTileBufs * kTok * 4 : 0);  // [2][128][2]
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

// 128 x n products with fp32 sums; format 0: fp16 (or e4m3, in an 8-bit product),
// 1: bf16.
__device__ constexpr uint32_t idesc(uint32_t format, int n, bool b_mn_major) {
  return (1u << 4) | (format << 7) | (format << 10) | (b_mn_major ? 1u << 16 : 0u) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// D[tmem] (+)= A[smem] * B[smem], e4m3 inputs (32 summed values), fp32 sums.
__device__ __forceinline__ void mma_e4m3_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate));
}

__device__ __forceinline__ void tmem_ld32_start(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
// The registers pass through the wait, so that nothing reads them before it.
__device__ __forceinline__ void tmem_ld32_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                 "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                 "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                 "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                 "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])::"memory");
}

__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e != 0;
}

template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Two fp32 operations in one instruction.
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split(F2 x, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x.v));
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void sts64(uint32_t addr, uint32_t a, uint32_t b) {
  asm volatile("st.shared.v2.b32 [%0], {%1,%2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
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
  return __all_sync(
      0xffffffffu, mbar_wait_sleep(bar, parity, status, kStatusAttnTimeout, abort_flag));
}

// One CTA's share of one job: K / V tiles k0 .. k0 + nt of (sequence b, kv head h,
// row tile).
struct Segment {
  int b, h, n, len, ctx, nb, k0, nt, rows, mt;
  int row0;      // first of the job's rows, node * G + head of the group
  int q_row0;    // first query row of the sequence
  const int* table;
  int64_t c0, c1;  // CTAs that share the job
  int64_t units;
};

// K / V tiles of softmax group w: all of them with two row tiles, every other one
// with one.
__device__ __forceinline__ int group_tiles(int nt, int mt, int w) {
  return mt == 2 ? nt : (nt + 1 - w) >> 1;
}

__device__ __forceinline__ Segment segment_at(const Args& a, const int64_t* pre, int64_t u,
                                              int64_t u_end, int64_t piece, bool skip) {
  Segment g;
  g.b = find_seq(pre, a.B, u);
  const SeqShape s = seq_shape<kTok>(a, g.b, kTileRows);
  const int64_t local = u - pre[g.b];
  const int job = (int)divide(local, s.nb);
  g.k0 = (int)(local - (int64_t)job * s.nb);
  g.units = min((int64_t)s.nb - g.k0, u_end - u);
  g.h = job / s.tiles;
  g.row0 = (job - g.h * s.tiles) * kTileRows;
  g.n = s.n;
  g.len = s.len;
  g.nb = s.nb;
  g.ctx = s.len - s.n;
  g.table = a.table + (int64_t)g.b * a.table_stride;
  g.q_row0 = a.row_start[g.b];
  g.rows = min(kTileRows, s.n * a.G - g.row0);
  g.mt = g.rows > 128 ? 2 : 1;
  g.nt = skip ? 0 : max(0, min(g.k0 + (int)g.units, (s.len + kTok - 1) / kTok) - g.k0);
  const int64_t js = pre[g.b] + (int64_t)job * s.nb;
  g.c0 = divide(js, piece);
  g.c1 = divide(js + s.nb - 1, piece);
  return g;
}

// What the loading groups share with the others.
struct LoadSmem {
  uint32_t k, v;      // [2] operand tiles (shared addresses)
  uint32_t raw;       // this lane's place in V's codes
  uint32_t pairs;     // this warp's [128] scales of V over the reference, as fp16 pairs
  float* k_scale;     // [kTileBufs][128]
  float* v_ref;       // [kTileBufs]: log2 of V's reference / 2^6, or kEachItsOwn
  float* v_refs;      // [kTileBufs][128]: the same for each key
  uint64_t *k_full, *v_full, *k_free, *v_free;  // [2]
  uint64_t* r_full;   // [kTileBufs]
  volatile int* abort_flag;
  int* nonfinite;
};

// Four warps bring 64 tokens of every K / V tile of the CTA's jobs into shared
// memory, by asynchronous copies: K, and V of the bf16 cache, to their places; V's codes
// to a place of the lane's own, whence it unpacks them.  The next tile's copies are made
// as soon as there is room.  (Loads into registers, a tile ahead, kept waiting for one
// another: a warp has but a few counters for all its loads in flight.)
template <int D, bool FP8>
__device__ __forceinline__ void load_tiles(const Args& a, const int64_t* pre, int64_t u0,
                                           int64_t u_end, int64_t piece, const LoadSmem& sm,
                                           int group) {
  using S = TileSmem<D, FP8>;
  constexpr int RB = FP8 ? D : 2 * D;      // bytes of a cache row
  constexpr int LPT = RB / 16;             // lanes that share a row, 16 bytes each
  constexpr int TPW = 32 / LPT;            // rows of one warp-wide load
  constexpr int ROWS = 64 / (4 * TPW);     // copies of a lane for its part of a tile, of K and of V
  const int ct = threadIdx.x & 127, cw = ct >> 5, lane = ct & 31;
  // Lanes in fours along a row, then over two rows: the eight lanes of a store
  // phase then write different banks, also when each writes every other chunk.
  const int piece16 = LPT <= 4 ? lane % LPT : (lane & 3) | (lane >> 3 & (LPT / 4 - 1)) << 2;
  const int sub = 64 * group + cw * TPW +
                  (LPT <= 4 ? lane / LPT : (lane >> 2 & 1) | (lane >> 3) / (LPT / 4) << 1);
  // Token of this lane's i-th row.
  auto token_of = [&](int i) { return i * 4 * TPW + sub; };
  // Its 16-byte chunk of a tile row: of K, and of V (8-bit: the first of two).
  const int k_chunk = piece16 & 7, v_chunk = FP8 ? (2 * piece16) & 7 : piece16 & 7;
  const uint32_t k_tiles = sm.k + (piece16 >> 3) * S::kSlab;
  const uint32_t v_tiles = sm.v + (FP8 ? piece16 >> 2 : piece16 >> 3) * S::kSlab;
  const int64_t block_bytes = (int64_t)a.Hkv * 16 * RB;
  int kc = 0;
  for (int64_t u = u0; u < u_end;) {
    const Segment g = segment_at(a, pre, u, u_end, piece, *sm.abort_flag != 0);
    u += g.units;
    if (g.nt == 0) continue;
    const int blocks = (g.len + 15) >> 4;
    const int64_t first_row = (a.layer_blocks * a.Hkv + g.h) * 16;
    const uint8_t* k_base = a.k + first_row * RB + piece16 * 16;
    const uint8_t* v_base = a.v + first_row * RB + piece16 * 16;
    // Blocks past the end read the last one (hidden, and zeroed where it would
    // matter).
    auto fetch_pages = [&](int kt) {
      return __ldg(g.table + min((g.k0 + kt) * 8 + (lane & 7), blocks - 1));
    };
    auto row_at = [&](int tok, int pages) {
      const int64_t page = __shfl_sync(0xffffffffu, pages, tok >> 4);
      return page * block_bytes + (tok & 15) * RB;
    };
    // Room for a tile (of all the CTA's tiles), its copies.
    auto room = [&](uint64_t* free, int tile) {
      return tile < 2 ||
             warp_wait(free + (tile & 1), ((tile >> 1) + 1) & 1, a.status, sm.abort_flag);
    };
    auto copy_k = [&](int tile, int pages) {
      const uint32_t dst = k_tiles + (tile & 1) * S::kKTile;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int tok = token_of(i);
        copy16(dst + tok * 128 + ((k_chunk ^ (tok & 7)) << 4), k_base + row_at(tok, pages));
      }
    };
    auto copy_v = [&](int tile, int pages) {
      const uint32_t dst = FP8 ? sm.raw + (tile & 1) * 128 * D : v_tiles + (tile & 1) * S::kVTile;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int tok = token_of(i);
        copy16(FP8 ? dst + i * 512 : dst + tok * 128 + ((v_chunk ^ (tok & 7)) << 4),
               v_base + row_at(tok, pages));
      }
    };
    // Scales of tokens 4 lane .. 4 lane + 3 of a tile.
    auto load_scales = [&](const float* from, int pages) {
      const int64_t page = __shfl_sync(0xffffffffu, pages, lane >> 2);
      return __ldg(reinterpret_cast<const float4*>(from + first_row + page * a.Hkv * 16) +
                   (lane & 3));
    };
    float4 ks = make_float4(0.f, 0.f, 0.f, 0.f), vs = ks;
    // Page numbers run ahead of the rows they lead to.
    int pages = fetch_pages(0), next_pages = fetch_pages(1);
    if (!room(sm.k_free, kc)) continue;
    copy_k(kc, pages);
    copies_commit();
    if (!FP8 && !room(sm.v_free, kc)) continue;
    copy_v(kc, pages);
    copies_commit();
    if constexpr (FP8) {
      ks = load_scales(a.ks, pages);
      vs = load_scales(a.vs, pages);
    }
    for (int kt = 0; kt < g.nt; ++kt, ++kc) {
      const int st = kc & 1;
      const bool more = kt + 1 < g.nt;
      const int later_pages = fetch_pages(kt + 2);
      const int pos0 = (g.k0 + kt) * kTok;
      const bool tail = pos0 + kTok > g.ctx;
      if constexpr (FP8) {
        float kx[4] = {ks.x, ks.y, ks.z, ks.w}, vx[4] = {vs.x, vs.y, vs.z, vs.w};
        uint32_t top = 0u, low = 0xffffffffu;  // of the scales that are not 0
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // A row past the end gets the scale 0.  A key one of whose scales is not
          // a number gets NaN scores and a value of zero, so that only the rows
          // that see it get NaN.
          const bool fine = isfinite(kx[e]) && isfinite(vx[e]);
          if (!fine) kx[e] = __int_as_float(0x7fc00000);
          if (!fine || (tail && pos0 + 4 * lane + e >= g.len)) vx[e] = 0.f;
          top = max(top, __float_as_uint(vx[e]));
          if (vx[e] != 0.f) low = min(low, __float_as_uint(vx[e]));
        }
        // Reference 2^(x - 126) > the tile's largest scale.  x is kept from 43 on
        // (2^-83; 127 without any scale): sums of weights over the reference stay
        // far from overflow then, even for heads whose values are all zero.
        top = __reduce_max_sync(0xffffffffu, top);
        const int x = top == 0u ? 127 : max(43, (int)(top >> 23));
        low = __reduce_min_sync(0xffffffffu, low);
        const bool wide = top != 0u && x - max(43, (int)(low >> 23)) >= kSpan;
        uint32_t pair[4];  // each token's scale over the reference as two fp16 numbers
        int own[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          own[e] = wide && vx[e] != 0.f ? max(43, (int)(__float_as_uint(vx[e]) >> 23)) : x;
          const float y = vx[e] * (__int_as_float((253 - own[e]) << 23) * 64.f);  // 2^6 s / r
          pair[e] = pack_f16(y, y - __half2float(__float2half_rn(y)));
        }
        __syncwarp();
        sts128(sm.pairs + lane * 16, pair[0], pair[1], pair[2], pair[3]);
        __syncwarp();
        if (group == 0 && cw == 0) {
          const int slot = kc & (kTileBufs - 1);
          reinterpret_cast<float4*>(sm.k_scale + slot * kTok)[lane] =
              make_float4(kx[0], kx[1], kx[2], kx[3]);
          reinterpret_cast<float4*>(sm.v_refs + slot * kTok)[lane] =
                make_float4((float)(own[0] - 126 - 6), (float)(own[1] - 126 - 6),
                            (float)(own[2] - 126 - 6), (float)(own[3] - 126 - 6));
          if (lane == 0) sm.v_ref[slot] = wide ? kEachItsOwn : (float)(x - 126 - 6);
          mbar_arrive(sm.r_full + slot);
        }
        if (more) {
          ks = load_scales(a.ks, next_pages);
          vs = load_scales(a.vs, next_pages);
        }
      }
      copies_wait<1>();
      fence_proxy_async_smem();
      mbar_arrive(sm.k_full + st);
      if (more) {
        if (!room(sm.k_free, kc + 1)) break;
        copy_k(kc + 1, next_pages);
      }
      copies_commit();
      copies_wait<1>();
      const uint32_t v_dst = v_tiles + st * S::kVTile;
      if (FP8 && !room(sm.v_free, kc)) break;
      if (FP8 || tail) {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) {
          const int tok = token_of(i);
          const uint32_t c0 = v_dst + tok * 128 + ((v_chunk ^ (tok & 7)) << 4);
          const uint4 u = lds128(FP8 ? sm.raw + st * 128 * D + i * 512 : c0);
          uint32_t w[4] = {u.x, u.y, u.z, u.w};
          if constexpr (FP8) {
            // Scales are at most 2^6: values of 448 x 2^6 at most.
            const uint32_t pair = lds32(sm.pairs + tok * 4);
            const uint32_t hi = __byte_perm(pair, 0u, 0x1010), lo = __byte_perm(pair, 0u, 0x3232);
            if (tail && pair == 0u) w[0] = w[1] = w[2] = w[3] = 0u;  // codes may be NaN's there
            uint32_t f[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) codes_to_f16(w[j], f[2 * j], f[2 * j + 1]);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = hfma2(f[j], hi, hmul2(f[j], lo));
            sts128(c0, f[0], f[1], f[2], f[3]);
            sts128(c0 ^ 16u, f[4], f[5], f[6], f[7]);
          } else {
            // Value rows that a product must not meet: past the end anything may
            // lie there, and a node may hold an infinity or a NaN that its
            // siblings do not see (added to the rows that do see it at the end).
            bool bad = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (pos0 + tok >= g.len) w[j] = 0u;
              if ((w[j] & 0x7f80u) == 0x7f80u) { w[j] &= 0xffff0000u; bad = true; }
              if ((w[j] & 0x7f800000u) == 0x7f800000u) { w[j] &= 0xffffu; bad = true; }
            }
            if (bad) *sm.nonfinite = 1;
            sts128(c0, w[0], w[1], w[2], w[3]);
          }
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(sm.v_full + st);
      if (more) {
        if (!FP8 && !room(sm.v_free, kc + 1)) break;
        copy_v(kc + 1, next_pages);
      }
      copies_commit();
      pages = next_pages;
      next_pages = later_pages;
    }
  }
  copies_wait<0>();
}

// A step of a softmax thread's row in two passes over its scores, the maximum first:
// where keys are hidden, where the row's maximum moves, and for values with a
// reference each.  (A call, so that its registers stay out of the ordinary step's: with
// the keys' references in line the trees of 64 nodes took 185 to 215 us.)
struct StepEnd {
  float m, l;
  bool ok;
};

template <int D, bool FP8>
__device__ __noinline__ StepEnd two_pass_step(uint32_t s_addr, uint32_t o_addr, const float* sc,
                                              const float* refs, float mul, float m, float l,
                                              RowSight sight, int pos0, bool tail, bool has_sums,
                                              uint64_t* pv_bar, uint32_t pv_parity, int* status,
                                              volatile int* abort_flag) {
  constexpr float kUp = FP8 ? 7.f : 0.f;
  bool ok = true;
  float mx = -INFINITY;
#pragma unroll 1
  for (int c0 = 0; c0 < kStep; c0 += 32) {
    uint32_t v[32];
    __syncwarp();
    tmem_ld32_start(s_addr + c0, v);
    tmem_ld32_wait(v);
    const uint32_t seen = tail ? sight.at(pos0 + c0) : 0xffffffffu;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float x = __uint_as_float(v[i]);
      const float t = FP8 ? fmaf(x * sc[c0 + i], mul, refs[c0 + i]) : x * mul;
      mx = fmaxf(mx, seen >> i & 1 ? t : -INFINITY);
    }
  }
  float alpha = 1.f;
  if (mx > m) {
    alpha = ex2(m - mx);
    m = mx;
    l *= alpha;
  }
  if (__any_sync(0xffffffffu, alpha != 1.f) && has_sums) {
    ok = warp_wait(pv_bar, pv_parity, status, abort_flag);
    tc_fence_after();
#pragma unroll 1
    for (int c0 = 0; c0 < D; c0 += 16) {
      float v[16];
      __syncwarp();
      tmem_ld16(o_addr + c0, v);
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * alpha);
      tmem_st16(o_addr + c0, w);
    }
  }
  const float shift = kUp - m;
#pragma unroll 1
  for (int c0 = 0; c0 < kStep; c0 += 32) {
    uint32_t v[32];
    __syncwarp();
    tmem_ld32_start(s_addr + c0, v);
    tmem_ld32_wait(v);
    const uint32_t seen = tail ? sight.at(pos0 + c0) : 0xffffffffu;
    uint32_t w[16];
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float t[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = __uint_as_float(v[i + e]), r = FP8 ? refs[c0 + i + e] : 0.f;
        t[e] = ex2(FP8 ? fmaf(x * sc[c0 + i + e], mul, r + shift) : fmaf(x, mul, shift));
        if (!(seen >> (i + e) & 1)) t[e] = 0.f;
        // (the weights count the values' reference: 2^r of it out again)
        l = FP8 ? fmaf(t[e], ex2(-r), l) : l + t[e];
      }
      w[i / 2] = FP8 ? pack_f16(t[0], t[1]) : pack_bf16(t[0], t[1]);
    }
    tmem_st16(s_addr + c0 / 2, w);
  }
  return {m, l, ok};
}

template <int D, bool FP8>
__global__ void __launch_bounds__(kTileThreads, 1) attn_tiles_kernel(const Args a) {
  using S = TileSmem<D, FP8>;
  constexpr uint32_t kSlab = S::kSlab;
  constexpr float kUp = FP8 ? 7.f : 0.f;  // weights are held as 2^kUp w
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  float* k_scale = reinterpret_cast<float*>(smem + S::kScale);
  float* v_refs = reinterpret_cast<float*>(smem + S::kRefs);
  float* sm_ml = reinterpret_cast<float*>(smem + S::kMl);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
  uint64_t* k_full = bars;        // [2]
  uint64_t* v_full = bars + 2;    // [2]
  uint64_t* k_free = bars + 4;    // [2]
  uint64_t* v_free = bars + 6;    // [2]
  uint64_t* s_full = bars + 8;    // [group][2]
  uint64_t* p_full = bars + 12;   // [group][2]
  uint64_t* pv_done = bars + 16;  // [group][2]
  uint64_t* r_full = bars + 20;   // [kTileBufs]: a tile's scale references
  uint64_t* q_full = r_full + kTileBufs;
  int64_t* pre = reinterpret_cast<int64_t*>(smem + S::kPre);
  __shared__ int64_t s_sum[kTileThreads / 32];
  __shared__ float s_vref[kTileBufs];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_last, s_nonfinite;

  const int tid = threadIdx.x, warp = tid >> 5;
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(k_full + i, 256);
      mbar_init(v_full + i, 256);
      mbar_init(k_free + i, 2);
      mbar_init(v_free + i, 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
      mbar_init(pv_done + i, 1);
    }
    for (int i = 0; i < kTileBufs; ++i) mbar_init(r_full + i, 32);
    mbar_init(q_full, 256);
    fence_mbar_init();
    s_abort = 0;
    s_nonfinite = 0;
  }
  // Tensor memory is taken only once the kernels before are done, and the next
  // one is let in only then: neither ever waits for columns the other holds.
  grid_dep_wait();
  if (warp == 16) {
    tmem_alloc(&s_tmem, 512);
    tmem_relinquish();
  }
  scan_work<kTok, kTileThreads>(a, kTileRows, a.Hkv, pre, s_sum);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  grid_dep_launch();

  const int64_t total = pre[a.B];
  const int64_t piece = max((int64_t)1, divide(total + gridDim.x - 1, gridDim.x));
  const int64_t u0 = (int64_t)blockIdx.x * piece;
  const int64_t u_end = min(total, u0 + piece);
  volatile int* abort_flag = &s_abort;
  // The softmax groups and the warps that issue the scores leave every job together.
  // (A score warp without a tile in a job would not be missed otherwise: two jobs on,
  // the query rows' barrier shows it the parity it had before, and it waits for ever.)
  auto job_end = [] { named_bar_sync(3, 256 + 64); };

  if (warp >= 16) {
    // -------------------------------------------------------------- products
    // Warps 16, 17: scores of the two groups; 18, 19: their sums.  (One warp for all
    // took longer to issue than the products to run.)  A warp walks through its
    // steps together, on values that are the same in every lane: the product
    // instructions take their operands from uniform registers (45 cycles each
    // this way, 110 from one lane's own).  One lane issues.
    fewer_registers<kRegsIssue>();
    auto same = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
    const int w = same(warp & 1), is_sum = same((warp >> 1) & 1);
    const uint32_t tm = (uint32_t)same((int)tmem);
    // (addresses stay below 2^18: offsets add to a descriptor's address field)
    const uint64_t q_desc = umma_desc_sw128((uint32_t)same((int)smem_u32(smem + S::kQ)));
    const uint64_t k_desc = umma_desc_sw128((uint32_t)same((int)smem_u32(smem + S::kK)));
    const uint64_t v_desc = desc_v((uint32_t)same((int)smem_u32(smem + S::kV)), kSlab);
    const bool issuer = elect_one();
    uint64_t* const s_bar = s_full + 2 * w;
    uint64_t* const p_bar = p_full + 2 * w;
    uint64_t* const pv_bar = pv_done + 2 * w;
    int kc0 = 0, seg = 0, n = 0;  // tiles, segments and this group's steps so far
    for (int64_t u = u0; u < u_end;) {
      const Segment g = segment_at(a, pre, u, u_end, piece, *abort_flag != 0);
      u += g.units;
      const int nt = same(g.nt), two = same(g.mt == 2 ? 1 : 0);
      int steps = same(kSpt * group_tiles(nt, two + 1, w));
      if (!is_sum) {
        if (nt > 0 && !warp_wait(q_full, seg++ & 1, a.status, abort_flag)) steps = 0;
        const uint64_t qd = q_desc + (uint32_t)((w & two) * (S::kQTile >> 4));
        for (int j = 0; j < steps; ++j, ++n) {
          const int kc = kc0 + (two ? j / kSpt : w + j / kSpt * 2), sg = kc & 1;
          const int buf = n % kSb, part = j % kSpt;
          // The scores take the place of the weights of kSb steps before.
          if (j >= kSb && !warp_wait(pv_bar + buf, (n / kSb + 1) & 1, a.status, abort_flag)) break;
          if (part == 0 && !warp_wait(k_full + sg, (kc >> 1) & 1, a.status, abort_flag)) break;
          tc_fence_after();
          const uint64_t kd =
              k_desc + (uint32_t)(sg * (S::kKTile >> 4) + part * (kStep * 128 >> 4));
          const uint32_t d = tm + w * 128 + buf * kStep;
          if (issuer) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              if constexpr (FP8) {  // first the high parts of q, then the low ones
                const int half = ks / (D / 32), kk = ks % (D / 32);
                mma_e4m3_ss(d, qd + ((half * kSlab + kk * 32) >> 4), kd + (kk * 32 >> 4),
                            idesc(0, kStep, false), ks != 0);
              } else {
                const uint32_t off = ((ks >> 2) * kSlab + (ks & 3) * 32) >> 4;
                mma_bf16_ss(d, qd + off, kd + off, idesc(1, kStep, false), ks != 0);
              }
            }
            mma_commit(s_bar + buf);
            if (part == kSpt - 1) {  // two arrivals free a tile: one of each reading group
              mma_commit(k_free + sg);
              if (!two) mma_commit(k_free + sg);
            }
          }
          __syncwarp();
        }
        job_end();
      } else {
        for (int j = 0; j < steps; ++j, ++n) {
          const int kc = kc0 + (two ? j / kSpt : w + j / kSpt * 2), sg = kc & 1;
          const int buf = n % kSb, part = j % kSpt;
          // Weights first: they come only after the job before has been finished by both
          // groups, all its tiles of values read.  Until then the values' barrier may be
          // two phases behind this tile's, which a wait on its parity takes for done: with
          // one row tile this group does not wait for the other one's tiles.
          if (!warp_wait(p_bar + buf, (n / kSb) & 1, a.status, abort_flag)) break;
          if (part == 0 && !warp_wait(v_full + sg, (kc >> 1) & 1, a.status, abort_flag)) break;
          tc_fence_after();
          const uint64_t vd =
              v_desc + (uint32_t)(sg * (S::kVTile >> 4) + part * (kStep * 128 >> 4));
          const uint32_t d = tm + 256 + w * 128, p = tm + w * 128 + buf * kStep;
          if (issuer) {
#pragma unroll
            for (int ks = 0; ks < kStep / 16; ++ks)
              mma_bf16_ts(d, p + ks * 8, vd + ks * (2048 >> 4), idesc(FP8 ? 0 : 1, D, true),
                          j > 0 || ks != 0);
            mma_commit(pv_bar + buf);
            if (part == kSpt - 1) {
              mma_commit(v_free + sg);
              if (!two) mma_commit(v_free + sg);
            }
          }
          __syncwarp();
        }
      }
      kc0 += nt;
    }
    __syncwarp();
  } else if (warp >= 8) {
    fewer_registers<kRegsLoad>();
    LoadSmem sm;
    sm.k = smem_u32(smem + S::kK);
    sm.v = smem_u32(smem + S::kV);
    sm.raw = smem_u32(smem + S::kRaw) + (warp - 8) * 16 * D + (tid & 31) * 16;
    sm.pairs = smem_u32(smem + S::kPairs) + (warp - 8) * kTok * 4;
    sm.k_scale = k_scale;
    sm.v_ref = s_vref;
    sm.v_refs = v_refs;
    sm.k_full = k_full;
    sm.v_full = v_full;
    sm.k_free = k_free;
    sm.v_free = v_free;
    sm.r_full = r_full;
    sm.abort_flag = abort_flag;
    sm.nonfinite = &s_nonfinite;
    load_tiles<D, FP8>(a, pre, u0, u_end, piece, sm, (warp - 8) >> 2);
  } else {
    // -------------------------------------------------------------- softmax
    more_registers<kRegsSoftmax>();
    const int wg = warp >> 2;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t o_addr = lane_base + 256 + wg * 128;
    int kc0 = 0, n = 0;  // tiles and this group's steps so far
    for (int64_t u = u0; u < u_end;) {
      const Segment g = segment_at(a, pre, u, u_end, piece, *abort_flag != 0);
      u += g.units;
      // This thread's row.
      const int row = g.mt == 2 ? tid : tid & 127;
      const bool live_row = row < g.rows;
      const bool live_warp = (g.mt == 2 ? warp : warp & 3) * 32 < g.rows;
      const int rr = g.row0 + (live_row ? row : 0);
      const int node = node_of(a, rr);
      const int64_t q_row = g.q_row0 + node;
      const int head = g.h * a.G + rr - node * a.G;
      float row_scale = a.scale_log2;
      // The warp's 32 query rows into shared memory, D / 8 lanes a row.  (Each thread
      // its own row instead: 32 lines an instruction, 5 us before the first product.)
      {
        constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes of a row, rows of a load
        const int lane = tid & 31, c = lane % LPR, sub = lane / LPR;
        const int first = (g.mt == 2 ? warp : warp & 3) * 32;  // its row in the job
        const bool writes = g.mt == 2 || wg == 0;
        const uint32_t dst = smem_u32(smem + S::kQ) + (g.mt == 2 ? wg : 0) * S::kQTile;
        const __nv_bfloat16* q_base =
            a.q + (int64_t)g.q_row0 * a.q_stride + (int64_t)g.h * a.G * D + 8 * c;
        constexpr int kBatch = 8;  // loads in flight
#pragma unroll 1
        for (int i0 = 0; i0 < 32 / RPI; i0 += kBatch) {
          uint4 y[kBatch];
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int r = first + (i0 + i) * RPI + sub;
            const int node = node_of(a, g.row0 + r);
            y[i] = make_uint4(0u, 0u, 0u, 0u);
            if (r < g.rows)
              y[i] = *reinterpret_cast<const uint4*>(
                  q_base + node * a.q_stride + (g.row0 + r - node * a.G) * D);
          }
          float up[kBatch];
          if constexpr (FP8) {
            uint32_t top[kBatch];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
              const uint32_t both = __vmaxu2(__vmaxu2(y[i].x & 0x7fff7fffu, y[i].y & 0x7fff7fffu),
                                             __vmaxu2(y[i].z & 0x7fff7fffu, y[i].w & 0x7fff7fffu));
              top[i] = max(both & 0xffffu, both >> 16);
            }
#pragma unroll
            for (int o = 1; o < LPR; o <<= 1)
#pragma unroll
              for (int i = 0; i < kBatch; ++i)
                top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
              const QScale qs = q_scale(top[i]);
              up[i] = qs.up;
              // (for the thread that has this row)
              const float down = __shfl_sync(0xffffffffu, qs.down, lane % RPI * LPR);
              if (lane / RPI == i0 + i) row_scale *= down;
            }
          }
          if (!writes) continue;
#pragma unroll
          for (int i = 0; i < kBatch; ++i) {
            const int r = (first + (i0 + i) * RPI + sub) & 127;
            if constexpr (FP8) {
              uint32_t hi[2], lo[2];
              split_e4m3(y[i].x, y[i].y, up[i], hi[0], lo[0]);
              split_e4m3(y[i].z, y[i].w, up[i], hi[1], lo[1]);
              const uint32_t at = dst + r * 128 + (((c >> 1) ^ (r & 7)) << 4) + (c & 1) * 8;
              sts64(at, hi[0], hi[1]);
              sts64(at + kSlab, lo[0], lo[1]);
            } else {
              sts128(dst + (c >> 3) * kSlab + r * 128 + (((c & 7) ^ (r & 7)) << 4), y[i].x, y[i].y,
                     y[i].z, y[i].w);
            }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        if (g.nt > 0) mbar_arrive(q_full);
      }
      RowSight sight;
      sight.len = g.len;
      sight.ctx = g.ctx;
      sight.node = node;
      sight.masked = a.masks != nullptr;
      sight.mask = sight.masked && live_row ? (uint64_t)a.masks[q_row] : 0;

      float m = kNegBig, l = 0.f;
      const int tiles = group_tiles(g.nt, g.mt, wg);
      bool ok = true;
      for (int j = 0; j < kSpt * tiles; ++j, ++n) {
        const int kt = g.mt == 2 ? j / kSpt : wg + j / kSpt * 2;
        const int buf = n % kSb;
        const int kc = kc0 + kt;
        const int pos0 = (g.k0 + kt) * kTok + j % kSpt * kStep;
        const uint32_t s_addr = lane_base + wg * 128 + buf * kStep;
        ok = warp_wait(s_full + 2 * wg + buf, (n / kSb) & 1, a.status, abort_flag) &&
             (!FP8 || j % kSpt != 0 || warp_wait(r_full + (kc & (kTileBufs - 1)), (kc / kTileBufs) & 1, a.status,
                                   abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (live_warp) {
          // Score in base 2, with log2 of the values' reference, less `shift`.
          const float mul = row_scale;
          const float lv = FP8 ? s_vref[kc & (kTileBufs - 1)] : 0.f;
          const float* sc = k_scale + (kc & (kTileBufs - 1)) * kTok + j % kSpt * kStep;
          const bool tail = pos0 + kStep > g.ctx;
          const bool wide = FP8 && lv == kEachItsOwn;
          const float* refs = v_refs + (kc & (kTileBufs - 1)) * kTok + j % kSpt * kStep;
          bool again = __any_sync(0xffffffffu, tail || wide || m == kNegBig);
          float sum = 0.f;
          if (!again) {
            const F2 mul2v = f2(mul, mul);
            const float shift = lv + kUp - m;
            const F2 shift2 = f2(shift, shift);
            F2 sum2 = f2(0.f, 0.f);
            float mx = -INFINITY;
            uint32_t p[kStep / 2];
            uint32_t v[2][32];
            tmem_ld32_start(s_addr, v[0]);
#pragma unroll
            for (int c = 0; c < kStep / 32; ++c) {
              tmem_ld32_wait(v[c & 1]);
              if (c + 1 < kStep / 32) tmem_ld32_start(s_addr + 32 * (c + 1), v[(c + 1) & 1]);
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const uint32_t* y = v[c & 1] + i;
                F2 x0 = f2(__uint_as_float(y[0]), __uint_as_float(y[1]));
                F2 x1 = f2(__uint_as_float(y[2]), __uint_as_float(y[3]));
                if constexpr (FP8) {
                  const float4 k4 = *reinterpret_cast<const float4*>(sc + 32 * c + i);
                  x0 = mul2(x0, f2(k4.x, k4.y));
                  x1 = mul2(x1, f2(k4.z, k4.w));
                }
                x0 = fma2(x0, mul2v, shift2);
                x1 = fma2(x1, mul2v, shift2);
                float t[4];
                split(x0, t[0], t[1]);
                split(x1, t[2], t[3]);
                mx = fmaxf(fmaxf(mx, fmaxf(t[0], t[1])), fmaxf(t[2], t[3]));
#pragma unroll
                for (int e = 0; e < 4; ++e) t[e] = ex2(t[e]);
                sum2 = add2(sum2, add2(f2(t[0], t[1]), f2(t[2], t[3])));
                p[16 * c + i / 2] = FP8 ? pack_f16(t[0], t[1]) : pack_bf16(t[0], t[1]);
                p[16 * c + i / 2 + 1] = FP8 ? pack_f16(t[2], t[3]) : pack_bf16(t[2], t[3]);
              }
            }
            again = __any_sync(0xffffffffu, mx > 8.f + kUp);
            if (!again) {
#pragma unroll
              for (int c = 0; c < kStep / 2; c += 16) {
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i] = p[c + i];
                tmem_st16(s_addr + c, w);
              }
              float s0, s1;
              split(sum2, s0, s1);
              sum = s0 + s1;
            }
          }
          if (again) {
            const StepEnd e = two_pass_step<D, FP8>(
                s_addr, o_addr, sc, refs, mul, m, l, sight, pos0, tail, j > 0,
                pv_done + 2 * wg + (n - 1) % kSb, ((n - 1) / kSb) & 1, a.status, abort_flag);
            m = e.m;
            l = e.l;
            ok = e.ok;
          } else {
            // (the weights count the values' reference: 2^lv of it out again)
            l += FP8 ? sum * ex2(-lv) : sum;
          }
          tmem_st_wait();
        }
        if (!ok) break;
        tc_fence_before();
        mbar_arrive(p_full + 2 * wg + buf);
      }
      if (tiles > 0 && ok)
        ok = warp_wait(pv_done + 2 * wg + (n - 1) % kSb, ((n - 1) / kSb) & 1, a.status, abort_flag);
      tc_fence_after();
      // Join the groups (one row tile) and the CTAs that share the job.
      sm_ml[(wg * 128 + (tid & 127)) * 2] = m;
      sm_ml[(wg * 128 + (tid & 127)) * 2 + 1] = l;
      tc_fence_before();
      named_bar_sync(2, 256);
      tc_fence_after();
      ok = ok && !*abort_flag;
      const bool whole = g.c0 == g.c1;
      const int64_t c0 = g.c0, c1 = g.c1;
      // With one row tile each group joins and stores half of the dims.
      const int d_lo = g.mt == 2 ? 0 : wg * (D / 2), d_hi = g.mt == 2 ? D : d_lo + D / 2;
      float* slot = a.part + ((int64_t)blockIdx.x * 2 + (blockIdx.x == c0 ? 1 : 0)) * kTileRows *
                                 (D + 2);
      auto put = [&](int d, float (&y)[16], float inv, bool none) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 16; ++i) y[i] = none ? 0.f : y[i] * inv;
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
          w[i / 2] = pack_bf16(y[i], y[i + 1]);
          w[i / 2 + 1] = pack_bf16(y[i + 2], y[i + 3]);
        }
        __nv_bfloat16* dst = a.out + q_row * a.out_stride + (int64_t)head * D + d;
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
        float f[2] = {0.f, 0.f}, M = m, L = l;
        if (g.mt == 2) {
          f[wg] = 1.f;
        } else {
          const float m0 = sm_ml[r * 2], m1 = sm_ml[(128 + r) * 2];
          M = fmaxf(m0, m1);
          f[0] = ex2(m0 - M);
          f[1] = ex2(m1 - M);
          L = sm_ml[r * 2 + 1] * f[0] + sm_ml[(128 + r) * 2 + 1] * f[1];
        }
        if (!whole && live_row && (g.mt == 2 || wg == 0)) {
          slot[row] = M;
          slot[kTileRows + row] = L;
        }
        const bool more = !FP8 && *(volatile int*)&s_nonfinite;
#pragma unroll 1
        for (int d = d_lo; d < d_hi; d += 16) {
          float y[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) y[i] = 0.f;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if ((g.mt == 2 && w != wg) || group_tiles(g.nt, g.mt, w) == 0) continue;
            float v[16];
            __syncwarp();
            tmem_ld16(lane_base + 256 + w * 128 + d, v);
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = fmaf(v[i], f[w], y[i]);
          }
          if (more && live_row) {
            // The infinities and NaNs that were kept out of the products.
            const int last = min((g.k0 + g.nt) * kTok, g.len);
            for (int pos = max(g.k0, g.ctx / kTok) * kTok; pos < last; ++pos) {
              if (!(sight.at(pos) & 1)) continue;
              const int64_t vr =
                  ((a.layer_blocks + g.table[pos >> 4]) * a.Hkv + g.h) * 16 + (pos & 15);
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
            put(d, y, 1.f / L, L == 0.f);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) slot[(2 + d + i) * kTileRows + row] = y[i];
          }
        }
      }
      if (!whole) {
        __threadfence();
        named_bar_sync(2, 256);
        if (tid == 0) {
          s_last = atomicAdd(a.counters + c0, 1) == (int)(c1 - c0);
          if (s_last) a.counters[c0] = 0;
        }
        named_bar_sync(2, 256);
        if (s_last && live_row && ok) {
          __threadfence();
          constexpr int P = 4;  // parts whose loads are in flight together
          auto part_of = [&](int64_t c) {
            return a.part + (c * 2 + (c == c0 ? 1 : 0)) * kTileRows * (D + 2) + row;
          };
          float M = kNegBig, L = 0.f;
          for (int64_t c = c0; c <= c1; c += P) {
            float pm[P], pl[P], m_new = M;
#pragma unroll
            for (int i = 0; i < P; ++i) {
              pm[i] = c + i <= c1 ? __ldcg(part_of(c + i)) : kNegBig;
              pl[i] = c + i <= c1 ? __ldcg(part_of(c + i) + kTileRows) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < P; ++i) m_new = fmaxf(m_new, pm[i]);
            L *= ex2(M - m_new);
#pragma unroll
            for (int i = 0; i < P; ++i) L += pl[i] * ex2(pm[i] - m_new);
            M = m_new;
          }
#pragma unroll 1
          for (int d = d_lo; d < d_hi; d += 16) {
            float y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = 0.f;
            for (int64_t c = c0; c <= c1; c += P) {
              float v[P][16], f[P];
#pragma unroll
              for (int k = 0; k < P; ++k) {
                f[k] = c + k <= c1 ? ex2(__ldcg(part_of(c + k)) - M) : 0.f;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  v[k][i] = c + k <= c1 ? __ldcg(part_of(c + k) + (2 + d + i) * kTileRows) : 0.f;
              }
#pragma unroll
              for (int k = 0; k < P; ++k)
#pragma unroll
                for (int i = 0; i < 16; ++i) y[i] = fmaf(v[k][i], f[k], y[i]);
            }
            put(d, y, 1.f / L, L == 0.f);
          }
        }
      }
      kc0 += g.nt;
      // The next job's query rows and statistics take the same places: not
      // before both groups are done with these.
      tc_fence_before();
      job_end();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 16) tmem_dealloc(tmem, 512);
}

template <int D, bool FP8>
void launch_tiles(const Args& a, cudaStream_t stream) {
  const int smem = TileSmem<D, FP8>::bytes(a.B);
  static PerDevice allowed, checked;
  allow_smem(attn_tiles_kernel<D, FP8>, TileSmem<D, FP8>::bytes(kMaxBatch), allowed);
  checked.once(0, [] {
    cudaFuncAttributes attr;
    CB_CUDA_CHECK(cudaFuncGetAttributes(&attr, attn_tiles_kernel<D, FP8>));
    if (attr.numRegs < kRegsLaunch)  // the groups' shares would never come free
      throw std::runtime_error("attn_tiles_kernel was built with too few registers a thread");
  });
  launch_kernel(attn_tiles_kernel<D, FP8>, dim3(num_sms()), dim3(kTileThreads), smem, stream, a);
}

template void launch_tiles<64, false>(const Args&, cudaStream_t);
template void launch_tiles<64, true>(const Args&, cudaStream_t);
template void launch_tiles<128, false>(const Args&, cudaStream_t);
template void launch_tiles<128, true>(const Args&, cudaStream_t);

}  // namespace tree
}  // namespace cb

// What the attention kernels over new tokens share: arguments, the split of the
// work, and small device helpers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "mma_frag.cuh"

namespace cb {
namespace tree {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegBig = -1e30f;
constexpr int kMaxBatch = 2048;

struct Args {
  const __nv_bfloat16* q;
  int64_t q_stride;
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  const int* table;
  int64_t table_stride;
  int table_width;
  const int* seq_lens;
  const int* row_start;
  const int64_t* masks;
  __nv_bfloat16* out;
  int64_t out_stride;
  float* part;    // two partial results for each CTA
  int* counters;  // [grid], zero between launches
  int* status;
  int64_t layer_blocks;
  int B, Hkv, G;
  uint32_t per_g;  // 2^32 / G, rounded up; 0 for G = 1
  int out_vec;  // output rows are 16-byte aligned
  float scale_log2;
};

// Four codes as fp16, exact: those of the word's lower half, those of its upper half.
// (The conversion runs at the rate of an integer instruction; moving the bits into place
// takes three and a half for every pair.)
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\n"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The power of two that puts a query row's largest value into [2^7, 2^8), from the
// bits of its largest bf16 magnitude, and the way back.  A row with an infinity or
// a NaN gets NaN scores.
struct QScale {
  float up, down;
};
__device__ __forceinline__ QScale q_scale(uint32_t top) {
  const int e = (int)(top >> 7);
  const int sh = e == 0 || e == 255 ? 0 : min(100, 127 + 7 - e);
  QScale s;
  s.up = __int_as_float((127 + sh) << 23);
  s.down = e == 255 ? __int_as_float(0x7fc00000) : __int_as_float((127 - sh) << 23);
  return s;
}

// Four bf16 values (two words) times `up` as e4m3 numbers: hi + lo has all eight
// bits of a value that is at least 2^-9 of the row's largest, and is within 2^-18
// of the largest otherwise.
__device__ __forceinline__ void split_e4m3(uint32_t a0, uint32_t a1, float up, uint32_t& hi,
                                           uint32_t& lo) {
  const float x[4] = {__uint_as_float(a0 << 16) * up, __uint_as_float(a0 & 0xffff0000u) * up,
                      __uint_as_float(a1 << 16) * up, __uint_as_float(a1 & 0xffff0000u) * up};
  uint32_t h = 0u, l = 0u;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t h8 = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * k], x[2 * k + 1]),
                                                 __NV_SATFINITE, __NV_E4M3);
    const float2 back =
        __half22float2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)h8, __NV_E4M3));
    const uint32_t l8 = __nv_cvt_float2_to_fp8x2(
        make_float2(x[2 * k] - back.x, x[2 * k + 1] - back.y), __NV_SATFINITE, __NV_E4M3);
    h |= h8 << (16 * k);
    l |= l8 << (16 * k);
  }
  hi = h;
  lo = l;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Asynchronous copies global -> shared, each lane for itself.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Node of a query row, node * G + head of the group, below 2^32 / G.
__device__ __forceinline__ int node_of(const Args& a, int r) {
  return a.G == 1 ? r : (int)__umulhi((uint32_t)r, a.per_g);
}

// n rows, len keys in nb units of UNIT tokens (one at least), read by `tiles`
// row tiles.
struct SeqShape {
  int n, len, nb, tiles;
};

template <int UNIT>
__device__ __forceinline__ SeqShape seq_shape(const Args& a, int b, int rows) {
  SeqShape s;
  s.n = max(0, a.row_start[b + 1] - a.row_start[b]);
  s.len = min(max(0, a.seq_lens[b]), a.table_width * 16);
  s.nb = max(1, (s.len + UNIT - 1) / UNIT);
  s.tiles = (s.n * a.G + rows - 1) / rows;
  return s;
}

// pre[b] = units of work of `heads` kv heads before sequence b; pre[B] = all of it.
// seqs[b], if asked for: its keys and first row; seqs[B].y: the end of the rows.
template <int UNIT, int THREADS>
__device__ __forceinline__ void scan_work(const Args& a, int rows, int heads, int64_t* pre,
                                          int64_t* warp_sum, int2* seqs = nullptr) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t carry = 0;
  if (tid == 0) pre[0] = 0;
  for (int base = 0; base < a.B; base += THREADS) {
    const int b = base + tid;
    int64_t u = 0;
    if (b < a.B) {
      const SeqShape s = seq_shape<UNIT>(a, b, rows);
      u = (int64_t)heads * s.tiles * s.nb;
      if (seqs != nullptr) {
        const int row0 = a.row_start[b];
        seqs[b] = make_int2(s.len, row0);
        if (b == a.B - 1) seqs[a.B] = make_int2(0, row0 + s.n);
      }
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, u, o);
      if (lane >= o) u += x;
    }
    if (lane == 31) warp_sum[warp] = u;
    __syncthreads();
    int64_t before = carry;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) before += warp_sum[w];
      carry += warp_sum[w];
    }
    if (b < a.B) pre[b + 1] = before + u;
    __syncthreads();
  }
}

// The sequence that unit u belongs to: pre[b] <= u < pre[b + 1].  Sequences
// without rows share their successor's offset: the search ends on the last of
// them, the one with the work.
__device__ __forceinline__ int find_seq(const int64_t* pre, int B, int64_t u) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= u) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Work is counted in 64 bits but hardly ever needs them.
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if (((a | b) >> 32) == 0) return (int64_t)((uint32_t)a / (uint32_t)b);
  return a / b;
}

// More than 16 query rows of a kv head and sequence.
template <int D, bool FP8>
void launch_tiles(const Args& a, cudaStream_t stream);

}  // namespace tree
}  // namespace cb

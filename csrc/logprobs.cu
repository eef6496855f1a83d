// Log-probabilities of given tokens, entropy and the top alternatives of logit
// rows, in one pass over the logits.
//
//   S = sum 2^(x log2e - r),  W = sum 2^(x log2e - r) (x log2e - r)
//   log2 p(t) = (x_t log2e - r) - log2 S,   entropy = ln 2 (log2 S - W / S)
//
// hold for every reference r near the row's maximum: each thread keeps its own
// (r, S, W) and moves r only when a value is 2^8 times over it, so the common
// path is one fused multiply-add and one exponential a value.  The same r stands
// in every term, so its own rounding cancels, as long as 2^(that rounding) is a
// finite number: below 2^30 r is rounded by 2^5 at most, so S stays below 2^72.
// If the row's maximum is 2^29 or more in magnitude, other floats are so far from it
// (32 at least) that S is the number of values equal to it.  At the end r moves to the
// maximum itself, the thread's and then the row's.  Values of -2^30 or
// less beside a maximum above -2^29 weigh nothing in any frame, and set none.
//
// Top k: each thread notes the chunk of its own largest value.  Of the largest
// values of 32 groups of threads the k-th is a bound below the row's k-th largest,
// and only threads whose own largest value reaches it can hold any of the row's
// top k: their values alone are read a second time, and the few that reach the bound
// are ranked by counting, each against all.  (Sorting the threads' maxima instead, for
// a tighter bound, cost more than the few values it spared.)  Order: larger value
// first, then lower index (-0 = 0; a NaN comes before everything).
//
// A row is cut in slices, one for each CTA, when there are few rows; the last
// CTA of a row joins them.
//
// Bound: memory for many rows (2047 rows of 128256 bf16 logits, 525 MB: 98 us without
// alternatives, 5.3 TB/s; 110 us with one), where the exponentials take about 60 us and
// 16-bit logits' maxima are taken two at a time.  Latency for few: one row 9 us with
// alternatives, 64 rows 16 us, for two trips to memory, two joins of a CTA and a launch.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cfloat>

#include "common.cuh"
#include "host_utils.h"

namespace cb {
namespace lp {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 32;
constexpr int kCand = 1024;
constexpr float kLog2e = 1.4426950408889634f;

using Key = unsigned long long;  // ordered value, then inverted index

struct Args {
  const void* x;
  int64_t ld;
  int V, slices, slice_len, top_k;
  const int* tokens;
  float* logprob;
  float* entropy;
  int* top_ids;
  float* top_lp;
  float* part;  // [R][slices][4 + 2 * kMaxTop]: m, r, S, W, keys
  int* counters;
};

__device__ __forceinline__ uint32_t order_bits(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);  // -0 becomes 0
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t o) {
  if (o == 0xffffffffu) return __int_as_float(0x7fc00000);
  return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ Key make_key(float x, int i) {
  return ((Key)order_bits(x) << 32) | (uint32_t)~i;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Descending sort of one key a lane.
__device__ __forceinline__ Key warp_sort(Key v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      const Key o = __shfl_xor_sync(0xffffffffu, v, stride);
      const bool first = (lane & stride) == 0;
      const bool down = (lane & size) == 0;
      v = (first == down) ? (v > o ? v : o) : (v > o ? o : v);
    }
  }
  return v;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ Key warp_merge(Key a, Key b) {
  const int lane = threadIdx.x & 31;
  const Key r = __shfl_sync(0xffffffffu, b, 31 - lane);
  Key v = a > r ? a : r;
#pragma unroll
  for (int stride = 16; stride > 0; stride >>= 1) {
    const Key o = __shfl_xor_sync(0xffffffffu, v, stride);
    v = (lane & stride) == 0 ? (v > o ? v : o) : (v > o ? o : v);
  }
  return v;
}
// The 32 largest of every warp's descending list, in every warp's registers.
__device__ __forceinline__ Key block_merge(Key v, Key* lists) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int n = kWarps; n > 1; n >>= 1) {
    __syncthreads();
    lists[threadIdx.x] = v;
    __syncthreads();
    if (warp < n / 2) v = warp_merge(v, lists[(warp + n / 2) * 32 + lane]);
  }
  __syncthreads();
  if (warp == 0) lists[lane] = v;
  __syncthreads();
  return lists[lane];
}

// The k-th largest of 32 groups' largest keys, groups by lane (the lowest indices of
// equal values, in the first warp's chunks, are in groups of their own): at least k
// keys reach it.  Zero if there are fewer than k groups with a key.
__device__ __forceinline__ Key block_bound(Key key, int k, Key* lists) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  lists[threadIdx.x] = key;
  __syncthreads();
  if (warp == 0) {
#pragma unroll
    for (int w = 1; w < kWarps; ++w) {
      const Key o = lists[w * 32 + lane];
      key = o > key ? o : key;
    }
    __syncwarp();
    lists[lane] = key;
    __syncwarp();
    int before = 0;
#pragma unroll 8
    for (int i = 0; i < 32; ++i) before += lists[i] > key || (lists[i] == key && i < lane);
    __syncwarp();
    if (before == k - 1) lists[0] = key;
  }
  __syncthreads();
  return lists[0];
}

// Candidates by their place: out[0 .. k) = the k largest keys, descending (all
// different; zeros after the last).
__device__ __forceinline__ void block_rank(const Key* cand, int count, int k, Key* out) {
  if (threadIdx.x < 32) out[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kThreads) {
    const Key key = cand[i];
    int before = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) before += cand[j] > key;
    if (before < k) out[before] = key;
  }
  __syncthreads();
}

// Running sums in the frame r; m is the largest value so far.
struct Stat {
  float m, r, s, w;
};
constexpr float kLowest = -1073741824.f;  // -2^30: r of a thread without a larger value
constexpr float kHuge = 536870912.f;      // 2^29

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  Stat o;
  o.m = max_nan(a.m, b.m);
  o.r = fmaxf(a.r, b.r);
  const float da = fmaxf(a.r - o.r, -200.f), db = fmaxf(b.r - o.r, -200.f);
  const float fa = ex2(da), fb = ex2(db);
  o.s = a.s * fa + b.s * fb;
  o.w = fa * fmaf(a.s, da, a.w) + fb * fmaf(b.s, db, b.w);
  return o;
}
__device__ __forceinline__ Stat warp_join(Stat v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat u;
    u.m = __shfl_xor_sync(0xffffffffu, v.m, o);
    u.r = __shfl_xor_sync(0xffffffffu, v.r, o);
    u.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    u.w = __shfl_xor_sync(0xffffffffu, v.w, o);
    v = join(v, u);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ float value(const T* p) {
  if constexpr (std::is_same<T, float>::value) return *p;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
  else return __bfloat162float(*p);
}

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// 16 bytes of logits as floats.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
  float v[N];
  // The largest of them, a NaN if there is one; with the values no lower than -2^30
  // from here on if that comes cheap (`bounded`).
  static constexpr bool bounded = std::is_same<T, __nv_bfloat16>::value;
  __device__ __forceinline__ float set_top(uint4 u) {
    if constexpr (bounded) {
      const uint32_t t = max_nan_bf16x2(max_nan_bf16x2(u.x, u.y), max_nan_bf16x2(u.z, u.w));
      constexpr uint32_t kLow = 0xce80ce80u;  // -2^30, twice
      u.x = max_bf16x2(u.x, kLow);
      u.y = max_bf16x2(u.y, kLow);
      u.z = max_bf16x2(u.z, kLow);
      u.w = max_bf16x2(u.w, kLow);
      set(u);
      return max_nan(__uint_as_float(t << 16), __uint_as_float(t & 0xffff0000u));
    } else {
      set(u);
      float top = v[0];
#pragma unroll
      for (int i = 1; i < N; ++i) top = max_nan(top, v[i]);
      return top;
    }
  }
  __device__ __forceinline__ void set(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, float>::value) {
        v[i] = __uint_as_float(w[i]);
      } else if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
};

// CTAS of an SM: 2 leave a thread 64 registers, its loads of four chunks and the sums
// of the last ones side by side; 3 are better where an SM works through many rows, and
// the end of one hides behind the others (2047 rows of 128256: 110 us against 122;
// 64 rows of 151936: 17.4 against 15.9).
template <typename T, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) token_logprobs_kernel(const Args a) {
  constexpr int N = Chunk<T>::N;
  constexpr int U = 4;  // chunks in flight for each thread
  __shared__ Key lists[kThreads];
  __shared__ Key cand[kCand];
  __shared__ Stat stats[kWarps];
  __shared__ uint16_t owners[kThreads];
  __shared__ int s_count, s_owners, s_last;
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y, slice = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ld;
  const int lo = min(a.V, slice * a.slice_len), hi = min(a.V, lo + a.slice_len);
  // [lo, v0): before the first 16-byte boundary; [v0, v1): whole chunks.
  const int skew = (int)((reinterpret_cast<uintptr_t>(x + lo) & 15) / sizeof(T));
  const int v0 = min(hi, lo + (skew ? N - skew : 0));
  const int chunks = (hi - v0) / N;
  const int v1 = v0 + chunks * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + v0);
  if (tid == 0) s_count = s_owners = 0;

  Stat st = {-INFINITY, kLowest, 0.f, 0.f};
  int best = tid;  // chunk of the largest value among the chunks
  float best_v = -INFINITY;
  bool nan = false;
  auto raise = [&](float top) {
    const float r = top * kLog2e;
    const float d = fmaxf(st.r - r, -200.f);
    const float f = ex2(d);
    st.w = f * fmaf(st.s, d, st.w);
    st.s *= f;
    st.r = r;
  };
  auto add = [&](float v, bool bounded, float& s, float& w) {
    float d = fmaf(v, kLog2e, -st.r);
    if (!bounded) d = fmaxf(d, -200.f);  // -inf: a weight of 0, not a NaN
    const float e = ex2(d);
    s += e;
    w = fmaf(e, d, w);
  };
  auto take = [&](const uint4& raw, int c) {
    Chunk<T> u;
    const float top = u.set_top(raw);
    nan |= top != top;
    if (top > best_v) {
      best_v = top;
      best = c;
    }
    if (top * kLog2e > st.r + 8.f && top < kHuge) raise(top);
    // A chunk's sums on their own first: W counts the lag of r, up to 8 S, and every sum
    // with it is rounded by that much.
    float s = 0.f, w = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) add(u.v[i], Chunk<T>::bounded, s, w);
    st.s += s;
    st.w += w;
  };
  // Edges: fewer than 2 N elements, one for each of the first threads.
  const int n0 = v0 - lo;
  const int edge = tid < n0 ? lo + tid : (tid - n0 < hi - v1 ? v1 + tid - n0 : -1);
  float edge_v = -INFINITY;
  if (edge >= 0) {
    edge_v = value(x + edge);
    nan |= edge_v != edge_v;
    if (edge_v * kLog2e > st.r && edge_v < kHuge) raise(edge_v);
    add(edge_v, false, st.s, st.w);
  }
  int c = tid;
  for (; c + (U - 1) * kThreads < chunks; c += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i) raw[i] = __ldg(xv + c + i * kThreads);
#pragma unroll
    for (int i = 0; i < U; ++i) take(raw[i], c + i * kThreads);
  }
  {
    uint4 raw[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (c + i * kThreads < chunks) raw[i] = __ldg(xv + c + i * kThreads);
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (c + i * kThreads < chunks) take(raw[i], c + i * kThreads);
  }
  st.m = nan ? __int_as_float(0x7fc00000) : fmaxf(best_v, edge_v);
  if (st.m * kLog2e > st.r && st.m < kHuge) raise(st.m);  // no lag from here on

  // This thread's largest value with its index.
  Key key = 0;
  auto chunk_keys = [&](int at, auto&& use) {
    Chunk<T> u;
    u.set(__ldg(xv + at));
#pragma unroll
    for (int i = 0; i < N; ++i) use(make_key(u.v[i], v0 + at * N + i));
  };
  auto keep_largest = [&](Key k2) { key = k2 > key ? k2 : key; };
  if (a.top_k > 0) {
    if (edge >= 0) key = make_key(edge_v, edge);
    if (nan) {
      for (int i = tid; i < chunks; i += kThreads) chunk_keys(i, keep_largest);
    } else if (best < chunks) {
      chunk_keys(best, keep_largest);
    }
  }

  st = warp_join(st);
  if (lane == 0) stats[warp] = st;
  Key top = 0;
  if (a.top_k > 0) {
    const Key bound = block_bound(key, a.top_k, lists);
    auto offer = [&](Key k2) {
      if (k2 >= bound && k2 > 0) {
        const int at = atomicAdd(&s_count, 1);
        if (at < kCand) cand[at] = k2;
      }
    };
    if (edge >= 0) offer(make_key(edge_v, edge));
    if (key >= bound && key > 0) owners[atomicAdd(&s_owners, 1)] = (uint16_t)tid;
    __syncthreads();
    const int each = (chunks + kThreads - 1) / kThreads, all = s_owners * each;
    for (int i = tid; i < all; i += kThreads) {
      const int at = owners[i / each] + i % each * kThreads;
      if (at < chunks) chunk_keys(at, offer);
    }
    __syncthreads();
    const int count = s_count;
    if (count <= kCand) {
      block_rank(cand, count, a.top_k, lists);
      top = lists[lane];
    } else {
      // More values over the bound than the list holds (many of a row's
      // largest values in a few threads' chunks): one pass for each place.
      Key last = ~(Key)0;
      for (int j = 0; j < a.top_k; ++j) {
        key = edge >= 0 ? make_key(edge_v, edge) : 0;
        if (key >= last) key = 0;
        for (int i = tid; i < chunks; i += kThreads)
          chunk_keys(i, [&](Key k2) { key = k2 < last && k2 > key ? k2 : key; });
        const Key found = block_merge(warp_sort(key), lists);
        last = __shfl_sync(0xffffffffu, found, 0);
        if (lane == j) top = last;
      }
    }
  } else {
    __syncthreads();
  }
  if (warp == 0) {
    st = lane < kWarps ? stats[lane] : Stat{-INFINITY, kLowest, 0.f, 0.f};
    st = warp_join(st);
  }

  if (a.slices > 1) {
    constexpr int P = 4 + 2 * kMaxTop;
    float* part = a.part + ((int64_t)row * a.slices + slice) * P;
    if (warp == 0) {
      if (lane == 0) *reinterpret_cast<float4*>(part) = make_float4(st.m, st.r, st.s, st.w);
      if (lane < a.top_k) reinterpret_cast<Key*>(part + 4)[lane] = top;
      __threadfence();
      __syncwarp();
      if (lane == 0) {
        s_last = atomicAdd(a.counters + row, 1) == a.slices - 1;
        if (s_last) a.counters[row] = 0;
      }
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    const float* parts = a.part + (int64_t)row * a.slices * P;
    if (a.top_k > 0) {
      // The same again, with the slices' lists for the threads' chunks.
      auto list = [&](int i) { return reinterpret_cast<const Key*>(parts + (int64_t)i * P + 4); };
      if (tid == 0) s_count = 0;
      key = 0;
      for (int i = tid; i < a.slices; i += kThreads) keep_largest(__ldcg(list(i)));
      const Key bound = block_bound(key, a.top_k, lists);
      for (int i = tid; i < a.slices * a.top_k; i += kThreads) {
        const Key k2 = __ldcg(list(i / a.top_k) + i % a.top_k);
        if (k2 >= bound && k2 > 0) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kCand) cand[at] = k2;
        }
      }
      __syncthreads();
      if (s_count <= kCand) {
        block_rank(cand, s_count, a.top_k, lists);
        top = lists[lane];
      } else {
        top = 0;
        for (int i = warp; i < a.slices; i += kWarps)
          top = warp_merge(top, lane < a.top_k ? __ldcg(list(i) + lane) : 0);
        top = block_merge(top, lists);
      }
    }
    if (warp == 0) {
      st = {-INFINITY, kLowest, 0.f, 0.f};
      for (int i = lane; i < a.slices; i += 32) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(parts + i * P));
        st = join(st, Stat{f.x, f.y, f.z, f.w});
      }
      st = warp_join(st);
    }
  }

  // From here on warp 0 holds the row's sums and list.
  if (warp == 0 && lane == 0) stats[0] = st;
  __syncthreads();
  const float m = stats[0].m;
  // NaN or +inf in the row: no distribution.  Nothing but -inf: every token
  // has probability 0.
  const bool bad = !(m < INFINITY), empty = m == -INFINITY;
  const bool far = !bad && !empty && fabsf(m) >= kHuge;
  if (far) {
    int same = 0;
    for (int i = tid; i < a.V; i += kThreads) same += value(x + i) == m;
    same = __reduce_add_sync(0xffffffffu, same);
    if (lane == 0) lists[warp] = same;
    __syncthreads();
    if (tid == 0) {
      Key total = 0;
      for (int w = 0; w < kWarps; ++w) total += lists[w];
      stats[0] = Stat{m, 0.f, (float)total, 0.f};
    }
    __syncthreads();
    st = stats[0];
  }
  if (warp != 0) return;
  // From the rounded reference to the maximum: S counts the maximum itself as 1 and is
  // no less, so that no probability passes 1 and no entropy falls below 0.
  if (!bad && !empty && !far) {
    const float d = fmaf(m, kLog2e, -st.r), f = ex2(-d);
    st.w = f * fmaf(-st.s, d, st.w);
    st.s *= f;
  }
  constexpr float kLn2 = 0.6931471805599453f;
  const float log2_s = log2f(fmaxf(st.s, 1.f));
  const float none = __int_as_float(0x7fc00000);
  auto lp_of = [&](float v) {
    if (bad) return none;
    if (empty) return -INFINITY;
    return fmaf(-log2_s, kLn2, v - m);
  };
  if (lane == 0) {
    const int t = a.tokens[row];
    a.logprob[row] = t >= 0 && t < a.V ? lp_of(value(x + t)) : none;
    a.entropy[row] = bad ? none : (empty ? 0.f : fmaxf(log2_s - st.w / st.s, 0.f) * kLn2);
  }
  if (lane < a.top_k) {
    a.top_ids[(int64_t)row * a.top_k + lane] = (int)~(uint32_t)top;
    a.top_lp[(int64_t)row * a.top_k + lane] = lp_of(order_value((uint32_t)(top >> 32)));
  }
}

template <typename T>
void launch(const Args& a, int rows, cudaStream_t stream) {
  const dim3 grid((unsigned)a.slices, (unsigned)rows), block(kThreads);
  if (rows >= 8 * num_sms())
    launch_kernel(token_logprobs_kernel<T, 3>, grid, block, 0, stream, a);
  else
    launch_kernel(token_logprobs_kernel<T, 2>, grid, block, 0, stream, a);
}

}  // namespace lp

// {slices of a row, workspace floats, workspace counters} of token_logprobs.
std::vector<int64_t> token_logprobs_plan(int64_t rows, int64_t vocab, int64_t elem_size) {
  // Two CTAs for each SM, all at once (64 rows, top 20: 15.9 us; three or four for each
  // SM, that do not all fit, 22 and 27), slices of one chunk a thread at least.
  const int64_t least = lp::kThreads * (16 / elem_size);
  int64_t s = std::max<int64_t>(1, 2 * num_sms() / std::max<int64_t>(1, rows));
  s = std::min(s, std::max<int64_t>(1, vocab / least));
  return {s, s > 1 ? rows * s * (4 + 2 * lp::kMaxTop) : 0, s > 1 ? rows : 0};
}

// Log-probability [R], entropy [R], ids of the top alternatives [R, k] and theirs.
// (The results are allocated here: from Python that took longer than one row does.)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> token_logprobs(
    at::Tensor logits, at::Tensor tokens, int64_t top_k, at::Tensor ws, at::Tensor counters) {
  TORCH_CHECK(logits.is_cuda() && logits.dim() == 2 && logits.stride(1) == 1 && logits.size(1) > 0,
              "logits must be [rows, vocab] with inner stride 1");
  const auto type = logits.scalar_type();
  TORCH_CHECK(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat,
              "logits must be bf16, fp16 or fp32");
  const int64_t R = logits.size(0), V = logits.size(1);
  TORCH_CHECK(V < (int64_t(1) << 31) - 4096, "vocabulary too large");
  TORCH_CHECK(top_k >= 0 && top_k <= lp::kMaxTop && top_k <= V,
              "top_k must be in 0..32 and at most the vocabulary");
  TORCH_CHECK(tokens.scalar_type() == at::kInt && tokens.is_contiguous() && tokens.numel() == R &&
                  tokens.device() == logits.device(),
              "tokens must be int32, one per row");
  TORCH_CHECK(R <= 65535, "at most 65535 rows in one call");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  at::Tensor logprob = at::empty({R}, f32), entropy = at::empty({R}, f32);
  at::Tensor top_ids = at::empty({R, top_k}, f32.dtype(at::kInt));
  at::Tensor top_lp = at::empty({R, top_k}, f32);
  if (R == 0) return {logprob, entropy, top_ids, top_lp};
  const int64_t es = (int64_t)logits.element_size();
  const std::vector<int64_t> plan = token_logprobs_plan(R, V, es);
  TORCH_CHECK(ws.scalar_type() == at::kFloat && counters.scalar_type() == at::kInt &&
                  ws.device() == logits.device() && counters.device() == logits.device() &&
                  ws.numel() >= plan[1] && counters.numel() >= plan[2] &&
                  (plan[0] == 1 || reinterpret_cast<uintptr_t>(ws.data_ptr()) % 16 == 0),
              "workspace too small, or not 16-byte aligned");
  lp::Args a;
  a.x = logits.data_ptr();
  a.ld = logits.stride(0);
  a.V = (int)V;
  a.slices = (int)plan[0];
  a.slice_len = (int)((V + plan[0] - 1) / plan[0]);
  a.top_k = (int)top_k;
  a.tokens = tokens.data_ptr<int>();
  a.logprob = logprob.data_ptr<float>();
  a.entropy = entropy.data_ptr<float>();
  a.top_ids = top_ids.data_ptr<int>();
  a.top_lp = top_lp.data_ptr<float>();
  a.part = ws.data_ptr<float>();
  a.counters = counters.data_ptr<int>();
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (type == at::kFloat) lp::launch<float>(a, (int)R, stream);
  else if (type == at::kHalf) lp::launch<__half>(a, (int)R, stream);
  else lp::launch<__nv_bfloat16>(a, (int)R, stream);
  return {logprob, entropy, top_ids, top_lp};
}

}  // namespace cb

// Log-probabilities of given tokens, entropy and the top alternatives of logit
// rows, in one pass over the logits.
//
//   m = max x,  S = sum e^(x - m),  W = sum e^(x - m) (x - m)
//   logprob(t) = (x_t - m) - ln S,   entropy = ln S - W / S
//
// held as a running (m, S, W) by every thread and joined at the end.  The k-th
// largest of the threads' largest values is a bound below the row's k-th
// largest: only the at most k threads whose largest value reaches it can hold
// any of the row's top k.  Order: larger value first, then lower index
// (-0 = 0; a NaN comes before everything).  A row is cut in slices, one for each
// CTA, when there are few rows; the last CTA of a row joins them.
#include <torch/extension.h>
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
  float* part;  // [R][slices][4 + 2 * kMaxTop]
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

struct Stat {
  float m, s, w;
};
// Joins two running sums; m may be -inf (nothing but -inf so far).
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
  Stat r;
  r.m = max_nan(a.m, b.m);
  const float ref = fmaxf(r.m, -FLT_MAX);
  const float da = fmaxf(a.m, -FLT_MAX) - ref, db = fmaxf(b.m, -FLT_MAX) - ref;
  const float fa = exp2f(da * kLog2e), fb = exp2f(db * kLog2e);
  r.s = a.s * fa + b.s * fb;
  r.w = (fa > 0.f ? fa * (a.w + a.s * da) : 0.f) + (fb > 0.f ? fb * (b.w + b.s * db) : 0.f);
  return r;
}

template <typename T>
__device__ __forceinline__ float value(const T* p) {
  if constexpr (std::is_same<T, float>::value) return *p;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(*p);
  else return __bfloat162float(*p);
}

// 16 bytes of logits as floats.
template <typename T>
struct Chunk {
  static constexpr int N = 16 / sizeof(T);
  float v[N];
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

template <typename T>
__global__ void __launch_bounds__(kThreads) token_logprobs_kernel(const Args a) {
  constexpr int N = Chunk<T>::N;
  __shared__ Key lists[kThreads];
  __shared__ Key cand[kCand];
  __shared__ Stat stats[kWarps];
  __shared__ int s_count, s_last;
  grid_dep_launch();
  grid_dep_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y, slice = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.x) + (int64_t)row * a.ld;
  const int lo = slice * a.slice_len, hi = min(a.V, lo + a.slice_len);
  // [lo, v0): before the first 16-byte boundary; [v0, v1): whole chunks.
  const int skew = (int)((reinterpret_cast<uintptr_t>(x + lo) & 15) / sizeof(T));
  const int v0 = min(hi, lo + (skew ? N - skew : 0));
  const int chunks = (hi - v0) / N;
  const int v1 = v0 + chunks * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + v0);

  Stat st = {-INFINITY, 0.f, 0.f};
  float ref = -FLT_MAX;
  auto raise = [&](float to) {
    const float n = fmaxf(to, -FLT_MAX);
    const float d = ref - n;
    const float f = exp2f(d * kLog2e);
    st.w = f > 0.f ? f * (st.w + st.s * d) : 0.f;
    st.s *= f;
    st.m = max_nan(st.m, to);
    ref = n;
  };
  auto add = [&](float v) {
    const float d = fmaxf(v - ref, -1e4f);
    const float e = exp2f(d * kLog2e);
    st.s += e;
    st.w = fmaf(e, d, st.w);
  };
  // Edges: fewer than 2 N elements, one for each of the first threads.
  const int edge = tid < v0 - lo ? lo + tid : (tid - (v0 - lo) < hi - v1 ? v1 + tid - (v0 - lo) : -1);
  float edge_v = -INFINITY;
  if (edge >= 0) {
    edge_v = value(x + edge);
    if (!(edge_v <= st.m)) raise(edge_v);
    add(edge_v);
  }
  for (int c = tid; c < chunks; c += kThreads) {
    Chunk<T> u;
    u.set(__ldg(xv + c));
    float top = u.v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = max_nan(top, u.v[i]);
    if (!(top <= st.m)) raise(top);
#pragma unroll
    for (int i = 0; i < N; ++i) add(u.v[i]);
  }
  // Row statistics.
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Stat other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o);
    other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    other.w = __shfl_xor_sync(0xffffffffu, st.w, o);
    st = join(st, other);
  }
  if (lane == 0) stats[warp] = st;
  __syncthreads();
  st = stats[0];
  for (int w = 1; w < kWarps; ++w) st = join(st, stats[w]);

  Key top = 0;
  if (a.top_k > 0) {
    Key key = edge >= 0 ? make_key(edge_v, edge) : 0;
    for (int c = tid; c < chunks; c += kThreads) {
      Chunk<T> u;
      u.set(__ldg(xv + c));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const Key k2 = make_key(u.v[i], v0 + c * N + i);
        key = k2 > key ? k2 : key;
      }
    }
    const Key bound_list = block_merge(warp_sort(key), lists);
    const Key bound = __shfl_sync(0xffffffffu, bound_list, a.top_k - 1);
    if (tid == 0) s_count = 0;
    __syncthreads();
    if (key >= bound && key > 0) {
      if (edge >= 0) {
        const Key k2 = make_key(edge_v, edge);
        if (k2 >= bound) {
          const int at = atomicAdd(&s_count, 1);
          if (at < kCand) cand[at] = k2;
        }
      }
      for (int c = tid; c < chunks; c += kThreads) {
        Chunk<T> u;
        u.set(__ldg(xv + c));
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const Key k2 = make_key(u.v[i], v0 + c * N + i);
          if (k2 >= bound) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kCand) cand[at] = k2;
          }
        }
      }
    }
    __syncthreads();
    const int count = s_count;
    if (count <= kCand) {
      for (int i = warp * 32; i < count; i += kThreads)
        top = warp_merge(top, warp_sort(i + lane < count ? cand[i + lane] : 0));
      top = block_merge(top, lists);
    } else {
      // More values over the bound than the list holds (many of a row's
      // largest values in a few threads' chunks): one pass for each place.
      Key last = ~(Key)0;
      for (int j = 0; j < a.top_k; ++j) {
        Key k1 = edge >= 0 ? make_key(edge_v, edge) : 0;
        if (k1 >= last) k1 = 0;
        for (int c = tid; c < chunks; c += kThreads) {
          Chunk<T> u;
          u.set(__ldg(xv + c));
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const Key k2 = make_key(u.v[i], v0 + c * N + i);
            if (k2 < last && k2 > k1) k1 = k2;
          }
        }
        const Key found = block_merge(warp_sort(k1), lists);
        last = __shfl_sync(0xffffffffu, found, 0);
        if (lane == j) top = last;
      }
    }
  }

  if (a.slices > 1) {
    constexpr int P = 4 + 2 * kMaxTop;
    float* part = a.part + ((int64_t)row * a.slices + slice) * P;
    if (warp == 0) {
      if (lane == 0) {
        part[0] = st.m;
        part[1] = st.s;
        part[2] = st.w;
      }
      reinterpret_cast<Key*>(part + 4)[lane] = top;
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
    if (warp == 0) {
      st = {-INFINITY, 0.f, 0.f};
      top = 0;
      for (int i = 0; i < a.slices; ++i) {
        const float* p = a.part + ((int64_t)row * a.slices + i) * P;
        const Stat o = {__ldcg(p), __ldcg(p + 1), __ldcg(p + 2)};
        st = join(st, o);
        if (a.top_k > 0)
          top = warp_merge(top, __ldcg(reinterpret_cast<const Key*>(p + 4) + lane));
      }
    }
  }
  if (warp != 0) return;
  // NaN or +inf in the row: no distribution.  Nothing but -inf: every token
  // has probability 0.
  const bool bad = !(st.m < INFINITY);
  const bool empty = st.m == -INFINITY;
  const float ln_s = logf(st.s);
  const float nan = __int_as_float(0x7fc00000);
  auto lp_of = [&](float v) { return bad ? nan : (empty ? -INFINITY : (v - st.m) - ln_s); };
  if (lane == 0) {
    const int t = a.tokens[row];
    a.logprob[row] = t >= 0 && t < a.V ? lp_of(value(x + t)) : nan;
    a.entropy[row] = bad ? nan : (empty ? 0.f : ln_s - st.w / st.s);
  }
  if (lane < a.top_k) {
    a.top_ids[(int64_t)row * a.top_k + lane] = (int)~(uint32_t)top;
    a.top_lp[(int64_t)row * a.top_k + lane] = lp_of(order_value((uint32_t)(top >> 32)));
  }
}

}  // namespace lp

// {slices of a row, workspace floats, workspace counters} of token_logprobs.
std::vector<int64_t> token_logprobs_plan(int64_t rows, int64_t vocab, int64_t elem_size) {
  // About four CTAs for each SM, slices of two chunks a thread at least.
  const int64_t least = 2 * lp::kThreads * (16 / elem_size);
  int64_t s = std::max<int64_t>(1, 4 * num_sms() / std::max<int64_t>(1, rows));
  s = std::min(s, std::max<int64_t>(1, vocab / least));
  return {s, s > 1 ? rows * s * (4 + 2 * lp::kMaxTop) : 0, s > 1 ? rows : 0};
}

void token_logprobs(torch::Tensor logits, torch::Tensor tokens, int64_t top_k,
                    torch::Tensor logprob, torch::Tensor entropy, torch::Tensor top_ids,
                    torch::Tensor top_lp, torch::Tensor ws, torch::Tensor counters) {
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
  TORCH_CHECK(logprob.scalar_type() == at::kFloat && entropy.scalar_type() == at::kFloat &&
                  top_ids.scalar_type() == at::kInt && top_lp.scalar_type() == at::kFloat &&
                  logprob.numel() >= R && entropy.numel() >= R && top_ids.numel() >= R * top_k &&
                  top_lp.numel() >= R * top_k && logprob.is_contiguous() &&
                  entropy.is_contiguous() && top_ids.is_contiguous() && top_lp.is_contiguous(),
              "outputs must be contiguous fp32 [R], [R], int32 [R, k], fp32 [R, k]");
  if (R == 0) return;
  TORCH_CHECK(R <= 65535, "at most 65535 rows in one call");
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t es = (int64_t)logits.element_size();
  const std::vector<int64_t> plan = token_logprobs_plan(R, V, es);
  TORCH_CHECK(ws.numel() >= plan[1] && counters.numel() >= plan[2], "workspace too small");
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
  const dim3 grid((unsigned)plan[0], (unsigned)R);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  const dim3 block(lp::kThreads);
  if (type == at::kFloat) launch_kernel(lp::token_logprobs_kernel<float>, grid, block, 0, stream, a);
  else if (type == at::kHalf)
    launch_kernel(lp::token_logprobs_kernel<__half>, grid, block, 0, stream, a);
  else launch_kernel(lp::token_logprobs_kernel<__nv_bfloat16>, grid, block, 0, stream, a);
}

}  // namespace cb

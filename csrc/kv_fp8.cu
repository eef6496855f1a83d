// The 8-bit paged KV cache: quantising write and read-back.
//
// Cache layout: codes [L, NB, Hkv, 16, D] e4m3 and one fp32 scale for every
// (token, kv head) row, [L, NB, Hkv, 16], for K and for V: D + 4 bytes a row
// in place of 2 D.
//
//   a = max |y|,  s = max(a * fl(1/448), 2^-100),  code = e4m3(y * fl(1/s))
//
// with y the rotated key or the value in fp32.  The floor keeps 1/s and
// log2 s finite for a row of zeros.  A row that holds a NaN or an infinity gets
// s = NaN and zero codes: it reads back as NaN, and an attention row that does
// not see it never multiplies by it.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "host_utils.h"

namespace cb {

using bf16 = __nv_bfloat16;

constexpr float kE4M3Max = 448.f;
constexpr float kScaleMin = 7.888609052210118e-31f;  // 2^-100

struct WriteArgs {
  const bf16* qkv;
  int64_t ldq;
  bf16* q_out;  // rotated q rows (qkv itself: in place)
  int64_t ldqo;
  const int* positions;
  const float* cos_sin;
  const int* slots;
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  int64_t layer_blocks;  // layer * NB
  int T, Hq, Hkv, rot, interleaved;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ uint4 pack8_bf16(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&p);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ uint2 pack8_e4m3(const float (&v)[8], float inv) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(
        make_float2(v[4 * i] * inv, v[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(
        make_float2(v[4 * i + 2] * inv, v[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[i] = lo | (hi << 16);
  }
  return make_uint2(w[0], w[1]);
}

// D / 16 lanes share one head row; each holds two chunks of 8 values: the two
// halves of 8 rotation pairs (half layout), or 16 neighbours (interleaved
// pairs, and everything that is not rotated).
// A thread handles HPT heads of its token, all loaded before the first is used
// (and before the cosines arrive); with few tokens the heads of a token spread
// over gridDim.y CTAs instead.
// Bound: memory.  8192 tokens of 32 + 2 x 8 heads of 128: 189 MB in 35 us, 5.5 TB/s.
// A few tokens: two dependent trips to memory, 2 us behind another kernel.
template <int D, int HPT>
__global__ void __launch_bounds__(128) rope_kv_write_fp8_kernel(const WriteArgs a) {
  constexpr int LPH = D / 16;
  constexpr int GROUPS = 128 / LPH;
  grid_dep_launch();
  grid_dep_wait();
  const int t = blockIdx.x;
  const int p = threadIdx.x % LPH;
  const int slot = a.slots[t];
  const bool rotated = 16 * p < a.rot;
  const int half = a.rot / 2;
  const bool split = rotated && !a.interleaved;
  const int d0 = split ? 8 * p : 16 * p;
  const int d1 = split ? half + 8 * p : 16 * p + 8;
  const int heads = a.Hq + 2 * a.Hkv;
  const bf16* row = a.qkv + (int64_t)t * a.ldq;
  const int h0 = blockIdx.y * HPT * GROUPS + threadIdx.x / LPH;
  uint4 raw[HPT][2];
#pragma unroll
  for (int k = 0; k < HPT; ++k) {
    const int h = h0 + k * GROUPS;
    if (h < heads) {
      raw[k][0] = *reinterpret_cast<const uint4*>(row + (int64_t)h * D + d0);
      raw[k][1] = *reinterpret_cast<const uint4*>(row + (int64_t)h * D + d1);
    } else {
      raw[k][0] = raw[k][1] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  alignas(16) float c[8], sn[8];
  if (rotated) {
    const float* cs = a.cos_sin + (int64_t)a.positions[t] * a.rot + 8 * p;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(c + i) = __ldg(reinterpret_cast<const float4*>(cs + i));
      *reinterpret_cast<float4*>(sn + i) = __ldg(reinterpret_cast<const float4*>(cs + half + i));
    }
  }
#pragma unroll
  for (int k = 0; k < HPT; ++k) {
    const int h = h0 + k * GROUPS;
    const bool live = h < heads && (h < a.Hq || slot >= 0);
    float y0[8], y1[8];
    unpack8(raw[k][0], y0);
    unpack8(raw[k][1], y1);
    if (rotated && h < a.Hq + a.Hkv) {
      // Products and sums are rounded one by one (no contraction), so that
      // codes do not depend on how the compiler fuses them.
      if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float u0 = y0[2 * i], u1 = y0[2 * i + 1];
          y0[2 * i] = __fsub_rn(__fmul_rn(u0, c[i]), __fmul_rn(u1, sn[i]));
          y0[2 * i + 1] = __fadd_rn(__fmul_rn(u1, c[i]), __fmul_rn(u0, sn[i]));
          const float w0 = y1[2 * i], w1 = y1[2 * i + 1];
          y1[2 * i] = __fsub_rn(__fmul_rn(w0, c[4 + i]), __fmul_rn(w1, sn[4 + i]));
          y1[2 * i + 1] = __fadd_rn(__fmul_rn(w1, c[4 + i]), __fmul_rn(w0, sn[4 + i]));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u0 = y0[i], u1 = y1[i];
          y0[i] = __fsub_rn(__fmul_rn(u0, c[i]), __fmul_rn(u1, sn[i]));
          y1[i] = __fadd_rn(__fmul_rn(u1, c[i]), __fmul_rn(u0, sn[i]));
        }
      }
    }
    // Largest magnitude over the row's lanes, on the bit patterns: an infinity
    // or a NaN is larger than every finite value.
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      top = max(top, __float_as_uint(y0[i]) & 0x7fffffffu);
      top = max(top, __float_as_uint(y1[i]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) continue;
    if (h < a.Hq) {
      bf16* dst = a.q_out + (int64_t)t * a.ldqo + (int64_t)h * D;
      *reinterpret_cast<uint4*>(dst + d0) = pack8_bf16(y0);
      *reinterpret_cast<uint4*>(dst + d1) = pack8_bf16(y1);
      continue;
    }
    const bool fine = top < 0x7f800000u;
    float s = fmaxf(__uint_as_float(top) * (1.f / kE4M3Max), kScaleMin);
    const float inv = __frcp_rn(s);
    uint2 w0 = make_uint2(0u, 0u), w1 = w0;
    if (fine) {
      w0 = pack8_e4m3(y0, inv);
      w1 = pack8_e4m3(y1, inv);
    } else {
      s = __int_as_float(0x7fc00000);
    }
    const bool is_k = h < a.Hq + a.Hkv;
    const int kh = h - a.Hq - (is_k ? 0 : a.Hkv);
    const int64_t r = ((a.layer_blocks + (slot >> 4)) * a.Hkv + kh) * 16 + (slot & 15);
    uint8_t* dst = (is_k ? a.k : a.v) + r * D;
    *reinterpret_cast<uint2*>(dst + d0) = w0;
    *reinterpret_cast<uint2*>(dst + d1) = w1;
    if (p == 0) (is_k ? a.ks : a.vs)[r] = s;
  }
}

struct ReadArgs {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  bf16* k_out;  // [N, Hkv, 16, D]
  bf16* v_out;
  const int* blocks;
  int64_t layer_blocks;
  uint32_t items;      // 8-code pieces of K and V together: 2 N per_block
  uint32_t per_block;  // pieces of one block of one of them: Hkv * 16 * D / 8
};

// A thread turns pieces of 8 codes into 8 bf16 values each: 8-byte loads and
// 16-byte stores, both whole lines for a warp, and kReadPieces of them in
// flight.  Pieces run over [block][K, V][head][token][dim].
// Bound: memory, two thirds of it writes.  4096 blocks of 8 heads of 128: 407 MB in
// 80 us, 5.1 TB/s.
constexpr int kReadPieces = 8;

template <int D>
__global__ void __launch_bounds__(256) kv_read_fp8_kernel(const ReadArgs a) {
  grid_dep_launch();
  grid_dep_wait();
  const uint32_t base = blockIdx.x * (256 * kReadPieces) + threadIdx.x;
  uint2 code[kReadPieces];
  float scale[kReadPieces];
#pragma unroll
  for (int j = 0; j < kReadPieces; ++j) {
    const uint32_t i = base + j * 256;
    code[j] = make_uint2(0u, 0u);
    scale[j] = 0.f;
    if (i < a.items) {
      const uint32_t pair = i / a.per_block;
      const uint32_t c = i - pair * a.per_block;
      const int blk = a.blocks[pair >> 1];
      if (blk >= 0) {
        const int64_t src = (a.layer_blocks + blk) * a.per_block + c;
        code[j] = __ldg(reinterpret_cast<const uint2*>(pair & 1 ? a.v : a.k) + src);
        scale[j] = __ldg((pair & 1 ? a.vs : a.ks) + src / (D / 8));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kReadPieces; ++j) {
    const uint32_t i = base + j * 256;
    if (i >= a.items) continue;
    const uint32_t pair = i / a.per_block;
    const uint32_t c = i - pair * a.per_block;
    float y[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t word = w < 2 ? code[j].x : code[j].y;
      const __half2 h2 = __nv_cvt_fp8x2_to_halfraw2(
          (__nv_fp8x2_storage_t)(word >> (16 * (w & 1))), __NV_E4M3);
      const float2 f = __half22float2(h2);
      y[2 * w] = f.x * scale[j];
      y[2 * w + 1] = f.y * scale[j];
    }
    uint4* dst = reinterpret_cast<uint4*>(pair & 1 ? a.v_out : a.k_out);
    dst[(int64_t)(pair >> 1) * a.per_block + c] = pack8_bf16(y);
  }
}

// ---------------------------------------------------------------- host side

static void check_fp8_cache(const at::Tensor& k, const at::Tensor& v,
                            const at::Tensor& ks, const at::Tensor& vs) {
  TORCH_CHECK(k.is_cuda() && k.scalar_type() == at::kFloat8_e4m3fn &&
                  v.scalar_type() == at::kFloat8_e4m3fn,
              "k/v cache must be float8_e4m3fn on the GPU");
  TORCH_CHECK(k.dim() == 5 && k.size(3) == 16 && k.is_contiguous() && v.is_contiguous() &&
                  v.sizes() == k.sizes(),
              "k/v cache must be [L, NB, Hkv, 16, D] contiguous, of one shape");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(k.data_ptr()) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(v.data_ptr()) % 8 == 0,
              "k/v cache must be 8-byte aligned");
  TORCH_CHECK(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.dim() == 4 &&
                  ks.is_contiguous() && vs.is_contiguous() && ks.sizes() == vs.sizes() &&
                  ks.size(0) == k.size(0) && ks.size(1) == k.size(1) && ks.size(2) == k.size(2) &&
                  ks.size(3) == 16,
              "k/v scales must be fp32 [L, NB, Hkv, 16] contiguous");
  TORCH_CHECK(v.device() == k.device() && ks.device() == k.device() && vs.device() == k.device(),
              "cache and scales must be on one device");
}

// Few tokens: one head a thread, so that the heads' loads and the row maxima of
// one token run side by side; from four CTAs an SM on, three heads a thread, with more
// loads in flight (32 + 2 x 8 heads of 128; 64 tokens: 1.9 us against 2.3, 592: 3.4
// against 4.1; 1024: 4.8 against 4.2, 8192: 35 against 33).
template <int D>
static void launch_write(const WriteArgs& a, cudaStream_t stream) {
  constexpr int groups = 128 / (D / 16);
  const int heads = a.Hq + 2 * a.Hkv;
  if (a.T < 4 * num_sms()) {
    const dim3 grid((unsigned)a.T, (heads + groups - 1) / groups);
    launch_kernel(rope_kv_write_fp8_kernel<D, 1>, grid, dim3(128), 0, stream, a);
  } else {
    const dim3 grid((unsigned)a.T, (heads + 3 * groups - 1) / (3 * groups));
    launch_kernel(rope_kv_write_fp8_kernel<D, 3>, grid, dim3(128), 0, stream, a);
  }
}

void rope_kv_write_fp8(at::Tensor qkv, at::Tensor positions, at::Tensor cos_sin,
                       at::Tensor slots, at::Tensor k_cache, at::Tensor v_cache,
                       at::Tensor k_scale, at::Tensor v_scale, int64_t layer, int64_t Hq,
                       int64_t Hkv, int64_t D, int64_t rot, bool interleaved,
                       c10::optional<at::Tensor> q_out) {
  check_fp8_cache(k_cache, v_cache, k_scale, v_scale);
  TORCH_CHECK(qkv.dim() == 2 && qkv.scalar_type() == at::kBFloat16 && qkv.stride(1) == 1 &&
                  qkv.size(1) == (Hq + 2 * Hkv) * D,
              "qkv must be bf16 [T, (Hq + 2 Hkv) D] with inner stride 1");
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256");
  TORCH_CHECK(k_cache.size(2) == Hkv && k_cache.size(4) == D && Hq >= 0,
              "cache heads / head_dim mismatch");
  TORCH_CHECK(rot > 0 && rot % 16 == 0 && rot <= D, "rotary dim must be a multiple of 16, <= D");
  TORCH_CHECK(layer >= 0 && layer < k_cache.size(0), "layer outside the cache");
  const int64_t T = qkv.size(0);
  TORCH_CHECK(positions.scalar_type() == at::kInt && slots.scalar_type() == at::kInt &&
                  positions.is_contiguous() && slots.is_contiguous() && positions.numel() >= T &&
                  slots.numel() >= T,
              "positions / slots must be int32, one per row");
  TORCH_CHECK(cos_sin.scalar_type() == at::kFloat && cos_sin.is_contiguous() &&
                  cos_sin.dim() == 2 && cos_sin.size(1) == rot,
              "cos_sin must be fp32 [positions, rot]");
  at::Tensor qo = q_out.has_value() ? *q_out : qkv;
  TORCH_CHECK(qo.scalar_type() == at::kBFloat16 && qo.dim() == 2 && qo.stride(1) == 1 &&
                  qo.size(0) >= T && qo.size(1) >= Hq * D,
              "q_out must be bf16 [T, Hq D] with inner stride 1");
  TORCH_CHECK((qkv.stride(0) * 2) % 16 == 0 && (qo.stride(0) * 2) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(qo.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(cos_sin.data_ptr()) % 16 == 0,
              "qkv / q_out rows and cos_sin must be 16-byte aligned");
  TORCH_CHECK(qkv.device() == k_cache.device() && qo.device() == qkv.device() &&
                  positions.device() == qkv.device() && slots.device() == qkv.device() &&
                  cos_sin.device() == qkv.device(),
              "all tensors must be on one device");
  if (T == 0) return;
  const c10::cuda::CUDAGuard guard(qkv.device());
  WriteArgs a;
  a.qkv = reinterpret_cast<const bf16*>(qkv.data_ptr());
  a.ldq = qkv.stride(0);
  a.q_out = reinterpret_cast<bf16*>(qo.data_ptr());
  a.ldqo = qo.stride(0);
  a.positions = positions.data_ptr<int>();
  a.cos_sin = cos_sin.data_ptr<float>();
  a.slots = slots.data_ptr<int>();
  a.k = reinterpret_cast<uint8_t*>(k_cache.data_ptr());
  a.v = reinterpret_cast<uint8_t*>(v_cache.data_ptr());
  a.ks = k_scale.data_ptr<float>();
  a.vs = v_scale.data_ptr<float>();
  a.layer_blocks = layer * k_cache.size(1);
  a.T = (int)T;
  a.Hq = (int)Hq;
  a.Hkv = (int)Hkv;
  a.rot = (int)rot;
  a.interleaved = interleaved ? 1 : 0;
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  if (D == 64) launch_write<64>(a, stream);
  else if (D == 128) launch_write<128>(a, stream);
  else launch_write<256>(a, stream);
}

void kv_read_fp8(at::Tensor k_cache, at::Tensor v_cache, at::Tensor k_scale,
                 at::Tensor v_scale, at::Tensor blocks, int64_t layer, at::Tensor k_out,
                 at::Tensor v_out) {
  check_fp8_cache(k_cache, v_cache, k_scale, v_scale);
  const int64_t N = blocks.numel(), Hkv = k_cache.size(2), D = k_cache.size(4);
  TORCH_CHECK(D == 64 || D == 128 || D == 256, "head_dim must be 64, 128 or 256");
  TORCH_CHECK(layer >= 0 && layer < k_cache.size(0), "layer outside the cache");
  TORCH_CHECK(blocks.scalar_type() == at::kInt && blocks.is_contiguous(),
              "blocks must be contiguous int32");
  for (const at::Tensor* o : {&k_out, &v_out}) {
    TORCH_CHECK(o->scalar_type() == at::kBFloat16 && o->is_contiguous() &&
                    o->numel() >= N * Hkv * 16 * D &&
                    reinterpret_cast<uintptr_t>(o->data_ptr()) % 16 == 0,
                "k_out / v_out must be contiguous bf16 with room for [N, Hkv, 16, D]");
    TORCH_CHECK(o->device() == k_cache.device(), "all tensors must be on one device");
  }
  TORCH_CHECK(blocks.device() == k_cache.device(), "all tensors must be on one device");
  if (N == 0 || Hkv == 0) return;
  const c10::cuda::CUDAGuard guard(k_cache.device());
  ReadArgs a;
  a.k = reinterpret_cast<const uint8_t*>(k_cache.data_ptr());
  a.v = reinterpret_cast<const uint8_t*>(v_cache.data_ptr());
  a.ks = k_scale.data_ptr<float>();
  a.vs = v_scale.data_ptr<float>();
  a.layer_blocks = layer * k_cache.size(1);
  a.per_block = (uint32_t)(Hkv * 2 * D);
  cudaStream_t stream = at::cuda::getCurrentCUDAStream();
  // Pieces are counted in 32 bits: a call past that is cut into several launches.
  const int64_t most = ((int64_t(1) << 31) - 1) / (2 * a.per_block);
  for (int64_t n0 = 0; n0 < N; n0 += most) {
    const int64_t n = std::min(most, N - n0);
    a.k_out = reinterpret_cast<bf16*>(k_out.data_ptr()) + n0 * Hkv * 16 * D;
    a.v_out = reinterpret_cast<bf16*>(v_out.data_ptr()) + n0 * Hkv * 16 * D;
    a.blocks = blocks.data_ptr<int>() + n0;
    a.items = (uint32_t)(2 * n * a.per_block);
    const dim3 grid((a.items + 256 * kReadPieces - 1) / (256 * kReadPieces));
    if (D == 64) launch_kernel(kv_read_fp8_kernel<64>, grid, dim3(256), 0, stream, a);
    else if (D == 128) launch_kernel(kv_read_fp8_kernel<128>, grid, dim3(256), 0, stream, a);
    else launch_kernel(kv_read_fp8_kernel<256>, grid, dim3(256), 0, stream, a);
  }
}

}  // namespace cb

// AdamW over many tensors in one launch, with states in 8 bits or in 32 (sm_100a).
//
// The update is that of adamw.cu (decoupled weight decay, here one per tensor):
//   m = b1 m + (1 - b1) g;   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// p is fp32, g fp32 or bf16, and a bf16 copy of p is written in the same pass. lr and the step
// count live on the device; the last CTA of the step counts it.
//
// 8-bit states hold blocks of 256 values of one tensor under one power-of-two scale (an exponent
// byte e: 2^(e - 127)); a power of two costs a floating format no precision, makes scaling exact
// and needs no division. The first moment is e4m3. The second is eight unsigned bits, 5 of
// exponent and 3 of mantissa in units of 1 (value 0..7 below 8, then (8 + m) 2^(x - 1)): it has no
// sign to store, and 34 binades leave a value 2^33 below the block's largest its own code; e4m3
// would keep 18, and a second moment that became zero under a first moment that did not would
// throw its weight out by lr / eps. A non-zero second moment never becomes zero here.
// Values are rounded up or down with probabilities that keep their mean: with b2 = 0.999 a step
// moves v by a tenth of a percent, and rounding to nearest in steps of 12 percent would never let
// it move. The 16 + 16 random bits of a value are a hash of its place, the step and the seed, so a
// step can be repeated bit for bit. m and v are computed without fused multiply-adds, in the
// order of the formula: a value next to a rounding border lands on the same side everywhere.
//
// A warp takes one block: eight values a lane. The tensors' addresses are kernel arguments, so
// nothing is copied to the device and nothing is remembered from one call to the next.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "../common/common.cuh"

namespace llmt {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = 256;  // values per scale, and per warp

template <int CAP>
struct Batch {
  MultiTensor t[CAP];
  int count;
};

__device__ __forceinline__ float pow2_of(uint32_t e) { return __uint_as_float(e << 23); }

// Smallest exponent byte e under which the block's largest magnitude `top` (its bits) is at most
// the format's largest value: 2^places * (1 + limit / 2^23).
__device__ __forceinline__ uint32_t scale_byte(uint32_t top, int places, uint32_t limit) {
  const int e = (int)(top >> 23) - places + ((top & 0x7fffffu) > limit ? 1 : 0);
  return (uint32_t)min(max(e, 1), 253);
}
__device__ __forceinline__ uint32_t scale_byte_m(uint32_t top) { return scale_byte(top, 8, 0x600000u); }   // 448
__device__ __forceinline__ uint32_t scale_byte_v(uint32_t top) { return scale_byte(top, 33, 0x700000u); }  // 1.875 2^33

// Both codes are the top bits of an fp32 number: scaled so that the format's subnormals are fp32's
// subnormals, adding 20 random bits below the kept ones and cutting rounds up with the right
// probability, in the normal and the subnormal range alike.
__device__ __forceinline__ uint32_t encode_m(float m, uint32_t e, uint32_t noise) {
  if (m != m) return 0x7fu;
  const float y = __fmul_rn(__fmul_rn(fabsf(m), pow2_of(254u - e)), 0x1p-120f);
  return min((__float_as_uint(y) + noise) >> 20, 126u) | (m < 0.f ? 0x80u : 0u);
}
__device__ __forceinline__ uint32_t encode_v(float v, uint32_t e, uint32_t noise) {
  const float y = __fmul_rn(__fmul_rn(v, pow2_of(254u - e)), 0x1p-129f);
  const uint32_t c = min((__float_as_uint(y) + noise) >> 20, 255u);
  return v > 0.f ? max(c, 1u) : c;
}
__device__ __forceinline__ float decode_m(uint32_t code, float scale) {
  const float y = __uint_as_float((code & 0x7fu) << 20) * 0x1p120f;
  const float x = (code & 0x7fu) == 0x7fu ? NAN : y * scale;
  return code & 0x80u ? -x : x;
}
__device__ __forceinline__ float decode_v(uint32_t code, float scale) {
  return __uint_as_float(code << 20) * 0x1p64f * 0x1p65f * scale;
}

// 32 mixed bits of place i: two rounds of multiplication and xor-shift; the odd constants are
// digits of e, of the square root of two and of the golden ratio.
__device__ __forceinline__ uint32_t place_hash(int64_t i, uint32_t seed) {
  uint32_t x = ((uint32_t)i ^ ((uint32_t)(i >> 32) * 0x6A09E667u)) * 0x9E3779B1u + seed;
  x = (x ^ (x >> 16)) * 0xB7E15163u;
  x = (x ^ (x >> 15)) * 0x6A09E667u;
  return x ^ (x >> 16);
}

struct StepConst {
  float b1, c1, b2, c2, eps, step_size, root, lr, grad_scale;
  uint32_t seed;
};

__device__ __forceinline__ void update(const StepConst& k, float decay, float g, float& p, float& m, float& v) {
  g = __fmul_rn(g, k.grad_scale);
  m = __fadd_rn(__fmul_rn(m, k.b1), __fmul_rn(g, k.c1));
  v = __fadd_rn(__fmul_rn(v, k.b2), __fmul_rn(__fmul_rn(g, k.c2), g));
  p = p * decay - k.step_size * (m / (sqrtf(v) * k.root + k.eps));
}

__device__ __forceinline__ StepConst step_const(const MultiHyper& h) {
  const float t = (float)(*h.step + 1), lr = *h.lr;
  StepConst k;
  k.b1 = h.b1;
  k.c1 = h.c1;
  k.b2 = h.b2;
  k.c2 = h.c2;
  k.eps = h.eps;
  k.lr = lr;
  k.step_size = lr / (1.f - powf(h.b1, t));
  k.root = 1.f / sqrtf(1.f - powf(h.b2, t));
  k.grad_scale = h.grad_scale * (h.grad_scale_dev ? *h.grad_scale_dev : 1.f);
  k.seed = (uint32_t)(*h.step + 1) * 0xB7E15163u + h.seed * 0x3C6EF373u;
  return k;
}

template <typename G, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads) adamw_multi_kernel(const __grid_constant__ Batch<CAP> batch, MultiHyper h,
                                                               MultiState s, int64_t blocks, bool last_launch) {
  const StepConst k = step_const(h);
  const int lane = threadIdx.x & 31;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t w = blockIdx.x * (int64_t)(kThreads / 32) + (threadIdx.x >> 5); w < blocks; w += stride) {
    int lo = 0, hi = batch.count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (batch.t[mid].first_work <= w) lo = mid;
      else hi = mid - 1;
    }
    const MultiTensor& t = batch.t[lo];
    const int64_t in_t = w - t.first_work, at = in_t * kBlock;
    const int64_t blk = t.first_block + in_t;  // in the state buffers
    const int n = (int)min((int64_t)kBlock, t.n - at);
    const float decay = 1.f - k.lr * t.wd;
    float m[8], v[8];
    float sm = 1.f, sv = 1.f;
    if (BITS == 8) {
      sm = pow2_of(s.ms[blk]);
      sv = pow2_of(s.vs[blk]);
    }
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = lane + 32 * j;
      m[j] = v[j] = 0.f;
      if (i >= n) continue;
      const int64_t si = blk * kBlock + i;
      float p = t.p[at + i];
      float g;
      if constexpr (sizeof(G) == 4) g = static_cast<const float*>(t.g)[at + i];
      else g = __bfloat162float(static_cast<const bf16*>(t.g)[at + i]);
      if (BITS == 8) {
        m[j] = decode_m(static_cast<const uint8_t*>(s.m)[si], sm);
        v[j] = decode_v(static_cast<const uint8_t*>(s.v)[si], sv);
      } else {
        m[j] = static_cast<const float*>(s.m)[si];
        v[j] = static_cast<const float*>(s.v)[si];
      }
      update(k, decay, g, p, m[j], v[j]);
      t.p[at + i] = p;
      if (t.p16) static_cast<bf16*>(t.p16)[at + i] = __float2bfloat16_rn(p);
      if (h.zero_grad) {
        if constexpr (sizeof(G) == 4) static_cast<float*>(t.g)[at + i] = 0.f;
        else static_cast<bf16*>(t.g)[at + i] = __float2bfloat16_rn(0.f);
      }
      if (BITS == 32) {
        static_cast<float*>(s.m)[si] = m[j];
        static_cast<float*>(s.v)[si] = v[j];
      }
      // (a NaN does not set the scale)
      if (fabsf(m[j]) <= INFINITY) top_m = max(top_m, __float_as_uint(fabsf(m[j])));
      if (v[j] <= INFINITY) top_v = max(top_v, __float_as_uint(v[j]));
    }
    if (BITS == 8) {
      const uint32_t em = scale_byte_m(__reduce_max_sync(0xffffffffu, top_m));
      const uint32_t ev = scale_byte_v(__reduce_max_sync(0xffffffffu, top_v));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int i = lane + 32 * j;
        if (i >= n) continue;
        const int64_t si = blk * kBlock + i;
        const uint32_t r = place_hash(si, k.seed);
        static_cast<uint8_t*>(s.m)[si] = (uint8_t)encode_m(m[j], em, ((r >> 16) << 4) | 8u);
        static_cast<uint8_t*>(s.v)[si] = (uint8_t)encode_v(v[j], ev, ((r & 0xffffu) << 4) | 8u);
      }
      if (lane == 0) {
        s.ms[blk] = (uint8_t)em;
        s.vs[blk] = (uint8_t)ev;
      }
    }
  }
  if (!last_launch) return;
  // every CTA has read the step count; the last one to finish counts the step and re-arms the ticket
  __syncthreads();
  if (threadIdx.x == 0 && atomicAdd(h.ticket, 1u) == gridDim.x - 1) {
    *h.ticket = 0;
    *h.step += 1;
  }
}

__global__ void __launch_bounds__(kThreads) state_values_kernel(const uint8_t* m, const uint8_t* ms, const uint8_t* v,
                                                                const uint8_t* vs, void* mo, void* vo, bool f32, int64_t n8) {
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < n8; i += (int64_t)gridDim.x * kThreads) {
    const uint2 a = reinterpret_cast<const uint2*>(m)[i], b = reinterpret_cast<const uint2*>(v)[i];
    const float sm = pow2_of(ms[i / (kBlock / 8)]), sv = pow2_of(vs[i / (kBlock / 8)]);
    float x[8], y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = decode_m(((j < 4 ? a.x : a.y) >> (8 * (j & 3))) & 255u, sm);
      y[j] = decode_v(((j < 4 ? b.x : b.y) >> (8 * (j & 3))) & 255u, sv);
    }
    if (f32) {
      for (int j = 0; j < 2; ++j) {
        st_f4(static_cast<float*>(mo) + 8 * i + 4 * j, make_float4(x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]));
        st_f4(static_cast<float*>(vo) + 8 * i + 4 * j, make_float4(y[4 * j], y[4 * j + 1], y[4 * j + 2], y[4 * j + 3]));
      }
    } else {  // exact: 4 significant bits, and an exponent that bf16 has
      reinterpret_cast<BF16x8*>(mo)[i] = float_to_bf16x8(x);
      reinterpret_cast<BF16x8*>(vo)[i] = float_to_bf16x8(y);
    }
  }
}

// Codes of fp32 states, to the nearest (a loaded checkpoint: values that came from codes stay).
__global__ void __launch_bounds__(kThreads) encode_states_kernel(const float* m, const float* v, uint8_t* mc, uint8_t* ms,
                                                                 uint8_t* vc, uint8_t* vs, int64_t blocks) {
  const int lane = threadIdx.x & 31;
  const int64_t stride = (int64_t)gridDim.x * (kThreads / 32);
  for (int64_t blk = blockIdx.x * (int64_t)(kThreads / 32) + (threadIdx.x >> 5); blk < blocks; blk += stride) {
    float x[8], y[8];
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = m[blk * kBlock + lane + 32 * j];
      y[j] = v[blk * kBlock + lane + 32 * j];
      if (fabsf(x[j]) <= INFINITY) top_m = max(top_m, __float_as_uint(fabsf(x[j])));
      if (y[j] <= INFINITY && y[j] >= 0.f) top_v = max(top_v, __float_as_uint(fabsf(y[j])));
    }
    const uint32_t em = scale_byte_m(__reduce_max_sync(0xffffffffu, top_m));
    const uint32_t ev = scale_byte_v(__reduce_max_sync(0xffffffffu, top_v));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mc[blk * kBlock + lane + 32 * j] = (uint8_t)encode_m(x[j], em, 1u << 19);
      vc[blk * kBlock + lane + 32 * j] = (uint8_t)encode_v(fabsf(y[j]), ev, 1u << 19);
    }
    if (lane == 0) {
      ms[blk] = (uint8_t)em;
      vs[blk] = (uint8_t)ev;
    }
  }
}

template <typename G, int BITS, int CAP>
cudaError_t launch(const MultiTensor* t, int count, const MultiHyper& h, const MultiState& s, bool last, cudaStream_t st) {
  Batch<CAP> b;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    b.t[i] = t[i];
    b.t[i].first_work = (int32_t)blocks;
    blocks += cdiv(t[i].n, (int64_t)kBlock);
  }
  b.count = count;
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(blocks, kThreads / 32), sm_count() * 8));
  adamw_multi_kernel<G, BITS, CAP><<<grid, kThreads, 0, st>>>(b, h, s, blocks, last);
  return cudaGetLastError();
}

template <typename G, int BITS>
cudaError_t launches(const MultiTensor* t, int count, const MultiHyper& h, const MultiState& s, cudaStream_t st) {
  constexpr int kSmall = 64, kLarge = 640;  // 3.1 KB and 30.7 KB of kernel arguments
  for (int i = 0; i < count; i += kLarge) {
    const int k = std::min(kLarge, count - i);
    const bool last = i + k == count;
    const cudaError_t e = k <= kSmall ? launch<G, BITS, kSmall>(t + i, k, h, s, last, st)
                                      : launch<G, BITS, kLarge>(t + i, k, h, s, last, st);
    if (e) return e;
  }
  return cudaSuccess;
}

}  // namespace

cudaError_t adamw_multi(const MultiTensor* t, int count, bool grad_bf16, int bits, const MultiHyper& h, const MultiState& s,
                        cudaStream_t st) {
  LLMT_REQUIRE(count > 0, "adamw_multi: no tensors");
  LLMT_REQUIRE(bits == 8 || bits == 32, "adamw_multi: states have 8 or 32 bits");
  if (grad_bf16) return bits == 8 ? launches<bf16, 8>(t, count, h, s, st) : launches<bf16, 32>(t, count, h, s, st);
  return bits == 8 ? launches<float, 8>(t, count, h, s, st) : launches<float, 32>(t, count, h, s, st);
}

cudaError_t adamw_state_values(const uint8_t* m, const uint8_t* ms, const uint8_t* v, const uint8_t* vs, void* mo, void* vo,
                               bool f32, int64_t n, cudaStream_t st) {
  if (n == 0) return cudaSuccess;
  const int grid = (int)std::min<int64_t>(cdiv(n / 8, kThreads), sm_count() * 8);
  state_values_kernel<<<grid, kThreads, 0, st>>>(m, ms, v, vs, mo, vo, f32, n / 8);
  return cudaGetLastError();
}

cudaError_t adamw_encode_states(const float* m, const float* v, uint8_t* mc, uint8_t* ms, uint8_t* vc, uint8_t* vs,
                                int64_t blocks, cudaStream_t st) {
  if (blocks == 0) return cudaSuccess;
  const int grid = (int)std::min<int64_t>(cdiv(blocks, kThreads / 32), sm_count() * 8);
  encode_states_kernel<<<grid, kThreads, 0, st>>>(m, v, mc, ms, vc, vs, blocks);
  return cudaGetLastError();
}

}  // namespace llmt

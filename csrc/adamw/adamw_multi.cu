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

// Both codes are bits 20 to 27 of an fp32 number: scaled so that the format's subnormals are fp32's
// subnormals, adding 20 random bits below the kept ones and cutting rounds up with the right
// probability, in the normal and the subnormal range alike. Here they are shifted to the top byte, where
// four of them are gathered by byte permutations, as the noise is made. noise: bits 8 to 23 random, bit 7 set (half a last step). A block's scale keeps
// every finite value within the format; infinities and NaN are put right afterwards (code_of_bad_*).
__device__ __forceinline__ uint32_t encode_m(float m, float unscale, uint32_t noise) {  // without the sign
  return (__float_as_uint(__fmul_rn(__fmul_rn(fabsf(m), unscale), 0x1p-120f)) << 4) + noise;
}
__device__ __forceinline__ uint32_t encode_v(float v, float unscale, uint32_t noise) {
  const uint32_t y = (__float_as_uint(__fmul_rn(__fmul_rn(v, unscale), 0x1p-129f)) << 4) + noise;
  return max(y, min(__float_as_uint(v), 1u) << 24);  // v >= 0: a non-zero one keeps a non-zero code
}
__device__ __forceinline__ uint32_t code_of_bad_m(float m, uint32_t code) { return m != m ? 0x7fu : fabsf(m) == INFINITY ? 126u : code; }
__device__ __forceinline__ uint32_t code_of_bad_v(float v, uint32_t code) { return v <= 3.4028235e38f ? code : 255u; }
__device__ __forceinline__ uint32_t sign_m(float m) { return (__float_as_uint(m) >> 24) & 0x80u; }

__device__ __forceinline__ float2 decode_m2(uint32_t codes, float scale) {  // two codes in the low 16 bits
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);  // exact
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return make_float2(f.x * scale, f.y * scale);
}
__device__ __forceinline__ float decode_m(uint32_t code, float scale) { return decode_m2(code & 0xffu, scale).x; }
// scale_2_29: 2^29 times the block's scale (codes are units of 2^-129 as fp32 bits; two exact steps).
__device__ __forceinline__ float decode_v(uint32_t code, float scale_2_29) {
  return __uint_as_float(code << 20) * 0x1p100f * scale_2_29;
}

// 32 mixed bits of place i: two rounds of multiplication and xor-shift; the odd constants are
// digits of e, of the square root of two and of the golden ratio.
__device__ __forceinline__ uint32_t high_mix(int64_t i) { return (uint32_t)(i >> 32) * 0x6A09E667u; }
__device__ __forceinline__ uint32_t place_hash(uint32_t low, uint32_t high, uint32_t seed) {
  uint32_t x = (low ^ high) * 0x9E3779B1u + seed;
  x = (x ^ (x >> 16)) * 0xB7E15163u;
  x = (x ^ (x >> 15)) * 0x6A09E667u;
  return x ^ (x >> 16);
}

struct StepConst {
  float b1, c1, b2, c2, eps, step_size, root, lr, grad_scale;
  uint32_t seed;
};

// The moments as written. With 32-bit states the square root and the quotient are correctly rounded, as in adamw.cu.
// With 8-bit states, themselves rounded to 2^-4, they are the approximate ones (2^-22 of the update; 374M values
// 1069 us, 1097 correctly rounded), of the kind that keeps subnormal second moments: flushed to zero, those would
// throw their weights out by lr / eps.
template <int BITS>
__device__ __forceinline__ void update(const StepConst& k, float decay, float g, float& p, float& m, float& v) {
  g = __fmul_rn(g, k.grad_scale);
  m = __fadd_rn(__fmul_rn(m, k.b1), __fmul_rn(g, k.c1));
  v = __fadd_rn(__fmul_rn(v, k.b2), __fmul_rn(__fmul_rn(g, k.c2), g));
  if constexpr (BITS == 32) {
    p = p * decay - k.step_size * (m / (sqrtf(v) * k.root + k.eps));
  } else {
    float root;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
    p = p * decay - k.step_size * __fdividef(m, root * k.root + k.eps);
  }
}

// 1 - b^t from the fp64 logarithm of b: of b rounded to fp32 the difference would lose 1.3e-5 of itself at
// b = 0.999, 1.4e-3 at 0.99999. (log 0 = -inf gives 1.)
__device__ __forceinline__ float one_less_power(double log_b, int t) { return -expm1f((float)(log_b * (double)t)); }

__device__ __forceinline__ StepConst step_const(const MultiHyper& h) {
  const int t = *h.step + 1;
  const float lr = *h.lr;
  StepConst k;
  k.b1 = h.b1;
  k.c1 = h.c1;
  k.b2 = h.b2;
  k.c2 = h.c2;
  k.eps = h.eps;
  k.lr = lr;
  k.step_size = lr / one_less_power(h.log_b1, t);
  k.root = 1.f / sqrtf(one_less_power(h.log_b2, t));
  k.grad_scale = h.grad_scale * (h.grad_scale_dev ? *h.grad_scale_dev : 1.f);
  k.seed = (uint32_t)t * 0xB7E15163u + h.seed * 0x3C6EF373u;
  return k;
}

// 32 bytes at once (the widest load and store of sm_100): a lane's eight fp32 values.
__device__ __forceinline__ void ld8(const float* p, float (&x)[8]) {
  asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
               : "l"(p));
}
__device__ __forceinline__ void st8(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}

// Exponent bytes of a block (the whole warp calls it).
struct Scales {
  uint32_t m, v;
};
__device__ __forceinline__ Scales block_scales(float top_m, float top_v) {
  return {scale_byte_m(__reduce_max_sync(0xffffffffu, __float_as_uint(top_m))),
          scale_byte_v(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v)))};
}
// The random bits of each moment from a place's 32: the upper 16 and the lower 16.
__device__ __forceinline__ uint32_t noise_m(uint32_t r) { return __byte_perm(r, 0x80u, 0x5324); }
__device__ __forceinline__ uint32_t noise_v(uint32_t r) { return __byte_perm(r, 0x80u, 0x5104); }
// The top bytes of four words.
__device__ __forceinline__ uint32_t top_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}

// A whole block of a tensor on 32-byte borders (16 for 16-bit gradients and copies): all its loads are
// issued before anything is computed.
template <typename G, int BITS>
__device__ __forceinline__ void whole_block(const MultiTensor& t, const MultiHyper& h, const MultiState& s, const StepConst& k,
                                            int64_t at, int64_t blk, int lane) {
  const float decay = 1.f - k.lr * t.wd;
  const int64_t i = at + 8 * lane, si = blk * kBlock + 8 * lane;
  float p[8], g[8], m[8], v[8];
  uint4 g16;
  if constexpr (sizeof(G) == 4) ld8(static_cast<const float*>(t.g) + i, g);
  else g16 = *reinterpret_cast<const uint4*>(static_cast<const bf16*>(t.g) + i);
  ld8(t.p + i, p);
  uint2 mc, vc;
  uint32_t em = 0, ev = 0;
  if constexpr (BITS == 8) {
    mc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(s.m) + si);
    vc = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(s.v) + si);
    em = s.ms[blk];
    ev = s.vs[blk];
  } else {
    ld8(static_cast<const float*>(s.m) + si, m);
    ld8(static_cast<const float*>(s.v) + si, v);
  }
  if constexpr (sizeof(G) == 2) {
    const uint32_t u[4] = {g16.x, g16.y, g16.z, g16.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[2 * j] = __uint_as_float(u[j] << 16);
      g[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
    }
  }
  if constexpr (BITS == 8) {
    const float sm = pow2_of(em), sv = pow2_of(ev + 29u);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = decode_m2((j < 2 ? mc.x : mc.y) >> (16 * (j & 1)), sm);
      m[2 * j] = f.x;
      m[2 * j + 1] = f.y;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = decode_v(((j < 4 ? vc.x : vc.y) >> (8 * (j & 3))) & 0xffu, sv);
  }
  float top_m = 0.f, top_v = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    update<BITS>(k, decay, g[j], p[j], m[j], v[j]);
    top_m = fmaxf(top_m, fabsf(m[j]));  // (a NaN does not set the scale)
    top_v = fmaxf(top_v, v[j]);
  }
  st8(t.p + i, p);
  if (t.p16) {
    BF16x8 o = float_to_bf16x8(p);
    *reinterpret_cast<BF16x8*>(static_cast<bf16*>(t.p16) + i) = o;
  }
  if (h.zero_grad) {
    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if constexpr (sizeof(G) == 4) st8(static_cast<float*>(t.g) + i, z);
    else *reinterpret_cast<uint4*>(static_cast<bf16*>(t.g) + i) = make_uint4(0u, 0u, 0u, 0u);
  }
  if constexpr (BITS == 8) {
    const Scales e = block_scales(top_m, top_v);
    const float um = pow2_of(254u - e.m), uv = pow2_of(254u - e.v);
    const uint32_t high = high_mix(si), low = (uint32_t)si;  // one high word for the block
    uint32_t cm[2], cv[2];
    float bad = 0.f;  // becomes NaN where a moment is infinite or NaN
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t a[4], b[4], sg[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t r = place_hash(low + 4 * q + j, high, k.seed);
        a[j] = encode_m(m[4 * q + j], um, noise_m(r));
        b[j] = encode_v(v[4 * q + j], uv, noise_v(r));
        sg[j] = __float_as_uint(m[4 * q + j]);
        bad = fmaf(m[4 * q + j], 0.f, fmaf(v[4 * q + j], 0.f, bad));
      }
      cm[q] = top_bytes(a[0], a[1], a[2], a[3]) | (top_bytes(sg[0], sg[1], sg[2], sg[3]) & 0x80808080u);
      cv[q] = top_bytes(b[0], b[1], b[2], b[3]);
    }
    if (bad != bad) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int sh = 8 * (j & 3);
        const uint32_t c = code_of_bad_m(m[j], (cm[j >> 2] >> sh) & 0x7fu) | sign_m(m[j]);
        cm[j >> 2] = (cm[j >> 2] & ~(0xffu << sh)) | c << sh;
        cv[j >> 2] = (cv[j >> 2] & ~(0xffu << sh)) | code_of_bad_v(v[j], (cv[j >> 2] >> sh) & 0xffu) << sh;
      }
    }
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(s.m) + si) = make_uint2(cm[0], cm[1]);
    *reinterpret_cast<uint2*>(static_cast<uint8_t*>(s.v) + si) = make_uint2(cv[0], cv[1]);
    if (lane == 0) {
      s.ms[blk] = (uint8_t)e.m;
      s.vs[blk] = (uint8_t)e.v;
    }
  } else {
    st8(static_cast<float*>(s.m) + si, m);
    st8(static_cast<float*>(s.v) + si, v);
  }
}

// Starts bringing a block into L2: one 128-byte line a lane. With 8-bit states the warps' own loads (registers
// for one block each) are not enough bytes in flight: with the next block asked for under the present one's
// arithmetic they wait for L2 instead of memory (2.39 -> 1.85 ms in runs of 8). With 32-bit states they are
// enough.
template <typename G, int BITS>
__device__ __forceinline__ void prefetch_block(const MultiTensor& t, const MultiState& s, int64_t at, int64_t blk, int lane) {
  constexpr int kStateLine = BITS == 32 ? 32 : 128;  // values in a line
  const char* a;
  if (lane < 8) a = reinterpret_cast<const char*>(t.p + at) + 128 * lane;
  else if (lane < 16) a = static_cast<const char*>(t.g) + sizeof(G) * at + 128 * (lane - 8);
  else if (lane < 24) a = static_cast<const char*>(s.m) + BITS / 8 * (blk * kBlock) + 128 * (lane - 16);
  else a = static_cast<const char*>(s.v) + BITS / 8 * (blk * kBlock) + 128 * (lane - 24);
  const int lines = lane < 8 ? 8 : lane < 16 ? 2 * (int)sizeof(G) : kBlock / kStateLine;
  if ((lane & 7) < lines) asm volatile("prefetch.global.L2 [%0];" ::"l"(a));
}

// A tensor's last block, or any block of a tensor off those borders: value by value, 32 apart.
template <typename G, int BITS>
__device__ __noinline__ void any_block(MultiTensor t, MultiHyper h, MultiState s, StepConst k, int64_t at, int64_t blk, int n,
                                       int lane) {
  const float decay = 1.f - k.lr * t.wd;
  const float sm = BITS == 8 ? pow2_of(s.ms[blk]) : 1.f, sv = BITS == 8 ? pow2_of(s.vs[blk] + 29u) : 1.f;
  float m[8], v[8], top_m = 0.f, top_v = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int i = lane + 32 * j;
    m[j] = v[j] = 0.f;
    if (i >= n || !LLMT_IN(at + i, at + i + 1, t.n, 611) || !LLMT_IN(blk * kBlock + i, blk * kBlock + i + 1, s.n, 612)) continue;
    const int64_t si = blk * kBlock + i;
    float p = t.p[at + i], g;
    if constexpr (sizeof(G) == 4) g = static_cast<const float*>(t.g)[at + i];
    else g = __bfloat162float(static_cast<const bf16*>(t.g)[at + i]);
    if (BITS == 8) {
      m[j] = decode_m(static_cast<const uint8_t*>(s.m)[si], sm);
      v[j] = decode_v(static_cast<const uint8_t*>(s.v)[si], sv);
    } else {
      m[j] = static_cast<const float*>(s.m)[si];
      v[j] = static_cast<const float*>(s.v)[si];
    }
    update<BITS>(k, decay, g, p, m[j], v[j]);
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
    top_m = fmaxf(top_m, fabsf(m[j]));
    top_v = fmaxf(top_v, v[j]);
  }
  if (BITS == 8) {
    const Scales e = block_scales(top_m, top_v);
    const float um = pow2_of(254u - e.m), uv = pow2_of(254u - e.v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t si = blk * kBlock + lane + 32 * j;
      if (lane + 32 * j >= n) continue;
      const uint32_t r = place_hash((uint32_t)si, high_mix(si), k.seed);
      static_cast<uint8_t*>(s.m)[si] = (uint8_t)(code_of_bad_m(m[j], encode_m(m[j], um, noise_m(r)) >> 24) | sign_m(m[j]));
      static_cast<uint8_t*>(s.v)[si] = (uint8_t)code_of_bad_v(v[j], encode_v(v[j], uv, noise_v(r)) >> 24);
    }
    if (lane == 0) {
      s.ms[blk] = (uint8_t)e.m;
      s.vs[blk] = (uint8_t)e.v;
    }
  }
}

// The tensor that block w of the launch lies in, by a whole warp: 32 tensors are looked at at once, twice at
// the most 1024, in place of ten dependent reads of the arguments.
template <int CAP>
__device__ __forceinline__ int find_tensor(const Batch<CAP>& batch, int64_t w, int lane) {
  static_assert(CAP <= 1024, "two steps of 32");
  const int step = (batch.count + 31) / 32;
  int i = lane * step;
  const int at = (__popc(__ballot_sync(0xffffffffu, i < batch.count && batch.t[min(i, CAP - 1)].first_work <= w)) - 1) * step;
  i = at + lane;
  return at + __popc(__ballot_sync(0xffffffffu, lane < step && i < batch.count && batch.t[min(i, CAP - 1)].first_work <= w)) - 1;
}

// Bound by memory: with 32-bit states 28 to 30 bytes a value, 103% of the measured copy rate for 0.94G values
// (3.89 ms); with 8-bit states 16 to 18 bytes, 97% for 374M values (1.07 ms), at 76% of the issue slots.
// A CTA takes a run of `rounds` blocks a warp, consecutive warps consecutive blocks, and ends: the memory
// serves a few hundred short runs, handed out in order, at its copy rate, but a persistent grid at 88%
// (4.57 ms), whether it sweeps through all tensors together or each CTA steps through runs of its own.
// Blocks brought to shared memory by asynchronous copies one ahead were slower with 8 bits (1.95 ms
// against 1.80, moments decoded) and no faster with 32.
template <typename G, int BITS, int CAP>
__global__ void __launch_bounds__(kThreads, 4) adamw_multi_kernel(const __grid_constant__ Batch<CAP> batch, MultiHyper h,
                                                                  MultiState s, int blocks, int rounds, bool last_launch) {
  constexpr int kWarps = kThreads / 32;
  const StepConst k = step_const(h);
  const int lane = threadIdx.x & 31;
  int tensor = -1;
  const int64_t stop = min((int64_t)blocks, (int64_t)(blockIdx.x + 1) * kWarps * rounds);
  for (int64_t w = (int64_t)blockIdx.x * kWarps * rounds + (threadIdx.x >> 5); w < stop; w += kWarps) {
    if (tensor < 0) tensor = find_tensor(batch, w, lane);
    while (tensor + 1 < batch.count && batch.t[tensor + 1].first_work <= w) ++tensor;
    const MultiTensor& t = batch.t[tensor];
    const int in_t = (int)w - t.first_work;
    const int64_t at = (int64_t)in_t * kBlock, blk = t.first_block + in_t;  // in the tensor, in the states
    const int n = (int)min((int64_t)kBlock, t.n - at);
    if (BITS == 8 && w + kWarps < stop && t.n - at >= (kWarps + 1) * kBlock)
      prefetch_block<G, BITS>(t, s, at + kWarps * kBlock, blk + kWarps, lane);
    if (!LLMT_IN(at, at + n, t.n, 613) || !LLMT_IN(blk * kBlock, (blk + 1) * kBlock, s.n, 614)) continue;
    if (t.wide && n == kBlock) whole_block<G, BITS>(t, h, s, k, at, blk, lane);
    else any_block<G, BITS>(t, h, s, k, at, blk, n, lane);
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
  const int64_t first = blockIdx.x * (int64_t)(4 * kThreads) + threadIdx.x;
#pragma unroll 4
  for (int64_t i = first; i < min(n8, first + 4 * kThreads); i += kThreads) {
    const uint2 a = reinterpret_cast<const uint2*>(m)[i], b = reinterpret_cast<const uint2*>(v)[i];
    const float sm = pow2_of(ms[i / (kBlock / 8)]), sv = pow2_of(vs[i / (kBlock / 8)] + 29u);
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
      mc[blk * kBlock + lane + 32 * j] = (uint8_t)(code_of_bad_m(x[j], encode_m(x[j], pow2_of(254u - em), 1u << 23) >> 24) | sign_m(x[j]));
      vc[blk * kBlock + lane + 32 * j] = (uint8_t)code_of_bad_v(y[j], encode_v(fabsf(y[j]), pow2_of(254u - ev), 1u << 23) >> 24);
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
    const uintptr_t g = (uintptr_t)t[i].g, p16 = (uintptr_t)t[i].p16;
    b.t[i].wide = (uintptr_t)t[i].p % 32 == 0 && g % (sizeof(G) == 4 ? 32 : 16) == 0 && p16 % 16 == 0;
    blocks += cdiv(t[i].n, (int64_t)kBlock);
  }
  b.count = count;
  LLMT_REQUIRE(blocks < 0x7fffffff, "adamw_multi: too many values for one launch");
  // whole waves of CTAs of at most `most` rounds. 8-bit blocks are small beside a CTA's start, in which the
  // arguments and the step's constants are waited for: 375M values with moments decoded take 1.85 ms in
  // runs of 8, 1.65 of 16, 1.61 of 32; 0.94G 32-bit values 3.90 ms in runs of 4, 3.97 of 8, 4.03 of 16
  constexpr int64_t most = BITS == 8 ? 32 : 4;
  const int64_t slots = (int64_t)sm_count() * 4 * (kThreads / 32), waves = cdiv(blocks, slots * most);
  const int rounds = (int)cdiv(blocks, slots * waves);
  const int grid = (int)cdiv(blocks, (int64_t)rounds * (kThreads / 32));
  adamw_multi_kernel<G, BITS, CAP><<<grid, kThreads, 0, st>>>(b, h, s, (int)blocks, rounds, last);
  return cudaGetLastError();
}

template <typename G, int BITS>
cudaError_t launches(const MultiTensor* t, int count, const MultiHyper& h, const MultiState& s, cudaStream_t st) {
  constexpr int kSmall = 64, kLarge = kTensorsPerLaunch;  // 3.1 KB and 30.7 KB of kernel arguments
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
  state_values_kernel<<<(unsigned)cdiv(n / 8, (int64_t)(4 * kThreads)), kThreads, 0, st>>>(m, ms, v, vs, mo, vo, f32, n / 8);
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

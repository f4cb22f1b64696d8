// Rotary positions for q and k in one launch (sm_100a): half and interleaved pairs, a part of the
// head, any frequencies, any positions, and the inverse rotation (the backward).
//
// Pair j of a head at position p turns by the angle p w_j:
//   y1 = x1 c - x2 s,  y2 = x2 c + x1 s    (inverse: s negated)
// x1, x2 are values j and j + rd / 2 (half) or 2 j and 2 j + 1 (interleaved) of the first rd values
// of the head; the others are handed on. c and s carry the scaling's factor.
//
// fp32 angles are no use at far positions (at 10^6 their spacing is 0.06), and a table of every
// position is as long as the context. So the position is cut into three digits,
// |p| = h 2^20 + m 2^10 + l, and the table holds e^(i digit w_j) of each digit, computed in 64 bits:
// rows 0 .. 1023 for l (times the factor), 1024 .. 2047 for m, 2048 .. 4095 for h: 2 MB for any position
// below 2^31, which stay in L2. The rotation is the product of the digits' rotations (one complex
// product up to 2^20, two beyond), three roundings of fp32 off at the most. A position outside
// (-2^31, 2^31) gives NaN.
#include <cuda_fp16.h>

#include "../common/common.cuh"

namespace llmt {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float2 cmul(float2 a, float2 b) {
  return make_float2(a.x * b.x - a.y * b.y, a.x * b.y + a.y * b.x);
}

__device__ __forceinline__ int64_t position(const RopeArgs& a, int b, int t) {
  if (!a.pos) return t;
  const int64_t i = b * a.psb + t * a.pst;
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[i] : static_cast<const int32_t*>(a.pos)[i];
}

// Cosine and sine (with the factor) of pair j at position p.
__device__ __forceinline__ float2 turn(const RopeArgs& a, int64_t p, int j) {
  const uint64_t u = p < 0 ? -(uint64_t)p : (uint64_t)p;
  if (u >> 31) return make_float2(NAN, NAN);
  const int pairs = a.rd / 2;
  const float2* tab = reinterpret_cast<const float2*>(a.table) + j;
  float2 c = cmul(tab[(int64_t)(u & 1023) * pairs], tab[(int64_t)(1024 + ((u >> 10) & 1023)) * pairs]);
  if (u >> 20) c = cmul(c, tab[(int64_t)(2048 + (u >> 20)) * pairs]);
  if ((p < 0) != a.inverse) c.y = -c.y;
  return c;
}

__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void put(bf16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void put(float& d, float v) { d = v; }

// One thread per (token, pair or value behind the rotated ones), looping over the heads.
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RopeArgs a, int64_t items, int per_token) {
  const int64_t it = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  if (it >= items) return;
  const int64_t n = it / per_token;
  const int i = (int)(it % per_token), b = (int)(n / a.T), t = (int)(n % a.T);
  const int pairs = a.rd / 2;
  const int heads = a.q.heads + a.k.heads;
  if (i >= pairs) {
    const int d = a.rd + i - pairs;
    for (int h = 0; h < heads; ++h) {
      const RopeHeads& x = h < a.q.heads ? a.q : a.k;
      const int hh = h < a.q.heads ? h : h - a.q.heads;
      static_cast<T*>(x.out)[b * x.osb + t * x.ost + hh * x.osh + d] =
          static_cast<const T*>(x.in)[b * x.isb + t * x.ist + hh * x.ish + d];
    }
    return;
  }
  const float2 c = turn(a, position(a, b, t), i);
  const int d1 = a.interleaved ? 2 * i : i, d2 = a.interleaved ? 2 * i + 1 : i + pairs;
  for (int h = 0; h < heads; ++h) {
    const RopeHeads& x = h < a.q.heads ? a.q : a.k;
    const int hh = h < a.q.heads ? h : h - a.q.heads;
    const T* in = static_cast<const T*>(x.in) + b * x.isb + t * x.ist + hh * x.ish;
    T* out = static_cast<T*>(x.out) + b * x.osb + t * x.ost + hh * x.osh;
    const float x1 = to_f(in[d1]), x2 = to_f(in[d2]);
    put(out[d1], x1 * c.x - x2 * c.y);
    put(out[d2], x2 * c.x + x1 * c.y);
  }
}

}  // namespace

cudaError_t rotary(const RopeArgs& a, int kind, cudaStream_t st) {
  LLMT_REQUIRE(a.rd > 0 && a.rd % 2 == 0 && a.rd <= a.hd, "rotary: rotary_dim must be even and at most head_dim");
  const int64_t tokens = (int64_t)a.B * a.T;
  if (tokens == 0 || a.q.heads + a.k.heads == 0) return cudaSuccess;
  const int per_token = a.rd / 2 + (a.hd - a.rd);
  const int64_t items = tokens * per_token;
  LLMT_REQUIRE(cdiv(items, (int64_t)kThreads) <= 0x7fffffff, "rotary: too many values");
  const unsigned grid = (unsigned)cdiv(items, (int64_t)kThreads);
  switch (kind) {
    case 0: rotary_kernel<bf16><<<grid, kThreads, 0, st>>>(a, items, per_token); break;
    case 1: rotary_kernel<__half><<<grid, kThreads, 0, st>>>(a, items, per_token); break;
    default: rotary_kernel<float><<<grid, kThreads, 0, st>>>(a, items, per_token); break;
  }
  return cudaGetLastError();
}

}  // namespace llmt

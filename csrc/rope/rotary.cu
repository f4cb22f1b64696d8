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
//
// Bound by memory: each value is read and written once. A thread has 8 pairs (4 of fp32) of one token,
// computes their cosines and sines once and turns the same pairs of several heads, all of whose loads
// (16 bytes each) are issued before the first is used. Where a head's rotated part is not made of such
// pieces, or an address is off their borders, a thread has single pairs.
#include <cuda_fp16.h>

#include <type_traits>

#include "../common/common.cuh"

namespace llmt {
namespace {

constexpr int kThreads = 256;
#ifdef LLMT_DEBUG_BOUNDS
constexpr bool kGuarded = true;
#else
constexpr bool kGuarded = false;
#endif

// Complex product, each part one rounded product and one fused multiply-add: spelled out, so that a value
// has the same bits whichever way it is reached.
__device__ __forceinline__ float2 cmul(float2 a, float2 b) {
  return make_float2(fmaf(a.x, b.x, -__fmul_rn(a.y, b.y)), fmaf(a.x, b.y, __fmul_rn(a.y, b.x)));
}

__device__ __forceinline__ int64_t position(const RopeArgs& a, int b, int t) {
  if (!a.pos) return t;
  const int64_t i = b * a.psb + t * a.pst;
  return a.pos64 ? static_cast<const int64_t*>(a.pos)[i] : static_cast<const int32_t*>(a.pos)[i];
}

// Cosines and sines (with the factor) of pairs j .. j + N - 1 at position p.
template <int N>
__device__ __forceinline__ void turns(const RopeArgs& a, int64_t p, int j, float2 (&c)[N]) {
  const uint64_t u = p < 0 ? -(uint64_t)p : (uint64_t)p;
  if (u >> 31) {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = make_float2(NAN, NAN);
    return;
  }
  const int64_t pairs = a.rd / 2;
  const float2* tab = reinterpret_cast<const float2*>(a.table) + j;
  auto row = [&](int64_t r, float2 (&d)[N]) {
    const float2* e = tab + r * pairs;
    if constexpr (N == 1) {
      d[0] = e[0];
    } else {  // rows of whole pieces: 16-byte borders
#pragma unroll
      for (int i = 0; i < N; i += 2) {
        const float4 f = *reinterpret_cast<const float4*>(e + i);
        d[i] = make_float2(f.x, f.y);
        d[i + 1] = make_float2(f.z, f.w);
      }
    }
  };
  float2 m[N];
  row((int64_t)(u & 1023), c);
  row((int64_t)(1024 + ((u >> 10) & 1023)), m);
#pragma unroll
  for (int i = 0; i < N; ++i) c[i] = cmul(c[i], m[i]);
  if (u >> 20) {
    row((int64_t)(2048 + (u >> 20)), m);
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = cmul(c[i], m[i]);
  }
  if ((p < 0) != a.inverse) {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i].y = -c[i].y;
  }
}

__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void put(bf16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half& d, float v) { d = __float2half_rn(v); }
__device__ __forceinline__ void put(float& d, float v) { d = v; }

// Values 2 i and 2 i + 1 of a 16-byte piece.
template <typename T>
__device__ __forceinline__ float2 pair_of(const uint4& x, int i) {
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
  if constexpr (sizeof(T) == 4) {
    return make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
  } else if constexpr (std::is_same_v<T, bf16>) {
    return make_float2(__uint_as_float(u[i] << 16), __uint_as_float(u[i] & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
  }
}
template <typename T>
__device__ __forceinline__ void put_pair(uint32_t (&u)[4], int i, float2 f) {
  if constexpr (sizeof(T) == 4) {
    u[2 * i] = __float_as_uint(f.x);
    u[2 * i + 1] = __float_as_uint(f.y);
  } else if constexpr (std::is_same_v<T, bf16>) {
    u[i] = pack_bf16x2(f.x, f.y);
  } else {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <typename T>
struct Head {
  const T* in;
  T* out;
  int64_t at_in, at_out, in_n, out_n;  // its first elements and the buffers' extents (the bounds-checked build)
  __device__ __forceinline__ bool reads(int d, int n) const { return LLMT_IN(at_in + d, at_in + d + n, in_n, 621); }
  __device__ __forceinline__ bool writes(int d, int n) const { return LLMT_IN(at_out + d, at_out + d + n, out_n, 622); }
};
// Head h of the token, q's heads first and then k's.
template <typename T>
__device__ __forceinline__ Head<T> head_of(const RopeArgs& a, int b, int t, int h) {
  const bool of_q = h < a.q.heads;
  const RopeHeads& x = of_q ? a.q : a.k;
  const int64_t i = of_q ? h : h - a.q.heads;
  const int64_t at_in = b * x.isb + t * x.ist + i * x.ish, at_out = b * x.osb + t * x.ost + i * x.osh;
  return {static_cast<const T*>(x.in) + at_in, static_cast<T*>(x.out) + at_out, at_in, at_out, x.in_n, x.out_n};
}

// WIDE: a thread has two pieces of a head, N values each: the pairs' two sides (half), or N pairs beside
// one another (interleaved), or, past the rotated part, 2 N values to hand on. Else one pair or one value.
// HEADS heads at a time, `per` in all; items are (token, group of heads, place in the head), place fastest.
template <typename T, bool WIDE, bool INTER, int HEADS>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RopeArgs a, int64_t items, int places, int groups, int per) {
  constexpr int N = WIDE ? 16 / (int)sizeof(T) : 1;
  const int64_t it = blockIdx.x * (int64_t)kThreads + threadIdx.x;
  if (it >= items) return;
  const int place = (int)(it % places);
  const int64_t rest = it / places;
  const int group = (int)(rest % groups);
  const int64_t n = rest / groups;
  const int b = (int)(n / a.T), t = (int)(n % a.T);
  const int pairs = a.rd / 2, turned = pairs / N;
  const int h0 = group * per, h1 = min(h0 + per, a.q.heads + a.k.heads);
  const bool turn = place < turned;
  int d1, d2;  // the first values of the two pieces
  if (turn) {
    d1 = INTER ? 2 * N * place : N * place;
    d2 = INTER ? d1 + N : d1 + pairs;
  } else {
    d1 = a.rd + (WIDE ? 2 * N * (place - turned) : place - turned);
    d2 = d1 + N;
  }
  const bool second = turn || (WIDE && d2 < a.hd);
  float2 c[N];
  if (turn) turns<N>(a, position(a, b, t), N * place, c);
  for (int h = h0; h < h1; h += HEADS) {
    if constexpr (WIDE) {
      uint4 x[HEADS], y[HEADS];
      T* out[HEADS];
#pragma unroll
      for (int i = 0; i < HEADS; ++i) {
        if (h + i >= h1) continue;
        const Head<T> p = head_of<T>(a, b, t, h + i);
        out[i] = p.out;
        if (!p.reads(d1, N) || !p.writes(d1, N) || (second && !(p.reads(d2, N) && p.writes(d2, N)))) {
          out[i] = nullptr;
          continue;
        }
        x[i] = *reinterpret_cast<const uint4*>(p.in + d1);
        if (second) y[i] = *reinterpret_cast<const uint4*>(p.in + d2);
      }
#pragma unroll
      for (int i = 0; i < HEADS; ++i) {
        if (h + i >= h1 || (kGuarded && !out[i])) continue;
        if (turn) {
          uint32_t u[4], v[4];
#pragma unroll
          for (int j = 0; j < N / 2; ++j) {
            float2 f = pair_of<T>(x[i], j), g = pair_of<T>(y[i], j);
            if constexpr (INTER) {
              f = cmul(c[j], f);
              g = cmul(c[N / 2 + j], g);
            } else {
              const float2 e = cmul(c[2 * j], make_float2(f.x, g.x)), o = cmul(c[2 * j + 1], make_float2(f.y, g.y));
              f = make_float2(e.x, o.x);
              g = make_float2(e.y, o.y);
            }
            put_pair<T>(u, j, f);
            put_pair<T>(v, j, g);
          }
          x[i] = make_uint4(u[0], u[1], u[2], u[3]);
          y[i] = make_uint4(v[0], v[1], v[2], v[3]);
        }
        *reinterpret_cast<uint4*>(out[i] + d1) = x[i];
        if (second) *reinterpret_cast<uint4*>(out[i] + d2) = y[i];
      }
    } else {
      const Head<T> p = head_of<T>(a, b, t, h);
      if (!p.reads(d1, 1) || !p.writes(d1, 1) || (turn && !(p.reads(d2, 1) && p.writes(d2, 1)))) continue;
      if (turn) {
        const float2 y = cmul(c[0], make_float2(to_f(p.in[d1]), to_f(p.in[d2])));
        put(p.out[d1], y.x);
        put(p.out[d2], y.y);
      } else {
        p.out[d1] = p.in[d1];
      }
    }
  }
}

// Whether every head's pieces lie on 16-byte borders.
bool on_borders(const RopeHeads& x, int e) {
  if (x.heads == 0) return true;
  const int64_t n = 16 / e;
  return (uintptr_t)x.in % 16 == 0 && (uintptr_t)x.out % 16 == 0 && x.isb % n == 0 && x.ist % n == 0 && x.ish % n == 0 &&
         x.osb % n == 0 && x.ost % n == 0 && x.osh % n == 0;
}

template <typename T, bool INTER>
cudaError_t run(const RopeArgs& a, cudaStream_t st) {
  const int n = 16 / (int)sizeof(T), heads = a.q.heads + a.k.heads;
  const bool wide = (a.rd / 2) % n == 0 && (a.hd - a.rd) % n == 0 && on_borders(a.q, sizeof(T)) && on_borders(a.k, sizeof(T));
  // the handed-on part is not touched where every head stays in place
  const bool stays = (a.q.heads == 0 || a.q.in == a.q.out) && (a.k.heads == 0 || a.k.in == a.k.out);
  const int kept = stays ? 0 : a.hd - a.rd;
  const int places = wide ? a.rd / 2 / n + (kept + 2 * n - 1) / (2 * n) : a.rd / 2 + kept;
  const int64_t tokens = (int64_t)a.B * a.T;
  // heads a thread turns: as many as leave each SM 1024 threads, 8 at the most (12.3 us with 4096 a SM, 11.1 with 512,
  // 10.2 with 1024: 4092 tokens of 32 x 64, half of each head)
  const int64_t fill = (int64_t)sm_count() * 1024;
  int per = 8;
  while (per > 1 && tokens * places * cdiv((int64_t)heads, (int64_t)per) < fill) per /= 2;
  const int groups = (int)cdiv((int64_t)heads, (int64_t)per);
  const int64_t items = tokens * places * groups;
  LLMT_REQUIRE(cdiv(items, (int64_t)kThreads) <= 0x7fffffff, "rotary: too many values");
  const unsigned grid = (unsigned)cdiv(items, (int64_t)kThreads);
  if (!wide) rotary_kernel<T, false, INTER, 1><<<grid, kThreads, 0, st>>>(a, items, places, groups, per);
  else if (per == 2) rotary_kernel<T, true, INTER, 2><<<grid, kThreads, 0, st>>>(a, items, places, groups, per);
  else if (per >= 4) rotary_kernel<T, true, INTER, 4><<<grid, kThreads, 0, st>>>(a, items, places, groups, per);
  else rotary_kernel<T, true, INTER, 1><<<grid, kThreads, 0, st>>>(a, items, places, groups, per);
  return cudaGetLastError();
}

}  // namespace

cudaError_t rotary(const RopeArgs& a, int kind, cudaStream_t st) {
  LLMT_REQUIRE(a.rd > 0 && a.rd % 2 == 0 && a.rd <= a.hd, "rotary: rotary_dim must be even and at most head_dim");
  if ((int64_t)a.B * a.T == 0 || a.q.heads + a.k.heads == 0) return cudaSuccess;
  switch (kind) {
    case 0: return a.interleaved ? run<bf16, true>(a, st) : run<bf16, false>(a, st);
    case 1: return a.interleaved ? run<__half, true>(a, st) : run<__half, false>(a, st);
    default: return a.interleaved ? run<float, true>(a, st) : run<float, false>(a, st);
  }
}

}  // namespace llmt

// Post-training losses over rows of logits (sm_100a): token log-probabilities, a clipped policy
// loss with a KL term, and a preference loss over pairs of sequences, each with its gradient.
//
// For a row z (one token, V logits) with target id y:
//   M = max z,  S = sum exp(z - M),  logp = (z[y] - M) - log S
//   gradient of a loss whose slope in logp is c:  dz = c (onehot(y) - exp(z - M) / S)
// Policy, per token with weight w (1 / tokens that count, or per sequence):
//   r = exp(logp - old),  d = ref - logp
//   loss = w [ -min(r A, clip(r, 1 - lo, 1 + hi) A) + k (e^d - 1 - d) ]
//   c    = w [ -r A where r A <= clip(r) A, else 0;  + k (1 - e^d) ]
// Preference, for the pair of sequences p (chosen) and P + p (rejected):
//   gain = sum over tokens that count of (logp - ref)  [/ their number],  D = gain_p - gain_(P+p)
//   sigmoid: (1 - s) softplus(-b D) + s softplus(b D);  hinge: max(0, 1 - b D);  ipo: (D - 1 / 2b)^2
//   c of a token = +-f'(D) / P [/ number]
// A token counts where its mask is set and its target is an id of the vocabulary; the logits of
// every other row are not read (they may hold anything), and its gradient is zero.
//
// Each row is summed by one CTA; sums, maxima and slopes are fp32, the sums over tokens fp64, and
// the gradient is rounded once, to the logits' type. No atomics touch a result: equal inputs give
// equal bits.
#include <cuda_fp16.h>

#include "../common/common.cuh"

namespace llmt {
namespace {

constexpr int kRowThreads = 512;
constexpr int kPairThreads = 256;

// e^x through the exponential of two. log2(e) in one fp32 number is 1.3e-8 short, which makes every
// e^-8 of a row's sum 1e-7 too large: a bias that the sum of a long sequence's log-probabilities
// shows (3.8e-5 of a reward over 700 tokens; 7e-6 with the second part of the constant).
__device__ __forceinline__ float exp_(float x) {
  const float t = fmaf(x, 1.44269502f, x * 1.92596299e-8f);
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return y;
}

// ---------------------------------------------------------------- 16-byte pieces of a row
template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <>
__device__ __forceinline__ float to_f<bf16>(bf16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }
template <>
__device__ __forceinline__ bf16 from_f<bf16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

template <typename T>
struct alignas(16) Piece {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// A row seen as 16-byte pieces at aligned addresses: piece c holds elements [c N - off, c N - off + N),
// the first and the last one perhaps only in part.
template <typename T>
struct RowView {
  static constexpr int N = Piece<T>::N;
  T* p;
  int V, off, pieces;
  __device__ RowView(T* row, int v) : p(row), V(v) {
    off = (int)(((uintptr_t)row & 15) / sizeof(T));
    pieces = (off + v + N - 1) / N;
  }
  __device__ __forceinline__ bool whole(int c) const { return c * N >= off && (c + 1) * N - off <= V; }
  __device__ __forceinline__ Piece<T> load(int c) const {
    const int e0 = c * N - off;
    if (whole(c)) return *reinterpret_cast<const Piece<T>*>(p + e0);
    Piece<T> r;
#pragma unroll
    for (int j = 0; j < N; ++j) r.v[j] = (e0 + j >= 0 && e0 + j < V) ? p[e0 + j] : from_f<T>(-INFINITY);
    return r;
  }
  // Stores the piece that `like` (another view of as many elements) has at c.
  __device__ __forceinline__ void store(const RowView& like, int c, const Piece<T>& x) const {
    const int e0 = c * N - like.off;
    if (like.off == off && whole(c)) {
      *reinterpret_cast<Piece<T>*>(p + e0) = x;
      return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (e0 + j >= 0 && e0 + j < V) p[e0 + j] = x.v[j];
  }
};

// ---------------------------------------------------------------- tokens
__device__ __forceinline__ bool token_counts(const TokenBatch& a, int b, int t, int64_t* y) {
  *y = a.tgt.p[b * a.tgt.sb + t * a.tgt.st];
  const bool on = a.mask.p == nullptr || a.mask.p[b * a.mask.sb + t * a.mask.st] != 0;
  return on && *y >= 0 && *y < a.V;
}

// One CTA per sequence: the number of its tokens that count. Also re-arms the loss sum's ticket.
__global__ void __launch_bounds__(256) count_tokens_kernel(TokenBatch a, int* count, unsigned* ticket) {
  const int b = blockIdx.x;
  int n = 0;
  int64_t y;
  for (int t = threadIdx.x; t < a.T; t += blockDim.x) n += token_counts(a, b, t, &y) ? 1 : 0;
  n = __reduce_add_sync(0xffffffffu, n);
  __shared__ int part[8];
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) n += part[i];
    count[b] = n;
    if (b == 0 && ticket) *ticket = 0;
  }
}

// Weight of a token of sequence b: the whole CTA calls it (it sums the counts of all sequences).
__device__ __forceinline__ float token_weight(const int* count, int B, int b, int reduction) {
  if (reduction == LOSS_SUM) return 1.f;
  __shared__ int s_sum, s_full;
  if (threadIdx.x < 32) {
    int sum = 0, full = 0;
    for (int i = threadIdx.x; i < B; i += 32) {
      sum += count[i];
      full += count[i] > 0 ? 1 : 0;
    }
    sum = __reduce_add_sync(0xffffffffu, sum);
    full = __reduce_add_sync(0xffffffffu, full);
    if (threadIdx.x == 0) {
      s_sum = sum;
      s_full = full;
    }
  }
  __syncthreads();
  if (reduction == LOSS_TOKEN) return 1.f / (float)s_sum;
  return 1.f / ((float)count[b] * (float)s_full);
}

// Loss and slope of one token, both with the weight in.
__device__ __forceinline__ void policy_token(const PolicyArgs& q, int b, int t, float logp, float w, float* loss,
                                             float* slope) {
  const float A = q.adv.p[b * q.adv.sb + t * q.adv.st];
  const float old = q.old.p ? q.old.p[b * q.old.sb + t * q.old.st] : logp;
  const float r = expf(logp - old);
  const float free = r * A, held = fminf(fmaxf(r, 1.f - q.clip_lo), 1.f + q.clip_hi) * A;
  // written so that a NaN ratio or advantage stays one (fminf and fmaxf drop it)
  float l = r != r ? r : -(free <= held ? free : held);
  float c = free <= held || r != r ? -free : 0.f;
  if (q.ref.p) {
    const float d = q.ref.p[b * q.ref.sb + t * q.ref.st] - logp;
    const float e = expm1f(d);  // e^d - 1 - d without losing a small d
    l += q.kl_coef * (e - d);
    c -= q.kl_coef * e;
  }
  *loss = l * w;
  *slope = c * w;
}

// Sum of n floats by one CTA in a fixed order, in fp64.
__device__ __forceinline__ double cta_sum(double s) {
  __shared__ double part[32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  s = part[0];
  for (int i = 1; i < (int)(blockDim.x >> 5); ++i) s += part[i];
  return s;
}

// The CTA that is the last of `total` to come here sums x[0, n) into *out, times scale.
__device__ __forceinline__ void last_one_sums(unsigned* ticket, unsigned total, const float* x, int64_t n, float scale,
                                              float* out) {
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(ticket, 1u) == total - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) s += (double)__ldcg(x + i);
  s = cta_sum(s);
  if (threadIdx.x == 0) *out = (float)(s * (double)scale);
}

// ---------------------------------------------------------------- rows
struct MaxSum {
  float m, s;
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s};
  return {m, a.s * exp_(a.m - m) + b.s * exp_(b.m - m)};
}

template <typename T>
__device__ __forceinline__ void zero_row(const RowView<T>& out) {
  Piece<T> z;
#pragma unroll
  for (int j = 0; j < Piece<T>::N; ++j) z.v[j] = from_f<T>(0.f);
  for (int c = threadIdx.x; c < out.pieces; c += blockDim.x) out.store(out, c, z);
}

template <typename T>
__device__ __forceinline__ void write_gradient(const RowView<T>& in, const RowView<T>& out, int64_t y, float m, float s,
                                               float c) {
  const float k = -c / s;
  for (int i = threadIdx.x; i < in.pieces; i += blockDim.x) {
    const Piece<T> x = in.load(i);
    Piece<T> d;
    const int64_t hit = y + in.off - (int64_t)i * Piece<T>::N;
#pragma unroll
    for (int j = 0; j < Piece<T>::N; ++j) {
      float g = k * exp_(to_f(x.v[j]) - m);
      if (hit == j) g += c;
      d.v[j] = from_f<T>(g);
    }
    out.store(in, i, d);
  }
}

// One CTA per row: its maximum, sum and log-probability; with POLICY the loss and slope of its
// token, with GRAD also the row of the gradient.
template <typename T, bool POLICY, bool GRAD>
__global__ void __launch_bounds__(kRowThreads) token_rows_kernel(TokenBatch a, PolicyArgs q, RowOut o) {
  const int64_t n = blockIdx.x;
  const int b = (int)(n / a.T), t = (int)(n % a.T);
  int64_t y;
  const bool counts = token_counts(a, b, t, &y);
  const RowView<T> in((T*)a.z + b * a.zsb + t * a.zst, a.V);
  const RowView<T> out(GRAD ? (T*)o.dz + b * o.sb + t * o.st : (T*)a.z, a.V);
  if (n == 0 && !POLICY && threadIdx.x == 0 && o.ticket) *o.ticket = 0;
  if (!counts) {
    if (threadIdx.x == 0) {
      o.logp[n] = 0.f;
      if (o.stats) o.stats[n] = make_float2(0.f, 1.f);
      if (POLICY) o.loss_rows[n] = 0.f, o.coef[n] = 0.f;
    }
    if (GRAD) zero_row(out);
  } else {
    const float zy = to_f(in.p[y]);
    MaxSum ms = {-INFINITY, 0.f};
    for (int i = threadIdx.x; i < in.pieces; i += blockDim.x) {
      const Piece<T> x = in.load(i);
      float f[Piece<T>::N], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int j = 0; j < Piece<T>::N; ++j) {
        f[j] = to_f(x.v[j]);
        top = fmaxf(top, f[j]);
      }
      const float at = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int j = 0; j < Piece<T>::N; ++j) sum += exp_(f[j] - at);
      ms = join(ms, {top, sum});
    }
#pragma unroll
    for (int w = 16; w > 0; w >>= 1)
      ms = join(ms, {__shfl_xor_sync(0xffffffffu, ms.m, w), __shfl_xor_sync(0xffffffffu, ms.s, w)});
    __shared__ MaxSum part[kRowThreads / 32];
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ms;
    __syncthreads();
    ms = part[0];
    for (int i = 1; i < (int)(blockDim.x >> 5); ++i) ms = join(ms, part[i]);
    const float logp = (zy - ms.m) - logf(ms.s);
    float loss = 0.f, slope = 0.f;
    if (POLICY) policy_token(q, b, t, logp, token_weight(o.count, a.B, b, q.reduction), &loss, &slope);
    if (threadIdx.x == 0) {
      o.logp[n] = logp;
      if (o.stats) o.stats[n] = make_float2(ms.m, ms.s);
      if (POLICY) o.loss_rows[n] = loss, o.coef[n] = slope;
    }
    if (GRAD) {
      if (slope == 0.f) zero_row(out);
      else write_gradient(in, out, y, ms.m, ms.s, slope * (o.grad_out ? *o.grad_out : 1.f));
    }
  }
  if (POLICY) last_one_sums(o.ticket, gridDim.x, o.loss_rows, gridDim.x, 1.f, o.loss);
}

// Gradient rows from the saved maxima and sums and the slope of each token. With skip_one the
// buffer already holds the gradient for an incoming gradient of 1.
template <typename T>
__global__ void __launch_bounds__(kRowThreads) grad_rows_kernel(TokenBatch a, RowOut o, bool skip_one) {
  const float g = o.grad_out ? *o.grad_out : 1.f;
  if (skip_one && g == 1.f) return;
  // the last rows first: the pass before this one left them in L2
  const int64_t n = gridDim.x - 1 - (int64_t)blockIdx.x;
  const int b = (int)(n / a.T), t = (int)(n % a.T);
  const RowView<T> in((T*)a.z + b * a.zsb + t * a.zst, a.V);
  const RowView<T> out((T*)o.dz + b * o.sb + t * o.st, a.V);
  const float c = o.coef[n];
  if (c == 0.f) {
    zero_row(out);
    return;
  }
  const float2 ms = o.stats[n];
  write_gradient(in, out, a.tgt.p[b * a.tgt.sb + t * a.tgt.st], ms.x, ms.y, c * g);
}

// ---------------------------------------------------------------- losses on log-probabilities
__global__ void __launch_bounds__(kPairThreads) policy_tokens_kernel(TokenBatch a, PolicyArgs q, const float* logp, RowOut o) {
  const int b = blockIdx.x;
  const float w = token_weight(o.count, a.B, b, q.reduction);
  for (int t = threadIdx.x; t < a.T; t += blockDim.x) {
    const int64_t n = (int64_t)b * a.T + t;
    int64_t y;
    float loss = 0.f, slope = 0.f;
    if (token_counts(a, b, t, &y)) policy_token(q, b, t, logp[n], w, &loss, &slope);
    o.loss_rows[n] = loss;
    o.coef[n] = slope;
  }
  __syncthreads();
  last_one_sums(o.ticket, gridDim.x, o.loss_rows, (int64_t)a.B * a.T, 1.f, o.loss);
}

// One CTA per pair.
__global__ void __launch_bounds__(kPairThreads) preference_kernel(TokenBatch a, PreferenceArgs q, const float* logp, RowOut o) {
  const int p = blockIdx.x, P = gridDim.x;
  double gain[2];
  int number[2];
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int b = p + side * P;
    double s = 0.0;
    int count = 0;
    for (int t = threadIdx.x; t < a.T; t += blockDim.x) {
      int64_t y;
      if (!token_counts(a, b, t, &y)) continue;
      s += (double)(logp[(int64_t)b * a.T + t] - (q.ref.p ? q.ref.p[b * q.ref.sb + t * q.ref.st] : 0.f));
      ++count;
    }
    gain[side] = cta_sum(s);
    number[side] = (int)cta_sum((double)count);
    if (q.average) gain[side] /= (double)max(number[side], 1);
  }
  const float D = (float)(gain[0] - gain[1]), x = q.beta * D;
  float loss, slope;  // of the pair, slope in D
  if (q.kind == PREF_SIGMOID) {
    const float s = q.smoothing, soft = log1pf(expf(-fabsf(x)));
    loss = (1.f - s) * (soft + fmaxf(-x, 0.f)) + s * (soft + fmaxf(x, 0.f));
    slope = q.beta * (s / (1.f + expf(-x)) - (1.f - s) / (1.f + expf(x)));
  } else if (q.kind == PREF_HINGE) {
    loss = x != x ? x : fmaxf(0.f, 1.f - x);
    slope = x < 1.f ? -q.beta : (x != x ? x : 0.f);
  } else {
    const float off = D - 0.5f / q.beta;
    loss = off * off;
    slope = 2.f * off;
  }
#pragma unroll 1
  for (int side = 0; side < 2; ++side) {
    const int b = p + side * P;
    const float c = (side ? -slope : slope) / (float)P / (q.average ? (float)max(number[side], 1) : 1.f);
    for (int t = threadIdx.x; t < a.T; t += blockDim.x) {
      int64_t y;
      o.coef[(int64_t)b * a.T + t] = token_counts(a, b, t, &y) ? c : 0.f;
    }
    if (threadIdx.x == 0) o.rewards[b] = (float)((double)q.beta * gain[side]);
  }
  if (threadIdx.x == 0) o.loss_rows[p] = loss;
  last_one_sums(o.ticket, P, o.loss_rows, P, 1.f / (float)P, o.loss);
}

template <bool POLICY, bool GRAD>
cudaError_t rows(const TokenBatch& a, const PolicyArgs& q, const RowOut& o, cudaStream_t st) {
  const unsigned n = (unsigned)((int64_t)a.B * a.T);
  switch (a.dtype) {
    case 0: token_rows_kernel<bf16, POLICY, GRAD><<<n, kRowThreads, 0, st>>>(a, q, o); break;
    case 1: token_rows_kernel<__half, POLICY, GRAD><<<n, kRowThreads, 0, st>>>(a, q, o); break;
    default: token_rows_kernel<float, POLICY, GRAD><<<n, kRowThreads, 0, st>>>(a, q, o); break;
  }
  return cudaGetLastError();
}

cudaError_t check(const TokenBatch& a) {
  LLMT_REQUIRE(a.B > 0 && a.T > 0 && a.V > 0, "loss rows: empty batch");
  LLMT_REQUIRE((int64_t)a.B * a.T <= 0x7fffffff, "loss rows: more than 2^31 - 1 tokens");
  return cudaSuccess;
}

}  // namespace

cudaError_t logprob_rows(const TokenBatch& a, const RowOut& o, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  return rows<false, false>(a, PolicyArgs{}, o, st);
}

cudaError_t policy_rows(const TokenBatch& a, const PolicyArgs& q, const RowOut& o, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  count_tokens_kernel<<<a.B, 256, 0, st>>>(a, o.count, o.ticket);
  if (cudaError_t e = cudaGetLastError()) return e;
  return o.dz ? rows<true, true>(a, q, o, st) : rows<true, false>(a, q, o, st);
}

cudaError_t policy_tokens(const TokenBatch& a, const PolicyArgs& q, const float* logp, const RowOut& o, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  count_tokens_kernel<<<a.B, 256, 0, st>>>(a, o.count, o.ticket);
  if (cudaError_t e = cudaGetLastError()) return e;
  policy_tokens_kernel<<<a.B, kPairThreads, 0, st>>>(a, q, logp, o);
  return cudaGetLastError();
}

cudaError_t preference_tokens(const TokenBatch& a, const PreferenceArgs& q, const float* logp, const RowOut& o,
                              bool ticket_ready, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  LLMT_REQUIRE(a.B % 2 == 0, "preference loss: the batch holds the chosen sequences, then as many rejected ones");
  if (!ticket_ready)
    if (cudaError_t e = cudaMemsetAsync(o.ticket, 0, sizeof(unsigned), st)) return e;
  preference_kernel<<<a.B / 2, kPairThreads, 0, st>>>(a, q, logp, o);
  return cudaGetLastError();
}

cudaError_t grad_rows(const TokenBatch& a, const RowOut& o, bool skip_one, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  const unsigned n = (unsigned)((int64_t)a.B * a.T);
  switch (a.dtype) {
    case 0: grad_rows_kernel<bf16><<<n, kRowThreads, 0, st>>>(a, o, skip_one); break;
    case 1: grad_rows_kernel<__half><<<n, kRowThreads, 0, st>>>(a, o, skip_one); break;
    default: grad_rows_kernel<float><<<n, kRowThreads, 0, st>>>(a, o, skip_one); break;
  }
  return cudaGetLastError();
}

}  // namespace llmt

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
// Bound by memory: the logits of the rows that count once, all of the gradient once. A CTA streams its row
// through two 32 KB tiles of shared memory by bulk copies, summing one while the next arrives, and
// goes back from the last tile to the first for the gradient: the last two are still there, the others are
// read again from L2 or memory. Three CTAs of 256 threads a SM work on different rows. (2 x 32 KB and 3 CTAs
// 338 us for 4 x 1024 x 128256 bf16; 3 x 32 KB and 2 CTAs 342, 4 x 16 KB 363, 2 x 24 KB and 4 CTAs 355; a row held
// by a cluster of 64 KB slices, read once but waited for as a whole, 410; gradients stored without the streaming
// hint 357.) Where there are few rows a cluster of up to 8 CTAs shares one, and exchanges the maximum and
// sum of each warp through distributed shared memory. Sums, maxima and slopes are fp32, the sums over
// tokens fp64, and the gradient is rounded once, to the logits' type. No atomics touch a result: equal inputs
// give equal bits.
#include <cuda_fp16.h>

#include <type_traits>

#include "../common/common.cuh"
#include "../common/sm100.cuh"

namespace llmt {
namespace {

constexpr int kMaxThreads = 256;        // of a CTA of a row: with 512, the 40 registers left to each cost 13%
constexpr int kTileBytes = 32 * 1024;   // of a row, two in a CTA's shared memory, three CTAs a SM
constexpr int kSliceBytes = 2 * kTileBytes;
constexpr int kMaxCluster = 8;
constexpr int kFill = 4;                // CTAs a SM up to which few rows are split further
constexpr int kPairThreads = 256;

// Exponentials. Errors of one sign matter here: those of 700 tokens' log-probabilities add up in the
// reward of their sequence. log2(e) in one fp32 number is 1.3e-8 short, which makes an e^-8 1e-7 too large: it is
// held in two parts, the second what the first leaves (a product with a constant to more than its type's digits:
// Dekker, Numerische Mathematik 18, 1971). The exponential of two is up to 8e-7 off, and short in the mean: the
// terms of a row by 3.1e-8 to 4.9e-8 where its logits are normal with a spread of 0.5 to 3, by 1.8e-8 to 4.4e-8 where they are
// uniform (64 to 20000 ids, all types). A row's logarithm takes the middle of that back (kShort).
constexpr double kLog2eExact = 1.4426950408889634074;
constexpr float kLog2e = (float)kLog2eExact, kLog2eLow = (float)(kLog2eExact - (double)kLog2e);
constexpr double kShort = 4e-8;
// e^x for x <= 0 (e^-87 below that), of the few factors that join a row's sums. With expf, which is not free of
// errors of one sign here, log-probabilities of 5110 ids came out 1.4e-8 off in the mean. Reduced as by Cody and Waite
// (Software Manual for the Elementary Functions, 1980): x = n ln 2 + r, |r| <= ln 2 / 2, ln 2 in two parts; e^r by its
// series up to r^7 (what is left, r^8 / 40320, is 6e-10 in the mean); 2^n exactly.
__device__ __forceinline__ float join_exp(float x) {
  constexpr double ln2 = 0.693147180559945309417;
  constexpr float high = (float)ln2, low = (float)(ln2 - (double)high);
  x = fmaxf(x, -87.f);
  const float n = rintf(x * kLog2e);
  const float r = fmaf(-n, low, fmaf(-n, high, x));
  float p = 1.f / 5040;
  p = fmaf(p, r, 1.f / 720);
  p = fmaf(p, r, 1.f / 120);
  p = fmaf(p, r, 1.f / 24);
  p = fmaf(p, r, 1.f / 6);
  p = fmaf(p, r, 0.5f);
  p = fmaf(p, r, 1.f);
  p = fmaf(p, r, 1.f);
  return p * __int_as_float(((int)n + 127) << 23);
}
// sum + e^(z - at), two values at a time.
__device__ __forceinline__ float2 add_exp(float2 z, float2 minus_at, float2 sum) {
  const float2 x = sm100::add2(z, minus_at);
  const float2 t = sm100::fma2(x, make_float2(kLog2e, kLog2e), sm100::mul2(x, make_float2(kLog2eLow, kLog2eLow)));
  return sm100::add2(sum, make_float2(sm100::ex2_approx(t.x), sm100::ex2_approx(t.y)));
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

// 16 bytes of a row in registers: N values of T, in pairs.
template <typename T>
struct Piece {
  static constexpr int N = 16 / sizeof(T);
  uint32_t u[4];
};
template <typename T>
__device__ __forceinline__ float2 pair_of(const Piece<T>& x, int i) {
  if constexpr (sizeof(T) == 4) {
    return make_float2(__uint_as_float(x.u[2 * i]), __uint_as_float(x.u[2 * i + 1]));
  } else if constexpr (std::is_same_v<T, bf16>) {
    return make_float2(__uint_as_float(x.u[i] << 16), __uint_as_float(x.u[i] & 0xffff0000u));
  } else {
    const uint32_t u = x.u[i];
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
}
template <typename T>
__device__ __forceinline__ void put_pair(Piece<T>& x, int i, float2 f) {
  if constexpr (sizeof(T) == 4) {
    x.u[2 * i] = __float_as_uint(f.x);
    x.u[2 * i + 1] = __float_as_uint(f.y);
  } else if constexpr (std::is_same_v<T, bf16>) {
    x.u[i] = pack_bf16x2(f.x, f.y);
  } else {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    x.u[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Larger of two values, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same_v<T, bf16>) asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <typename T>
__device__ __forceinline__ float piece_max(const Piece<T>& x, float m) {
  if constexpr (sizeof(T) == 4) {
    const float2 p = pair_of(x, 0), q = pair_of(x, 1);
    return max_nan(m, max_nan(max_nan(p.x, p.y), max_nan(q.x, q.y)));
  } else {
    Piece<T> r;
    r.u[0] = max2_nan<T>(max2_nan<T>(x.u[0], x.u[1]), max2_nan<T>(x.u[2], x.u[3]));
    const float2 p = pair_of(r, 0);
    return max_nan(m, max_nan(p.x, p.y));
  }
}

// A row seen as 16-byte pieces at aligned addresses: piece c holds elements [c N - off, c N - off + N),
// the first and the last one perhaps only in part. at and n: the row's first element and the number of
// elements of the buffer (the bounds-checked build's extents).
template <typename T>
struct RowView {
  static constexpr int N = Piece<T>::N;
  T* p;
  int V, off, pieces, whole_lo, whole_hi;
  int64_t at, n;
  __device__ RowView(T* base, int64_t at_, int64_t n_, int v) : p(base + at_), V(v), at(at_), n(n_) {
    off = (int)(((uintptr_t)p & 15) / sizeof(T));
    pieces = (off + v + N - 1) / N;
    whole_lo = off ? 1 : 0;
    whole_hi = (off + v) / N;
  }
  // Address of piece c (of whole pieces only, or to compare).
  __device__ __forceinline__ uint4* piece(int c) const { return reinterpret_cast<uint4*>(p + ((int64_t)c * N - off)); }
  // The element of place e of piece c, where the row has it.
  __device__ __forceinline__ bool has(int c, int e) const {
    const int i = c * N - off + e;
    return i >= 0 && i < V && LLMT_IN(at + i, at + i + 1, n, 602);
  }
  __device__ __forceinline__ T& element(int c, int e) const { return p[(int64_t)c * N - off + e]; }
};

// The pieces of a row's ends, element by element; the missing ones are of -inf.
template <typename T>
__device__ uint4 load_part(const RowView<T>& r, int c) {
  Piece<T> x;
  for (int j = 0; j < Piece<T>::N / 2; ++j)
    put_pair(x, j, make_float2(r.has(c, 2 * j) ? to_f(r.element(c, 2 * j)) : -INFINITY,
                               r.has(c, 2 * j + 1) ? to_f(r.element(c, 2 * j + 1)) : -INFINITY));
  return make_uint4(x.u[0], x.u[1], x.u[2], x.u[3]);
}
// Stores x, the piece c of a row that `like` views, into another view of it, element by element.
template <typename T>
__device__ void store_part(const RowView<T>& out, const RowView<T>& like, int c, const Piece<T>& x) {
  for (int j = 0; j < Piece<T>::N; ++j) {
    const int i = c * Piece<T>::N - like.off + j;
    const float2 f = pair_of(x, j / 2);  // back to the type it came from: exact
    if (i >= 0 && i < out.V && LLMT_IN(out.at + i, out.at + i + 1, out.n, 604)) out.p[i] = from_f<T>(j & 1 ? f.y : f.x);
  }
}

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
  pdl_trigger();
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

// Few tokens, averaged over tokens, are counted by each row's CTA while its row is on the way, in place of a
// kernel before it (the call for 80 rows 16.2 -> 14.4 us of host time).
__host__ __device__ inline bool counted_here(const TokenBatch& a, int reduction) {
  return reduction == LOSS_SUM || (reduction == LOSS_TOKEN && (int64_t)a.B * a.T <= kTokensCountedInRows);
}
__device__ __forceinline__ float token_weight_here(const TokenBatch& a, int reduction) {  // by one warp
  if (reduction == LOSS_SUM) return 1.f;
  const int n = a.B * a.T;
  int sum = 0;
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < n; i += 32) {
    int64_t y;
    sum += token_counts(a, i / a.T, i % a.T, &y) ? 1 : 0;
  }
  return 1.f / (float)__reduce_add_sync(0xffffffffu, sum);
}

// Weight of a token of sequence b, by one warp (it sums the counts of all sequences).
__device__ __forceinline__ float token_weight(const int* count, int B, int b, int reduction) {
  if (reduction == LOSS_SUM) return 1.f;
  int sum = 0, full = 0;
  for (int i = threadIdx.x & 31; i < B; i += 32) {
    const int c = count[i];
    sum += c;
    full += c > 0 ? 1 : 0;
  }
  sum = __reduce_add_sync(0xffffffffu, sum);
  if (reduction == LOSS_TOKEN) return 1.f / (float)sum;
  full = __reduce_add_sync(0xffffffffu, full);
  return 1.f / ((float)count[b] * (float)full);
}

// What the policy loss reads of one token.
struct PolicyToken {
  float adv, old, ref;
};
__device__ __forceinline__ PolicyToken load_token(const PolicyArgs& q, int b, int t) {
  PolicyToken k;
  k.adv = q.adv.p[b * q.adv.sb + t * q.adv.st];
  k.old = q.old.p ? q.old.p[b * q.old.sb + t * q.old.st] : 0.f;
  k.ref = q.ref.p ? q.ref.p[b * q.ref.sb + t * q.ref.st] : 0.f;
  return k;
}

// Loss and slope of one token, both with the weight in.
__device__ __forceinline__ void policy_token(const PolicyArgs& q, PolicyToken k, float logp, float w, float* loss,
                                             float* slope) {
  const float A = k.adv, r = q.old.p ? expf(logp - k.old) : (logp == logp ? 1.f : logp);
  // an advantage of zero takes no part, a ratio past fp32 included (inf * 0 would be NaN)
  const float free = A == 0.f ? 0.f : r * A;
  const float held = A == 0.f ? 0.f : fminf(fmaxf(r, 1.f - q.clip_lo), 1.f + q.clip_hi) * A;
  // a NaN ratio or advantage, or an infinite advantage under a ratio of zero, is one in the loss and in the slope:
  // fminf, fmaxf and comparisons drop it
  const bool bad = r != r || free != free;
  float l = bad ? NAN : -(free <= held ? free : held);
  float c = bad ? NAN : free <= held ? -free : 0.f;
  if (q.ref.p) {
    const float d = k.ref - logp;
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

// CTAs come here with the part that they have done of `total`; the one that completes it sums x[0, n)
// into *out, times scale.
__device__ __forceinline__ void last_one_sums(unsigned* ticket, unsigned done, unsigned total, const float* x, int64_t n,
                                              float scale, float* out) {
  __shared__ bool last;
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(ticket, done) + done == total;
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
struct alignas(8) MaxSum {  // written to other CTAs as one 8-byte vector
  float m, s;
};

// The pieces of a CTA of a row's cluster: [lo, hi), in tiles of the shared memory's size.
template <typename T, int THREADS>
struct Slice {
  static constexpr int kTile = kTileBytes / 16;
  int lo, hi;
  __device__ Slice(const RowView<T>& v, int rank, int ctas) {
    const int per = (v.pieces + ctas - 1) / ctas;
    lo = min(rank * per, v.pieces);
    hi = min(lo + per, v.pieces);
  }
  __device__ __forceinline__ int tiles() const { return max(1, (hi - lo + kTile - 1) / kTile); }
  __device__ __forceinline__ int begin(int tile) const { return lo + tile * kTile; }
  __device__ __forceinline__ int end(int tile) const { return min(hi, lo + (tile + 1) * kTile); }
  // Whether this thread is the one that has piece c.
  __device__ __forceinline__ bool owns(int c) const { return c >= lo && c < hi && (c - lo) % kTile % THREADS == (int)threadIdx.x; }
};

// Brings a tile into shared memory: its whole pieces in one bulk copy, the row's ragged ends by their
// threads. Complete after Tiles::wait. last: the tile is not read again (its lines leave L2 first).
template <typename T, int THREADS>
__device__ __forceinline__ void fill_tile(const RowView<T>& in, const Slice<T, THREADS>& s, int tile, uint4* buf, uint64_t* bar, bool last) {
  const int b = s.begin(tile), e = s.end(tile);
  const int wb = max(b, in.whole_lo), we = min(e, in.whole_hi);
  if (threadIdx.x == 0) {
    const uint32_t bytes = we > wb ? (uint32_t)(we - wb) * 16u : 0u;
    const bool inside = bytes == 0 || LLMT_IN(in.at + wb * RowView<T>::N - in.off, in.at + we * RowView<T>::N - in.off, in.n, 601);
    sm100::bar_arrive_expect_tx(bar, inside ? bytes : 0u);
    if (bytes && inside) {
      const T* src = in.p + (wb * RowView<T>::N - in.off);
      if (last) sm100::bulk_load_once(buf + (wb - b), src, bytes, bar);
      else sm100::bulk_load(buf + (wb - b), src, bytes, bar);
    }
  }
  if (b < in.whole_lo && b < e && threadIdx.x == 0) buf[0] = load_part(in, b);
  if (e > in.whole_hi && e - 1 >= b && e - 1 >= in.whole_lo && threadIdx.x == (unsigned)((e - 1 - b) % THREADS))
    buf[e - 1 - b] = load_part(in, e - 1);
}

// Pieces [b, e) of `like`, value(i) each, into the view `out` of the same row: whole pieces as such, the
// row's ends, and everything where the two views lie differently, by elements.
template <typename T, int THREADS, typename Value>
__device__ __forceinline__ void store_pieces(const RowView<T>& out, const RowView<T>& like, int b, int e, Value value) {
  if (out.off != like.off) {
    for (int i = b + (int)threadIdx.x; i < e; i += THREADS) store_part(out, like, i, value(i));
    return;
  }
  const int we = min(e, out.whole_hi);
  uint4* const base = out.piece(0);
  const int wb = max(b, out.whole_lo);
  const bool inside = we <= wb || LLMT_IN(out.at + (int64_t)wb * Piece<T>::N - out.off, out.at + (int64_t)we * Piece<T>::N - out.off, out.n, 603);
  if (inside) {
#pragma unroll 4
    for (int i = b + (int)threadIdx.x; i < we; i += THREADS) {
      const Piece<T> d = value(i);
      if (i >= out.whole_lo) __stcs(base + i, make_uint4(d.u[0], d.u[1], d.u[2], d.u[3]));
    }
  }
  if (b < out.whole_lo && b < e && threadIdx.x == 0) store_part(out, like, b, value(b));
  if (e > out.whole_hi && e - 1 >= max(b, out.whole_lo) && threadIdx.x == (unsigned)((e - 1 - b) % THREADS))
    store_part(out, like, e - 1, value(e - 1));
}

template <typename T, int THREADS>
__device__ __forceinline__ void zero_row(const RowView<T>& out, int rank, int ctas) {
  const Slice<T, THREADS> s(out, rank, ctas);
  store_pieces<T, THREADS>(out, out, s.lo, s.hi, [](int) { return Piece<T>{{0u, 0u, 0u, 0u}}; });
}

// Two values of the gradient without the target's own term: k e^(z - M). The maximum is subtracted first, for
// every type: a multiply-add of z around a rounded M log2(e) would be off by 2^-24 of M log2(e) (1.3e-3 of the
// gradient at fp16 logits of 6e4, most of it at bf16 ones of 1e8), and at the maximum itself by enough to turn the
// sign of c (1 - p) of a token that is almost certain.
__device__ __forceinline__ float2 gradient_pair(float2 z, float m, float2 k2) {
  const float2 t = sm100::mul2(sm100::add2(z, make_float2(-m, -m)), make_float2(kLog2e, kLog2e));
  return sm100::mul2(k2, make_float2(sm100::ex2_approx(t.x), sm100::ex2_approx(t.y)));
}
template <typename T>
__device__ __forceinline__ Piece<T> gradient_piece(uint4 v, float m, float2 k2) {
  const Piece<T> x = {{v.x, v.y, v.z, v.w}};
  Piece<T> d;
#pragma unroll
  for (int h = 0; h < Piece<T>::N / 2; ++h) put_pair(d, h, gradient_pair(pair_of(x, h), m, k2));
  return d;
}
// The target's value once more, with its own term, by the thread that stored its piece.
template <typename T>
__device__ __forceinline__ void gradient_target(const RowView<T>& out, int y, float zy, float m, float k, float c) {
  out.p[y] = from_f<T>(gradient_pair(make_float2(zy, zy), m, make_float2(k, k)).x + c);
}

// Maximum and sum of the whole row from those of each warp, by one warp; a row with an infinite or NaN
// maximum has sum NaN (its log-probability and gradient then are).
__device__ __forceinline__ MaxSum join_warps(const MaxSum* part, int n) {
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x & 31; i < n; i += 32) m = max_nan(m, part[i].m);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, w));
  for (int i = threadIdx.x & 31; i < n; i += 32) s += part[i].s * join_exp(part[i].m - m);
  s = warp_sum(s);
  if (!(fabsf(m) < INFINITY)) s = NAN;
  return {m, s};
}

// The maximum's own term of a sum is exactly 1; the others are kShort short. The logarithm is in fp64:
// one rounded to fp32 lies on the grid of the result (the difference of two 16-bit logits does too),
// and what is added to it then only decides ties, always to one side.
__device__ __forceinline__ float row_logp(float zy, MaxSum r) {
  const double s = (double)r.s;
  return (float)((double)(zy - r.m) - (log(s) + kShort * (double)(1.f - 1.f / r.s)));
}

__device__ int g_error = 0;  // 1: a copy did not arrive within its wait's limit (the results are void)

// A row's tiles in a CTA's two buffers, tile t in buffer t & 1: the next one is on its way while one is worked on.
// One warp polls for a copy while the others rest at the CTA's barrier: eight polling warps take issue slots
// from the other rows' arithmetic. After a wait that ran out, one more for the copy: the CTA must not end under it.
template <typename T, int THREADS>
struct Tiles {
  const RowView<T>& in;
  const Slice<T, THREADS>& s;
  uint4* buf;
  uint64_t* bar;
  uint32_t phase = 0;  // bit b: of buffer b's barrier
  __device__ __forceinline__ void init() {
    if (threadIdx.x == 0) {
      sm100::bar_init(&bar[0], 1);
      sm100::bar_init(&bar[1], 1);
      sm100::fence_barrier_init();
      sm100::fence_proxy_async_smem();
    }
    __syncwarp();  // the other lanes of the warp that polls come to the barriers after they are made
  }
  __device__ __forceinline__ uint4* at(int tile) const { return buf + (tile & 1) * Slice<T, THREADS>::kTile; }
  __device__ __forceinline__ void fill(int tile, bool last) const { fill_tile(in, s, tile, at(tile), &bar[tile & 1], last); }
  // Into the buffer of a tile that the CTA has read.
  __device__ __forceinline__ void refill(int tile, bool last) const {
    __syncthreads();
    if (threadIdx.x == 0) sm100::fence_proxy_async_smem();
    fill(tile, last);
  }
  __device__ __forceinline__ const uint4* wait(int tile) {
    const int b = tile & 1;
    const uint32_t parity = phase >> b & 1;
    if (threadIdx.x < 32 && !sm100::wait_bar(&bar[b], parity, &g_error, 1)) sm100::wait_bar(&bar[b], parity, &g_error, 1);
    __syncthreads();
    sm100::bar_try_wait(&bar[b], parity);  // done: each thread sees the copy for itself
    phase ^= 1u << b;
    return at(tile);
  }
};

// One cluster per row: its maximum, sum and log-probability; with POLICY the loss and slope of its
// token, with GRAD also the row of the gradient, which goes back over the row's tiles: a slice of up to two is
// still in shared memory, of longer ones the tiles before the last two are read again. The CTAs on a SM work on
// different rows, so that one's copy runs under another's arithmetic.
template <typename T, int THREADS, bool POLICY, bool GRAD>
__global__ void __launch_bounds__(THREADS, 768 / THREADS) token_rows_kernel(TokenBatch a, PolicyArgs q, RowOut o, int ctas) {
  constexpr int kWarps = THREADS / 32;
  extern __shared__ uint4 buf[];
  __shared__ MaxSum part[kMaxCluster * kWarps];
  __shared__ float s_row[3];
  __shared__ uint64_t bar[2];
  const int64_t n = blockIdx.x / ctas;
  const int rank = (int)(blockIdx.x % ctas), warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
  const int b = (int)(n / a.T), t = (int)(n % a.T);
  int64_t y;
  const bool counts = token_counts(a, b, t, &y);  // the same for the whole cluster
  const RowView<T> in((T*)a.z, b * a.zsb + t * a.zst, a.zn, a.V);
  const RowView<T> out(GRAD ? (T*)o.dz : (T*)a.z, GRAD ? b * o.sb + t * o.st : 0, GRAD ? o.dn : a.zn, a.V);
  pdl_trigger();
  if (!counts) {
    pdl_wait();
    if (rank == 0 && threadIdx.x == 0) {
      if (n == 0 && !POLICY && o.ticket) *o.ticket = 0;
      o.logp[n] = 0.f;
      if (o.stats) o.stats[n] = make_float2(0.f, 1.f);
      if (POLICY) o.loss_rows[n] = 0.f, o.coef[n] = 0.f;
    }
    if (GRAD) zero_row<T, THREADS>(out, rank, ctas);
  } else {
    const Slice<T, THREADS> s(in, rank, ctas);
    const int tiles = s.tiles();
    Tiles<T, THREADS> held{in, s, buf, bar};
    held.init();
    held.fill(0, GRAD && tiles <= 2);  // thread 0 made the barriers
    if (tiles > 1) held.fill(1, GRAD && tiles <= 3);
    // (a CTA's shared memory may be written by others once it has begun)
    if (ctas > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    // what the token's loss needs, while the row is on its way
    const float zy = to_f(in.p[y]);
    PolicyToken token = {};
    float weight = 0.f;
    if (POLICY && warp == 0) {
      token = load_token(q, b, t);
      if (counted_here(a, q.reduction)) {
        weight = token_weight_here(a, q.reduction);
      } else {
        pdl_wait();  // the counts
        weight = token_weight(o.count, a.B, b, q.reduction);
      }
    }
    MaxSum ms = {-INFINITY, 0.f};
    for (int tile = 0; tile < tiles; ++tile) {
      const uint4* const x = held.wait(tile);
      const int count = s.end(tile) - s.begin(tile);
      float m = ms.m;
#pragma unroll 4
      for (int i = threadIdx.x; i < count; i += THREADS) {
        const uint4 v = x[i];
        m = piece_max(Piece<T>{{v.x, v.y, v.z, v.w}}, m);
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, w));
      const float at = m == -INFINITY ? 0.f : m;
      float2 sum = make_float2(ms.s == 0.f ? 0.f : ms.s * join_exp(ms.m - at), 0.f);
#pragma unroll 4
      for (int i = threadIdx.x; i < count; i += THREADS) {
        const uint4 v = x[i];
        const Piece<T> f = {{v.x, v.y, v.z, v.w}};
#pragma unroll
        for (int h = 0; h < Piece<T>::N / 2; ++h) sum = add_exp(pair_of(f, h), make_float2(-at, -at), sum);
      }
      ms.m = m;
      ms.s = sum.x + sum.y;
      if (tile + 2 < tiles) held.refill(tile + 2, GRAD && tile + 4 >= tiles);
    }
    ms.s = warp_sum(ms.s);
    // every warp's pair to every CTA of the cluster
    if (ctas > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (lane < ctas) {
      MaxSum* slot = &part[rank * kWarps + warp];
      if (ctas == 1) {
        *slot = ms;
      } else {
        const uint32_t to = sm100::cluster_map(slot, lane);
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(to), "f"(ms.m), "f"(ms.s) : "memory");
      }
    }
    if (ctas == 1) __syncthreads();
    else sm100::cluster_sync();
    pdl_wait();  // nothing is written before
    if (warp == 0) {
      ms = join_warps(part, ctas * kWarps);
      const float logp = row_logp(zy, ms);
      float loss = 0.f, slope = 0.f;
      if (POLICY) policy_token(q, token, logp, weight, &loss, &slope);
      if (lane == 0) {
        if (rank == 0) {
          if (n == 0 && !POLICY && o.ticket) *o.ticket = 0;
          o.logp[n] = logp;
          if (o.stats) o.stats[n] = make_float2(ms.m, ms.s);
          if (POLICY) o.loss_rows[n] = loss, o.coef[n] = slope;
        }
        s_row[0] = ms.m;
        s_row[1] = -slope / ms.s;
        s_row[2] = slope;
      }
    }
    if (GRAD) {
      __syncthreads();
      const float m = s_row[0], k = s_row[1], c = s_row[2];
      if (c == 0.f) {
        zero_row<T, THREADS>(out, rank, ctas);
      } else {
        for (int tile = tiles - 1; tile >= 0; --tile) {  // the last two are still there, the others in L2
          const uint4* const x = tile + 2 < tiles ? held.wait(tile) : held.at(tile);
          const int first = s.begin(tile);
          store_pieces<T, THREADS>(out, in, first, s.end(tile),
                                   [&](int i) { return gradient_piece<T>(x[i - first], m, make_float2(k, k)); });
          if (tile >= 2) held.refill(tile - 2, true);
        }
        if (s.owns(((int)y + in.off) / Piece<T>::N)) gradient_target(out, (int)y, zy, m, k, c);
      }
    }
  }
}

// The loss from its rows, in a fixed order. A kernel of its own: a ticket taken by each row's CTA needs a
// fence after the row's loss, and the fence waits for the CTA's gradient to reach memory (10 us of
// 110 at 4096 rows of 32000 bf16).
__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* x, int64_t n, float* out) {
  pdl_wait();
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) s += (double)x[i];
  s = cta_sum(s);
  if (threadIdx.x == 0) *out = (float)s;
}

// Gradient rows from the saved maxima and sums and the slope of each token. With skip_one the
// buffer already holds the gradient for an incoming gradient of 1.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 768 / THREADS) grad_rows_kernel(TokenBatch a, RowOut o, bool skip_one, int ctas) {
  extern __shared__ uint4 buf[];
  __shared__ uint64_t bar[2];
  pdl_trigger();
  const float g = o.grad_out ? *o.grad_out : 1.f;
  if (skip_one && g == 1.f) return;
  // the last rows first: the pass before this one left them in L2
  const int64_t n = (gridDim.x - 1 - (int64_t)blockIdx.x) / ctas;
  const int rank = (int)((gridDim.x - 1 - blockIdx.x) % ctas);
  const int b = (int)(n / a.T), t = (int)(n % a.T);
  int64_t y;
  const bool counts = token_counts(a, b, t, &y);
  const RowView<T> in((T*)a.z, b * a.zsb + t * a.zst, a.zn, a.V);
  const RowView<T> out((T*)o.dz, b * o.sb + t * o.st, o.dn, a.V);
  const Slice<T, THREADS> s(in, rank, ctas);
  const int tiles = s.tiles();
  const bool mine = counts && s.owns(((int)y + in.off) / Piece<T>::N);
  const float zy = mine ? to_f(in.p[y]) : 0.f;
  Tiles<T, THREADS> held{in, s, buf, bar};
  held.init();
  // the copies run while the slopes are waited for
  if (counts) {
    held.fill(tiles - 1, true);
    if (tiles > 1) held.fill(tiles - 2, true);
  }
  pdl_wait();
  const float c = o.coef[n] * g;
  if (!counts || c == 0.f) {
    if (counts) {  // a token without a slope: its copies must not outlive the CTA
      held.wait(tiles - 1);
      if (tiles > 1) held.wait(tiles - 2);
    }
    zero_row<T, THREADS>(out, rank, ctas);
    return;
  }
  const float2 ms = o.stats[n];
  const float k = -c / ms.y;
  for (int tile = tiles - 1; tile >= 0; --tile) {
    const uint4* const x = held.wait(tile);
    const int first = s.begin(tile);
    store_pieces<T, THREADS>(out, in, first, s.end(tile),
                             [&](int i) { return gradient_piece<T>(x[i - first], ms.x, make_float2(k, k)); });
    if (tile >= 2) held.refill(tile - 2, true);
  }
  if (mine) gradient_target(out, (int)y, zy, ms.x, k, c);
}

// ---------------------------------------------------------------- losses on log-probabilities
__global__ void __launch_bounds__(kPairThreads) policy_tokens_kernel(TokenBatch a, PolicyArgs q, const float* logp, RowOut o) {
  const int b = blockIdx.x;
  const float w = token_weight(o.count, a.B, b, q.reduction);  // each warp for itself
  for (int t = threadIdx.x; t < a.T; t += blockDim.x) {
    const int64_t n = (int64_t)b * a.T + t;
    int64_t y;
    float loss = 0.f, slope = 0.f;
    if (token_counts(a, b, t, &y)) policy_token(q, load_token(q, b, t), logp[n], w, &loss, &slope);
    o.loss_rows[n] = loss;
    o.coef[n] = slope;
  }
  __syncthreads();
  last_one_sums(o.ticket, 1, gridDim.x, o.loss_rows, (int64_t)a.B * a.T, 1.f, o.loss);
}

// One CTA per pair, half of its threads for each sequence.
__global__ void __launch_bounds__(kPairThreads) preference_kernel(TokenBatch a, PreferenceArgs q, const float* logp, RowOut o) {
  constexpr int kHalf = kPairThreads / 2;
  const int p = blockIdx.x, P = gridDim.x;
  const int side = threadIdx.x >= kHalf, own = p + side * P;
  pdl_trigger();
  // what does not depend on the log-probabilities, of the first four tokens of each thread
  bool counts[4];
  float ref[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = (int)threadIdx.x % kHalf + i * kHalf;
    int64_t y;
    counts[i] = t < a.T && token_counts(a, own, t, &y);
    ref[i] = counts[i] && q.ref.p ? q.ref.p[own * q.ref.sb + t * q.ref.st] : 0.f;
  }
  pdl_wait();  // the log-probabilities
  double s = 0.0;
  int n = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (counts[i]) {
      s += (double)(logp[(int64_t)own * a.T + threadIdx.x % kHalf + i * kHalf] - ref[i]);
      ++n;
    }
  for (int t = (int)threadIdx.x % kHalf + 4 * kHalf; t < a.T; t += kHalf) {
    int64_t y;
    if (!token_counts(a, own, t, &y)) continue;
    s += (double)(logp[(int64_t)own * a.T + t] - (q.ref.p ? q.ref.p[own * q.ref.sb + t * q.ref.st] : 0.f));
    ++n;
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
  n = __reduce_add_sync(0xffffffffu, n);
  __shared__ double sums[kPairThreads / 32];
  __shared__ int counted[kPairThreads / 32];
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s, counted[threadIdx.x >> 5] = n;
  __syncthreads();
  double gain[2] = {0.0, 0.0};
  int number[2] = {0, 0};
#pragma unroll
  for (int w = 0; w < kPairThreads / 32; ++w) {
    gain[w >= kHalf / 32] += sums[w];
    number[w >= kHalf / 32] += counted[w];
  }
  if (q.average) {
    gain[0] /= (double)max(number[0], 1);
    gain[1] /= (double)max(number[1], 1);
  }
  const float D = (float)(gain[0] - gain[1]), x = q.beta * D;
  float loss, slope;  // of the pair, slope in D
  if (q.kind == PREF_SIGMOID) {
    const float s = q.smoothing, soft = log1pf(expf(-fabsf(x)));
    loss = (1.f - s) * (soft + fmaxf(-x, 0.f));
    if (s > 0.f) loss += s * (soft + fmaxf(x, 0.f));  // (0 times the infinity of an impossible rejected token is 0)
    slope = q.beta * (s / (1.f + expf(-x)) - (1.f - s) / (1.f + expf(x)));
  } else if (q.kind == PREF_HINGE) {
    loss = x != x ? x : fmaxf(0.f, 1.f - x);
    slope = x < 1.f ? -q.beta : (x != x ? x : 0.f);
  } else {
    const float off = D - 0.5f / q.beta;
    loss = off * off;
    slope = 2.f * off;
  }
  const float c = (side ? -slope : slope) / (float)P / (q.average ? (float)max(side ? number[1] : number[0], 1) : 1.f);
  for (int t = (int)threadIdx.x % kHalf; t < a.T; t += kHalf) {
    int64_t y;
    o.coef[(int64_t)own * a.T + t] = token_counts(a, own, t, &y) ? c : 0.f;
  }
  if (threadIdx.x % kHalf == 0) o.rewards[own] = (float)((double)q.beta * (side ? gain[1] : gain[0]));
  if (P == 1) {
    if (threadIdx.x == 0) *o.loss = loss;
    return;
  }
  if (threadIdx.x == 0) o.loss_rows[p] = loss;
  last_one_sums(o.ticket, 1, P, o.loss_rows, P, 1.f / (float)P, o.loss);
}

// One CTA a row where there are enough of them for every SM, each streaming its row's tiles; few rows are
// split over clusters.
struct RowShape {
  int ctas, threads, bytes;
};
RowShape row_shape(const TokenBatch& a) {
  const int e = a.dtype == 2 ? 4 : 2;
  const int64_t pieces = cdiv((int64_t)a.V * e, 16) + 1, n = (int64_t)a.B * a.T;
  RowShape r{1, kMaxThreads, 0};
  while (r.ctas < kMaxCluster && n * r.ctas * 2 <= kFill * sm_count() && pieces >= 512 * r.ctas) r.ctas *= 2;
  const int64_t per = cdiv(pieces, (int64_t)r.ctas);
  r.threads = per <= 512 ? 128 : 256;
  r.bytes = (int)(per * 16 <= kTileBytes ? per * 16 : kSliceBytes);
  return r;
}

// pdl: may start while the kernel before it in the stream, one of this file, runs.
template <auto KERNEL, typename... A>
cudaError_t launch_rows(const TokenBatch& a, RowShape r, bool pdl, cudaStream_t st, A... args) {
  const int64_t n = (int64_t)a.B * a.T;
  LLMT_REQUIRE(n * r.ctas <= 0x7fffffff, "loss rows: too many tokens");
  static std::atomic<uint64_t> ready{0};  // devices on which the kernel may have its shared memory
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (r.bytes > 48 * 1024 && (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
    if (cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceBytes)) return e;
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = (unsigned)(n * r.ctas);
  cfg.blockDim = r.threads;
  cfg.dynamicSmemBytes = r.bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {(unsigned)r.ctas, 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, KERNEL, args...);
}

template <typename T, bool POLICY, bool GRAD>
cudaError_t rows_of(const TokenBatch& a, RowShape r, const PolicyArgs& q, const RowOut& o, bool pdl, cudaStream_t st) {
  switch (r.threads) {
    case 128: return launch_rows<token_rows_kernel<T, 128, POLICY, GRAD>>(a, r, pdl, st, a, q, o, r.ctas);
    default: return launch_rows<token_rows_kernel<T, 256, POLICY, GRAD>>(a, r, pdl, st, a, q, o, r.ctas);
  }
}
template <bool POLICY, bool GRAD>
cudaError_t rows(const TokenBatch& a, const PolicyArgs& q, const RowOut& o, bool pdl, cudaStream_t st) {
  const RowShape r = row_shape(a);
  switch (a.dtype) {
    case 0: return rows_of<bf16, POLICY, GRAD>(a, r, q, o, pdl, st);
    case 1: return rows_of<__half, POLICY, GRAD>(a, r, q, o, pdl, st);
    default: return rows_of<float, POLICY, GRAD>(a, r, q, o, pdl, st);
  }
}
template <typename T>
cudaError_t grad_rows_of(const TokenBatch& a, const RowOut& o, bool skip_one, bool pdl, cudaStream_t st) {
  const RowShape r = row_shape(a);
  switch (r.threads) {
    case 128: return launch_rows<grad_rows_kernel<T, 128>>(a, r, pdl, st, a, o, skip_one, r.ctas);
    default: return launch_rows<grad_rows_kernel<T, 256>>(a, r, pdl, st, a, o, skip_one, r.ctas);
  }
}

cudaError_t check(const TokenBatch& a) {
  LLMT_REQUIRE(a.B > 0 && a.T > 0 && a.V > 0, "loss rows: empty batch");
  LLMT_REQUIRE((int64_t)a.B * a.T <= 0x7fffffff, "loss rows: more than 2^31 - 1 tokens");
  return cudaSuccess;
}

}  // namespace

cudaError_t logprob_rows(const TokenBatch& a, const RowOut& o, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  return rows<false, false>(a, PolicyArgs{}, o, false, st);
}

cudaError_t policy_rows(const TokenBatch& a, const PolicyArgs& q, const RowOut& o, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  const bool count = !counted_here(a, q.reduction);
  if (count) {
    count_tokens_kernel<<<a.B, 256, 0, st>>>(a, o.count, o.ticket);
    if (cudaError_t e = cudaGetLastError()) return e;
  }
  if (cudaError_t e = o.dz ? rows<true, true>(a, q, o, count, st) : rows<true, false>(a, q, o, count, st)) return e;
  const int64_t n = (int64_t)a.B * a.T;
  return launch_pdl_if(true, sum_rows_kernel, 1, n <= 2048 ? 128 : 1024, 0, st, (const float*)o.loss_rows, n, o.loss);
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
  return launch_pdl_if(ticket_ready, preference_kernel, a.B / 2, kPairThreads, 0, st, a, q, logp, o);
}

cudaError_t grad_rows(const TokenBatch& a, const RowOut& o, bool skip_one, bool after_loss, cudaStream_t st) {
  if (cudaError_t e = check(a)) return e;
  switch (a.dtype) {
    case 0: return grad_rows_of<bf16>(a, o, skip_one, after_loss, st);
    case 1: return grad_rows_of<__half>(a, o, skip_one, after_loss, st);
    default: return grad_rows_of<float>(a, o, skip_one, after_loss, st);
  }
}

int loss_error_code(bool reset) {
  int v = 0;
  cudaMemcpyFromSymbol(&v, g_error, sizeof(int));
  if (reset) {
    const int z = 0;
    cudaMemcpyToSymbol(g_error, &z, sizeof(int));
  }
  return v;
}

}  // namespace llmt

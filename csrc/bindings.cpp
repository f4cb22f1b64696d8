// PyTorch glue of the llmt native extension (module llmt._C).
//
// The only translation unit that includes torch: it validates tensors (device, dtype,
// layout), allocates outputs through the caching allocator, and calls the plain launch API
// of api.h on the current CUDA stream. Launch errors become Python exceptions.
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <numeric>

#include "api.h"

// Messages are put together here, numbers by std::to_string: a number streamed into TORCH_CHECK's
// message ends the process where torch and this module bring two copies of the C++ library's locales.
template <typename... A>
std::string message(const A&... a) {
  std::string s = "llmt: ";
  auto one = [&s](const auto& x) {
    using X = std::decay_t<decltype(x)>;
    if constexpr (std::is_same_v<X, at::ScalarType>) s += c10::toString(x);
    else if constexpr (std::is_arithmetic_v<X>) s += std::to_string(x);
    else s += x;
  };
  (one(a), ...);
  return s;
}
#define CHECK(cond, ...) TORCH_CHECK(cond, message(__VA_ARGS__))
#define CHECK_DT(t, dt) CHECK((t).scalar_type() == (dt), #t " has dtype ", (t).scalar_type(), ", expected ", (dt))

namespace {

cudaStream_t stream() { return c10::cuda::getCurrentCUDAStream().stream(); }

void ok(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return;
  if (e == cudaErrorInvalidValue && llmt::last_error()[0]) {
    TORCH_CHECK(false, "llmt: ", what, ": ", llmt::last_error());
  }
  TORCH_CHECK(false, "llmt: ", what, ": ", cudaGetErrorString(e));
}

// An uninitialised tensor on the current device, without the dispatcher (0.5 us in place of 1.2, which calls of
// a few microseconds show).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType dt) {
  return at::detail::empty_cuda(sizes, dt, at::Device(at::kCUDA, c10::cuda::current_device()), c10::nullopt);
}

void on_device(const at::Tensor& t, const char* name);
int float_kind(const at::Tensor& t, const char* name);
void all_on_device(std::initializer_list<std::pair<const c10::optional<at::Tensor>, const char*>> given);

void cuda2d(const at::Tensor& t, const char* name) {
  on_device(t, name);
  CHECK(t.dim() == 2 && t.stride(1) == 1, name, " must be 2D with unit inner stride");
}

// Every pointer a kernel dereferences must be memory of the launching device.
void on_device(const at::Tensor& t, const char* name) {
  CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  CHECK(t.get_device() == c10::cuda::current_device(), name, " is on cuda:", t.get_device(), ", the launch on cuda:",
        (int)c10::cuda::current_device());
}

const void* opt_ptr(const c10::optional<at::Tensor>& t, const char* name = "operand") {
  if (!(t.has_value() && t->defined())) return nullptr;
  on_device(*t, name);
  return t->data_ptr();
}

// Whether two tensors share a byte, at any strides (not negative): rows (values at unit stride along the last
// dimension, else single ones) at the distances that the other dimensions give. Searches the rows' distances, largest stride first, where what the smaller
// strides add can still reach the other row: a few steps where strides nest, as those of heads in packed rows do.
struct RowOverlap {
  struct Dim {
    int64_t stride, lo, hi;  // distance per step in bytes, steps
  };
  std::vector<Dim> dims;
  std::vector<int64_t> rest_lo, rest_hi;  // what the dimensions from one on add to a distance
  int64_t row_a = 0, row_b = 0;
  int left = 1 << 16;  // steps; layouts that need more count as overlapping

  static bool in_rows(const at::Tensor& t) { return t.dim() > 0 && t.stride(-1) == 1; }
  static int64_t row(const at::Tensor& t) { return t.element_size() * (in_rows(t) ? t.size(-1) : 1); }
  void add(const at::Tensor& t, int64_t sign) {
    for (int64_t i = 0; i < t.dim() - (in_rows(t) ? 1 : 0); ++i) {
      const int64_t s = t.stride(i) * t.element_size(), n = t.size(i) - 1;
      if (s == 0 || n == 0) continue;
      auto d = std::find_if(dims.begin(), dims.end(), [&](const Dim& x) { return x.stride == s; });
      if (d == dims.end()) d = dims.insert(d, {s, 0, 0});
      (sign > 0 ? d->hi : d->lo) += sign * n;
    }
  }
  bool from(size_t k, int64_t at) {  // at: bytes from b's row to a's so far
    if (at + rest_hi[k] <= -row_a || at + rest_lo[k] >= row_b) return false;
    if (k == dims.size()) return true;
    for (int64_t i = dims[k].lo; i <= dims[k].hi; ++i) {
      const int64_t x = at + i * dims[k].stride;
      if (x + rest_hi[k + 1] <= -row_a) {  // to the first step that reaches
        i += std::max<int64_t>(0, (-row_a - x - rest_hi[k + 1]) / dims[k].stride - 1);
        continue;
      }
      if (x + rest_lo[k + 1] >= row_b) break;
      if (--left < 0 || from(k + 1, x)) return true;
    }
    return false;
  }
  bool operator()(const at::Tensor& a, const at::Tensor& b) {
    if (a.numel() == 0 || b.numel() == 0) return false;
    row_a = row(a);
    row_b = row(b);
    add(a, 1);
    add(b, -1);
    std::sort(dims.begin(), dims.end(), [](const Dim& x, const Dim& y) { return x.stride > y.stride; });
    rest_lo.assign(dims.size() + 1, 0);
    rest_hi.assign(dims.size() + 1, 0);
    for (size_t k = dims.size(); k-- > 0;) {
      rest_lo[k] = rest_lo[k + 1] + dims[k].lo * dims[k].stride;
      rest_hi[k] = rest_hi[k + 1] + dims[k].hi * dims[k].stride;
    }
    return from(0, (const char*)a.data_ptr() - (const char*)b.data_ptr());
  }
};

void apart(const c10::optional<at::Tensor>& y, const c10::optional<at::Tensor>& x, const char* op, const char* y_name, const char* x_name) {
  if (y.has_value() && y->defined() && x.has_value() && x->defined())
    CHECK(!RowOverlap()(*y, *x), op, y_name, " overlaps ", x_name);
}

// ---------------------------------------------------------------- norms
std::vector<at::Tensor> add_rmsnorm_fwd(c10::optional<at::Tensor> a, at::Tensor r, at::Tensor w, double eps,
                                        bool write_s) {
  CHECK(r.is_cuda() && r.is_contiguous(), "r must be a contiguous CUDA tensor");
  on_device(r, "r");
  on_device(w, "w");
  if (a.has_value() && a->defined()) on_device(*a, "a");
  CHECK_DT(r, at::kFloat);
  CHECK_DT(w, at::kFloat);
  const int D = r.size(-1);
  const int64_t N = r.numel() / D;
  CHECK(w.numel() == D && w.is_contiguous(), "w must be contiguous with ", D, " elements");
  const bool has_a = a.has_value() && a->defined();
  if (has_a) {
    CHECK_DT((*a), at::kBFloat16);
    CHECK(a->is_contiguous() && a->numel() == r.numel(), "a must be contiguous and match r");
  }
  auto y = at::empty(r.sizes(), r.options().dtype(at::kBFloat16));
  auto rstd = at::empty({N}, r.options());
  at::Tensor s;
  if (write_s) s = at::empty_like(r);
  ok(llmt::add_rmsnorm_fwd(has_a ? a->data_ptr() : nullptr, r.data_ptr<float>(), w.data_ptr<float>(), y.data_ptr(),
                           write_s ? s.data_ptr<float>() : nullptr, rstd.data_ptr<float>(), N, D, (float)eps, stream()),
     "add_rmsnorm_fwd");
  return {y, s, rstd};
}

std::vector<at::Tensor> rmsnorm_bwd(at::Tensor dy, at::Tensor s, at::Tensor w, at::Tensor rstd,
                                    c10::optional<at::Tensor> ds_in, at::Tensor dw, at::Tensor ticket,
                                    bool write_ds16, bool accumulate) {
  CHECK_DT(dy, at::kBFloat16);
  CHECK_DT(s, at::kFloat);
  CHECK_DT(dw, at::kFloat);
  CHECK_DT(ticket, at::kInt);
  for (auto* t : {&dy, &s, &w, &rstd, &dw}) on_device(*t, "rmsnorm_bwd operand");
  if (ds_in.has_value() && ds_in->defined()) on_device(*ds_in, "ds_in");
  CHECK(dy.is_contiguous() && s.is_contiguous() && dy.numel() == s.numel(), "dy/s must be contiguous and match");
  const int D = s.size(-1);
  const int64_t N = s.numel() / D;
  CHECK(dw.numel() == D && dw.is_contiguous(), "dw must be contiguous with ", D, " elements");
  const bool has_dsin = ds_in.has_value() && ds_in->defined();
  if (has_dsin) {
    CHECK_DT((*ds_in), at::kFloat);
    CHECK(ds_in->is_contiguous() && ds_in->numel() == s.numel(), "ds_in must be contiguous and match s");
  }
  auto ds = at::empty_like(s);
  at::Tensor ds16;
  if (write_ds16) ds16 = at::empty(s.sizes(), s.options().dtype(at::kBFloat16));
  auto part = at::empty({llmt::rmsnorm_bwd_partials(N, D), D}, s.options());
  ok(llmt::rmsnorm_bwd(dy.data_ptr(), s.data_ptr<float>(), w.data_ptr<float>(), rstd.data_ptr<float>(),
                       has_dsin ? ds_in->data_ptr<float>() : nullptr, ds.data_ptr<float>(),
                       write_ds16 ? ds16.data_ptr() : nullptr, part.data_ptr<float>(), dw.data_ptr<float>(),
                       reinterpret_cast<unsigned*>(ticket.data_ptr<int>()), N, D, accumulate ? 1 : 0, stream()),
     "rmsnorm_bwd");
  return {ds, ds16};
}

// ---------------------------------------------------------------- elementwise
void swiglu_fwd(at::Tensor g, at::Tensor u, at::Tensor h) {
  cuda2d(g, "g");
  cuda2d(u, "u");
  cuda2d(h, "h");
  CHECK(g.stride(0) == u.stride(0), "g and u must share a row stride");
  CHECK_DT(g, at::kBFloat16);
  ok(llmt::swiglu_fwd(g.data_ptr(), u.data_ptr(), g.stride(0), h.data_ptr(), h.stride(0), g.size(0), g.size(1),
                      stream()),
     "swiglu_fwd");
}

void swiglu_bwd(at::Tensor dh, at::Tensor g, at::Tensor u, at::Tensor dg, at::Tensor du) {
  for (auto* t : {&dh, &g, &u, &dg, &du}) cuda2d(*t, "swiglu operand");
  CHECK(g.stride(0) == u.stride(0) && dg.stride(0) == du.stride(0), "paired row strides differ");
  ok(llmt::swiglu_bwd(dh.data_ptr(), dh.stride(0), g.data_ptr(), u.data_ptr(), g.stride(0), dg.data_ptr(),
                      du.data_ptr(), dg.stride(0), g.size(0), g.size(1), stream()),
     "swiglu_bwd");
}

void rope_inplace(at::Tensor qkv, at::Tensor cos_t, at::Tensor sin_t, int64_t T, int64_t n_rot_heads, int64_t hd,
                  bool backward) {
  CHECK_DT(qkv, at::kBFloat16);
  CHECK_DT(cos_t, at::kFloat);
  for (auto* t : {&qkv, &cos_t, &sin_t}) on_device(*t, "rope operand");
  CHECK(qkv.is_contiguous() && cos_t.is_contiguous() && sin_t.is_contiguous(), "rope operands must be contiguous");
  CHECK(cos_t.size(0) >= T && cos_t.size(1) == hd, "rope table too small");
  const int64_t ld = qkv.size(-1);
  ok(llmt::rope_inplace(qkv.data_ptr(), cos_t.data_ptr<float>(), sin_t.data_ptr<float>(), qkv.numel() / ld, (int)T,
                        (int)n_rot_heads, (int)hd, ld, backward, stream()),
     "rope_inplace");
}

void embedding_fwd(at::Tensor idx, at::Tensor W, at::Tensor x, c10::optional<at::Tensor> err, int64_t v0,
                   bool partial) {
  CHECK_DT(idx, at::kLong);
  CHECK_DT(W, at::kFloat);
  for (auto* t : {&idx, &W, &x}) on_device(*t, "embedding operand");
  CHECK(idx.is_contiguous() && W.is_contiguous() && x.is_contiguous(), "embedding operands must be contiguous");
  ok(llmt::embedding_fwd(idx.data_ptr<int64_t>(), W.data_ptr<float>(), x.data_ptr<float>(), idx.numel(), W.size(1),
                         W.size(0), v0, partial, err.has_value() && err->defined() ? err->data_ptr<int>() : nullptr,
                         stream()),
     "embedding_fwd");
}

void embedding_bwd(at::Tensor idx, at::Tensor dx, at::Tensor dW, int64_t v0) {
  CHECK_DT(dx, at::kFloat);
  CHECK_DT(dW, at::kFloat);
  for (auto* t : {&idx, &dx, &dW}) on_device(*t, "embedding operand");
  CHECK(idx.is_contiguous() && dx.is_contiguous() && dW.is_contiguous(), "embedding grads must be contiguous");
  ok(llmt::embedding_bwd(idx.data_ptr<int64_t>(), dx.data_ptr<float>(), dW.data_ptr<float>(), idx.numel(), dW.size(1),
                         dW.size(0), v0, stream()),
     "embedding_bwd");
}

// ---------------------------------------------------------------- rotary positions
llmt::RopeHeads rope_heads(const at::Tensor& x, const at::Tensor& y) {
  auto extent = [](const at::Tensor& t) {
    int64_t e = t.size(3);
    for (int i = 0; i < 3; ++i) e += t.stride(i) * (t.size(i) - 1);
    return t.numel() ? e : 0;
  };
  return {x.data_ptr(),  y.data_ptr(),  (int)x.size(2), x.stride(0), x.stride(1), x.stride(2),
          y.stride(0), y.stride(1), y.stride(2),    extent(x),   extent(y)};
}

// Rotates q and (when given) k, (B, T, heads, hd) with unit stride along hd, into q_out / k_out:
// new contiguous tensors, or given ones, which may be q and k themselves.
std::vector<at::Tensor> rotary(at::Tensor q, c10::optional<at::Tensor> k, c10::optional<at::Tensor> positions, at::Tensor table,
                               int64_t rotary_dim, bool interleaved, bool inverse, c10::optional<at::Tensor> q_out,
                               c10::optional<at::Tensor> k_out) {
  const bool has_k = k.has_value() && k->defined();
  CHECK(q.dim() == 4, "rotary: q must be (batch, tokens, heads, head_dim)");
  const int64_t B = q.size(0), T = q.size(1), hd = q.size(3);
  const int kind = float_kind(q, "q");
  CHECK(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= hd, "rotary: rotary_dim must be even and at most head_dim");
  CHECK(B <= 0x7fffffff && T <= 0x7fffffff && B * T <= 0x7fffffff, "rotary: more than 2^31 - 1 tokens");
  CHECK(table.scalar_type() == at::kFloat && table.is_contiguous() && table.dim() == 3 &&
            table.size(0) == llmt::kRopeTableRows && table.size(1) == rotary_dim / 2 && table.size(2) == 2,
        "rotary: table must be (", (int64_t)llmt::kRopeTableRows, ", rotary_dim / 2, 2) float32");
  auto shape = [&](const at::Tensor& x, const char* name) {
    CHECK(x.dim() == 4 && x.size(0) == B && x.size(1) == T && x.size(3) == hd, "rotary: ", name, " must be (", B, ", ", T, ", heads, ", hd, ")");
    CHECK(x.scalar_type() == q.scalar_type(), "rotary: q, k and their outputs must share a dtype");
    CHECK(hd == 1 || x.stride(3) == 1 || x.numel() == 0, "rotary: ", name, " must have unit stride along head_dim");
  };
  auto fresh_or = [&](const c10::optional<at::Tensor>& given, const at::Tensor& x, const char* name) {
    if (!(given.has_value() && given->defined())) return fresh({B, T, x.size(2), hd}, x.scalar_type());
    shape(*given, name);
    CHECK(given->size(2) == x.size(2), "rotary: ", name, " has other heads than its input");
    if (given->numel() > 0) {
      // strides that step over one another's extent, smallest first
      std::vector<std::pair<int64_t, int64_t>> d;
      for (int i = 0; i < 3; ++i)
        if (given->size(i) > 1) d.emplace_back(given->stride(i), given->size(i));
      std::sort(d.begin(), d.end());
      int64_t extent = hd;
      for (auto& s : d) {
        CHECK(s.first >= extent, "rotary: values of ", name, " overlap");
        extent += s.first * (s.second - 1);
      }
      auto end = [&](const at::Tensor& t) {
        int64_t e = hd;
        for (int i = 0; i < 3; ++i) e += t.stride(i) * (t.size(i) - 1);
        return (const char*)t.data_ptr() + e * t.element_size();
      };
      const bool same = given->data_ptr() == x.data_ptr() && given->strides() == x.strides();
      CHECK(same || (const char*)given->data_ptr() >= end(x) || end(*given) <= (const char*)x.data_ptr(),
            "rotary: ", name, " overlaps its input without being it");
    }
    return *given;
  };
  shape(q, "q");
  if (has_k) shape(*k, "k");
  CHECK(has_k || !k_out.has_value(), "rotary: k_out without k");
  for (auto* y : {&q_out, &k_out})
    if (y->has_value() && has_k && (*y)->numel() > 0 && k->numel() > 0 && q.numel() > 0) {
      const void* other = y == &q_out ? k->data_ptr() : q.data_ptr();
      CHECK((*y)->data_ptr() != other, "rotary: q_out is k, or k_out is q");
    }
  CHECK(!(q_out.has_value() && k_out.has_value() && q_out->numel() > 0 && q_out->data_ptr() == k_out->data_ptr()),
        "rotary: q_out and k_out are the same values");
  if (q_out.has_value() || k_out.has_value()) {
    const c10::optional<at::Tensor> given_q = q, given_table = table;
    apart(q_out, k, "rotary: ", "q_out", "k");
    apart(k_out, given_q, "rotary: ", "k_out", "q");
    apart(q_out, k_out, "rotary: ", "q_out", "k_out");
    for (auto* y : {&q_out, &k_out}) {
      const char* name = y == &q_out ? "q_out" : "k_out";
      apart(*y, positions, "rotary: ", name, "positions");
      apart(*y, given_table, "rotary: ", name, "the plan's table");
    }
  }
  llmt::RopeArgs a{};
  a.B = (int)B;
  a.T = (int)T;
  a.hd = (int)hd;
  a.rd = (int)rotary_dim;
  if (positions.has_value() && positions->defined()) {
    CHECK(positions->scalar_type() == at::kInt || positions->scalar_type() == at::kLong, "rotary: positions must be int32 or int64");
    CHECK(positions->dim() >= 1 && positions->dim() <= 2 && (positions->size(-1) == T || positions->size(-1) == 1) &&
              (positions->dim() == 1 || positions->size(0) == B || positions->size(0) == 1),
          "rotary: positions must be (", B, ", ", T, ") or broadcast to it");
    a.pos = positions->data_ptr();
    a.pos64 = positions->scalar_type() == at::kLong;
    a.pst = positions->size(-1) == 1 ? 0 : positions->stride(-1);
    a.psb = positions->dim() == 1 || positions->size(0) == 1 ? 0 : positions->stride(0);
    if (T > 1 && positions->size(-1) == 1) CHECK(false, "rotary: one position for ", T, " tokens");
  }
  all_on_device({{q, "q"}, {k, "k"}, {positions, "positions"}, {table, "table"}, {q_out, "q_out"}, {k_out, "k_out"}});
  at::Tensor qo = fresh_or(q_out, q, "q_out"), ko;
  a.q = rope_heads(q, qo);
  if (has_k) {
    ko = fresh_or(k_out, *k, "k_out");
    a.k = rope_heads(*k, ko);
  }
  a.table = table.data_ptr<float>();
  a.interleaved = interleaved;
  a.inverse = inverse;
  if (B * T > 0) ok(llmt::rotary(a, kind, stream()), "rotary");
  return {qo, ko};
}

// ---------------------------------------------------------------- optimizer
void adamw_step(at::Tensor p, at::Tensor g, at::Tensor m, at::Tensor v, c10::optional<at::Tensor> p16, at::Tensor lr,
                at::Tensor step, double b1, double b2, double eps, double wd, double grad_scale, bool zero_grad,
                int64_t max_blocks) {
  for (auto* t : {&p, &g, &m, &v, &lr, &step}) on_device(*t, "adamw operand");
  for (auto* t : {&p, &g, &m, &v}) {
    CHECK_DT((*t), at::kFloat);
    CHECK(t->is_contiguous() && t->numel() == p.numel(), "adamw buffers must be contiguous and equal-sized");
  }
  CHECK_DT(lr, at::kFloat);
  CHECK_DT(step, at::kInt);
  void* p16p = nullptr;
  if (p16.has_value() && p16->defined()) {
    CHECK_DT((*p16), at::kBFloat16);
    CHECK(p16->numel() == p.numel() && p16->is_contiguous(), "adamw: bf16 copy size mismatch");
    p16p = p16->data_ptr();
  }
  llmt::AdamHyper h{(float)b1, (float)b2, (float)eps, (float)wd, (float)grad_scale};
  ok(llmt::adamw_step(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr<float>(), v.data_ptr<float>(), p16p,
                      p.numel(), lr.data_ptr<float>(), step.data_ptr<int>(), h, zero_grad, stream(), (int)max_blocks),
     "adamw_step");
}

// The tensors of a MultiAdamW: their sizes and places in the states are fixed, their addresses are
// read at every step.
struct MultiPlan {
  std::vector<at::Tensor> p, p16;
  std::vector<double> wd;
  std::vector<int64_t> numel, first_block;
  int64_t blocks = 0;
  std::vector<uint32_t> order;    // of the parameters and (from p.size() on) their copies, by address when last looked at
  std::vector<uintptr_t> places;  // their addresses in this step, 0 for those left out

  size_t bytes(size_t i) const { return i < p.size() ? 4 * numel[i] : 2 * numel[i - p.size()]; }
  // Gradients that lie over a parameter or a copy would be read after its update, by another warp. A parameter
  // that is its own gradient is not: each value is read and written by one thread, unless it is cleared after.
  // Mostly the gradients lie elsewhere altogether.
  void check_apart(const std::vector<llmt::MultiTensor>& t, const std::vector<uint32_t>& index, size_t grad_bytes, bool cleared) {
    struct Span {
      uintptr_t first = UINTPTR_MAX, last = 0;
      void cover(uintptr_t at, size_t n) { first = std::min(first, at), last = std::max(last, at + n); }
      bool meets(const Span& x) const { return first < x.last && x.first < last; }
    };
    Span grads, masters, copies;
    for (const auto& x : t) grads.cover((uintptr_t)x.g, grad_bytes * x.n);
    for (size_t i = 0; i < places.size(); ++i) {
      if (!places[i]) places[i] = (uintptr_t)(i < p.size() ? p[i] : p16[i - p.size()]).data_ptr();
      (i < p.size() ? masters : copies).cover(places[i], bytes(i));
    }
    if (!grads.meets(masters) && !grads.meets(copies)) return;
    auto ascending = [this](uint32_t a, uint32_t b) { return places[a] < places[b]; };
    if (!std::is_sorted(order.begin(), order.end(), ascending)) std::sort(order.begin(), order.end(), ascending);
    std::vector<uintptr_t> ends(order.size());
    for (size_t i = 0; i < order.size(); ++i) ends[i] = places[order[i]] + bytes(order[i]);
    for (size_t i = 0; i < t.size(); ++i) {
      const uintptr_t first = (uintptr_t)t[i].g, last = first + grad_bytes * t[i].n;
      // the first tensor that ends behind the gradient's beginning (without branches: 12 -> 6 us of host time for 336 gradients)
      const uintptr_t* at = ends.data();
      for (size_t n = ends.size(); n > 0;) {
        const size_t half = (n + 1) / 2;
        at += at[half - 1] <= first ? half : 0;
        n -= half;
      }
      const size_t k = at - ends.data();
      if (k == ends.size() || places[order[k]] >= last) continue;
      const bool own = !cleared && first == (uintptr_t)t[i].p && last == ends[k];
      CHECK(own, "adamw: gradient ", index[i], " overlaps a parameter or its bf16 copy");
    }
  }

  MultiPlan(std::vector<at::Tensor> p_, std::vector<at::Tensor> p16_, std::vector<double> wd_)
      : p(std::move(p_)), p16(std::move(p16_)), wd(std::move(wd_)) {
    CHECK(!p.empty(), "adamw: no tensors");
    CHECK(p16.empty() || p16.size() == p.size(), "adamw: one bf16 copy per tensor, or none");
    CHECK(wd.size() == p.size(), "adamw: one weight decay per tensor");
    std::vector<std::pair<const char*, const char*>> spans;
    for (size_t i = 0; i < p.size(); ++i) {
      CHECK(p[i].scalar_type() == at::kFloat, "adamw: parameter ", i, " has dtype ", p[i].scalar_type(), ", expected Float");
      CHECK(p[i].is_contiguous(), "adamw: parameter ", i, " must be contiguous");
      CHECK(p[i].numel() > 0, "adamw: parameter ", i, " is empty");
      if (!p16.empty()) {
        CHECK(p16[i].scalar_type() == at::kBFloat16 && p16[i].is_contiguous() && p16[i].numel() == p[i].numel(),
              "adamw: bf16 copy ", i, " must be contiguous bf16 of its parameter's size");
        spans.emplace_back((const char*)p16[i].data_ptr(), (const char*)p16[i].data_ptr() + 2 * p16[i].numel());
      }
      spans.emplace_back((const char*)p[i].data_ptr(), (const char*)p[i].data_ptr() + 4 * p[i].numel());
      numel.push_back(p[i].numel());
      first_block.push_back(blocks);
      blocks += (p[i].numel() + 255) / 256;
    }
    CHECK(blocks < 0x7fffffff, "adamw: more than 2^31 - 1 blocks of 256 values");
    order.resize(p.size() + p16.size());
    std::iota(order.begin(), order.end(), 0u);
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i) CHECK(spans[i].first >= spans[i - 1].second, "adamw: two tensors share memory");
  }

  // grads: one per tensor, None leaves that tensor and its states as they are. Returns the kernels launched.
  int64_t step(const pybind11::list& grads, int64_t bits, at::Tensor m, at::Tensor v, c10::optional<at::Tensor> ms,
               c10::optional<at::Tensor> vs, at::Tensor lr, at::Tensor step, at::Tensor ticket, double b1, double b2, double eps,
               double grad_scale, c10::optional<at::Tensor> grad_scale_dev, int64_t seed, bool zero_grad) {
    CHECK(grads.size() == p.size(), "adamw: ", grads.size(), " gradients for ", p.size(), " tensors");
    CHECK(bits == 8 || bits == 32, "adamw: states have 8 or 32 bits");
    std::vector<llmt::MultiTensor> t;
    std::vector<uint32_t> index;
    t.reserve(p.size());
    index.reserve(p.size());
    places.assign(order.size(), 0);
    bool any = false, bf16 = false;
    int64_t elsewhere = -1;
    const int dev = m.get_device();
    for (size_t i = 0; i < p.size(); ++i) {
      pybind11::handle h = grads[i];
      if (h.is_none()) continue;
      CHECK(THPVariable_Check(h.ptr()), "adamw: gradient ", i, " is not a tensor");
      const at::Tensor& g = THPVariable_Unpack(h.ptr());
      const bool half = g.scalar_type() == at::kBFloat16;
      CHECK(half || g.scalar_type() == at::kFloat, "adamw: gradient ", i, " has dtype ", g.scalar_type(), ", expected Float or BFloat16");
      CHECK(!any || half == bf16, "adamw: gradients of two dtypes in one step");
      any = true;
      bf16 = half;
      CHECK(g.numel() == numel[i] && g.is_contiguous(), "adamw: gradient ", i, " must be contiguous with ", numel[i], " values");
      CHECK(p[i].numel() == numel[i] && p[i].is_contiguous() && p[i].scalar_type() == at::kFloat, "adamw: parameter ", i, " changed its size, layout or type");
      if (!(g.is_cuda() && p[i].is_cuda() && g.get_device() == dev && p[i].get_device() == dev)) elsewhere = (int64_t)i;
      if (!p16.empty()) {
        CHECK(p16[i].numel() == numel[i] && p16[i].is_contiguous() && p16[i].scalar_type() == at::kBFloat16, "adamw: bf16 copy ", i, " changed");
        if (!(p16[i].is_cuda() && p16[i].get_device() == dev)) elsewhere = (int64_t)i;
      }
      t.push_back({static_cast<float*>(p[i].data_ptr()), g.data_ptr(), p16.empty() ? nullptr : p16[i].data_ptr(), numel[i],
                   (int32_t)first_block[i], 0, (float)wd[i], false});
      CHECK(t.back().p && t.back().g && (p16.empty() || t.back().p16), "adamw: tensor ", i, " has no memory (its parameter, gradient or bf16 copy was freed)");
      index.push_back((uint32_t)i);
      places[i] = (uintptr_t)t.back().p;
      if (!p16.empty()) places[p.size() + i] = (uintptr_t)t.back().p16;
    }
    if (zero_grad) {  // cleared by one tensor's blocks while another's read it
      std::vector<std::pair<const char*, const char*>> spans;
      spans.reserve(t.size());
      for (const auto& x : t) {
        const char* g = static_cast<const char*>(x.g);
        spans.emplace_back(g, g + (bf16 ? 2 : 4) * x.n);
      }
      std::sort(spans.begin(), spans.end());
      for (size_t i = 1; i < spans.size(); ++i)
        CHECK(spans[i].first >= spans[i - 1].second, "adamw: zero_grad with one gradient for two tensors");
    }
    check_apart(t, index, bf16 ? 2 : 4, zero_grad);
    const int64_t n = 256 * blocks;
    const at::ScalarType dt_m = bits == 8 ? at::kFloat8_e4m3fn : at::kFloat, dt_v = bits == 8 ? at::kByte : at::kFloat;
    CHECK(m.scalar_type() == dt_m && v.scalar_type() == dt_v && m.numel() == n && v.numel() == n && m.is_contiguous() &&
              v.is_contiguous(),
          "adamw: states of another type or size");
    if (bits == 8)
      for (auto* x : {&ms, &vs})
        CHECK(x->has_value() && (*x)->scalar_type() == at::kByte && (*x)->numel() == blocks && (*x)->is_contiguous(),
              "adamw: one scale byte per block of 256 values");
    CHECK(lr.scalar_type() == at::kFloat && step.scalar_type() == at::kInt && ticket.scalar_type() == at::kInt,
          "adamw: lr must be float32, the step count and the ticket int32");
    if (grad_scale_dev.has_value())
      CHECK(grad_scale_dev->scalar_type() == at::kFloat && grad_scale_dev->numel() == 1, "adamw: grad_scale must be one float32 value");
    for (auto* x : {&m, &v, &lr, &step, &ticket}) on_device(*x, "adamw state");
    CHECK(elsewhere < 0, "adamw: tensor ", elsewhere, " is not on the states' device");
    if (t.empty()) {
      step.add_(1);
      return 0;
    }
    llmt::MultiHyper h{(float)b1, (float)(1.0 - b1), (float)b2, (float)(1.0 - b2), (float)eps, (float)grad_scale,
                       std::log(b1), std::log(b2), lr.data_ptr<float>(),
                       static_cast<const float*>(opt_ptr(grad_scale_dev, "grad_scale")),
                       step.data_ptr<int>(), reinterpret_cast<unsigned*>(ticket.data_ptr<int>()), (uint32_t)seed, zero_grad};
    llmt::MultiState s{m.data_ptr(), v.data_ptr(), static_cast<uint8_t*>(const_cast<void*>(opt_ptr(ms, "scale"))),
                       static_cast<uint8_t*>(const_cast<void*>(opt_ptr(vs, "scale"))), n};
    ok(llmt::adamw_multi(t.data(), (int)t.size(), bf16, (int)bits, h, s, stream()), "adamw_multi");
    return ((int64_t)t.size() + llmt::kTensorsPerLaunch - 1) / llmt::kTensorsPerLaunch;
  }
};

void check_codes(const at::Tensor& m, const at::Tensor& ms, const at::Tensor& v, const at::Tensor& vs) {
  for (auto* t : {&m, &ms, &v, &vs}) {
    CHECK(t->element_size() == 1 && t->is_contiguous(), "adamw: codes and scales are contiguous bytes");
    on_device(*t, "adamw state");
  }
  CHECK(m.numel() == v.numel() && m.numel() == 256 * ms.numel() && ms.numel() == vs.numel(),
        "adamw: one scale byte per block of 256 codes");
}

// (m, v) that the codes stand for, bf16 (exact) or fp32.
std::vector<at::Tensor> adamw_state_values(at::Tensor m, at::Tensor ms, at::Tensor v, at::Tensor vs, bool f32) {
  check_codes(m, ms, v, vs);
  auto o = m.options().dtype(f32 ? at::kFloat : at::kBFloat16);
  auto mo = at::empty(m.sizes(), o), vo = at::empty(v.sizes(), o);
  ok(llmt::adamw_state_values(static_cast<const uint8_t*>(m.data_ptr()), static_cast<const uint8_t*>(ms.data_ptr()),
                              static_cast<const uint8_t*>(v.data_ptr()), static_cast<const uint8_t*>(vs.data_ptr()),
                              mo.data_ptr(), vo.data_ptr(), f32, m.numel(), stream()),
     "adamw_state_values");
  return {mo, vo};
}

void adamw_encode_states(at::Tensor m32, at::Tensor v32, at::Tensor m, at::Tensor ms, at::Tensor v, at::Tensor vs) {
  check_codes(m, ms, v, vs);
  for (auto* t : {&m32, &v32}) {
    CHECK_DT((*t), at::kFloat);
    CHECK(t->is_contiguous() && t->numel() == m.numel(), "adamw: fp32 states must be contiguous and match the codes");
    on_device(*t, "adamw state");
  }
  ok(llmt::adamw_encode_states(m32.data_ptr<float>(), v32.data_ptr<float>(), static_cast<uint8_t*>(m.data_ptr()),
                               static_cast<uint8_t*>(ms.data_ptr()), static_cast<uint8_t*>(v.data_ptr()),
                               static_cast<uint8_t*>(vs.data_ptr()), ms.numel(), stream()),
     "adamw_encode_states");
}

void cast_bf16(at::Tensor x, at::Tensor y, int64_t max_blocks) {
  CHECK_DT(x, at::kFloat);
  CHECK_DT(y, at::kBFloat16);
  on_device(x, "x");
  on_device(y, "y");
  CHECK(x.numel() == y.numel() && x.is_contiguous() && y.is_contiguous(), "cast_bf16: bad args");
  ok(llmt::cast_bf16(x.data_ptr<float>(), y.data_ptr(), x.numel(), stream(), (int)max_blocks), "cast_bf16");
}

// ---------------------------------------------------------------- cross entropy
void ce_fwd_rows(at::Tensor logits, at::Tensor targets, at::Tensor lse, at::Tensor loss) {
  cuda2d(logits, "logits");
  CHECK_DT(logits, at::kBFloat16);
  CHECK_DT(targets, at::kLong);
  ok(llmt::ce_fwd_rows(logits.data_ptr(), logits.stride(0), targets.data_ptr<int64_t>(), lse.data_ptr<float>(),
                       loss.data_ptr<float>(), logits.size(0), logits.size(1), stream()),
     "ce_fwd_rows");
}

void ce_bwd_rows(at::Tensor logits, at::Tensor targets, at::Tensor lse, c10::optional<at::Tensor> grad_out,
                 double scale) {
  cuda2d(logits, "logits");
  CHECK_DT(logits, at::kBFloat16);
  ok(llmt::ce_bwd_rows(logits.data_ptr(), logits.stride(0), targets.data_ptr<int64_t>(), lse.data_ptr<float>(),
                       static_cast<const float*>(opt_ptr(grad_out, "grad_out")), (float)scale, logits.size(0), logits.size(1),
                       stream()),
     "ce_bwd_rows");
}

void ce_combine(at::Tensor part, at::Tensor tlogit, at::Tensor tgt, at::Tensor lse, at::Tensor loss, int64_t nblk,
                int64_t V) {
  for (auto* t : {&part, &tlogit, &tgt, &lse, &loss}) on_device(*t, "ce_combine operand");
  ok(llmt::ce_combine(part.data_ptr<float>(), tlogit.data_ptr<float>(), tgt.data_ptr<int64_t>(), lse.data_ptr<float>(),
                      loss.data_ptr<float>(), (int)lse.numel(), (int)nblk, (int)V, stream()),
     "ce_combine");
}

// ---------------------------------------------------------------- post-training losses
int float_kind(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return 0;
    case at::kHalf: return 1;
    case at::kFloat: return 2;
    default: CHECK(false, name, " has dtype ", t.scalar_type(), ", expected bfloat16, float16 or float32");
  }
  return -1;
}

// A (B, T) operand, broadcast where it has fewer or unit dimensions; empty when not given.
template <typename E>
llmt::Strided<E> strided_bt(const c10::optional<at::Tensor>& t, at::ScalarType dt, int64_t B, int64_t T, const char* name) {
  if (!(t.has_value() && t->defined())) return {nullptr, 0, 0};
  CHECK(t->scalar_type() == dt, name, " has dtype ", t->scalar_type(), ", expected ", dt);
  CHECK(t->dim() <= 2, name, " must be (batch, tokens) or broadcast to it");
  int64_t sb = 0, st = 0;
  if (t->dim() >= 1) {
    const int64_t n = t->size(-1);
    CHECK(n == T || n == 1, name, " has ", n, " tokens, the logits ", T);
    st = n == 1 ? 0 : t->stride(-1);
  }
  if (t->dim() == 2) {
    CHECK(t->size(0) == B || t->size(0) == 1, name, " has ", t->size(0), " sequences, the logits ", B);
    sb = t->size(0) == 1 ? 0 : t->stride(0);
  }
  return {static_cast<const E*>(t->data_ptr()), sb, st};
}

// Shapes and types are checked first, so that they are told apart from a tensor of another device.
void all_on_device(std::initializer_list<std::pair<const c10::optional<at::Tensor>, const char*>> given) {
  for (const auto& g : given)
    if (g.first.has_value() && g.first->defined()) on_device(*g.first, g.second);
}

void no_grad_wanted(const c10::optional<at::Tensor>& t, const char* name) {
  CHECK(!(t.has_value() && t->defined() && t->requires_grad()), name, " requires a gradient, which this loss does not give: detach it");
}

llmt::TokenBatch token_batch(const at::Tensor& targets, const c10::optional<at::Tensor>& mask, int64_t B, int64_t T, int64_t V) {
  CHECK(B > 0 && T > 0, "empty batch (", B, " sequences of ", T, " tokens)");
  CHECK(V > 0 && V < (int64_t(1) << 30), "a vocabulary of ", V, " ids");
  CHECK(B * T <= 0x7fffffff, "more than 2^31 - 1 tokens");
  CHECK(targets.dim() == 2 && targets.size(0) == B && targets.size(1) == T, "targets must be (", B, ", ", T, ")");
  llmt::TokenBatch a{};
  a.B = (int)B;
  a.T = (int)T;
  a.V = (int)V;
  a.tgt = strided_bt<int64_t>(targets, at::kLong, B, T, "targets");
  a.mask = strided_bt<uint8_t>(mask, at::kBool, B, T, "mask");
  return a;
}

llmt::TokenBatch logit_batch(const at::Tensor& logits, const at::Tensor& targets, const c10::optional<at::Tensor>& mask) {
  CHECK(logits.dim() == 3, "logits must be (batch, tokens, vocabulary)");
  llmt::TokenBatch a = token_batch(targets, mask, logits.size(0), logits.size(1), logits.size(2));
  CHECK(logits.stride(2) == 1 || logits.size(2) == 1, "logits must have unit stride along the vocabulary");
  a.dtype = float_kind(logits, "logits");
  a.z = logits.data_ptr();
  a.zsb = logits.stride(0);
  a.zst = logits.stride(1);
  a.zn = (logits.size(0) - 1) * a.zsb + (logits.size(1) - 1) * a.zst + a.V;
  return a;
}

// The rows written to: `out`, or a new contiguous tensor. Rows of `out` may not overlap one
// another; `out` may be the logits themselves, but not other rows of theirs.
at::Tensor gradient_rows(const at::Tensor& logits, const c10::optional<at::Tensor>& out, llmt::RowOut& o) {
  at::Tensor d;
  if (out.has_value() && out->defined()) {
    d = *out;
    CHECK(d.scalar_type() == logits.scalar_type() && d.sizes() == logits.sizes(), "out must match the logits");
    const int64_t B = d.size(0), T = d.size(1), V = d.size(2), sb = d.stride(0), st = d.stride(1);
    CHECK(d.stride(2) == 1 || V == 1, "out must have unit stride along the vocabulary");
    const bool rows_in = T == 1 || (st >= V && (B == 1 || sb >= (T - 1) * st + V));
    const bool rows_out = B == 1 || (sb >= V && (T == 1 || st >= (B - 1) * sb + V));
    CHECK(rows_in || rows_out, "rows of out overlap");
    const bool same = d.data_ptr() == logits.data_ptr() && d.strides() == logits.strides();
    const int64_t e = d.element_size();
    auto last = [&](const at::Tensor& t) {
      return (const char*)t.data_ptr() + e * ((B - 1) * t.stride(0) + (T - 1) * t.stride(1) + V);
    };
    CHECK(same || (const char*)d.data_ptr() >= last(logits) || last(d) <= (const char*)logits.data_ptr(),
          "out overlaps the logits without being the same rows");
  } else {
    d = fresh(logits.sizes(), logits.scalar_type());
  }
  o.dz = d.data_ptr();
  o.sb = d.stride(0);
  o.st = d.stride(1);
  o.dn = (d.size(0) - 1) * o.sb + (d.size(1) - 1) * o.st + d.size(2);
  return d;
}

const float* grad_scalar(const c10::optional<at::Tensor>& g) {
  if (!(g.has_value() && g->defined())) return nullptr;
  CHECK(g->scalar_type() == at::kFloat && g->numel() == 1, "grad_out must be one float32 value");
  return g->data_ptr<float>();
}

// (logp (B, T), stats (B, T, 2)) of rows of logits.
std::vector<at::Tensor> logprob_rows(at::Tensor logits, at::Tensor targets, c10::optional<at::Tensor> mask) {
  llmt::TokenBatch a = logit_batch(logits, targets, mask);
  all_on_device({{logits, "logits"}, {targets, "targets"}, {mask, "mask"}});
  auto logp = fresh({a.B, a.T}, at::kFloat), stats = fresh({a.B, a.T, 2}, at::kFloat);
  llmt::RowOut o{};
  o.logp = logp.data_ptr<float>();
  o.stats = reinterpret_cast<float2*>(stats.data_ptr<float>());
  ok(llmt::logprob_rows(a, o, stream()), "logprob_rows");
  return {logp, stats};
}

llmt::PolicyArgs policy_args(const c10::optional<at::Tensor>& old, const at::Tensor& adv, const c10::optional<at::Tensor>& ref,
                             int64_t B, int64_t T, double clip_lo, double clip_hi, double kl, int64_t reduction) {
  no_grad_wanted(old, "old_logp");
  no_grad_wanted(adv, "advantages");
  no_grad_wanted(ref, "ref_logp");
  CHECK(clip_lo >= 0 && clip_lo <= 1 && clip_hi >= 0, "clip must be (low in [0, 1], high >= 0)");
  CHECK(reduction >= 0 && reduction <= 2, "unknown reduction");
  CHECK(kl == 0 || (ref.has_value() && ref->defined()), "kl_coef without ref_logp");
  llmt::PolicyArgs q{};
  q.old = strided_bt<float>(old, at::kFloat, B, T, "old_logp");
  q.adv = strided_bt<float>(adv, at::kFloat, B, T, "advantages");
  q.ref = strided_bt<float>(ref, at::kFloat, B, T, "ref_logp");
  q.clip_lo = (float)clip_lo;
  q.clip_hi = (float)clip_hi;
  q.kl_coef = (float)kl;
  q.reduction = (int)reduction;
  return q;
}

// (loss, logp, dlogits, coef, stats): dlogits undefined unless `grad`, the last two unless `keep`.
std::vector<at::Tensor> policy_rows(at::Tensor logits, at::Tensor targets, c10::optional<at::Tensor> old, at::Tensor adv,
                                    c10::optional<at::Tensor> ref, c10::optional<at::Tensor> mask, double clip_lo,
                                    double clip_hi, double kl, int64_t reduction, bool grad, c10::optional<at::Tensor> out,
                                    bool keep) {
  llmt::TokenBatch a = logit_batch(logits, targets, mask);
  const llmt::PolicyArgs q = policy_args(old, adv, ref, a.B, a.T, clip_lo, clip_hi, kl, reduction);
  CHECK(grad || !out.has_value(), "out without grad");
  llmt::RowOut o{};
  at::Tensor d, coef, stats;
  if (grad && out.has_value()) d = gradient_rows(logits, out, o);
  if (out.has_value()) {
    const c10::optional<at::Tensor> ids = targets, advantages = adv;
    for (const auto& x : {std::make_pair(&ids, "targets"), {&mask, "mask"}, {&old, "old_logp"}, {&advantages, "advantages"}, {&ref, "ref_logp"}})
      apart(out, *x.first, "", "out", x.second);
  }
  all_on_device({{logits, "logits"}, {targets, "targets"}, {mask, "mask"}, {old, "old_logp"}, {adv, "advantages"},
                 {ref, "ref_logp"}, {out, "out"}});
  if (grad && !d.defined()) d = gradient_rows(logits, out, o);
  const int64_t n = (int64_t)a.B * a.T;
  auto loss = fresh({}, at::kFloat), logp = fresh({a.B, a.T}, at::kFloat);
  // one scratch buffer: the rows' losses, the counts and the ticket, and the slopes where nobody keeps them
  auto scratch = fresh({n + a.B + 1 + (keep ? 0 : n)}, at::kFloat);
  o.logp = logp.data_ptr<float>();
  o.loss = loss.data_ptr<float>();
  o.loss_rows = scratch.data_ptr<float>();
  o.count = reinterpret_cast<int*>(o.loss_rows + n);
  o.ticket = reinterpret_cast<unsigned*>(o.count + a.B);
  o.coef = o.loss_rows + n + a.B + 1;
  if (keep) {
    coef = fresh({a.B, a.T}, at::kFloat);
    stats = fresh({a.B, a.T, 2}, at::kFloat);
    o.coef = coef.data_ptr<float>();
    o.stats = reinterpret_cast<float2*>(stats.data_ptr<float>());
  }
  ok(llmt::policy_rows(a, q, o, stream()), "policy_rows");
  return {loss, logp, d, coef, stats};
}

// (loss, coef) of log-probabilities.
std::vector<at::Tensor> policy_tokens(at::Tensor logp, at::Tensor targets, int64_t V, c10::optional<at::Tensor> old,
                                      at::Tensor adv, c10::optional<at::Tensor> ref, c10::optional<at::Tensor> mask,
                                      double clip_lo, double clip_hi, double kl, int64_t reduction) {
  CHECK_DT(logp, at::kFloat);
  CHECK(logp.dim() == 2 && logp.is_contiguous(), "logp must be a contiguous (batch, tokens) tensor");
  llmt::TokenBatch a = token_batch(targets, mask, logp.size(0), logp.size(1), V);
  const llmt::PolicyArgs q = policy_args(old, adv, ref, a.B, a.T, clip_lo, clip_hi, kl, reduction);
  all_on_device({{logp, "logp"}, {targets, "targets"}, {mask, "mask"}, {old, "old_logp"}, {adv, "advantages"},
                 {ref, "ref_logp"}});
  auto loss = fresh({}, at::kFloat), coef = fresh({a.B, a.T}, at::kFloat), rows = fresh({(int64_t)a.B * a.T}, at::kFloat),
       words = fresh({a.B + 1}, at::kInt);
  llmt::RowOut o{};
  o.loss = loss.data_ptr<float>();
  o.loss_rows = rows.data_ptr<float>();
  o.coef = coef.data_ptr<float>();
  o.count = words.data_ptr<int>();
  o.ticket = reinterpret_cast<unsigned*>(o.count + a.B);
  ok(llmt::policy_tokens(a, q, logp.data_ptr<float>(), o, stream()), "policy_tokens");
  return {loss, coef};
}

llmt::PreferenceArgs preference_args(const c10::optional<at::Tensor>& ref, int64_t B, int64_t T, double beta,
                                     double smoothing, int64_t kind, bool average) {
  no_grad_wanted(ref, "ref_logp");
  CHECK(B % 2 == 0, "the batch holds the chosen sequences, then as many rejected ones: got ", B);
  CHECK(beta > 0, "beta must be positive");
  CHECK(smoothing >= 0 && smoothing < 0.5, "label_smoothing must be in [0, 0.5)");
  CHECK(kind >= 0 && kind <= 2, "unknown preference loss");
  CHECK(smoothing == 0 || kind == llmt::PREF_SIGMOID, "label_smoothing goes with the sigmoid loss");
  llmt::PreferenceArgs q{};
  q.ref = strided_bt<float>(ref, at::kFloat, B, T, "ref_logp");
  q.beta = (float)beta;
  q.smoothing = (float)smoothing;
  q.kind = (int)kind;
  q.average = average;
  return q;
}

// (loss, logp, rewards, dlogits, coef, stats): dlogits undefined unless `grad`, the last two unless `keep`.
std::vector<at::Tensor> preference_rows(at::Tensor logits, at::Tensor targets, c10::optional<at::Tensor> ref,
                                        c10::optional<at::Tensor> mask, double beta, double smoothing, int64_t kind,
                                        bool average, bool grad, c10::optional<at::Tensor> out, bool keep) {
  llmt::TokenBatch a = logit_batch(logits, targets, mask);
  const llmt::PreferenceArgs q = preference_args(ref, a.B, a.T, beta, smoothing, kind, average);
  CHECK(grad || !out.has_value(), "out without grad");
  llmt::RowOut o{};
  at::Tensor d, coef, stats;
  if (grad && out.has_value()) d = gradient_rows(logits, out, o);
  if (out.has_value()) {
    const c10::optional<at::Tensor> ids = targets;
    for (const auto& x : {std::make_pair(&ids, "targets"), {&mask, "mask"}, {&ref, "ref_logp"}}) apart(out, *x.first, "", "out", x.second);
  }
  all_on_device({{logits, "logits"}, {targets, "targets"}, {mask, "mask"}, {ref, "ref_logp"}, {out, "out"}});
  if (grad && !d.defined()) d = gradient_rows(logits, out, o);
  const int64_t n = (int64_t)a.B * a.T;
  auto loss = fresh({}, at::kFloat), logp = fresh({a.B, a.T}, at::kFloat), rewards = fresh({a.B}, at::kFloat);
  auto scratch = fresh({(keep ? 0 : 3 * n) + a.B / 2 + 1}, at::kFloat);  // stats, slopes, the pairs' losses, the ticket
  float* p = scratch.data_ptr<float>();
  if (keep) {
    coef = fresh({a.B, a.T}, at::kFloat);
    stats = fresh({a.B, a.T, 2}, at::kFloat);
    o.coef = coef.data_ptr<float>();
    o.stats = reinterpret_cast<float2*>(stats.data_ptr<float>());
  } else {
    o.stats = reinterpret_cast<float2*>(p);
    o.coef = p + 2 * n;
    p += 3 * n;
  }
  o.logp = logp.data_ptr<float>();
  o.loss = loss.data_ptr<float>();
  o.rewards = rewards.data_ptr<float>();
  o.loss_rows = p;
  o.ticket = reinterpret_cast<unsigned*>(p + a.B / 2);
  llmt::RowOut first = o;
  first.dz = nullptr;
  ok(llmt::logprob_rows(a, first, stream()), "preference_rows");
  ok(llmt::preference_tokens(a, q, o.logp, o, true, stream()), "preference_rows");
  if (grad) ok(llmt::grad_rows(a, o, false, true, stream()), "preference_rows");
  return {loss, logp, rewards, d, coef, stats};
}

// (loss, coef, rewards) of log-probabilities.
std::vector<at::Tensor> preference_tokens(at::Tensor logp, at::Tensor targets, int64_t V, c10::optional<at::Tensor> ref,
                                          c10::optional<at::Tensor> mask, double beta, double smoothing, int64_t kind,
                                          bool average) {
  CHECK_DT(logp, at::kFloat);
  CHECK(logp.dim() == 2 && logp.is_contiguous(), "logp must be a contiguous (batch, tokens) tensor");
  llmt::TokenBatch a = token_batch(targets, mask, logp.size(0), logp.size(1), V);
  const llmt::PreferenceArgs q = preference_args(ref, a.B, a.T, beta, smoothing, kind, average);
  all_on_device({{logp, "logp"}, {targets, "targets"}, {mask, "mask"}, {ref, "ref_logp"}});
  auto loss = fresh({}, at::kFloat), coef = fresh({a.B, a.T}, at::kFloat), rewards = fresh({a.B}, at::kFloat),
       scratch = fresh({a.B / 2 + 1}, at::kFloat);
  llmt::RowOut o{};
  o.loss = loss.data_ptr<float>();
  o.loss_rows = scratch.data_ptr<float>();
  o.coef = coef.data_ptr<float>();
  o.rewards = rewards.data_ptr<float>();
  o.ticket = reinterpret_cast<unsigned*>(o.loss_rows + a.B / 2);
  ok(llmt::preference_tokens(a, q, logp.data_ptr<float>(), o, false, stream()), "preference_tokens");
  return {loss, coef, rewards};
}

// Gradient rows coef (onehot - softmax) * grad_out from saved stats; with skip_one `out` holds
// them already where grad_out is 1.
at::Tensor grad_rows(at::Tensor logits, at::Tensor targets, c10::optional<at::Tensor> mask, at::Tensor coef,
                     at::Tensor stats, c10::optional<at::Tensor> grad_out, c10::optional<at::Tensor> out, bool skip_one) {
  llmt::TokenBatch a = logit_batch(logits, targets, mask);
  const int64_t n = (int64_t)a.B * a.T;
  for (auto* t : {&coef, &stats}) {
    CHECK_DT((*t), at::kFloat);
    CHECK(t->is_contiguous() && t->numel() == (t == &coef ? n : 2 * n), "grad_rows: coef (batch, tokens), stats (batch, tokens, 2)");
  }
  const float* g = grad_scalar(grad_out);
  llmt::RowOut o{};
  all_on_device({{logits, "logits"}, {targets, "targets"}, {mask, "mask"}, {coef, "coef"}, {stats, "stats"},
                 {grad_out, "grad_out"}, {out, "out"}});
  at::Tensor d = gradient_rows(logits, out, o);
  o.coef = coef.data_ptr<float>();
  o.stats = reinterpret_cast<float2*>(stats.data_ptr<float>());
  o.grad_out = g;
  ok(llmt::grad_rows(a, o, skip_one, false, stream()), "grad_rows");
  return d;
}

// ---------------------------------------------------------------- fp8 quantization
void fp8_quant(at::Tensor x, at::Tensor q, c10::optional<at::Tensor> qt, at::Tensor inv, at::Tensor scratch) {
  cuda2d(x, "x");
  CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat, "fp8_quant: x must be bf16 or fp32");
  CHECK(x.stride(1) == 1, "fp8_quant: x rows must be contiguous");
  const int64_t rows = x.size(0), cols = x.size(1);
  on_device(q, "q");
  CHECK_DT(q, at::kFloat8_e4m3fn);
  CHECK(q.is_contiguous() && q.numel() == rows * cols, "fp8_quant: q must be a contiguous rows x cols tensor");
  void* qtp = nullptr;
  if (qt.has_value() && qt->defined()) {
    on_device(*qt, "qt");
    CHECK_DT((*qt), at::kFloat8_e4m3fn);
    CHECK(qt->is_contiguous() && qt->numel() == rows * cols, "fp8_quant: qt must be a contiguous cols x rows tensor");
    qtp = qt->data_ptr();
  }
  for (auto* t : {&inv, &scratch}) {
    on_device(*t, "fp8_quant scale buffer");
    CHECK_DT((*t), at::kFloat);
  }
  CHECK(scratch.numel() >= llmt::fp8_amax_slots(), "fp8_quant: scratch needs fp8_amax_slots() floats");
  ok(llmt::fp8_quant(x.data_ptr(), x.scalar_type() == at::kFloat, (int)rows, (int)cols, x.stride(0), q.data_ptr(), qtp,
                     inv.data_ptr<float>(), scratch.data_ptr<float>(), stream()),
     "fp8_quant");
}

void mx_quant(int64_t kind, at::Tensor x, c10::optional<at::Tensor> q, c10::optional<at::Tensor> sf,
              c10::optional<at::Tensor> qt, c10::optional<at::Tensor> sft, c10::optional<at::Tensor> g,
              c10::optional<at::Tensor> scratch, bool interleave64, bool stochastic, int64_t seed,
              c10::optional<at::Tensor> seed_dev) {
  cuda2d(x, "x");
  CHECK(x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kFloat, "mx_quant: x must be bf16 or fp32");
  const int64_t rows = x.size(0), cols = x.size(1);
  const int64_t per = kind == 3 ? 2 : 1;
  auto bytes = [&](c10::optional<at::Tensor>& t, int64_t n, const char* name) -> void* {
    if (!t.has_value() || !t->defined()) return nullptr;
    on_device(*t, name);
    CHECK(t->element_size() == 1 && t->is_contiguous() && t->numel() >= n, name, ": contiguous bytes, at least ", n);
    return t->data_ptr();
  };
  void* qp = bytes(q, rows * cols / per, "q");
  void* qtp = bytes(qt, rows * cols / per, "qt");
  void* sfp = bytes(sf, qp ? llmt::mx_sf_bytes((int)kind, rows, cols) : 0, "sf");
  void* sftp = bytes(sft, qtp ? llmt::mx_sf_bytes((int)kind, cols, rows) : 0, "sft");
  float* gp = nullptr;
  float* sp = nullptr;
  if (kind == 3) {
    CHECK(g.has_value() && scratch.has_value(), "mx_quant: NVFP4 needs g and scratch");
    for (auto* t : {&*g, &*scratch}) {
      on_device(*t, "mx_quant scale buffer");
      CHECK_DT((*t), at::kFloat);
    }
    CHECK(scratch->numel() >= llmt::fp8_amax_slots(), "mx_quant: scratch too small");
    gp = g->data_ptr<float>();
    sp = scratch->data_ptr<float>();
  }
  ok(llmt::mx_quant((int)kind, x.data_ptr(), x.scalar_type() == at::kFloat, (int)rows, (int)cols, x.stride(0), qp, sfp, qtp,
                    sftp, gp, sp, interleave64, stochastic, (uint64_t)seed,
                    static_cast<const int64_t*>(opt_ptr(seed_dev, "seed_dev")), stream()),
     "mx_quant");
}

// ---------------------------------------------------------------- GEMM
void gemm(at::Tensor a, at::Tensor b, bool ta, bool tb, int64_t epi, at::Tensor out, bool accumulate,
          c10::optional<at::Tensor> aux, c10::optional<at::Tensor> out2, int64_t split, c10::optional<at::Tensor> cos_t,
          c10::optional<at::Tensor> sin_t, int64_t T, int64_t hd, int64_t rot_cols, c10::optional<at::Tensor> tgt,
          c10::optional<at::Tensor> lse, c10::optional<at::Tensor> grad_out, c10::optional<at::Tensor> part,
          c10::optional<at::Tensor> tlogit, double alpha, int64_t bn, int64_t splits, c10::optional<at::Tensor> peer,
          int64_t tp_rank, int64_t rows_per_rank, c10::optional<at::Tensor> scale_a, c10::optional<at::Tensor> scale_b,
          int64_t kind, c10::optional<at::Tensor> sfa, c10::optional<at::Tensor> sfb, c10::optional<at::Tensor> ag_src,
          c10::optional<at::Tensor> ag_dst, c10::optional<at::Tensor> ag_flags, int64_t ag_expect, int64_t ag_tp,
          c10::optional<at::Tensor> row_scale) {
  cuda2d(a, "a");
  cuda2d(b, "b");
  const bool bs = kind == 2 || kind == 3;
  const bool f8 = !bs && a.scalar_type() == at::kFloat8_e4m3fn;
  CHECK(kind == 0 || bs, "gemm: kind must be 0 (by dtype), 2 (MXFP8) or 3 (NVFP4)");
  if (bs) {
    CHECK(!ta && tb, "block-scaled gemm: both operands K-major (a: M x K, b: N x K)");
    CHECK(a.element_size() == 1 && b.element_size() == 1, "block-scaled gemm: byte operands");
    CHECK(sfa.has_value() && sfb.has_value(), "block-scaled gemm needs sfa and sfb");
    for (auto* t : {&*sfa, &*sfb}) {
      on_device(*t, "scale factors");
      CHECK(t->element_size() == 1 && t->is_contiguous(), "scale factors: contiguous bytes");
    }
    if (kind == 3) {
      CHECK(scale_a.has_value() && scale_b.has_value(), "NVFP4 gemm needs the decode scales");
      for (auto* t : {&*scale_a, &*scale_b}) {
        on_device(*t, "decode scale");
        CHECK_DT((*t), at::kFloat);
      }
    }
  } else if (f8) {
    CHECK_DT(b, at::kFloat8_e4m3fn);
    CHECK(!ta && tb, "fp8 gemm: both operands K-major (a: M x K, b: N x K)");
    CHECK(scale_a.has_value() && scale_b.has_value(), "fp8 gemm needs scale_a and scale_b");
    for (auto* t : {&*scale_a, &*scale_b}) {
      on_device(*t, "fp8 scale");
      CHECK_DT((*t), at::kFloat);
    }
  } else {
    CHECK_DT(a, at::kBFloat16);
    CHECK_DT(b, at::kBFloat16);
  }
  on_device(out, "out");
  const int kmul = kind == 3 ? 2 : 1;  // NVFP4 bytes hold two elements
  const int M = ta ? a.size(1) : a.size(0);
  const int K = (ta ? a.size(0) : a.size(1)) * kmul;
  int N = tb ? b.size(0) : b.size(1);
  const int Kb = (tb ? b.size(1) : b.size(0)) * kmul;
  CHECK(K == Kb, "gemm inner dims differ: ", K, " vs ", Kb);
  if (epi == llmt::EPI_SWIGLU) {
    CHECK(tb && b.size(0) == 2 * split, "SWIGLU gemm: b must be W13 (2*ffn, K)");
    N = (int)split;
  }
  switch (epi) {
    case llmt::EPI_BF16: case llmt::EPI_ROPE: case llmt::EPI_CE_BWD: case llmt::EPI_SWIGLU:
      CHECK_DT(out, at::kBFloat16);
      CHECK(out.dim() == 2 && out.size(0) >= M && out.size(1) >= N && out.stride(1) == 1 && out.stride(0) % 8 == 0,
            "gemm: bf16 output must be (M, N) row-major with a 16-byte-multiple pitch");
      break;
    case llmt::EPI_F32:
      CHECK_DT(out, at::kFloat);
      CHECK(out.dim() == 2 && out.size(0) >= M && out.size(1) >= N && out.stride(1) == 1 && out.stride(0) % 4 == 0,
            "gemm: fp32 output must be (M, N) row-major with a 16-byte-multiple pitch");
      break;
    case llmt::EPI_SWIGLU_BWD: case llmt::EPI_CE_FWD: break;
    case llmt::EPI_PEER_RS:
      CHECK(peer.has_value() && peer->defined() && peer->scalar_type() == at::kLong, "PEER_RS gemm needs peer slots");
      CHECK(out.dim() == 2 && out.size(1) == N && out.is_contiguous(), "PEER_RS: out is this rank's slot buffer (., N)");
      break;
    default: CHECK(false, "gemm: unknown epilogue ", epi);
  }
  llmt::GemmArgs g{};
  g.out = out.data_ptr();
  g.ldo = out.dim() == 2 ? out.stride(0) : N;
  g.accumulate = accumulate ? 1 : 0;
  g.split = (int)split;
  g.alpha = (float)alpha;
  if (aux.has_value() && aux->defined()) {
    on_device(*aux, "aux");
    CHECK_DT((*aux), at::kBFloat16);
    g.aux = aux->data_ptr();
    g.ld_aux = aux->stride(0);
  }
  if (out2.has_value() && out2->defined()) {
    on_device(*out2, "out2");
    CHECK_DT((*out2), at::kBFloat16);
    g.out2 = out2->data_ptr();
    g.ldo2 = out2->stride(0);
  }
  g.cos_t = static_cast<const float*>(opt_ptr(cos_t, "cos_t"));
  g.sin_t = static_cast<const float*>(opt_ptr(sin_t, "sin_t"));
  g.T = (int)T;
  g.hd = (int)hd;
  g.rot_cols = (int)rot_cols;
  g.tgt = static_cast<const int64_t*>(opt_ptr(tgt, "tgt"));
  g.lse = static_cast<const float*>(opt_ptr(lse, "lse"));
  g.grad_out = static_cast<const float*>(opt_ptr(grad_out, "grad_out"));
  g.part = static_cast<float*>(const_cast<void*>(opt_ptr(part, "part")));
  g.tlogit = static_cast<float*>(const_cast<void*>(opt_ptr(tlogit, "tlogit")));
  g.peer = reinterpret_cast<void* const*>(const_cast<void*>(opt_ptr(peer, "peer")));
  g.tp_rank = (int)tp_rank;
  g.rows_per_rank = (int)rows_per_rank;
  if (ag_src.has_value() && ag_src->defined()) {
    // fused all-gather: this rank's rows (rows_per_rank, K) bf16; a is this rank's gather buffer
    cuda2d(*ag_src, "ag_src");
    CHECK(kind == 0 && !f8, "fused all-gather: bf16 operands only");
    CHECK_DT((*ag_src), at::kBFloat16);
    CHECK(!ta && ag_src->size(0) == rows_per_rank && ag_src->size(1) == a.size(1) && ag_src->stride(1) == 1,
          "ag_src must be this rank's (rows_per_rank, K) rows of a row-major A");
    CHECK(ag_dst.has_value() && ag_flags.has_value() && ag_dst->scalar_type() == at::kLong &&
              ag_flags->scalar_type() == at::kLong && ag_dst->numel() == ag_tp && ag_flags->numel() == ag_tp,
          "fused all-gather needs ag_dst and ag_flags: int64 device arrays of ag_tp pointers");
    on_device(*ag_dst, "ag_dst");
    on_device(*ag_flags, "ag_flags");
    g.ag_src = ag_src->data_ptr();
    g.ag_lds = ag_src->stride(0);
    g.ag_dst = reinterpret_cast<void* const*>(ag_dst->data_ptr());
    g.ag_flags = reinterpret_cast<uint32_t* const*>(ag_flags->data_ptr());
    g.ag_expect = (uint32_t)ag_expect;
    g.ag_tp = (int)ag_tp;
  }
  if (epi == llmt::EPI_ROPE) CHECK(g.cos_t && g.sin_t && T > 0, "ROPE gemm needs rope tables and T");
  if (epi == llmt::EPI_SWIGLU) CHECK(g.aux && aux->stride(0) % 8 == 0, "SWIGLU gemm needs the gu save buffer");
  if (epi == llmt::EPI_SWIGLU_BWD) CHECK(g.aux && g.out2 && split == N, "SWIGLU_BWD gemm args");
  if (epi == llmt::EPI_CE_FWD) {
    CHECK(g.tgt && g.part && g.tlogit, "CE_FWD gemm args");
    const int BN = bn ? (int)bn : llmt::gemm_pick_bn(M, N, (int)epi);
    CHECK(part->numel() >= (int64_t)M * ((N + BN - 1) / BN) * 2, "CE_FWD partial buffer too small");
  }
  if (epi == llmt::EPI_CE_BWD) CHECK(g.tgt && g.lse, "CE_BWD gemm args");
  if (row_scale.has_value() && row_scale->defined()) {
    CHECK(epi == llmt::EPI_CE_BWD, "row_scale goes with the CE_BWD epilogue");
    CHECK(row_scale->scalar_type() == at::kFloat && row_scale->is_contiguous() && row_scale->numel() == M,
          "row_scale must be ", M, " contiguous float32 values");
    g.row_scale = static_cast<const float*>(opt_ptr(row_scale, "row_scale"));
  }
  if (bs) {
    if (kind == 3) {
      g.scale_a = scale_a->data_ptr<float>();
      g.scale_b = scale_b->data_ptr<float>();
    }
    g.sfa = static_cast<const uint8_t*>(sfa->data_ptr());
    g.sfb = static_cast<const uint8_t*>(sfb->data_ptr());
    const int kbytes = K / kmul;
    const int64_t need_a = llmt::mx_sf_bytes((int)kind, M, K), need_b = llmt::mx_sf_bytes((int)kind, b.size(0), K);
    CHECK(sfa->numel() >= need_a && sfb->numel() >= need_b, "block-scaled gemm: scale buffers too small");
    (void)kbytes;
    ok(llmt::gemm_bs((int)kind, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), M, N, K, (int)epi, g, stream(),
                     (int)splits),
       "gemm_bs");
    return;
  }
  if (f8) {
    g.scale_a = scale_a->data_ptr<float>();
    g.scale_b = scale_b->data_ptr<float>();
    ok(llmt::gemm_fp8(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), M, N, K, (int)epi, (int)bn, g, stream(),
                      (int)splits),
       "gemm_fp8");
    return;
  }
  ok(llmt::gemm(a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), ta, tb, M, N, K, (int)epi, (int)bn, g, stream(),
                (int)splits),
     "gemm");
}

// ---------------------------------------------------------------- attention
std::vector<at::Tensor> flash_attn_fwd(at::Tensor qkv, int64_t B, int64_t T, int64_t H, int64_t KV, int64_t hd,
                                       bool causal, double scale) {
  cuda2d(qkv, "qkv");
  CHECK_DT(qkv, at::kBFloat16);
  CHECK(qkv.size(0) == B * T && qkv.size(1) >= (H + 2 * KV) * hd, "flash_attn_fwd: qkv shape mismatch");
  auto o = at::empty({B * T, H * hd}, qkv.options());
  auto lse = at::empty({B, H, T}, qkv.options().dtype(at::kFloat));
  ok(llmt::flash_attn_fwd(qkv.data_ptr(), qkv.stride(0), o.data_ptr(), lse.data_ptr<float>(), (int)B, (int)T, (int)H,
                          (int)KV, (int)hd, causal, (float)scale, stream()),
     "flash_attn_fwd");
  return {o, lse};
}

at::Tensor flash_attn_bwd(at::Tensor dO, at::Tensor qkv, at::Tensor o, at::Tensor lse, at::Tensor cos_t,
                          at::Tensor sin_t, int64_t B, int64_t T, int64_t H, int64_t KV, int64_t hd, bool causal,
                          double scale) {
  CHECK_DT(dO, at::kBFloat16);
  CHECK_DT(qkv, at::kBFloat16);
  CHECK_DT(o, at::kBFloat16);
  CHECK_DT(lse, at::kFloat);
  for (auto* t : {&dO, &qkv, &o, &lse, &cos_t, &sin_t}) on_device(*t, "flash_attn_bwd operand");
  CHECK(dO.is_contiguous() && o.is_contiguous() && qkv.is_contiguous() && lse.is_contiguous(),
        "flash_attn_bwd: operands must be contiguous");
  CHECK(dO.numel() == B * T * H * hd && o.numel() == dO.numel(), "flash_attn_bwd: dO/o shape");
  CHECK(qkv.size(0) == B * T && qkv.size(1) == (H + 2 * KV) * hd, "flash_attn_bwd: qkv shape");
  CHECK(cos_t.size(0) >= T && cos_t.size(1) == hd && cos_t.is_contiguous() && sin_t.is_contiguous(),
        "flash_attn_bwd: rope tables");
  auto dqkv = at::empty_like(qkv);
  auto dsum = at::empty({2, B, H, T}, lse.options());
  auto dq_acc = at::empty({B * T, H * hd}, lse.options());
  ok(llmt::flash_attn_bwd(dO.data_ptr(), qkv.data_ptr(), qkv.stride(0), o.data_ptr(), lse.data_ptr<float>(),
                          cos_t.data_ptr<float>(), sin_t.data_ptr<float>(), dqkv.data_ptr(), dsum.data_ptr<float>(),
                          dq_acc.data_ptr<float>(), (int)B, (int)T, (int)H, (int)KV, (int)hd, causal, (float)scale,
                          stream()),
     "flash_attn_bwd");
  return dqkv;
}

// ---------------------------------------------------------------- data-parallel transport
pybind11::tuple ipc_alloc(int64_t bytes) {
  void* ptr = nullptr;
  char h[64];
  ok(llmt::ipc_alloc((size_t)bytes, &ptr, h), "ipc_alloc");
  return pybind11::make_tuple((int64_t)reinterpret_cast<uintptr_t>(ptr), pybind11::bytes(h, 64));
}

int64_t ipc_open(pybind11::bytes handle) {
  std::string h = handle;
  CHECK(h.size() == 64, "ipc handle must be 64 bytes");
  void* ptr = nullptr;
  ok(llmt::ipc_open(h.data(), &ptr), "ipc_open");
  return (int64_t)reinterpret_cast<uintptr_t>(ptr);
}

void ipc_close(int64_t ptr) { ok(llmt::ipc_close(reinterpret_cast<void*>(ptr)), "ipc_close"); }
void ipc_free(int64_t ptr) { ok(llmt::ipc_free(reinterpret_cast<void*>(ptr)), "ipc_free"); }

// Non-owning tensor over device memory this library allocated (the Python owner frees it).
at::Tensor tensor_from_ptr(int64_t ptr, int64_t numel, at::ScalarType dtype, int64_t device) {
  return at::from_blob(reinterpret_cast<void*>(ptr), {numel},
                       at::TensorOptions().dtype(dtype).device(at::Device(at::kCUDA, (int)device)));
}

void dp_barrier(at::Tensor pads_dev, int64_t my_pad, at::Tensor epoch, int64_t rank, int64_t world, int64_t code) {
  CHECK_DT(pads_dev, at::kLong);
  CHECK_DT(epoch, at::kInt);
  ok(llmt::dp_barrier(reinterpret_cast<uint32_t* const*>(pads_dev.data_ptr<int64_t>()),
                      reinterpret_cast<uint32_t*>(my_pad), reinterpret_cast<uint32_t*>(epoch.data_ptr<int>()),
                      (int)rank, (int)world, (int)code, stream()),
     "dp_barrier");
}

void dp_fused_adamw(at::Tensor grads_dev, at::Tensor shadows_dev, at::Tensor master, at::Tensor m, at::Tensor v,
                    int64_t lo, int64_t n, at::Tensor lr, at::Tensor step, double b1, double b2, double eps, double wd,
                    double grad_scale, int64_t world, int64_t max_blocks, bool clear) {
  CHECK_DT(grads_dev, at::kLong);
  CHECK_DT(shadows_dev, at::kLong);
  CHECK(grads_dev.numel() == world && shadows_dev.numel() == world, "peer pointer arrays must have world entries");
  CHECK(m.numel() >= n && v.numel() >= n && master.numel() >= lo + n, "shard bounds exceed the buffers");
  llmt::AdamHyper h{(float)b1, (float)b2, (float)eps, (float)wd, (float)grad_scale};
  ok(llmt::dp_fused_adamw(reinterpret_cast<float* const*>(grads_dev.data_ptr<int64_t>()),
                          reinterpret_cast<void* const*>(shadows_dev.data_ptr<int64_t>()), master.data_ptr<float>(),
                          m.data_ptr<float>(), v.data_ptr<float>(), lo, n, lr.data_ptr<float>(), step.data_ptr<int>(),
                          h, (int)world, stream(), (int)max_blocks, clear),
     "dp_fused_adamw");
}

void dp_nvls_adamw(int64_t g_mc, int64_t w_mc, at::Tensor master, at::Tensor m, at::Tensor v, int64_t lo, int64_t n,
                   at::Tensor lr, at::Tensor step, double b1, double b2, double eps, double wd, double grad_scale,
                   int64_t max_blocks) {
  on_device(master, "master");
  on_device(m, "m");
  on_device(v, "v");
  CHECK(g_mc != 0 && w_mc != 0, "dp_nvls_adamw: multicast addresses are null (no NVLS support)");
  CHECK(m.numel() >= n && v.numel() >= n && master.numel() >= lo + n, "shard bounds exceed the buffers");
  llmt::AdamHyper h{(float)b1, (float)b2, (float)eps, (float)wd, (float)grad_scale};
  ok(llmt::dp_nvls_adamw(reinterpret_cast<const void*>(g_mc), reinterpret_cast<void*>(w_mc), master.data_ptr<float>(),
                         m.data_ptr<float>(), v.data_ptr<float>(), lo, n, lr.data_ptr<float>(), step.data_ptr<int>(), h,
                         stream(), (int)max_blocks),
     "dp_nvls_adamw");
}

#ifdef LLMT_DEBUG_BOUNDS
// Self-test of the bounds-checked build: a store at index `i` of an n-float buffer, guarded by
// LLMT_IN. With i >= n the guard records the site and skips the store (nothing is written out
// of bounds); the record is read back with bounds_error(). Only this build has it.
void bounds_probe(at::Tensor buf, int64_t i) {
  on_device(buf, "buf");
  CHECK_DT(buf, at::kFloat);
  ok(llmt::bounds_probe(buf.data_ptr<float>(), buf.numel(), i, stream()), "bounds_probe");
}
#endif

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  namespace py = pybind11;
  using namespace pybind11::literals;
  m.doc() = "llmt native sm_100a kernels";
  m.def("add_rmsnorm_fwd", &add_rmsnorm_fwd, "a"_a, "r"_a, "w"_a, "eps"_a, "write_s"_a);
  m.def("rmsnorm_bwd", &rmsnorm_bwd, "dy"_a, "s"_a, "w"_a, "rstd"_a, "ds_in"_a, "dw"_a, "ticket"_a, "write_ds16"_a,
        "accumulate"_a);
  m.def("swiglu_fwd", &swiglu_fwd);
  m.def("swiglu_bwd", &swiglu_bwd);
  m.def("rope_inplace", &rope_inplace);
  m.def("embedding_fwd", &embedding_fwd, "idx"_a, "W"_a, "x"_a, "err"_a = py::none(), "v0"_a = 0,
        "partial"_a = false);
  m.def("embedding_bwd", &embedding_bwd, "idx"_a, "dx"_a, "dW"_a, "v0"_a = 0);
  m.def("adamw_step", &adamw_step, "p"_a, "g"_a, "m"_a, "v"_a, "p16"_a, "lr"_a, "step"_a, "b1"_a, "b2"_a, "eps"_a,
        "wd"_a, "grad_scale"_a, "zero_grad"_a = false, "max_blocks"_a = 0);
  m.def("cast_bf16", &cast_bf16, "x"_a, "y"_a, "max_blocks"_a = 0);
  m.def("ce_fwd_rows", &ce_fwd_rows);
  m.def("ce_bwd_rows", &ce_bwd_rows);
  m.def("ce_combine", &ce_combine);
  py::class_<MultiPlan>(m, "MultiPlan")
      .def(py::init<std::vector<at::Tensor>, std::vector<at::Tensor>, std::vector<double>>(), "p"_a, "p16"_a, "wd"_a)
      .def_readonly("blocks", &MultiPlan::blocks)
      .def_readonly("first_block", &MultiPlan::first_block)
      .def("step", &MultiPlan::step);
  m.def("adamw_state_values", &adamw_state_values, "m"_a, "ms"_a, "v"_a, "vs"_a, "f32"_a = false);
  m.def("adamw_encode_states", &adamw_encode_states, "m32"_a, "v32"_a, "m"_a, "ms"_a, "v"_a, "vs"_a);
  m.def("rotary", &rotary, "q"_a, "k"_a, "positions"_a, "table"_a, "rotary_dim"_a, "interleaved"_a, "inverse"_a,
        "q_out"_a = py::none(), "k_out"_a = py::none());
  m.def("loss_error_code", &llmt::loss_error_code, "reset"_a = false);
  m.def("logprob_rows", &logprob_rows, "logits"_a, "targets"_a, "mask"_a = py::none());
  m.attr("tokens_counted_in_rows") = (int)llmt::kTokensCountedInRows;
  m.def("policy_rows", &policy_rows, "logits"_a, "targets"_a, "old"_a, "adv"_a, "ref"_a, "mask"_a, "clip_lo"_a,
        "clip_hi"_a, "kl"_a, "reduction"_a, "grad"_a, "out"_a = py::none(), "keep"_a = false);
  m.def("policy_tokens", &policy_tokens, "logp"_a, "targets"_a, "V"_a, "old"_a, "adv"_a, "ref"_a, "mask"_a, "clip_lo"_a,
        "clip_hi"_a, "kl"_a, "reduction"_a);
  m.def("preference_rows", &preference_rows, "logits"_a, "targets"_a, "ref"_a, "mask"_a, "beta"_a, "smoothing"_a,
        "kind"_a, "average"_a, "grad"_a, "out"_a = py::none(), "keep"_a = false);
  m.def("preference_tokens", &preference_tokens, "logp"_a, "targets"_a, "V"_a, "ref"_a, "mask"_a, "beta"_a, "smoothing"_a,
        "kind"_a, "average"_a);
  m.def("grad_rows", &grad_rows, "logits"_a, "targets"_a, "mask"_a, "coef"_a, "stats"_a, "grad_out"_a = py::none(),
        "out"_a = py::none(), "skip_one"_a = false);
  m.def("gemm", &gemm, "a"_a, "b"_a, "ta"_a, "tb"_a, "epi"_a, "out"_a, "accumulate"_a = false, "aux"_a = py::none(),
        "out2"_a = py::none(), "split"_a = 0, "cos_t"_a = py::none(), "sin_t"_a = py::none(), "T"_a = 0, "hd"_a = 0,
        "rot_cols"_a = 0, "tgt"_a = py::none(), "lse"_a = py::none(), "grad_out"_a = py::none(), "part"_a = py::none(),
        "tlogit"_a = py::none(), "alpha"_a = 1.0, "bn"_a = 0, "splits"_a = 0, "peer"_a = py::none(), "tp_rank"_a = 0, "rows_per_rank"_a = 0,
        "scale_a"_a = py::none(), "scale_b"_a = py::none(), "kind"_a = 0, "sfa"_a = py::none(), "sfb"_a = py::none(),
        "ag_src"_a = py::none(), "ag_dst"_a = py::none(), "ag_flags"_a = py::none(), "ag_expect"_a = 0, "ag_tp"_a = 0,
        "row_scale"_a = py::none());
  m.def("mx_sf_bytes", &llmt::mx_sf_bytes);
  m.def("mx_quant", &mx_quant, "kind"_a, "x"_a, "q"_a, "sf"_a, "qt"_a, "sft"_a, "g"_a, "scratch"_a,
        "interleave64"_a = false, "stochastic"_a = false, "seed"_a = 0, "seed_dev"_a = py::none());
  m.def("fp8_amax_slots", &llmt::fp8_amax_slots);
  m.def("fp8_quant", &fp8_quant, "x"_a, "q"_a, "qt"_a, "inv"_a, "scratch"_a);
  m.def("gemm_error_code", &llmt::gemm_error_code, "reset"_a = false);
  m.def("gemm_plan", [](int64_t M, int64_t N, int64_t K, int64_t epi, bool can_split) {
    int bn = 0, splits = 1;
    llmt::gemm_plan((int)M, (int)N, (int)K, (int)epi, can_split, &bn, &splits);
    return std::make_tuple(bn, splits);
  });
  m.def("flash_attn_fwd", &flash_attn_fwd);
  m.def("flash_attn_bwd", &flash_attn_bwd);
  m.def("attn_error_code", &llmt::attn_error_code, "reset"_a = false);
  m.def("set_reserved_sms", &llmt::set_reserved_sms, "n"_a);
  m.def("reserved_sms", &llmt::reserved_sms);
  m.def("tp_allgather_rows", [](at::Tensor src, at::Tensor dst, int64_t tp, int64_t row0) {
    on_device(src, "src");
    CHECK(src.is_contiguous() && src.scalar_type() == at::kBFloat16 && src.dim() == 2, "tp_allgather_rows: src");
    ok(llmt::tp_allgather_rows(src.data_ptr(), reinterpret_cast<void* const*>(dst.data_ptr<int64_t>()), (int)tp, row0,
                               src.size(0), (int)src.size(1), stream()),
       "tp_allgather_rows");
  });
  m.def("tp_scatter_rows", [](at::Tensor src, at::Tensor slots, int64_t tp, int64_t rank) {
    on_device(src, "src");
    CHECK(src.is_contiguous() && src.scalar_type() == at::kBFloat16 && src.dim() == 2 && src.size(0) % tp == 0,
          "tp_scatter_rows: src");
    ok(llmt::tp_scatter_rows(src.data_ptr(), reinterpret_cast<void* const*>(slots.data_ptr<int64_t>()), (int)tp,
                             (int)rank, src.size(0) / tp, (int)src.size(1), stream()),
       "tp_scatter_rows");
  });
  m.def("tp_sum_slots", [](at::Tensor slots, at::Tensor out, int64_t tp) {
    on_device(slots, "slots");
    on_device(out, "out");
    CHECK(out.is_contiguous() && slots.is_contiguous() && slots.numel() == tp * out.numel(), "tp_sum_slots: shapes");
    ok(llmt::tp_sum_slots(slots.data_ptr(), out.data_ptr(), (int)tp, out.size(0), (int)out.size(1), stream()),
       "tp_sum_slots");
  });
  m.def("sm_count", &llmt::sm_count);
  m.def("ipc_alloc", &ipc_alloc);
  m.def("ipc_open", &ipc_open);
  m.def("ipc_close", &ipc_close);
  m.def("ipc_free", &ipc_free);
  m.def("tensor_from_ptr", &tensor_from_ptr);
  m.def("dp_barrier", &dp_barrier);
  m.def("dp_fused_adamw", &dp_fused_adamw, "grads_dev"_a, "shadows_dev"_a, "master"_a, "m"_a, "v"_a, "lo"_a, "n"_a,
        "lr"_a, "step"_a, "b1"_a, "b2"_a, "eps"_a, "wd"_a, "grad_scale"_a, "world"_a, "max_blocks"_a = 0,
        "clear"_a = true);
  m.def("dp_error_code", &llmt::dp_error_code, "reset"_a = false);
  m.def("bounds_error", &llmt::bounds_error, "reset"_a = false);
  m.def("bounds_checking", &llmt::bounds_checking);
#ifdef LLMT_DEBUG_BOUNDS
  m.def("bounds_probe", &bounds_probe, "buf"_a, "i"_a);
#endif
  m.def("dp_nvls_adamw", &dp_nvls_adamw, "g_mc"_a, "w_mc"_a, "master"_a, "m"_a, "v"_a, "lo"_a, "n"_a, "lr"_a, "step"_a,
        "b1"_a, "b2"_a, "eps"_a, "wd"_a, "grad_scale"_a, "max_blocks"_a = 0);
}

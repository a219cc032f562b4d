// Python binding of the mxfp4 products, the quantisation and the token sort,
// with their autograd nodes, over the C ABI of libqmoe.so.
//
// Every function takes its arguments as the Python wrappers do and a flag:
// without it, it returns None for anything but tensors the entry points can
// read as they are (GPU, contiguous, aligned, of the right types and sizes),
// and the wrapper then checks, converts or refuses; with it, such a call is an
// error.  Tracers, which would not see a launch, and tangents are refused.  A
// call made this way costs the host about 5 us where ctypes cost 11, and the
// token sort and the way back with their gradients 46 to 79 from run to run
// where Python autograd nodes cost 136, which is what a small call's time is
// made of.
//
// Launches go to the tensors' device and its current stream; nothing
// synchronises; outputs and tables come from torch's allocator.
#include <torch/extension.h>

#include <ATen/ops/arange.h>
#include <ATen/ops/index_select.h>
#include <ATen/ops/searchsorted.h>
#include <ATen/ops/zeros.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "qmoe.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

constexpr int64_t kSortedMinRows = 64;  // gathered rows from which the grouped GEMM takes sorted calls
// Rows of one matrix that the matrix-vector kernel takes: it reads the weights
// once per row, mostly from the caches after the first, the kernel for few rows
// once in all but with a longer start.  Two rows of 4096 x 2048 take 4.7 us
// either way, four 6.4 and 4.7, four of 1024 x 2048 3.4 and 4.0.  Transposed
// products take the GEMM from one row on (4096 x 2048: 20 and 14.2 us).
constexpr int64_t kQmvMaxRows = 4, kQmvMaxWork = int64_t(1) << 24;

// Rows above which products of two mxfp4 operands leave the kernel for few rows,
// and rows per expert from which laying the scales out in lines pays.
constexpr int64_t kFewRows = 64, kLineRows = 32;

struct Failure : std::runtime_error {
  int code;
  Failure(int c, const char* what)
      : std::runtime_error(std::string(what) + ": " + qmoe_last_error() + " (code " + std::to_string(c) + ")"), code(c) {}
  explicit Failure(const char* refused) : std::runtime_error(refused), code(QMOE_ERR_UNSUPPORTED) {}
};
void ok(int rc, const char* what) {
  if (rc != QMOE_OK) throw Failure(rc, what);
}

int type_of(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return QMOE_BF16;
    case at::kHalf: return QMOE_FP16;
    case at::kFloat: return QMOE_FP32;
    default: return -1;
  }
}
// A tensor the kernels can read as it is.
bool plain(const Tensor& t) {
  return t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg() && !t.is_conj() &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}
bool plain(const Tensor& t, at::ScalarType type) { return t.scalar_type() == type && plain(t); }
bool words(const Tensor& t) { return (t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32) && plain(t); }
// Scale bytes need no alignment.
bool bytes(const Tensor& t) {
  return t.scalar_type() == at::kByte && t.is_cuda() && t.layout() == at::kStrided && t.is_contiguous();
}
bool get(py::handle h, Tensor* t) {
  if (!THPVariable_Check(h.ptr())) return false;
  *t = THPVariable_Unpack(h.ptr());
  return true;
}
template <class T>
const T* ptr(const Tensor& t) {
  return t.defined() ? static_cast<const T*>(t.const_data_ptr()) : nullptr;
}
void* stream(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor ready(Tensor t) {
  t = t.resolve_neg().contiguous();
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 ? t.clone() : t;
}
// A gradient of t is asked for.  Tangents (forward mode) would be lost: refused.
bool records(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(/*level=*/0).defined(),
                              "forward-mode automatic differentiation is not supported here");
  return t.requires_grad() && at::GradMode::is_enabled();
}

// A tracer sees the allocation of a result and not the launch that fills it: refused.
void refuse_recorders() {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  if (torch::jit::tracer::isTracing() || TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY).has_value())
    throw Failure("torch.jit.trace and make_fx cannot record these kernels");
}

py::object none(bool must) {
  TORCH_CHECK(!must, "the arguments are not what the kernels read");
  return py::none();
}
py::object give(const Tensor& t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(t)); }

// Gradients are not differentiable again: where a graph of them is recorded, it ends in an error.
variable_list first_order(variable_list grads, const variable_list& from) {
  if (!at::GradMode::is_enabled()) return grads;
  bool any = false;
  for (const auto& t : from) any |= t.defined() && t.requires_grad();
  if (!any) return grads;
  for (auto& g : grads) {
    if (!g.defined()) continue;
    auto node = std::make_shared<torch::autograd::DelayedError>(
        "trying to differentiate twice a function that was marked with @once_differentiable", 1);
    g = (*node)({g.detach().requires_grad_(true)})[0];
  }
  return grads;
}

// ------------------------------------------------------------ quantisation

std::pair<Tensor, Tensor> quantize_run(const Tensor& x) {
  const int64_t K = x.size(-1);
  auto sizes = x.sizes().vec();
  sizes.back() = K / 8;
  Tensor w = at::empty(sizes, x.options().dtype(at::kInt).requires_grad(false));
  sizes.back() = K / 32;
  Tensor s = at::empty(sizes, x.options().dtype(at::kByte).requires_grad(false));
  ok(qmoe_mxfp4_quantize(x.const_data_ptr(), type_of(x), K ? x.numel() / K : 0, K,
                         static_cast<uint32_t*>(w.data_ptr()), s.data_ptr<uint8_t>(), stream(x)),
     "qmoe_mxfp4_quantize");
  return {w, s};
}

py::object quantize(py::handle x_, bool must) {
  refuse_recorders();
  Tensor x;
  if (!get(x_, &x) || type_of(x) < 0 || x.dim() < 1 || x.size(-1) % 32 || !plain(x)) return none(must);
  const c10::hip::HIPGuard guard(x.get_device());
  const auto [w, s] = quantize_run(x);
  return py::make_tuple(give(w), give(s));
}

py::object dequantize(py::handle w_, py::handle s_, int type, bool must) {
  refuse_recorders();
  Tensor w, s;
  if (!get(w_, &w) || !get(s_, &s) || !words(w) || !bytes(s) || w.dim() < 1 || w.dim() != s.dim() ||
      w.device() != s.device() || w.size(-1) % 4 || s.size(-1) != w.size(-1) / 4 ||
      w.sizes().slice(0, w.dim() - 1) != s.sizes().slice(0, s.dim() - 1))
    return none(must);
  const c10::hip::HIPGuard guard(w.get_device());
  const int64_t K = w.size(-1) * 8;
  auto sizes = w.sizes().vec();
  sizes.back() = K;
  const at::ScalarType types[] = {at::kBFloat16, at::kHalf, at::kFloat};
  Tensor out = at::empty(sizes, w.options().dtype(types[type]));
  ok(qmoe_mxfp4_dequantize(ptr<uint32_t>(w), ptr<uint8_t>(s), K ? w.numel() / w.size(-1) : 0, K, type, out.data_ptr(),
                           stream(w)),
     "qmoe_mxfp4_dequantize");
  return give(out);
}

// --------------------------------------------------------------- token sort

Tensor sort_run(const Tensor& x, const Tensor& inv) {
  const int64_t n = inv.numel(), T = x.size(0), D = x.size(1);
  Tensor xs = at::empty({n, D}, x.options().requires_grad(false));
  ok(qmoe_sort_rows(x.const_data_ptr(), T, ptr<int32_t>(inv), T ? n / T : 0, D, type_of(x), xs.data_ptr(), stream(x)),
     "qmoe_sort_rows");
  return xs;
}
Tensor sum_run(const Tensor& rows, const Tensor& inv, const Tensor& scores, const Tensor& first, int64_t T, int64_t k,
               at::ScalarType out) {
  Tensor y = at::empty({T, rows.size(1)}, rows.options().dtype(out).requires_grad(false));
  ok(qmoe_unsort_sum(rows.const_data_ptr(), rows.size(0), type_of(rows), ptr<int32_t>(inv), ptr<float>(scores),
                     ptr<int32_t>(first), T, k, rows.size(1), type_of(y), y.data_ptr(), stream(rows)),
     "qmoe_unsort_sum");
  return y;
}

struct Sort : torch::autograd::Function<Sort> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& inv) {
    ctx->save_for_backward({inv});
    ctx->saved_data["T"] = x.size(0);
    return sort_run(x, inv);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const Tensor inv = ctx->get_saved_variables()[0];
    const int64_t T = ctx->saved_data["T"].toInt();
    const Tensor d = ready(grads[0]);
    const c10::hip::HIPGuard guard(d.get_device());
    Tensor dx = sum_run(d, inv, {}, {}, T, T ? d.size(0) / T : 0, d.scalar_type());
    return first_order({dx, Tensor()}, grads);
  }
};

struct Unsort : torch::autograd::Function<Unsort> {
  static Tensor forward(AutogradContext* ctx, const Tensor& xs, const Tensor& inv, const Tensor& scores) {
    const bool ds = scores.requires_grad();
    ctx->save_for_backward({ds ? xs : Tensor(), inv, scores});
    ctx->saved_data["dxs"] = xs.requires_grad();
    ctx->saved_data["ds"] = ds;
    return sum_run(xs, inv, scores, {}, scores.size(0), scores.size(1), xs.scalar_type());
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &xs = saved[0], &inv = saved[1], &scores = saved[2];
    const Tensor dy = ready(grads[0]);
    const c10::hip::HIPGuard guard(dy.get_device());
    const int64_t T = scores.size(0), k = scores.size(1), n = T * k, D = dy.size(1);
    Tensor dxs, ds;
    if (ctx->saved_data["dxs"].toBool()) dxs = at::empty({n, D}, dy.options().requires_grad(false));
    if (ctx->saved_data["ds"].toBool()) ds = at::empty({T, k}, scores.options().requires_grad(false));
    ok(qmoe_unsort_grad(dy.const_data_ptr(), xs.defined() ? xs.const_data_ptr() : nullptr, n, type_of(dy),
                        ptr<int32_t>(inv), ptr<float>(scores), T, k, D, dxs.defined() ? dxs.data_ptr() : nullptr,
                        ds.defined() ? ds.data_ptr<float>() : nullptr, stream(dy)),
       "qmoe_unsort_grad");
    auto from = grads;
    from.push_back(xs);
    from.push_back(scores);
    return first_order({dxs, Tensor(), ds}, from);
  }
};

bool pairs(const Tensor& t, const Tensor& rows, int64_t n) {
  return plain(t, at::kInt) && t.dim() == 1 && t.numel() == n && t.device() == rows.device();
}

py::object sort_tokens(py::handle x_, py::handle order_, py::handle inv_, bool must) {
  refuse_recorders();
  Tensor x, order, inv;
  if (!get(x_, &x) || !get(order_, &order) || !get(inv_, &inv) || type_of(x) < 0 || x.dim() != 2 || !plain(x))
    return none(must);
  const int64_t n = order.numel(), T = x.size(0);
  if ((T ? n % T : n) || !pairs(order, x, n) || !pairs(inv, x, n)) return none(must);
  const c10::hip::HIPGuard guard(x.get_device());
  return give(records(x) ? Sort::apply(x, inv) : sort_run(x, inv));
}

py::object unsort_tokens(py::handle xs_, py::handle order_, py::handle inv_, py::handle scores_, bool must) {
  refuse_recorders();
  Tensor xs, order, inv, scores;
  if (!get(xs_, &xs) || !get(order_, &order) || !get(inv_, &inv) || !get(scores_, &scores) || type_of(xs) < 0 ||
      xs.dim() != 2 || !plain(xs))
    return none(must);
  const int64_t n = xs.size(0);
  if (!pairs(order, xs, n) || !pairs(inv, xs, n) || !plain(scores, at::kFloat) || scores.dim() != 2 ||
      scores.numel() != n || scores.device() != xs.device())
    return none(must);
  const c10::hip::HIPGuard guard(xs.get_device());
  if (records(xs) || records(scores)) return give(Unsort::apply(xs, inv, scores));
  return give(sum_run(xs, inv, scores, {}, scores.size(0), scores.size(1), xs.scalar_type()));
}

// ----------------------------------------------------------------- products

// Which activation row and which expert each of n output rows takes: x_rows,
// or row i / div; experts (undefined: expert 0 for all); and the tile table of
// sorted rows (undefined: not sorted, or one expert).  With inv activation row
// t's rows are known to be inv[t div .. (t + 1) div).
struct Rows {
  int64_t n = 0, div = 1, maxt = 0;
  Tensor x_rows, experts, offsets, tile_row, tile_exp, ntiles, inv;
};
struct Weights {
  Tensor w, s;
  int64_t E, N, K;
};

// The activation row of each row for the GEMMs; undefined: row r itself.
Tensor gemm_rows(const Rows& r, const Tensor& like) {
  if (r.x_rows.defined() || r.div == 1) return r.x_rows;
  return at::arange(r.n, like.options().dtype(at::kInt).requires_grad(false)).floor_divide_(r.div);
}

Tensor product_run(const Tensor& x_, const Weights& g, const Rows& r, bool transpose, at::ScalarType type) {
  Tensor x = x_;
  Tensor out = at::empty({r.n, transpose ? g.N : g.K}, x.options().dtype(type).requires_grad(false));
  if (out.numel() == 0) return out;
  if (x.size(1) == 0) return out.zero_();
  const int t = type_of(out);
  const bool few = transpose && (r.n == 1 || (r.n <= kQmvMaxRows && r.n * g.N * g.K <= kQmvMaxWork));
  if (!r.offsets.defined() && (r.experts.defined() || few)) {
    ok(qmoe_mxfp4_gather_qmv(ptr<uint16_t>(x), x.size(0), x.size(1), ptr<int32_t>(r.x_rows), (int32_t)r.div,
                             ptr<int32_t>(r.experts), r.n, ptr<uint32_t>(g.w), ptr<uint8_t>(g.s), (int32_t)g.E, g.N, g.K,
                             transpose, t, out.data_ptr(), stream(x)),
       "qmoe_mxfp4_gather_qmv");
    return out;
  }
  if (x.size(1) % 8) x = at::constant_pad_nd(x, {0, 8 - x.size(1) % 8});  // whole 16-byte units, zeros behind the row
  const Tensor rows = gemm_rows(r, x);
  ok(qmoe_mxfp4_gather_qmm(ptr<uint16_t>(x), x.size(0), x.size(1), ptr<int32_t>(rows), r.n, ptr<uint32_t>(g.w),
                           ptr<uint8_t>(g.s), (int32_t)g.E, g.N, g.K, transpose, ptr<int32_t>(r.offsets),
                           ptr<int32_t>(r.tile_row), ptr<int32_t>(r.tile_exp), ptr<int32_t>(r.ntiles), r.maxt, t,
                           out.data_ptr(), stream(x)),
     "qmoe_mxfp4_gather_qmm");
  return out;
}

// The rows of each of n_x activation rows, in ascending order: (order, first),
// activation row t's being order[first[t] .. first[t + 1]).  A stable radix sort
// of the rows' activation rows by the routing's counting sort, eleven bits a
// pass: no library sort, whose cleared counters a captured graph must not hold.
std::pair<Tensor, Tensor> rows_of(const Tensor& x_rows, int64_t n_x) {
  constexpr int64_t kBits = 11, kBins = 1 << kBits;
  const int64_t n = x_rows.numel(), maxt = kBins + 1;
  if (n == 0) return {x_rows, at::zeros({n_x + 1}, x_rows.options())};
  const Tensor at_ = x_rows.clamp(0, std::max<int64_t>(n_x - 1, 0));
  const int64_t bytes = qmoe_route_workspace_size(n, kBins);
  Tensor order;
  for (int64_t bit = 0; bit == 0 || (n_x - 1) >> bit; bit += kBits) {
    Tensor digit = at_.__rshift__(bit).bitwise_and_(kBins - 1);
    if (order.defined()) digit = digit.index_select(0, order);
    Tensor by = at::empty({n}, at_.options()), tmp = at::empty({2 * n + kBins + 1 + 2 * maxt + 1}, at_.options()),
           ws = at::empty({bytes}, at_.options().dtype(at::kByte));
    int32_t* p = tmp.data_ptr<int32_t>();
    // tiles as long as all the rows: one per bin at most
    ok(qmoe_route(digit.data_ptr<int32_t>(), n, kBins, (int32_t)n, by.data_ptr<int32_t>(), p, p + n, p + 2 * n,
                  p + 2 * n + kBins + 1, p + 2 * n + kBins + 1 + maxt, p + 2 * n + kBins + 1 + 2 * maxt, maxt,
                  ws.data_ptr(), bytes, stream(at_)),
       "qmoe_route");
    order = order.defined() ? order.index_select(0, by) : by;
  }
  return {order, at::searchsorted(at_.index_select(0, order), at::arange(n_x + 1, at_.options()), /*out_int32=*/true)};
}

struct Product : torch::autograd::Function<Product> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Weights& g, const Rows& r, bool transpose) {
    ctx->save_for_backward({g.w, g.s, r.x_rows, r.experts, r.offsets, r.tile_row, r.tile_exp, r.ntiles, r.inv});
    ctx->saved_data["sizes"] = std::vector<int64_t>{x.size(0), g.E, g.N, g.K, r.n, r.div, r.maxt, transpose};
    return product_run(x, g, r, transpose, at::kBFloat16);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto v = ctx->get_saved_variables();
    const auto z = ctx->saved_data["sizes"].toIntVector();
    const Weights g{v[0], v[1], z[1], z[2], z[3]};
    const int64_t n_x = z[0], div = z[5];
    Rows own;  // row r of the result's gradient for row r
    own.n = z[4], own.maxt = z[6], own.experts = v[3];
    own.offsets = v[4], own.tile_row = v[5], own.tile_exp = v[6], own.ntiles = v[7];
    const Tensor dy = ready(grads[0]);
    const c10::hip::HIPGuard guard(dy.get_device());
    Tensor dx;
    if (!v[2].defined() && div == 1) {
      dx = product_run(dy, g, own, !z[7], at::kBFloat16);
    } else {  // several rows share an activation row: their gradients are added in fp32, rounded once
      const Tensor dr = product_run(dy, g, own, !z[7], at::kFloat);
      if (!v[2].defined() || v[8].defined()) {
        dx = sum_run(dr, v[8], {}, {}, n_x, div, at::kBFloat16);
      } else {
        const auto [order, first] = rows_of(v[2], n_x);
        dx = sum_run(dr, order, {}, first, n_x, 0, at::kBFloat16);
      }
    }
    return first_order({dx, Tensor(), Tensor(), Tensor()}, grads);
  }
};

Tensor product(const Tensor& x, const Weights& g, const Rows& r, bool transpose) {
  return records(x) ? Product::apply(x, g, r, transpose) : product_run(x, g, r, transpose, at::kBFloat16);
}

Tensor qq_run(const Tensor& x, const Weights& g, const Rows& r) {
  Tensor out = at::empty({r.n, g.N}, x.options().requires_grad(false));
  if (out.numel() == 0) return out;
  if (g.K == 0) return out.zero_();
  Tensor xq, xs, lines;
  if (r.n > kFewRows && r.n >= kLineRows * g.E) {
    const int64_t words = (g.E * g.N + x.size(0)) * ((g.K + 127) / 128);
    xq = at::empty({x.size(0), g.K / 8}, x.options().dtype(at::kInt).requires_grad(false));
    lines = at::empty({words}, xq.options());
    const int rc = qmoe_mxfp4_quantize_lines(ptr<uint16_t>(x), x.size(0), g.K, static_cast<uint32_t*>(xq.data_ptr()),
                                             ptr<uint8_t>(g.s), (int32_t)g.E, g.N,
                                             static_cast<uint32_t*>(lines.data_ptr()), words, stream(x));
    if (rc == QMOE_ERR_UNSUPPORTED) lines = xq = Tensor();  // more than one launch holds: the scales stay in their rows
    else ok(rc, "qmoe_mxfp4_quantize_lines");
  }
  if (!lines.defined()) std::tie(xq, xs) = quantize_run(x);
  const Tensor rows = gemm_rows(r, x);
  ok(qmoe_mxfp4_gather_qqmm(ptr<uint32_t>(xq), ptr<uint8_t>(xs), x.size(0), ptr<int32_t>(rows), r.n, ptr<uint32_t>(g.w),
                            ptr<uint8_t>(g.s), (int32_t)g.E, g.N, g.K, ptr<int32_t>(r.offsets), ptr<int32_t>(r.tile_row),
                            ptr<int32_t>(r.tile_exp), ptr<int32_t>(r.ntiles), r.maxt, ptr<uint32_t>(lines),
                            out.data_ptr(), stream(x)),
     "qmoe_mxfp4_gather_qqmm");
  return out;
}

bool weights(py::handle w_, py::handle s_, const Tensor& x, int64_t dims, Weights* g) {
  if (!get(w_, &g->w) || !get(s_, &g->s) || !words(g->w) || !bytes(g->s) || g->w.dim() != dims || g->s.dim() != dims ||
      g->w.device() != x.device() || g->s.device() != x.device())
    return false;
  g->E = dims == 3 ? g->w.size(0) : 1;
  g->N = g->w.size(-2);
  g->K = g->w.size(-1) * 8;
  return g->K % 32 == 0 && g->s.size(-1) == g->K / 32 && g->s.size(-2) == g->N && (dims == 2 || g->s.size(0) == g->E);
}
Tensor as_rows(const Tensor& x) {
  if (x.dim() == 2) return x;
  int64_t n = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) n *= x.size(d);
  return x.reshape({n, x.size(-1)});
}

// x [.., C] times the weights of one matrix; qq: x quantised as well.
py::object matmul(py::handle x_, py::handle w_, py::handle s_, bool transpose, bool qq, bool must) {
  refuse_recorders();
  Tensor x;
  Weights g;
  if (!get(x_, &x) || !plain(x, at::kBFloat16) || x.dim() < 1 || !weights(w_, s_, x, 2, &g) ||
      x.size(-1) != (transpose ? g.K : g.N) || (qq && records(x)))
    return none(must);
  const c10::hip::HIPGuard guard(x.get_device());
  const Tensor x2 = as_rows(x);
  Rows r;
  r.n = x2.size(0);
  Tensor y = qq ? qq_run(x2, g, r) : product(x2, g, r, transpose);
  if (x.dim() != 2) {
    auto sizes = x.sizes().vec();
    sizes.back() = y.size(1);
    y = y.reshape(sizes);
  }
  return give(y);
}

bool table(const Tensor& experts, int64_t E, Rows* r) {
  const int64_t tr = qmoe_gemm_tile_rows(), n = r->n;
  if (E <= 0 || E > INT32_MAX || n > INT32_MAX) return false;
  r->maxt = (n + tr - 1) / tr + E;
  // one allocation, each table from a 256-byte boundary
  const auto pad = [](int64_t m) { return (m + 63) / 64 * 64; };
  const int64_t a = pad(E + 1), b = pad(r->maxt);
  const Tensor all = at::empty({a + 2 * b + 1}, experts.options());
  r->offsets = all.narrow(0, 0, E + 1);
  r->tile_row = all.narrow(0, a, r->maxt);
  r->tile_exp = all.narrow(0, a + b, r->maxt);
  r->ntiles = all.narrow(0, a + 2 * b, 1);
  ok(qmoe_build_tiles_clamped(ptr<int32_t>(experts), n, (int32_t)E, (int32_t)tr, r->offsets.data_ptr<int32_t>(),
                      r->tile_row.data_ptr<int32_t>(), r->tile_exp.data_ptr<int32_t>(), r->ntiles.data_ptr<int32_t>(),
                      r->maxt, stream(experts)),
     "qmoe_build_tiles_clamped");
  return true;
}

// The gather calls whose rows need no arranging: one row per batch index; the
// batch that of rhs, x's own or x's with its last dimensions broadcast, or
// lhs's; and either sorted or fewer rows than are worth sorting.
py::object gather(py::handle x_, py::handle w_, py::handle s_, py::handle lhs_, py::handle rhs_, bool transpose,
                  bool is_sorted, bool qq) {
  refuse_recorders();
  Tensor x, lhs, rhs;
  Weights g;
  if (!get(x_, &x) || !plain(x, at::kBFloat16) || x.dim() < 2 || x.size(-2) != 1 || !get(rhs_, &rhs) ||
      !plain(rhs, at::kInt) || rhs.device() != x.device() || !weights(w_, s_, x, 3, &g) ||
      x.size(-1) != (transpose ? g.K : g.N) || (qq && records(x)))
    return py::none();
  Rows r;
  r.n = rhs.numel();
  const int64_t n_x = x.numel() && x.size(-1) ? x.numel() / x.size(-1) : 0;
  if (r.n == 0 || n_x == 0 || g.E == 0) return py::none();
  if (lhs_.is_none()) {
    const int64_t bd = x.dim() - 2;
    if (bd != rhs.dim()) return py::none();
    int64_t d = 0;
    while (d < bd && x.size(d) == rhs.size(d)) ++d;
    for (int64_t i = d; i < bd; ++i) {
      if (x.size(i) != 1) return py::none();
      r.div *= rhs.size(i);
    }
  } else {
    if (!get(lhs_, &lhs) || !plain(lhs, at::kInt) || lhs.sizes() != rhs.sizes() || lhs.device() != x.device())
      return py::none();
    r.x_rows = lhs.reshape({-1});
  }
  if (!is_sorted && (qq || r.n >= kSortedMinRows)) return py::none();
  const c10::hip::HIPGuard guard(x.get_device());
  r.experts = rhs.reshape({-1});
  if ((qq || r.n >= kSortedMinRows) && !table(r.experts, g.E, &r)) return py::none();
  const Tensor x2 = as_rows(x);
  Tensor y = qq ? qq_run(x2, g, r) : product(x2, g, r, transpose);
  auto sizes = rhs.sizes().vec();
  sizes.push_back(1);
  sizes.push_back(y.size(1));
  return give(y.reshape(sizes));
}

// int64 ids as int32 ones clamped into [0, n).
Tensor narrow(const Tensor& ids, int64_t n) {
  TORCH_CHECK(ids.scalar_type() == at::kLong && ids.is_cuda() && ids.is_contiguous() && n >= 0 && n <= INT32_MAX,
              "the arguments are not what the kernels read");
  const c10::hip::HIPGuard guard(ids.get_device());
  Tensor out = at::empty(ids.sizes(), ids.options().dtype(at::kInt));
  ok(qmoe_narrow_ids(ptr<int64_t>(ids), ids.numel(), (int32_t)n, out.data_ptr<int32_t>(), stream(ids)), "qmoe_narrow_ids");
  return out;
}

// Rows already arranged by the wrapper: x [rows, C], x_rows / experts int32 or None, a tile table or None, and
// where the rows of activation row t are known, their places inv[t div .. (t + 1) div).
py::object rows_product(const Tensor& x, const Tensor& w, const Tensor& s, const std::optional<Tensor>& x_rows,
                        int64_t div, const std::optional<Tensor>& experts,
                        const std::optional<std::tuple<Tensor, Tensor, Tensor, Tensor, int64_t>>& tiles, int64_t n,
                        bool transpose, bool qq, const std::optional<Tensor>& inv) {
  refuse_recorders();
  if (records(x) && qq)
    throw Failure("the products of quantised activations have no gradient: detach x, or use quantized_matmul / gather_qmm");
  Weights g{w, s, w.size(0), w.size(1), w.size(2) * 8};
  Rows r;
  r.n = n;
  r.div = div;
  if (x_rows) r.x_rows = *x_rows;
  if (experts) r.experts = *experts;
  if (inv) r.inv = *inv;
  if (tiles) std::tie(r.offsets, r.tile_row, r.tile_exp, r.ntiles, r.maxt) = *tiles;
  TORCH_CHECK(plain(x, at::kBFloat16) && words(w) && bytes(s), "the arguments are not what the kernels read");
  for (const Tensor* t : {&r.x_rows, &r.experts, &r.offsets, &r.tile_row, &r.tile_exp, &r.ntiles, &r.inv})
    TORCH_CHECK(!t->defined() || (t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == x.device()),
                "the arguments are not what the kernels read");
  TORCH_CHECK((!x_rows || r.x_rows.numel() == n) && (!experts || r.experts.numel() == n) &&
                  (!inv || (r.inv.numel() == n && x.size(0) * div == n)), "the rows disagree");
  const c10::hip::HIPGuard guard(x.get_device());
  return give(qq ? qq_run(x, g, r) : product(x, g, r, transpose));
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Failure& f) {
      const py::module_ lib = py::module_::import("titan_amd._lib");
      const char* name = f.code == QMOE_ERR_UNSUPPORTED ? "QmoeUnsupported" : "QmoeError";
      const py::object type = lib.attr(name);
      PyErr_SetObject(type.ptr(), type(f.code, f.what()).ptr());
    }
  });
  m.def("quantize", &quantize);
  m.def("dequantize", &dequantize);
  m.def("sort_tokens", &sort_tokens);
  m.def("unsort_tokens", &unsort_tokens);
  m.def("matmul", &matmul);
  m.def("gather", &gather);
  m.def("narrow", &narrow);
  m.def("rows_product", &rows_product, py::arg("x"), py::arg("w"), py::arg("s"), py::arg("x_rows"), py::arg("div"),
        py::arg("experts"), py::arg("tiles"), py::arg("n"), py::arg("transpose"), py::arg("qq"),
        py::arg("inv") = py::none());
}

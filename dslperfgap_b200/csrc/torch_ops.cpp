// torch_ops.cpp — the `_dslpg_torch` extension: each op's common case
// (CUDA tensors of a supported dtype, the reference's usual arguments) done
// in C++: the checks, the output allocation through torch's caching
// allocator, and one call of the C-ABI entry point on the tensor's current
// stream. Under the reference's timing protocol (one synchronised call at a
// time) the host's work per call is part of every small-shape latency; here
// it is a pybind11 call plus at::empty instead of a Python wrapper.
//
// Every function takes the Python wrapper's arguments as they came and
// returns None for anything outside its case (a CPU tensor, another dtype, a
// list of dims, an eps the reference rejects, an empty tensor, ...); the
// Python wrapper then runs its own checks and raises exactly as before.
// Launch failures raise RuntimeError with dslpg_error_string's text.
#include <torch/extension.h>
#include <torch/csrc/Dtype.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>

#include "dslpg_b200.h"

namespace py = pybind11;

namespace {

int float_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DSLPG_F32;
    case at::kHalf: return DSLPG_F16;
    case at::kBFloat16: return DSLPG_BF16;
    default: return -1;
  }
}

// The tensor behind `h` if it is a CUDA tensor of a float dtype (on `dev`
// when dev >= 0), else nullopt.
std::optional<at::Tensor> cuda_float(const py::handle& h, int dev = -1) {
  if (!THPVariable_Check(h.ptr())) return std::nullopt;
  const at::Tensor& t = THPVariable_Unpack(h.ptr());
  if (!t.is_cuda() || float_code(t.scalar_type()) < 0) return std::nullopt;
  if (dev >= 0 && t.get_device() != dev) return std::nullopt;
  return t;
}

bool is_int(const py::handle& h) { return PyLong_Check(h.ptr()) && !PyBool_Check(h.ptr()); }

// Runs `call(stream)` on the tensor's device and current stream.
template <class F>
void launch(const at::Tensor& t, const char* what, F call) {
  const int dev = t.get_device();
  std::optional<c10::cuda::CUDAGuard> guard;
  if (c10::cuda::current_device() != dev) guard.emplace(dev);
  const int rc = call(c10::cuda::getCurrentCUDAStream(dev).stream());
  if (rc != 0) throw std::runtime_error(std::string(what) + " failed (" + std::to_string(rc) + "): " +
                                        dslpg_error_string(rc));
}

// [M, N, K] of a reduction over dim `d` (already in range) of `t`.
void mnk(const at::Tensor& t, int64_t d, int64_t& m, int64_t& n, int64_t& k) {
  m = 1;
  k = 1;
  for (int64_t i = 0; i < d; ++i) m *= t.size(i);
  n = t.size(d);
  for (int64_t i = d + 1; i < t.dim(); ++i) k *= t.size(i);
}

// dim as an index in [0, nd), or -1 when it is not an int in range.
int64_t norm_dim(const py::handle& h, int64_t nd) {
  if (!is_int(h) || nd < 1) return -1;
  const int64_t d = h.cast<int64_t>();
  if (d < -nd || d >= nd) return -1;
  return d < 0 ? d + nd : d;
}

std::vector<int64_t> reduced_shape(const at::Tensor& t, int64_t d, bool keepdim) {
  std::vector<int64_t> s;
  for (int64_t i = 0; i < t.dim(); ++i) {
    if (i != d) s.push_back(t.size(i));
    else if (keepdim) s.push_back(1);
  }
  return s;
}

py::object layer_norm(py::handle x_, py::handle w_, py::handle b_, py::handle eps_) {
  if (!PyFloat_Check(eps_.ptr()) || eps_.cast<double>() != 1e-5) return py::none();
  auto x = cuda_float(x_);
  if (!x) return py::none();
  auto w = cuda_float(w_, x->get_device());
  if (!w || w->dim() != 1 || x->dim() < 1 || x->size(-1) != w->size(0) || x->numel() == 0) return py::none();
  std::optional<at::Tensor> b;
  if (!b_.is_none()) {
    b = cuda_float(b_, x->get_device());
    if (!b || b->scalar_type() != w->scalar_type() || b->dim() != 1 || b->size(0) != w->size(0)) return py::none();
  }
  const at::Tensor xc = x->contiguous(), wc = w->contiguous();
  const at::Tensor bc = b ? b->contiguous() : at::Tensor();
  at::Tensor y = at::empty_like(xc);
  const int64_t n = wc.size(0);
  launch(xc, "dslpg_layer_norm_fwd", [&](cudaStream_t s) {
    return dslpg_layer_norm_fwd(xc.data_ptr(), wc.data_ptr(), b ? bc.data_ptr() : nullptr, y.data_ptr(),
                                xc.numel() / n, n, float_code(xc.scalar_type()), float_code(wc.scalar_type()), 1e-5f,
                                s);
  });
  return py::cast(y);
}

py::object rms_norm(py::handle x_, py::handle shape_, py::handle w_, py::handle eps_) {
  auto x = cuda_float(x_);
  if (!x || x->dim() < 1 || x->numel() == 0 || !(PyFloat_Check(eps_.ptr()) || is_int(eps_))) return py::none();
  const int64_t n = x->size(-1);
  if (is_int(shape_)) {
    if (shape_.cast<int64_t>() != n) return py::none();
  } else if (PyTuple_Check(shape_.ptr()) || PyList_Check(shape_.ptr())) {
    py::sequence seq = py::reinterpret_borrow<py::sequence>(shape_);
    if (seq.size() != 1 || !is_int(seq[0]) || seq[0].cast<int64_t>() != n) return py::none();
  } else {
    return py::none();
  }
  auto w = cuda_float(w_, x->get_device());
  if (!w || w->dim() != 1 || w->size(0) != n) return py::none();
  const double eps = eps_.cast<double>();
  const at::Tensor xc = x->contiguous(), wc = w->contiguous();
  at::Tensor y = at::empty_like(xc);
  launch(xc, "dslpg_rms_norm_fwd", [&](cudaStream_t s) {
    return dslpg_rms_norm_fwd(xc.data_ptr(), wc.data_ptr(), y.data_ptr(), xc.numel() / n, n,
                              float_code(xc.scalar_type()), float_code(wc.scalar_type()), static_cast<float>(eps), s);
  });
  return py::cast(y);
}

py::object softmax(py::handle x_) {
  auto x = cuda_float(x_);
  if (!x || x->dim() < 1 || x->numel() == 0) return py::none();
  const at::Tensor xc = x->contiguous();
  at::Tensor y = at::empty_like(xc);
  const int64_t n = xc.size(-1);
  launch(xc, "dslpg_softmax_fwd", [&](cudaStream_t s) {
    return dslpg_softmax_fwd(xc.data_ptr(), y.data_ptr(), xc.numel() / n, n, float_code(xc.scalar_type()), s);
  });
  return py::cast(y);
}

py::object log_softmax(py::handle x_, py::handle dim_, py::handle dtype_) {
  if (!dtype_.is_none()) return py::none();
  auto x = cuda_float(x_);
  if (!x || x->numel() == 0) return py::none();
  const int64_t d = norm_dim(dim_, x->dim());
  if (d < 0) return py::none();
  int64_t m, n, k;
  const at::Tensor xc = x->contiguous();
  mnk(xc, d, m, n, k);
  at::Tensor y = at::empty_like(xc);
  const int code = float_code(xc.scalar_type());
  launch(xc, "dslpg_log_softmax_fwd", [&](cudaStream_t s) {
    return dslpg_log_softmax_fwd(xc.data_ptr(), y.data_ptr(), m, n, k, code, code, s);
  });
  return py::cast(y);
}

py::object logsumexp(py::handle x_) {
  auto x = cuda_float(x_);
  if (!x || x->dim() < 1 || x->numel() == 0) return py::none();
  const at::Tensor xc = x->contiguous();
  const int64_t n = xc.size(-1);
  at::Tensor y = at::empty(reduced_shape(xc, xc.dim() - 1, false), xc.options());
  launch(xc, "dslpg_logsumexp_fwd", [&](cudaStream_t s) {
    return dslpg_logsumexp_fwd(xc.data_ptr(), y.data_ptr(), xc.numel() / n, n, float_code(xc.scalar_type()), s);
  });
  return py::cast(y);
}

// The reductions over one int dim (the reference's benchmark form).
bool red_args(py::handle x_, py::handle dim_, at::Tensor& xc, int64_t& d, int64_t& m, int64_t& n, int64_t& k) {
  auto x = cuda_float(x_);
  if (!x || x->numel() == 0) return false;
  d = norm_dim(dim_, x->dim());
  if (d < 0) return false;
  xc = x->contiguous();
  mnk(xc, d, m, n, k);
  return true;
}

py::object mean_reduction(py::handle x_, py::handle dim_, py::handle keepdim_, py::handle dtype_) {
  at::Tensor xc;
  int64_t d, m, n, k;
  if (!PyBool_Check(keepdim_.ptr()) || !red_args(x_, dim_, xc, d, m, n, k)) return py::none();
  at::ScalarType out_t = xc.scalar_type();
  if (!dtype_.is_none()) {
    if (!THPDtype_Check(dtype_.ptr())) return py::none();
    out_t = reinterpret_cast<THPDtype*>(dtype_.ptr())->scalar_type;
    if (float_code(out_t) < 0) return py::none();
  }
  at::Tensor y = at::empty(reduced_shape(xc, d, keepdim_.ptr() == Py_True), xc.options().dtype(out_t));
  launch(xc, "dslpg_mean_reduction", [&](cudaStream_t s) {
    return dslpg_mean_reduction(xc.data_ptr(), y.data_ptr(), m, n, k, float_code(xc.scalar_type()),
                                float_code(out_t), s);
  });
  return py::cast(y);
}

py::object max_reduction(py::handle x_, py::handle dim_, py::handle keepdim_) {
  at::Tensor xc;
  int64_t d, m, n, k;
  if (!PyBool_Check(keepdim_.ptr()) || !red_args(x_, dim_, xc, d, m, n, k)) return py::none();
  const auto shape = reduced_shape(xc, d, keepdim_.ptr() == Py_True);
  at::Tensor v = at::empty(shape, xc.options());
  at::Tensor i = at::empty(shape, xc.options().dtype(at::kLong));
  launch(xc, "dslpg_max_reduction", [&](cudaStream_t s) {
    return dslpg_max_reduction(xc.data_ptr(), v.data_ptr(), i.data_ptr<int64_t>(), m, n, k,
                               float_code(xc.scalar_type()), s);
  });
  return py::make_tuple(v, i);
}

py::object argmax(py::handle x_, py::handle dim_, py::handle keepdim_) {
  at::Tensor xc;
  int64_t d, m, n, k;
  if (!PyBool_Check(keepdim_.ptr()) || !red_args(x_, dim_, xc, d, m, n, k)) return py::none();
  at::Tensor i = at::empty(reduced_shape(xc, d, keepdim_.ptr() == Py_True), xc.options().dtype(at::kLong));
  launch(xc, "dslpg_argmax", [&](cudaStream_t s) {
    return dslpg_argmax(xc.data_ptr(), i.data_ptr<int64_t>(), m, n, k, float_code(xc.scalar_type()), s);
  });
  return py::cast(i);
}

bool is_number(const py::handle& h) { return PyFloat_Check(h.ptr()) || is_int(h); }

py::object cross_entropy_fwd(py::handle logits_, py::handle labels_, py::handle smoothing, py::handle logit_scale,
                             py::handle lse_square_scale, py::handle ignored_index, py::handle total_classes,
                             py::handle class_start_idx, py::handle block_size, py::handle has_smoothing,
                             py::handle split) {
  auto x = cuda_float(logits_);
  if (!x || x->dim() != 2 || x->size(0) == 0 || x->size(1) == 0 || !x->is_contiguous()) return py::none();
  if (!THPVariable_Check(labels_.ptr())) return py::none();
  const at::Tensor& lab = THPVariable_Unpack(labels_.ptr());
  const int lcode = lab.scalar_type() == at::kLong ? DSLPG_I64 : (lab.scalar_type() == at::kInt ? DSLPG_I32 : -1);
  if (lcode < 0 || !lab.is_cuda() || lab.get_device() != x->get_device() || lab.dim() != 1 ||
      lab.size(0) != x->size(0) || !lab.is_contiguous())
    return py::none();
  if (!is_number(smoothing) || !is_number(logit_scale) || !is_number(lse_square_scale) || !is_int(ignored_index) ||
      !is_number(total_classes) || !is_int(class_start_idx) || !is_int(block_size) || !PyBool_Check(has_smoothing.ptr()) ||
      !PyBool_Check(split.ptr()))
    return py::none();
  const int64_t bs = block_size.cast<int64_t>();
  if (bs <= 0) return py::none();
  const int64_t r = x->size(0), c = x->size(1);
  const auto opts = x->options().dtype(at::kFloat);
  at::Tensor loss = at::empty({r, c}, opts), lse = at::empty({r, c}, opts), z = at::empty({r, c}, opts);
  launch(*x, "dslpg_cross_entropy_fwd", [&](cudaStream_t s) {
    return dslpg_cross_entropy_fwd(x->data_ptr(), lab.data_ptr(), loss.data_ptr<float>(), lse.data_ptr<float>(),
                                   z.data_ptr<float>(), r, c, x->stride(0), float_code(x->scalar_type()), lcode,
                                   static_cast<float>(smoothing.cast<double>()),
                                   static_cast<float>(logit_scale.cast<double>()),
                                   static_cast<float>(lse_square_scale.cast<double>()), ignored_index.cast<int64_t>(),
                                   static_cast<float>(total_classes.cast<double>()), class_start_idx.cast<int64_t>(),
                                   bs, has_smoothing.ptr() == Py_True ? 1 : 0, split.ptr() == Py_True ? 1 : 0, s);
  });
  return py::make_tuple(loss, lse, z);
}

// A CUDA tensor of one of two dtypes on `dev`, else nullopt.
std::optional<at::Tensor> cuda_of(const py::handle& h, int dev, at::ScalarType a, at::ScalarType b) {
  if (!THPVariable_Check(h.ptr())) return std::nullopt;
  const at::Tensor& t = THPVariable_Unpack(h.ptr());
  if (!t.is_cuda() || t.get_device() != dev || (t.scalar_type() != a && t.scalar_type() != b)) return std::nullopt;
  return t;
}

// Checked q and k with their layout (rope, qk_norm_rope).
struct HeadRows {
  at::Tensor q, k, pos, freq;
  dslpg_heads h{};

  static void strides(const at::Tensor& t, int64_t* out) {
    const bool batched = t.dim() == 4;
    out[0] = batched ? t.stride(0) : 0;
    out[1] = t.stride(batched ? 1 : 0);
    out[2] = t.stride(batched ? 2 : 1);
  }

  bool take(py::handle q_, py::handle k_, py::handle pos_, py::handle freq_, py::handle sections, py::handle inter) {
    auto tq = cuda_float(q_);
    if (!tq || (tq->dim() != 3 && tq->dim() != 4) || !PyBool_Check(inter.ptr())) return false;
    const int dev = tq->get_device();
    auto tk = cuda_float(k_, dev);
    auto tp = cuda_of(pos_, dev, at::kLong, at::kInt);
    auto tf = cuda_of(freq_, dev, at::kFloat, at::kFloat);
    if (!tk || !tp || !tf || tk->scalar_type() != tq->scalar_type() || tk->dim() != tq->dim()) return false;
    const int64_t nd = tq->dim(), lead = nd - 2, d = tq->size(-1);
    for (int64_t i = 0; i < lead; ++i)
      if (tk->size(i) != tq->size(i)) return false;
    if (tq->numel() == 0 || tk->numel() == 0 || tk->size(-1) != d || d > 1024 || tq->stride(-1) != 1 ||
        tk->stride(-1) != 1 || tf->dim() != 1 || tf->stride(0) != 1 || tf->size(0) < 1 || 2 * tf->size(0) > d ||
        (tq->numel() + tk->numel()) / d > (1ll << 30))
      return false;
    h.axes = 1;
    h.sections[0] = tf->size(0);
    if (!sections.is_none()) {
      if (!PyTuple_Check(sections.ptr()) && !PyList_Check(sections.ptr())) return false;
      py::sequence seq = py::reinterpret_borrow<py::sequence>(sections);
      if (seq.size() < 1 || seq.size() > 4) return false;
      int64_t left = tf->size(0);
      for (size_t i = 0; i < seq.size(); ++i) {
        if (!is_int(seq[i])) return false;
        h.sections[i] = seq[i].cast<int64_t>();
        if (h.sections[i] < 0 || h.sections[i] > left) return false;
        left -= h.sections[i];
      }
      if (left != 0) return false;
      h.axes = static_cast<int32_t>(seq.size());
    }
    // positions: [axes,] tokens, or what broadcasts to that from the right
    const int64_t want = lead + (sections.is_none() ? 0 : 1);
    if (tp->dim() > want) return false;
    int64_t ps[3] = {0, 0, 0};  // axis, batch, seq
    for (int64_t i = 1; i <= tp->dim(); ++i) {
      const int64_t extent = i <= lead ? tq->size(lead - i) : h.axes;
      const int64_t size = tp->size(tp->dim() - i);
      if (size != extent && size != 1) return false;
      const int slot = i > lead ? 0 : (i == 1 ? 2 : 1);
      ps[slot] = size == 1 ? 0 : tp->stride(tp->dim() - i);
    }
    for (int i = 0; i < 3; ++i) h.position_strides[i] = ps[i];
    h.batch = lead == 2 ? tq->size(0) : 1;
    h.seq = tq->size(lead - 1);
    h.q_heads = tq->size(lead);
    h.k_heads = tk->size(lead);
    h.head_dim = d;
    h.rotary_dim = 2 * tf->size(0);
    strides(*tq, h.q_strides);
    strides(*tk, h.k_strides);
    h.interleaved = inter.ptr() == Py_True ? 1 : 0;
    h.dtype = float_code(tq->scalar_type());
    h.positions_dtype = tp->scalar_type() == at::kLong ? DSLPG_I64 : DSLPG_I32;
    q = *tq;
    k = *tk;
    pos = *tp;
    freq = *tf;
    return true;
  }

  // The norm weights: [head_dim] vectors of one float dtype.
  bool weights(py::handle qw_, py::handle kw_, at::Tensor& qw, at::Tensor& kw) {
    auto a = cuda_float(qw_, q.get_device()), b = cuda_float(kw_, q.get_device());
    if (!a || !b || a->scalar_type() != b->scalar_type() || a->dim() != 1 || b->dim() != 1 ||
        a->size(0) != h.head_dim || b->size(0) != h.head_dim || !a->is_contiguous() || !b->is_contiguous())
      return false;
    h.weight_dtype = float_code(a->scalar_type());
    qw = *a;
    kw = *b;
    return true;
  }

  at::Tensor dense(const at::Tensor& t) const { return at::empty(t.sizes(), t.options()); }
};

py::object rotate(bool bwd, py::handle q, py::handle k, py::handle pos, py::handle freq, py::handle sections,
                  py::handle inter) {
  HeadRows r;
  if (!r.take(q, k, pos, freq, sections, inter)) return py::none();
  at::Tensor yq = r.dense(r.q), yk = r.dense(r.k);
  launch(r.q, bwd ? "dslpg_rope_bwd" : "dslpg_rope_fwd", [&](cudaStream_t s) {
    return (bwd ? dslpg_rope_bwd : dslpg_rope_fwd)(r.q.data_ptr(), r.k.data_ptr(), r.pos.data_ptr(),
                                                   r.freq.data_ptr<float>(), yq.data_ptr(), yk.data_ptr(), &r.h, s);
  });
  return py::make_tuple(yq, yk);
}

py::object rope(py::handle q, py::handle k, py::handle pos, py::handle freq, py::handle sections, py::handle inter) {
  return rotate(false, q, k, pos, freq, sections, inter);
}

py::object rope_bwd(py::handle q, py::handle k, py::handle pos, py::handle freq, py::handle sections,
                    py::handle inter) {
  return rotate(true, q, k, pos, freq, sections, inter);
}

py::object qk_norm_rope(py::handle q, py::handle k, py::handle qw_, py::handle kw_, py::handle pos, py::handle freq,
                        py::handle eps, py::handle sections, py::handle inter) {
  HeadRows r;
  at::Tensor qw, kw;
  if (!(PyFloat_Check(eps.ptr()) || is_int(eps)) || !r.take(q, k, pos, freq, sections, inter) ||
      !r.weights(qw_, kw_, qw, kw))
    return py::none();
  at::Tensor yq = r.dense(r.q), yk = r.dense(r.k);
  launch(r.q, "dslpg_qk_norm_rope_fwd", [&](cudaStream_t s) {
    return dslpg_qk_norm_rope_fwd(r.q.data_ptr(), r.k.data_ptr(), qw.data_ptr(), kw.data_ptr(), r.pos.data_ptr(),
                                  r.freq.data_ptr<float>(), yq.data_ptr(), yk.data_ptr(), &r.h,
                                  static_cast<float>(eps.cast<double>()), s);
  });
  return py::make_tuple(yq, yk);
}

py::object qk_norm_rope_bwd(py::handle dq_, py::handle dk_, py::handle q, py::handle k, py::handle qw_,
                            py::handle kw_, py::handle pos, py::handle freq, py::handle eps, py::handle sections,
                            py::handle inter) {
  HeadRows r;
  at::Tensor qw, kw;
  if (!(PyFloat_Check(eps.ptr()) || is_int(eps)) || !r.take(q, k, pos, freq, sections, inter) ||
      !r.weights(qw_, kw_, qw, kw))
    return py::none();
  auto gq = cuda_float(dq_, r.q.get_device()), gk = cuda_float(dk_, r.q.get_device());
  if (!gq || !gk || gq->scalar_type() != r.q.scalar_type() || gk->scalar_type() != r.q.scalar_type() ||
      gq->sizes() != r.q.sizes() || gk->sizes() != r.k.sizes() || gq->stride(-1) != 1 || gk->stride(-1) != 1)
    return py::none();
  HeadRows::strides(*gq, r.h.dq_strides);
  HeadRows::strides(*gk, r.h.dk_strides);
  at::Tensor dq = r.dense(r.q), dk = r.dense(r.k);
  const auto f32 = r.q.options().dtype(at::kFloat);
  at::Tensor dqw = at::empty({r.h.head_dim}, f32), dkw = at::empty({r.h.head_dim}, f32);
  int64_t need = 0;
  if (dslpg_qk_norm_rope_bwd_workspace_bytes(r.h.head_dim, &need) != 0) return py::none();
  at::Tensor ws = at::empty({need}, r.q.options().dtype(at::kByte));
  launch(r.q, "dslpg_qk_norm_rope_bwd", [&](cudaStream_t s) {
    return dslpg_qk_norm_rope_bwd(gq->data_ptr(), gk->data_ptr(), r.q.data_ptr(), r.k.data_ptr(), qw.data_ptr(),
                                  kw.data_ptr(), r.pos.data_ptr(), r.freq.data_ptr<float>(), dq.data_ptr(),
                                  dk.data_ptr(), dqw.data_ptr<float>(), dkw.data_ptr<float>(), &r.h,
                                  static_cast<float>(eps.cast<double>()), ws.data_ptr(), need, s);
  });
  return py::make_tuple(dq, dk, dqw, dkw);
}

// A float32 CUDA vector of n values on `dev`.
std::optional<at::Tensor> f32_vector(const py::handle& h, int dev, int64_t n, bool dense = false) {
  auto t = cuda_of(h, dev, at::kFloat, at::kFloat);
  if (!t || t->dim() != 1 || t->size(0) != n || (dense && !t->is_contiguous())) return std::nullopt;
  return t;
}

// Logits and labels of the losses (policy_loss, preference_loss).
struct LossRows {
  at::Tensor logits, labels;
  dslpg_logit_rows r{};

  bool take(py::handle x_, py::handle labels_, py::handle scale, py::handle ignored) {
    auto x = cuda_float(x_);
    if (!x || x->dim() != 2 || x->size(0) == 0 || x->size(1) < 1 || x->size(1) > (1ll << 30) || x->stride(1) != 1 ||
        (x->size(0) > 1 && x->stride(0) < x->size(1)) || !is_number(scale) || !is_int(ignored))
      return false;
    auto lab = cuda_of(labels_, x->get_device(), at::kLong, at::kInt);
    if (!lab || lab->dim() != 1 || lab->size(0) != x->size(0) || !lab->is_contiguous()) return false;
    logits = *x;
    labels = *lab;
    r.logits = logits.data_ptr();
    r.labels = labels.data_ptr();
    r.n_rows = x->size(0);
    r.n_cols = x->size(1);
    r.row_stride = x->size(0) > 1 ? x->stride(0) : x->size(1);
    r.ignored_index = ignored.cast<int64_t>();
    r.logit_scale = scale.cast<double>();
    r.logits_dtype = float_code(x->scalar_type());
    r.labels_dtype = lab->scalar_type() == at::kLong ? DSLPG_I64 : DSLPG_I32;
    const double size = std::fabs(r.logit_scale);
    return size == 0.0 || (size >= 1e-30 && size <= 1e30);
  }
  int dev() const { return logits.get_device(); }
  at::Tensor f32(int64_t n) const { return at::empty({n}, logits.options().dtype(at::kFloat)); }
  at::Tensor grad() const { return at::empty(logits.sizes(), logits.options()); }
};

struct Policy {
  at::Tensor old, adv, ref;
  dslpg_policy_terms t{};

  bool take(const LossRows& r, py::handle old_, py::handle adv_, py::handle ref_, py::handle low, py::handle high,
            py::handle kl) {
    auto o = f32_vector(old_, r.dev(), r.r.n_rows), a = f32_vector(adv_, r.dev(), r.r.n_rows);
    if (!o || !a || !is_number(low) || !is_number(high) || !is_number(kl)) return false;
    if (!ref_.is_none()) {
      auto f = f32_vector(ref_, r.dev(), r.r.n_rows);
      if (!f) return false;
      ref = *f;
      t.ref_logp = ref.data_ptr<float>();
      t.ref_stride = ref.stride(0);
    }
    old = *o;
    adv = *a;
    t.old_logp = old.data_ptr<float>();
    t.advantages = adv.data_ptr<float>();
    t.old_stride = old.stride(0);
    t.advantages_stride = adv.stride(0);
    const double lo = low.cast<double>(), hi = high.cast<double>(), k = kl.cast<double>();
    t.clip_low = static_cast<float>(lo);
    t.clip_high = static_cast<float>(hi);
    t.kl_coef = static_cast<float>(k);
    return lo >= 0 && lo <= 1 && hi >= 0 && t.kl_coef - t.kl_coef == 0.f;
  }
};

py::object policy_loss_fwd(py::handle x, py::handle labels, py::handle old, py::handle adv, py::handle ref,
                           py::handle low, py::handle high, py::handle kl_coef, py::handle scale, py::handle ignored) {
  LossRows r;
  Policy p;
  if (!r.take(x, labels, scale, ignored) || !p.take(r, old, adv, ref, low, high, kl_coef)) return py::none();
  const int64_t n = r.r.n_rows;
  at::Tensor loss = r.f32(n), logp = r.f32(n), lse = r.f32(n), kl = r.f32(n);
  launch(r.logits, "dslpg_policy_loss_fwd", [&](cudaStream_t s) {
    return dslpg_policy_loss_fwd(&r.r, &p.t, loss.data_ptr<float>(), logp.data_ptr<float>(), lse.data_ptr<float>(),
                                 kl.data_ptr<float>(), s);
  });
  return py::make_tuple(loss, logp, lse, kl);
}

py::object policy_loss_bwd(py::handle dloss_, py::handle x, py::handle lse_, py::handle labels, py::handle old,
                           py::handle adv, py::handle ref, py::handle low, py::handle high, py::handle kl_coef,
                           py::handle scale, py::handle ignored) {
  LossRows r;
  Policy p;
  if (!r.take(x, labels, scale, ignored) || !p.take(r, old, adv, ref, low, high, kl_coef)) return py::none();
  auto dloss = f32_vector(dloss_, r.dev(), r.r.n_rows), lse = f32_vector(lse_, r.dev(), r.r.n_rows, true);
  if (!dloss || !lse) return py::none();
  at::Tensor dx = r.grad();
  launch(r.logits, "dslpg_policy_loss_bwd", [&](cudaStream_t s) {
    return dslpg_policy_loss_bwd(&r.r, &p.t, dloss->data_ptr<float>(), dloss->stride(0), lse->data_ptr<float>(),
                                 dx.data_ptr(), r.r.n_cols, s);
  });
  return py::cast(dx);
}

py::object policy_loss_fwd_bwd(py::handle x, py::handle labels, py::handle old, py::handle adv, py::handle dloss_,
                               py::handle ref, py::handle low, py::handle high, py::handle kl_coef, py::handle scale,
                               py::handle ignored) {
  LossRows r;
  Policy p;
  if (!r.take(x, labels, scale, ignored) || !p.take(r, old, adv, ref, low, high, kl_coef)) return py::none();
  const int64_t n = r.r.n_rows;
  auto dloss = f32_vector(dloss_, r.dev(), n);
  if (!dloss) return py::none();
  at::Tensor loss = r.f32(n), logp = r.f32(n), lse = r.f32(n), kl = r.f32(n), dx = r.grad();
  launch(r.logits, "dslpg_policy_loss_fwd_bwd", [&](cudaStream_t s) {
    return dslpg_policy_loss_fwd_bwd(&r.r, &p.t, dloss->data_ptr<float>(), dloss->stride(0), loss.data_ptr<float>(),
                                     logp.data_ptr<float>(), lse.data_ptr<float>(), kl.data_ptr<float>(),
                                     dx.data_ptr(), r.r.n_cols, s);
  });
  return py::make_tuple(loss, logp, lse, kl, dx);
}

struct Pairs {
  at::Tensor starts;
  dslpg_pair_terms t{};

  bool take(const LossRows& r, py::handle starts_, py::handle beta, py::handle smoothing) {
    auto st = cuda_of(starts_, r.dev(), at::kLong, at::kInt);
    if (!st || st->dim() != 1 || st->size(0) < 3 || st->size(0) % 2 == 0 || !st->is_contiguous() ||
        !is_number(beta) || !is_number(smoothing))
      return false;
    starts = *st;
    t.seq_starts = starts.data_ptr();
    t.starts_dtype = starts.scalar_type() == at::kLong ? DSLPG_I64 : DSLPG_I32;
    t.n_pairs = starts.size(0) / 2;
    const double s = smoothing.cast<double>();
    t.beta = static_cast<float>(beta.cast<double>());
    t.smoothing = static_cast<float>(s);
    return s >= 0 && s <= 1 && t.beta - t.beta == 0.f;
  }
};

py::object preference_loss_fwd(py::handle x, py::handle labels, py::handle starts, py::handle ref_, py::handle beta,
                               py::handle smoothing, py::handle scale, py::handle ignored) {
  LossRows r;
  Pairs p;
  if (!r.take(x, labels, scale, ignored) || !p.take(r, starts, beta, smoothing)) return py::none();
  auto ref = f32_vector(ref_, r.dev(), r.r.n_rows);
  if (!ref) return py::none();
  p.t.ref_logp = ref->data_ptr<float>();
  p.t.ref_stride = ref->stride(0);
  at::Tensor loss = r.f32(p.t.n_pairs), ratio = r.f32(2 * p.t.n_pairs), logp = r.f32(r.r.n_rows),
             lse = r.f32(r.r.n_rows);
  launch(r.logits, "dslpg_preference_loss_fwd", [&](cudaStream_t s) {
    return dslpg_preference_loss_fwd(&r.r, &p.t, loss.data_ptr<float>(), ratio.data_ptr<float>(),
                                     logp.data_ptr<float>(), lse.data_ptr<float>(), s);
  });
  return py::make_tuple(loss, ratio, logp, lse);
}

py::object preference_loss_bwd(py::handle dloss_, py::handle x, py::handle lse_, py::handle labels, py::handle starts,
                               py::handle ratio_, py::handle beta, py::handle smoothing, py::handle scale,
                               py::handle ignored) {
  LossRows r;
  Pairs p;
  if (!r.take(x, labels, scale, ignored) || !p.take(r, starts, beta, smoothing)) return py::none();
  auto dloss = f32_vector(dloss_, r.dev(), p.t.n_pairs), lse = f32_vector(lse_, r.dev(), r.r.n_rows, true),
       ratio = f32_vector(ratio_, r.dev(), 2 * p.t.n_pairs, true);
  if (!dloss || !lse || !ratio) return py::none();
  at::Tensor dx = r.grad();
  launch(r.logits, "dslpg_preference_loss_bwd", [&](cudaStream_t s) {
    return dslpg_preference_loss_bwd(&r.r, &p.t, dloss->data_ptr<float>(), dloss->stride(0), lse->data_ptr<float>(),
                                     ratio->data_ptr<float>(), dx.data_ptr(), r.r.n_cols, s);
  });
  return py::cast(dx);
}

}  // namespace

PYBIND11_MODULE(_dslpg_torch, m) {
  m.doc() = "C++ fast path of the dslperfgap_b200 wrappers (None = not handled here)";
  m.def("layer_norm", &layer_norm);
  m.def("rms_norm", &rms_norm);
  m.def("softmax", &softmax);
  m.def("log_softmax", &log_softmax);
  m.def("logsumexp", &logsumexp);
  m.def("mean_reduction", &mean_reduction);
  m.def("max_reduction", &max_reduction);
  m.def("argmax", &argmax);
  m.def("cross_entropy_fwd", &cross_entropy_fwd);
  m.def("policy_loss_fwd", &policy_loss_fwd);
  m.def("policy_loss_bwd", &policy_loss_bwd);
  m.def("policy_loss_fwd_bwd", &policy_loss_fwd_bwd);
  m.def("preference_loss_fwd", &preference_loss_fwd);
  m.def("preference_loss_bwd", &preference_loss_bwd);
  m.def("rope", &rope);
  m.def("rope_bwd", &rope_bwd);
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("qk_norm_rope_bwd", &qk_norm_rope_bwd);
}

// hcg_torch.cpp -- the device-tensor binding of the library as a Python
// extension (host code only): the checks and stride rules of the Python
// wrappers in hc.gfx950, made on the tensors' C++ attributes, and the
// current HIP stream of the device, so that a small call costs about the
// host time of the launch itself.
//
// gemm handles the common case only (three device tensors on the current
// device, fp16 or bf16 operands, a float32 C that can be written in place) and
// returns -1 for anything else, which the Python wrapper then takes through
// its general path; otherwise it returns hcg_gemm_algo's status (the message
// is hcg_last_error's).
//
// The language-model operators handle contiguous device tensors (an 8-bit
// product's operands: any rows that one stride reaches) on the current device
// with new outputs.  They return those, None for anything else (the
// Python wrapper's general path, which also names what is wrong with it), or
// the call's status where it is not HCG_OK.

#include <torch/extension.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>

#include <optional>

#include "hcg_fp8.h"
#include "hcg_gemm.h"
#include "hcg_lm.h"

namespace {

namespace py = pybind11;

int64_t gemm(const at::Tensor& a, const at::Tensor& b, const at::Tensor& c, int64_t algo) {
  if (a.dim() != 2 || b.dim() != 2 || c.dim() != 2) return -1;
  if (!a.is_cuda() || !b.is_cuda() || !c.is_cuda()) return -1;
  const c10::DeviceIndex dev = a.get_device();
  if (b.get_device() != dev || c.get_device() != dev || c10::hip::current_device() != dev) return -1;
  const at::ScalarType st = a.scalar_type();
  int dtype;
  if (st == at::kHalf)
    dtype = HCG_F16;
  else if (st == at::kBFloat16)
    dtype = HCG_BF16;
  else
    return -1;
  if (b.scalar_type() != st || c.scalar_type() != at::kFloat) return -1;
  const int64_t m = a.size(0), k = a.size(1), n = b.size(1);
  if (b.size(0) != k || c.size(0) != m || c.size(1) != n || m == 0 || n == 0) return -1;
  // Row-major views only (the Python wrapper copies other layouts first); a
  // one-row matrix's row stride is unused, so the smallest legal one is passed.
  if (k > 0 && (a.stride(1) != 1 || (m > 1 && a.stride(0) < k))) return -1;
  if (k > 0 && (b.stride(1) != 1 || (k > 1 && b.stride(0) < n))) return -1;
  if (!(c.stride(1) == 1 || n == 1) || !(m == 1 || c.stride(0) >= n)) return -1;
  const int64_t lda = m > 1 ? std::max<int64_t>(a.stride(0), k) : std::max<int64_t>(k, 1);
  const int64_t ldb = k > 1 ? std::max<int64_t>(b.stride(0), n) : std::max<int64_t>(n, 1);
  const int64_t ldc = m > 1 ? std::max<int64_t>(c.stride(0), n) : std::max<int64_t>(n, 1);
  hipStream_t stream = c10::hip::getCurrentHIPStream(dev).stream();
  return hcg_gemm_algo((int)algo, dtype, a.data_ptr(), lda, b.data_ptr(), ldb, static_cast<float*>(c.data_ptr()),
                       ldc, m, n, k, stream);
}

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kHalf: return HCG_F16;
    case at::kBFloat16: return HCG_BF16;
    case at::kFloat: return HCG_F32;
    default: return -1;
  }
}

// Contiguous, on the current device (`dev`, which it sets where it is -1).
bool here(const at::Tensor& t, c10::DeviceIndex& dev) {
  if (!t.is_cuda() || !t.is_contiguous()) return false;
  if (dev < 0) {
    dev = t.get_device();
    return dev == c10::hip::current_device();
  }
  return t.get_device() == dev;
}

int id_bytes(const at::Tensor& t) {
  return t.scalar_type() == at::kLong ? 8 : t.scalar_type() == at::kInt ? 4 : 0;
}

hipStream_t stream_of(c10::DeviceIndex dev) { return c10::hip::getCurrentHIPStream(dev).stream(); }

at::Tensor workspace(int64_t bytes, const at::Tensor& like) {
  return at::empty({bytes}, like.options().dtype(at::kByte));
}

py::object embedding(const at::Tensor& tokens, const at::Tensor& table, double scale) {
  c10::DeviceIndex dev = -1;
  const int dtype = dtype_of(table), ids = id_bytes(tokens);
  if (dtype < 0 || !ids || table.dim() != 2 || !here(table, dev) || !here(tokens, dev)) return py::none();
  const int64_t vocab = table.size(0), width = table.size(1);
  auto shape = tokens.sizes().vec();
  shape.push_back(width);
  at::Tensor out = at::empty(shape, table.options());
  const int64_t ld = std::max<int64_t>(width, 1);
  const int rc = hcg_embedding(dtype, table.data_ptr(), ld, vocab, width, ids, tokens.data_ptr(), tokens.numel(),
                               (float)scale, out.data_ptr(), ld, stream_of(dev));
  return rc ? py::cast(rc) : py::cast(out);
}

py::object embedding_grad(const at::Tensor& dy, const at::Tensor& tokens, int64_t vocab, double scale) {
  c10::DeviceIndex dev = -1;
  const int dtype = dtype_of(dy), ids = id_bytes(tokens);
  if (dtype < 0 || !ids || vocab < 0 || dy.dim() != tokens.dim() + 1 || !here(dy, dev) || !here(tokens, dev) ||
      dy.sizes().slice(0, tokens.dim()) != tokens.sizes())
    return py::none();
  const int64_t width = dy.size(-1), n = tokens.numel(), ld = std::max<int64_t>(width, 1);
  at::Tensor out = at::empty({vocab, width}, dy.options()), ws;
  const int64_t need = hcg_embedding_grad_workspace(dtype, n, vocab, width);
  if (need > 0) ws = workspace(need, dy);
  const int rc = hcg_embedding_grad(dtype, dy.data_ptr(), ld, n, width, ids, tokens.data_ptr(), vocab, -1,
                                    (float)scale, dtype, out.data_ptr(), ld, need > 0 ? ws.data_ptr() : nullptr, need,
                                    stream_of(dev));
  return rc ? py::cast(rc) : py::cast(out);
}

// A parameter vector of x's width and type, or float32.
bool param_fits(const at::Tensor& p, const at::Tensor& x, c10::DeviceIndex dev) {
  return here(p, dev) && p.dim() == 1 && p.size(0) == x.size(-1) &&
         (p.scalar_type() == x.scalar_type() || p.scalar_type() == at::kFloat);
}

py::object layer_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                      const std::optional<at::Tensor>& bias, double eps) {
  c10::DeviceIndex dev = -1;
  const int dtype = dtype_of(x);
  if (dtype < 0 || x.dim() < 1 || x.size(-1) == 0 || !here(x, dev)) return py::none();
  int pdtype = dtype;
  if (weight) {
    if (!param_fits(*weight, x, dev)) return py::none();
    pdtype = dtype_of(*weight);
  }
  if (bias) {
    if (!param_fits(*bias, x, dev) || (weight && dtype_of(*bias) != pdtype)) return py::none();
    pdtype = dtype_of(*bias);
  }
  const int64_t width = x.size(-1), rows = x.numel() / width;
  const auto shape = x.sizes().slice(0, x.dim() - 1);
  at::Tensor y = at::empty(x.sizes(), x.options());
  const auto f32 = x.options().dtype(at::kFloat);
  at::Tensor mean = at::empty(shape, f32), rstd = at::empty(shape, f32);
  const int rc = hcg_layer_norm(dtype, x.data_ptr(), width, rows, width, pdtype, weight ? weight->data_ptr() : nullptr,
                                bias ? bias->data_ptr() : nullptr, (float)eps, y.data_ptr(), width,
                                static_cast<float*>(mean.data_ptr()), static_cast<float*>(rstd.data_ptr()),
                                stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(y, mean, rstd));
}

py::object layer_norm_grad(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& mean, const at::Tensor& rstd,
                           const std::optional<at::Tensor>& weight) {
  c10::DeviceIndex dev = -1;
  const int dtype = dtype_of(x);
  if (dtype < 0 || x.dim() < 1 || x.size(-1) == 0 || !here(x, dev) || !here(dy, dev) || !here(mean, dev) ||
      !here(rstd, dev) || dy.sizes() != x.sizes() || dy.scalar_type() != x.scalar_type() ||
      mean.scalar_type() != at::kFloat || rstd.scalar_type() != at::kFloat)
    return py::none();
  const int64_t width = x.size(-1), rows = x.numel() / width;
  if (mean.numel() != rows || rstd.numel() != rows || (weight && !param_fits(*weight, x, dev))) return py::none();
  const int pdtype = weight ? dtype_of(*weight) : dtype;
  at::Tensor dx = at::empty(x.sizes(), x.options());
  const auto popt = weight ? weight->options() : x.options();
  at::Tensor dw = at::empty({width}, popt), db = at::empty({width}, popt), ws;
  const int64_t need = hcg_layer_norm_grad_workspace(rows, width);
  if (need > 0) ws = workspace(need, x);
  const int rc = hcg_layer_norm_grad(
      dtype, dy.data_ptr(), width, x.data_ptr(), width, rows, width, static_cast<const float*>(mean.data_ptr()),
      static_cast<const float*>(rstd.data_ptr()), pdtype, weight ? weight->data_ptr() : nullptr, dx.data_ptr(), width,
      dw.data_ptr(), db.data_ptr(), need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(dx, dw, db));
}

// What both calls of the head ask of their arguments; rows and a vocabulary of
// none are the Python wrapper's.
bool head_fits(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets, c10::DeviceIndex& dev) {
  const int dtype = dtype_of(x);
  return (dtype == HCG_F16 || dtype == HCG_BF16) && x.dim() >= 1 && weight.dim() == 2 && here(x, dev) &&
         here(weight, dev) && here(targets, dev) && weight.scalar_type() == x.scalar_type() &&
         x.size(-1) == weight.size(1) && id_bytes(targets) && targets.sizes() == x.sizes().slice(0, x.dim() - 1) &&
         x.numel() > 0 && weight.size(0) > 0;
}

py::object linear_cross_entropy(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets,
                                int64_t ignore) {
  c10::DeviceIndex dev = -1;
  if (!head_fits(x, weight, targets, dev)) return py::none();
  const int64_t width = x.size(-1), vocab = weight.size(0), tokens = targets.numel();
  const auto f32 = x.options().dtype(at::kFloat);
  at::Tensor loss = at::empty(targets.sizes(), f32), lse = at::empty(targets.sizes(), f32);
  const int64_t need = hcg_linear_cross_entropy_workspace(tokens, vocab, width, weight.data_ptr(), width, 0);
  at::Tensor ws = workspace(need, x);
  const int rc = hcg_linear_cross_entropy(dtype_of(x), x.data_ptr(), width, tokens, weight.data_ptr(), width, vocab,
                                          width, id_bytes(targets), targets.data_ptr(), ignore,
                                          static_cast<float*>(loss.data_ptr()), static_cast<float*>(lse.data_ptr()),
                                          ws.data_ptr(), need, stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(loss, lse));
}

py::object linear_cross_entropy_grad(const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets,
                                     int64_t ignore, bool mean, double grad_scale) {
  c10::DeviceIndex dev = -1;
  if (!head_fits(x, weight, targets, dev)) return py::none();
  const int64_t width = x.size(-1), vocab = weight.size(0), tokens = targets.numel();
  at::Tensor loss = at::empty({}, x.options().dtype(at::kFloat));
  at::Tensor dx = at::empty(x.sizes(), x.options()), dw = at::empty(weight.sizes(), x.options());
  const int64_t need = hcg_linear_cross_entropy_workspace(tokens, vocab, width, weight.data_ptr(), width, 1);
  at::Tensor ws = workspace(need, x);
  const int rc = hcg_linear_cross_entropy_grad(
      dtype_of(x), x.data_ptr(), width, tokens, weight.data_ptr(), width, vocab, width, id_bytes(targets),
      targets.data_ptr(), ignore, mean, (float)grad_scale, static_cast<float*>(loss.data_ptr()), dx.data_ptr(), width,
      dw.data_ptr(), width, ws.data_ptr(), need, stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(loss, dx, dw));
}

// What both forms of the root-mean-square norm make of their arguments.
struct Rms {
  int dtype, rdtype, pdtype;
  int64_t rows, width;
  at::Tensor h, rstd;
  const void* residual;
  void* sum;
};
bool rms_fits(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& residual,
              c10::DeviceIndex& dev, Rms& r) {
  r.dtype = r.rdtype = r.pdtype = dtype_of(x);
  if (r.dtype < 0 || x.dim() < 1 || x.size(-1) == 0 || !here(x, dev)) return false;
  if (weight) {
    if (!param_fits(*weight, x, dev)) return false;
    r.pdtype = dtype_of(*weight);
  }
  if (residual) {
    if (!here(*residual, dev) || residual->sizes() != x.sizes() ||
        (residual->scalar_type() != x.scalar_type() && residual->scalar_type() != at::kFloat))
      return false;
    r.rdtype = dtype_of(*residual);
  }
  r.width = x.size(-1);
  r.rows = x.numel() / r.width;
  r.h = residual ? at::empty(x.sizes(), residual->options()) : x;
  r.residual = residual ? residual->data_ptr() : nullptr;
  r.sum = residual ? r.h.data_ptr() : nullptr;
  r.rstd = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  return true;
}

py::object rms_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                    const std::optional<at::Tensor>& residual, double eps) {
  c10::DeviceIndex dev = -1;
  Rms r;
  if (!rms_fits(x, weight, residual, dev, r)) return py::none();
  at::Tensor y = at::empty(x.sizes(), x.options());
  const int rc = hcg_rms_norm(r.dtype, x.data_ptr(), r.width, r.rows, r.width, r.rdtype, r.residual, r.width, r.pdtype,
                              weight ? weight->data_ptr() : nullptr, (float)eps, y.data_ptr(), r.width, r.sum, r.width,
                              static_cast<float*>(r.rstd.data_ptr()), stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(y, r.h, r.rstd));
}

py::object rms_norm_grad(const at::Tensor& dy, const at::Tensor& h, const at::Tensor& rstd,
                         const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& dresidual) {
  c10::DeviceIndex dev = -1;
  const int dtype = dtype_of(dy), hdtype = dtype_of(h);
  if (dtype < 0 || dy.dim() < 1 || dy.size(-1) == 0 || !here(dy, dev) || !here(h, dev) || !here(rstd, dev) ||
      h.sizes() != dy.sizes() || (hdtype != dtype && hdtype != HCG_F32) || rstd.scalar_type() != at::kFloat)
    return py::none();
  const int64_t width = dy.size(-1), rows = dy.numel() / width;
  if (rstd.numel() != rows || (weight && !param_fits(*weight, dy, dev))) return py::none();
  if (dresidual && (!here(*dresidual, dev) || dresidual->sizes() != h.sizes() ||
                    dresidual->scalar_type() != h.scalar_type()))
    return py::none();
  const int pdtype = weight ? dtype_of(*weight) : dtype;
  at::Tensor dh = at::empty(h.sizes(), h.options()), dw = at::empty({width}, weight ? weight->options() : dy.options()),
             ws;
  const int64_t need = hcg_rms_norm_grad_workspace(rows, width);
  if (need > 0) ws = workspace(need, dy);
  const int rc = hcg_rms_norm_grad(dtype, dy.data_ptr(), width, hdtype, h.data_ptr(), width, rows, width,
                                   static_cast<const float*>(rstd.data_ptr()), pdtype,
                                   weight ? weight->data_ptr() : nullptr, dresidual ? dresidual->data_ptr() : nullptr,
                                   width, dh.data_ptr(), width, dw.data_ptr(), need > 0 ? ws.data_ptr() : nullptr, need,
                                   stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(dh, dw));
}

// New q (rows of whole 16 bytes) and scale (block by block in memory), as
// hc.gfx950.fp8 lays them out.
struct Quantized {
  at::Tensor q, scale;
  int64_t ldq, step;
};
Quantized new_quantized(const at::Tensor& like, c10::IntArrayRef lead, int64_t cols, c10::IntArrayRef down, int q_dtype,
                        int scale_dtype) {
  const auto strided = [](c10::IntArrayRef dims, int64_t last, int64_t first, at::ScalarType type, const at::Tensor& t,
                          int64_t last_stride) {
    auto shape = dims.vec();
    std::vector<int64_t> strides(shape.size() + 1, last_stride);
    int64_t step = first;
    for (size_t i = shape.size(); i-- > 0; step *= std::max<int64_t>(shape[i], 1)) strides[i] = step;
    shape.push_back(last);
    return at::empty_strided(shape, strides, t.options().dtype(type));
  };
  Quantized r;
  r.ldq = std::max<int64_t>((cols + 15) / 16 * 16, 1);
  r.step = 1;
  for (const int64_t n : down) r.step *= n;
  r.step = std::max<int64_t>(r.step, 1);
  r.q = strided(lead, cols, r.ldq, q_dtype == HCG_E5M2 ? at::kFloat8_e5m2 : at::kFloat8_e4m3fn, like, 1);
  r.scale = strided(down, (cols + HCG_FP8_BLOCK - 1) / HCG_FP8_BLOCK, 1,
                    scale_dtype == HCG_E8M0 ? at::kFloat8_e8m0fnu : at::kFloat, like, r.step);
  return r;
}

py::object rms_norm_fp8(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                        const std::optional<at::Tensor>& residual, double eps, int q_dtype, int scale_dtype) {
  c10::DeviceIndex dev = -1;
  Rms r;
  if (!rms_fits(x, weight, residual, dev, r)) return py::none();
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  const Quantized o = new_quantized(x, lead, r.width, lead, q_dtype, scale_dtype);
  const int rc = hcg_rms_norm_fp8(r.dtype, x.data_ptr(), r.width, r.rows, r.width, r.rdtype, r.residual, r.width,
                                  r.pdtype, weight ? weight->data_ptr() : nullptr, (float)eps, q_dtype, o.q.data_ptr(),
                                  o.ldq, scale_dtype, o.scale.data_ptr(), 1, o.step, r.sum, r.width,
                                  static_cast<float*>(r.rstd.data_ptr()), stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(o.q, o.scale, r.h, r.rstd));
}

py::object quantize_fp8(const at::Tensor& x, bool tile, bool transpose, int q_dtype, int scale_dtype) {
  c10::DeviceIndex dev = -1;
  const int dtype = dtype_of(x);
  if (dtype < 0 || x.dim() < 1 || x.numel() == 0 || !here(x, dev)) return py::none();
  const int64_t cols = x.size(-1), rows = x.numel() / cols;
  const int64_t turned[] = {cols}, tiles[] = {((transpose ? cols : rows) + HCG_FP8_BLOCK - 1) / HCG_FP8_BLOCK};
  const auto lead = transpose ? c10::IntArrayRef(turned, 1) : x.sizes().slice(0, x.dim() - 1);
  const Quantized o =
      new_quantized(x, lead, transpose ? rows : cols, tile ? c10::IntArrayRef(tiles, 1) : lead, q_dtype, scale_dtype);
  const int rc = hcg_quantize_fp8(dtype, x.data_ptr(), cols, rows, cols, transpose, tile, q_dtype, o.q.data_ptr(), o.ldq,
                                  scale_dtype, o.scale.data_ptr(), 1, o.step, stream_of(dev));
  return rc ? py::cast(rc) : py::object(py::make_tuple(o.q, o.scale));
}

// Whether the leading dimensions are rows that one stride reaches, which it gives.
bool rows_of(const at::Tensor& t, int64_t& stride) {
  stride = 1;
  int64_t next = -1;
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (next < 0)
      stride = t.stride(d);
    else if (t.stride(d) != next)
      return false;
    next = t.stride(d) * t.size(d);
  }
  return true;
}

py::object linear_fp8(const at::Tensor& x, const at::Tensor& x_scale, const at::Tensor& weight,
                      const at::Tensor& weight_scale, int out_dtype) {
  if (!x.is_cuda() || !x_scale.is_cuda() || !weight.is_cuda() || !weight_scale.is_cuda()) return py::none();
  const c10::DeviceIndex dev = x.get_device();
  if (x_scale.get_device() != dev || weight.get_device() != dev || weight_scale.get_device() != dev ||
      c10::hip::current_device() != dev)
    return py::none();
  const auto xt = x.scalar_type(), st = x_scale.scalar_type();
  if ((xt != at::kFloat8_e4m3fn && xt != at::kFloat8_e5m2) || weight.scalar_type() != at::kFloat8_e4m3fn ||
      (st != at::kFloat && st != at::kFloat8_e8m0fnu) || weight_scale.scalar_type() != st || x.dim() < 1 ||
      weight.dim() != 2 || weight_scale.dim() != 2 || x_scale.dim() != x.dim() || x.numel() == 0 || weight.numel() == 0)
    return py::none();
  const int64_t inputs = x.size(-1), outputs = weight.size(0), tokens = x.numel() / inputs;
  const int64_t blocks = (inputs + HCG_FP8_BLOCK - 1) / HCG_FP8_BLOCK;
  const int64_t tiles = (outputs + HCG_FP8_BLOCK - 1) / HCG_FP8_BLOCK;
  const bool tile = weight_scale.size(0) == tiles;
  int64_t ldx, xs_row;
  if (weight.size(1) != inputs || x_scale.size(-1) != blocks || weight_scale.size(1) != blocks ||
      (!tile && weight_scale.size(0) != outputs) ||
      x_scale.sizes().slice(0, x.dim() - 1) != x.sizes().slice(0, x.dim() - 1) || !rows_of(x, ldx) ||
      !rows_of(x_scale, xs_row) || (inputs > 1 && (x.stride(-1) != 1 || weight.stride(1) != 1)) ||
      (tokens > 1 && ldx < inputs) || (outputs > 1 && weight.stride(0) < inputs))
    return py::none();
  auto shape = x.sizes().vec();
  shape.back() = outputs;
  at::Tensor y = at::empty(shape, x.options().dtype(out_dtype == HCG_F16    ? at::kHalf
                                                    : out_dtype == HCG_BF16 ? at::kBFloat16
                                                                            : at::kFloat));
  at::Tensor ws;
  const int sdtype = st == at::kFloat ? HCG_F32 : HCG_E8M0;
  if (tokens == 1) ldx = inputs;
  const int64_t ldw = outputs == 1 ? inputs : weight.stride(0);
  const int64_t need =
      hcg_linear_fp8_workspace(HCG_FP8_AUTO, tokens, outputs, inputs, x.data_ptr(), ldx, weight.data_ptr(), ldw, sdtype,
                               xs_row, tile, weight_scale.data_ptr(), weight_scale.stride(0), weight_scale.stride(1),
                               out_dtype);
  if (need > 0) ws = workspace(need, x);
  const int rc =
      hcg_linear_fp8(HCG_FP8_AUTO, xt == at::kFloat8_e5m2 ? HCG_E5M2 : HCG_E4M3, x.data_ptr(), ldx, tokens,
                     weight.data_ptr(), ldw, outputs, inputs, sdtype, x_scale.data_ptr(), xs_row, x_scale.stride(-1), tile,
                     weight_scale.data_ptr(), weight_scale.stride(0), weight_scale.stride(1), out_dtype, y.data_ptr(),
                     outputs, need > 0 ? ws.data_ptr() : nullptr, need, stream_of(dev));
  return rc ? py::cast(rc) : py::cast(y);
}

}  // namespace

PYBIND11_MODULE(_hcg_torch, mod) {
  mod.def("gemm", &gemm, "C = A @ B on the current HIP stream; -1 when the case is not handled here");
  mod.def("embedding", &embedding);
  mod.def("embedding_grad", &embedding_grad);
  mod.def("layer_norm", &layer_norm);
  mod.def("layer_norm_grad", &layer_norm_grad);
  mod.def("linear_cross_entropy", &linear_cross_entropy);
  mod.def("linear_cross_entropy_grad", &linear_cross_entropy_grad);
  mod.def("rms_norm", &rms_norm);
  mod.def("rms_norm_grad", &rms_norm_grad);
  mod.def("rms_norm_fp8", &rms_norm_fp8);
  mod.def("quantize_fp8", &quantize_fp8);
  mod.def("linear_fp8", &linear_fp8);
}

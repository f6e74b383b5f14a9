// The Python binding of the decode operators (include/nsattn.h: nsa_linear4 .. nsa_kv4_attention) over torch
// tensors, module nanosaur2_web_b200._native.  A decode step is a few microseconds of GPU work per call; through
// ctypes the Python side of a call costs 14 to 38, here 5 to 10, so these operators are bound in C++ and the rest of
// the library through ctypes (_lib.py).  Arguments are checked here (shapes, types, devices) and in the C ABI
// (values, alignment, overlap); both raise NsaError.  ops.py documents the functions.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <string>

#include "nsattn.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

[[noreturn]] void raise(int status, const std::string& message) {
  static const py::handle cls = py::object(py::module_::import("nanosaur2_web_b200._lib").attr("NsaError")).release();
  const py::object error = cls(status, message);
  PyErr_SetObject(cls.ptr(), error.ptr());
  throw py::error_already_set();
}

[[noreturn]] void invalid(const std::string& message) { raise(NSA_ERR_INVALID_ARGUMENT, message); }

void check(nsa_status status) {
  if (status != NSA_OK) raise(status, nsa_last_error());
}

// The one CUDA device that all tensors of a call live on.
class Devices {
 public:
  Devices& operator()(const Tensor& t) {
    if (!t.is_cuda()) invalid("tensors must live on a CUDA device");
    const int i = t.get_device();
    if (index_ >= 0 && i != index_)
      invalid("tensors live on cuda:" + std::to_string(index_) + " and cuda:" + std::to_string(i) + ": one device is wanted");
    index_ = i;
    return *this;
  }
  Devices& operator()(const OptTensor& t) { return t ? (*this)(*t) : *this; }
  c10::DeviceIndex index() const { return (c10::DeviceIndex)index_; }

 private:
  int index_ = -1;
};

// Makes the device current for a call and gives its current stream.
struct OnDevice {
  c10::cuda::CUDAGuard guard;
  void* stream;
  explicit OnDevice(c10::DeviceIndex i) : guard(i), stream(c10::cuda::getCurrentCUDAStream(i).stream()) {}
};

int32_t dtype_code(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kFloat) return NSA_F32;
  if (t.scalar_type() == at::kBFloat16) return NSA_BF16;
  invalid(std::string(name) + " must be float32 or bfloat16");
}

int32_t int32_of(int64_t v, const char* name) {
  if (v < INT32_MIN || v > INT32_MAX) invalid(std::string(name) + " is out of range");
  return (int32_t)v;
}

void* data(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }

nsa_weight4 weight(const Tensor& codes, const Tensor& scales, int64_t N, int64_t K, int64_t group) {
  if (group != 32 && group != 64 && group != 128) invalid("group must be 32, 64 or 128");
  if (N < 1 || K < 1) invalid("N and K must be >= 1");
  const int64_t t = (N + 15) / 16, k = (K + 127) / 128;
  if (codes.scalar_type() != at::kByte || scales.scalar_type() != at::kBFloat16 ||
      codes.sizes() != at::IntArrayRef({t, k, 16, 64}) || scales.sizes() != at::IntArrayRef({t, k, 16, 128 / group}) ||
      !codes.is_contiguous() || !scales.is_contiguous())
    invalid("a " + std::to_string(group) + "-group weight [" + std::to_string(N) + ", " + std::to_string(K) +
            "] has contiguous codes uint8 [" + std::to_string(t) + ", " + std::to_string(k) + ", 16, 64] and scales bfloat16 [" +
            std::to_string(t) + ", " + std::to_string(k) + ", 16, " + std::to_string(128 / group) + "]");
  return {int32_of(N, "N"), int32_of(K, "K"), (int32_t)group, codes.data_ptr<uint8_t>(), scales.data_ptr()};
}

std::pair<Tensor, Tensor> quantize4(const Tensor& W, int64_t group, const OptTensor& codes_, const OptTensor& scales_) {
  const auto dev = Devices()(W)(codes_)(scales_).index();
  if (W.dim() != 2 || W.size(0) < 1 || W.size(1) < 1 || (W.size(1) > 1 && W.stride(1) != 1))
    invalid("W must be a non-empty [N, K] tensor with unit inner stride");
  const int64_t N = W.size(0), K = W.size(1), ld = N > 1 ? W.stride(0) : K;
  if (ld < K) invalid("the rows of W must not overlap");
  if (group != 32 && group != 64 && group != 128) invalid("group must be 32, 64 or 128");
  OnDevice on(dev);
  const int64_t t = (N + 15) / 16, k = (K + 127) / 128;
  Tensor codes = codes_ ? *codes_ : at::empty({t, k, 16, 64}, W.options().dtype(at::kByte));
  Tensor scales = scales_ ? *scales_ : at::empty({t, k, 16, 128 / group}, W.options().dtype(at::kBFloat16));
  const nsa_weight4 w = weight(codes, scales, N, K, group);
  check(nsa_quantize4(&w, W.data_ptr(), dtype_code(W, "W"), ld, on.stream));
  return {codes, scales};
}

Tensor expand4(const Tensor& codes, const Tensor& scales, int64_t N, int64_t K, int64_t group, const OptTensor& out_) {
  const auto dev = Devices()(codes)(scales)(out_).index();
  const nsa_weight4 w = weight(codes, scales, N, K, group);
  OnDevice on(dev);
  const Tensor out = out_ ? *out_ : at::empty({N, K}, scales.options());
  if (out.scalar_type() != at::kBFloat16 || out.sizes() != at::IntArrayRef({N, K}) || (K > 1 && out.stride(1) != 1) ||
      (N > 1 && out.stride(0) < K))
    invalid("out must be a bfloat16 [N, K] tensor with unit inner stride");
  check(nsa_expand4(&w, out.data_ptr(), N > 1 ? out.stride(0) : K, on.stream));
  return out;
}

Tensor linear4(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t N, int64_t K, int64_t group,
               const OptTensor& bias, const OptTensor& out_, bool resid, std::optional<at::ScalarType> out_dtype) {
  const auto dev = Devices()(x)(codes)(scales)(bias)(out_).index();
  const nsa_weight4 w = weight(codes, scales, N, K, group);
  if (x.scalar_type() != at::kBFloat16 || x.dim() != 2 || x.size(1) != K || (K > 1 && x.stride(1) != 1))
    invalid("x must be [M, " + std::to_string(K) + "] bf16 with unit inner stride");
  const int64_t M = x.size(0);
  if (bias && (bias->scalar_type() != at::kFloat || bias->sizes() != at::IntArrayRef({N}) || !bias->is_contiguous()))
    invalid("bias must be a contiguous float32 [" + std::to_string(N) + "] tensor");
  OnDevice on(dev);
  Tensor out;
  if (out_) {
    out = *out_;
    if (out.sizes() != at::IntArrayRef({M, N}) || (N > 1 && out.stride(1) != 1))
      invalid("out must be [" + std::to_string(M) + ", " + std::to_string(N) + "] with unit inner stride");
  } else {
    if (resid) invalid("resid needs out");
    out = at::empty({M, N}, x.options().dtype(out_dtype.value_or(at::kFloat)));
  }
  nsa_linear4_desc d{};
  d.M = int32_of(M, "M");
  d.lda = M > 1 ? x.stride(0) : K;
  d.ldc = M > 1 ? out.stride(0) : N;
  if (d.lda < K || d.ldc < N) invalid("the rows of x and out must not overlap");
  d.resid = resid;
  d.out_dtype = dtype_code(out, "out");
  check(nsa_linear4(&d, &w, x.data_ptr(), static_cast<const float*>(data(bias)), out.data_ptr(), on.stream));
  return out;
}

nsa_kv4_cache cache_of(const Tensor& codes, const Tensor& scales) {
  const auto c = codes.sizes(), s = scales.sizes();
  if (c.size() != 5 || c[1] != 2 || s.size() != 5 || s[0] != c[0] || s[1] != 2 || s[2] != c[2] || s[3] != c[3] ||
      s[4] != c[4] / 16 || codes.scalar_type() != at::kByte || scales.scalar_type() != at::kBFloat16 ||
      !codes.is_contiguous() || !scales.is_contiguous())
    invalid("the cache has contiguous codes uint8 [n_pages, 2, Hkv, P, D/2] and scales bfloat16 [n_pages, 2, Hkv, P, D/32]");
  return {int32_of(c[0], "n_pages"), int32_of(c[3], "P"), int32_of(c[2], "Hkv"), int32_of(2 * c[4], "D"),
          codes.data_ptr<uint8_t>(), scales.data_ptr()};
}

// The step; *table may be replaced by a contiguous copy (to be kept until the launch).
nsa_kv4_batch batch_of(int64_t B, int64_t L, Tensor* table, const Tensor& start, const OptTensor& count, int64_t positions) {
  if (table->dim() != 2 || table->size(0) != B || table->scalar_type() != at::kInt ||
      (table->size(1) > 1 && table->stride(1) != 1))
    invalid("table must be an int32 [" + std::to_string(B) + ", max_pages] tensor with unit inner stride");
  const auto vector = [&](const Tensor& t, const char* name) {
    if (t.dim() != 1 || t.size(0) != B || t.scalar_type() != at::kInt || (B > 1 && t.stride(0) != 1))
      invalid(std::string(name) + " must be a contiguous int32 [" + std::to_string(B) + "] tensor");
  };
  vector(start, "start");
  if (count) vector(*count, "count");
  const int64_t pages = table->size(1);
  if (B > 1 && table->stride(0) < pages) *table = table->contiguous();   // every sequence on the same pages
  nsa_kv4_batch b{};
  b.B = int32_of(B, "B");
  b.L = int32_of(L, "L");
  b.max_pages = int32_of(pages, "max_pages");
  b.table_ld = B > 1 ? table->stride(0) : pages;
  b.table = table->data_ptr<int32_t>();
  b.start = start.data_ptr<int32_t>();
  b.count = static_cast<const int32_t*>(data(count));
  b.positions = int32_of(positions, "positions");
  return b;
}

// A [B, L, columns] operand with unit inner stride; pitches of axes of length 1 are those of a contiguous one.
struct Rows {
  int64_t B, L, cols, ld, bstride;
};
Rows rows_of(const Tensor& t, const char* name) {
  if (t.dim() != 3 || (t.size(2) > 1 && t.stride(2) != 1))
    invalid(std::string(name) + " must be [B, L, columns] with unit inner stride");
  Rows r{t.size(0), t.size(1), t.size(2), 0, 0};
  r.ld = r.L > 1 ? t.stride(1) : r.cols;
  r.bstride = r.B > 1 ? t.stride(0) : r.L * r.ld;
  return r;
}
Rows result_rows(const Tensor& t, const char* name, int64_t B, int64_t L, int64_t cols) {
  const Rows r = rows_of(t, name);
  if (t.scalar_type() != at::kBFloat16 || r.B != B || r.L != L || r.cols != cols)
    invalid(std::string(name) + " must be a bfloat16 [" + std::to_string(B) + ", " + std::to_string(L) + ", " +
            std::to_string(cols) + "] tensor");
  return r;
}

Tensor kv4_append(const Tensor& qkv, const Tensor& codes, const Tensor& scales, Tensor table, const Tensor& start,
                  const OptTensor& count, int64_t Hq, const Tensor& q_norm, const Tensor& k_norm, const OptTensor& cs,
                  int64_t cs_rows, int64_t cs_D, int64_t sin_off, double eps, int64_t qOff, std::optional<int64_t> kOff_,
                  std::optional<int64_t> vOff_, const OptTensor& out_) {
  const auto dev = Devices()(qkv)(codes)(scales)(table)(start)(count)(q_norm)(k_norm)(cs)(out_).index();
  const nsa_kv4_cache c = cache_of(codes, scales);
  const int64_t D = c.D, Hkv = c.Hkv;
  const Rows x = rows_of(qkv, "qkv");
  if (Hq < 1 || Hq > (1 << 24) || qOff < 0) invalid("need Hq >= 1 and offsets >= 0");
  const int64_t kOff = kOff_.value_or(qOff + Hq * D), vOff = vOff_.value_or(kOff + Hkv * D);
  if (kOff < 0 || vOff < 0 || qOff + Hq * D > x.cols || kOff + Hkv * D > x.cols || vOff + Hkv * D > x.cols)
    invalid("the q, k and v heads must lie inside qkv's columns");
  for (const Tensor* w : {&q_norm, &k_norm})
    if (w->scalar_type() != at::kFloat || w->sizes() != at::IntArrayRef({D}) || !w->is_contiguous())
      invalid("q_norm and k_norm must be contiguous float32 [" + std::to_string(D) + "] tensors");
  if (cs && (cs_D != D || cs->scalar_type() != at::kFloat || !cs->is_contiguous() || sin_off < 0 || cs_rows < 1 ||
             cs_rows > cs->numel() || cs_rows * (D / 2) > cs->numel() - sin_off))
    invalid("cs must be a float32 table of one row or more of head dim " + std::to_string(D));
  OnDevice on(dev);
  const Tensor out = out_ ? *out_ : at::empty({x.B, x.L, Hq * D}, qkv.options().dtype(at::kBFloat16));
  const Rows o = result_rows(out, "out", x.B, x.L, Hq * D);
  const nsa_kv4_batch b = batch_of(x.B, x.L, &table, start, count, 0);
  nsa_kv4_append_desc d{};
  d.Hq = (int32_t)Hq;
  d.in_dtype = dtype_code(qkv, "qkv");
  d.ld = x.ld;
  d.bstride = x.bstride;
  d.qOff = qOff;
  d.kOff = kOff;
  d.vOff = vOff;
  d.qo_ld = o.ld;
  d.qo_bstride = o.bstride;
  d.sinOff = cs ? sin_off : 0;
  d.rope_rows = cs ? int32_of(cs_rows, "cs") : 0;
  d.eps = (float)eps;
  check(nsa_kv4_append(&d, &c, &b, qkv.data_ptr(), q_norm.data_ptr<float>(), k_norm.data_ptr<float>(),
                       static_cast<const float*>(data(cs)), out.data_ptr(), on.stream));
  return out;
}

Tensor kv4_read(const Tensor& codes, const Tensor& scales, int64_t positions, Tensor table, const Tensor& start, int64_t L,
                const OptTensor& count, const OptTensor& out_) {
  const auto dev = Devices()(codes)(scales)(table)(start)(count)(out_).index();
  const nsa_kv4_cache c = cache_of(codes, scales);
  if (table.dim() != 2 || L < 0) invalid("table must be [B, max_pages] and L >= 0");
  const int64_t B = table.size(0), width = 2 * (int64_t)c.Hkv * c.D;
  OnDevice on(dev);
  const Tensor out = out_ ? *out_ : at::zeros({B, L, width}, scales.options());
  const Rows o = result_rows(out, "out", B, L, width);
  const nsa_kv4_batch b = batch_of(B, L, &table, start, count, positions);
  check(nsa_kv4_read(&c, &b, out.data_ptr(), o.ld, o.bstride, on.stream));
  return out;
}

Tensor kv4_attention(const Tensor& q, const Tensor& codes, const Tensor& scales, int64_t positions, Tensor table,
                     const Tensor& start, const OptTensor& count, int64_t window, int64_t sinks, double scale, const OptTensor& out_,
                     const OptTensor& workspace_) {
  const auto dev = Devices()(q)(codes)(scales)(table)(start)(count)(out_)(workspace_).index();
  const nsa_kv4_cache c = cache_of(codes, scales);
  const Rows x = rows_of(q, "q");
  if (q.scalar_type() != at::kBFloat16 || c.D < 1 || x.cols % c.D || x.cols < c.D)
    invalid("q must be bfloat16 rows of whole heads of " + std::to_string(c.D));
  OnDevice on(dev);
  const Tensor out = out_ ? *out_ : at::empty({x.B, x.L, x.cols}, q.options());
  const Rows o = result_rows(out, "out", x.B, x.L, x.cols);
  const nsa_kv4_batch b = batch_of(x.B, x.L, &table, start, count, positions);
  nsa_kv4_attention_desc d{};
  d.Hq = int32_of(x.cols / c.D, "Hq");
  d.q_ld = x.ld;
  d.q_bstride = x.bstride;
  d.o_ld = o.ld;
  d.o_bstride = o.bstride;
  d.window = int32_of(window, "window");
  d.sinks = int32_of(sinks, "sinks");
  d.scale = (float)scale;
  if (scale != 0 && d.scale == 0.f) invalid("scale is 0 in fp32");
  OptTensor workspace = workspace_;
  if (!workspace) {
    const size_t need = nsa_kv4_attention_workspace_size(&d, &c, &b);
    if (need) workspace = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
  } else if (workspace->scalar_type() != at::kByte || !workspace->is_contiguous()) {
    invalid("workspace must be a contiguous uint8 tensor");
  }
  check(nsa_kv4_attention(&d, &c, &b, q.data_ptr(), out.data_ptr(), data(workspace),
                          workspace ? (size_t)workspace->numel() : 0, on.stream));
  return out;
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  m.def("quantize4", &quantize4);
  m.def("expand4", &expand4);
  m.def("linear4", &linear4);
  m.def("kv4_append", &kv4_append);
  m.def("kv4_read", &kv4_read);
  m.def("kv4_attention", &kv4_attention);
}

// Python binding of the decoder operators (decoder_ops.py): argument checks on the tensors
// themselves and the call into liblatchmoe_b200's C ABI, whose entry points arrive as addresses.
// A 16-token norm takes a few us on the GPU; checked in Python and passed through ctypes, its call
// took 9.3 us on the host, half of it checks.
#include <torch/csrc/utils/pybind.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>

#include <optional>
#include <string>

#include "latchmoe_b200.h"

namespace py = pybind11;

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

struct Library {
  decltype(&lm_last_error) last_error = nullptr;
  decltype(&lm_add_rms_norm) add_rms_norm = nullptr;
  decltype(&lm_build_page_tables) build_page_tables = nullptr;
  decltype(&lm_release_pages) release_pages = nullptr;
  decltype(&lm_rope_cache_write) rope_cache_write = nullptr;
  decltype(&lm_paged_attention) paged_attention = nullptr;
} lib;

void bind(const std::string& name, uint64_t address) {
#define LM_BIND(f) \
  if (name == "lm_" #f) lib.f = reinterpret_cast<decltype(lib.f)>(address);
  LM_BIND(last_error)
  LM_BIND(add_rms_norm)
  LM_BIND(build_page_tables)
  LM_BIND(release_pages)
  LM_BIND(rope_cache_write)
  LM_BIND(paged_attention)
#undef LM_BIND
}

[[noreturn]] void refuse(const std::string& what) { throw py::value_error(what); }

void done(const char* name, int rc) {
  if (rc < 0)
    throw std::runtime_error(std::string(name) + " failed (" + std::to_string(rc) + "): " +
                             lib.last_error());
}

std::string text(at::IntArrayRef v) {
  std::string s = "(";
  for (size_t i = 0; i < v.size(); ++i) s += (i ? ", " : "") + (v[i] < 0 ? "any" : std::to_string(v[i]));
  return s + ")";
}

// The checks of one call: all tensors on one CUDA device, the current one.
class Check {
 public:
  // dtype, device and shape (-1: any size)
  void tensor(const char* name, const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
    if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
    if (t.scalar_type() != type)
      refuse(std::string(name) + " must be " + c10::toString(type) + ", not " + c10::toString(t.scalar_type()));
    bool same = t.dim() == static_cast<int64_t>(shape.size());
    for (size_t i = 0; same && i < shape.size(); ++i) same = shape[i] < 0 || shape[i] == t.size(i);
    if (!same) refuse(std::string(name) + " must have shape " + text(shape) + ", not " + text(t.sizes()));
    if (device_ < 0) device_ = t.get_device();
    if (t.get_device() != device_) refuse(std::string(name) + " is on another device than the other tensors");
  }
  void dense(const char* name, const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
    tensor(name, t, type, shape);
    if (!t.is_contiguous()) refuse(std::string(name) + " must be contiguous");
  }
  // rows [T, n] that do not overlap; returns the row stride
  int64_t rows(const char* name, const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
    tensor(name, t, type, shape);
    if (t.size(1) > 1 && t.stride(1) != 1) refuse(std::string(name) + "'s rows must be contiguous");
    if (t.size(0) <= 1) return std::max(t.stride(0), t.size(1));
    if (t.stride(0) < t.size(1)) refuse(std::string(name) + "'s rows overlap");
    return t.stride(0);
  }
  // heads [.., D] with contiguous values
  void heads(const char* name, const Tensor& t, at::IntArrayRef shape) {
    tensor(name, t, at::kBFloat16, shape);
    if (t.numel() > 0 && t.stride(-1) != 1) refuse(std::string(name) + "'s heads must be contiguous");
  }
  int64_t table(const Tensor& t, int64_t requests) {
    tensor("block_tables", t, at::kInt, {requests, -1});
    if (t.size(1) == 0 || (t.size(1) > 1 && t.stride(1) != 1))
      refuse("block_tables' rows must be contiguous and not empty");
    return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1));
  }
  int32_t* err(const OptTensor& t) {
    if (!t) return nullptr;
    dense("err_word", *t, at::kInt, {1});
    return t->data_ptr<int32_t>();
  }
  // The library launches on the current device.
  void* stream() const {
    const auto current = c10::cuda::current_device();
    if (current != device_)
      refuse("the tensors are on cuda:" + std::to_string(device_) + ", which is not the current device");
    return c10::cuda::getCurrentCUDAStream(device_).stream();
  }

 private:
  int64_t device_ = -1;
};

// A dimension of one has no stride of its own (torch keeps whatever the tensor was cut from); the C ABI
// takes multiples of 8, so such a one passes as `of_one`.
int64_t stride(const Tensor& t, int64_t dim, int64_t of_one = 0) {
  return t.size(dim) == 1 ? of_one : t.stride(dim);
}

uint16_t* bits(const Tensor& t) { return static_cast<uint16_t*>(t.data_ptr()); }
uint16_t* bits(const OptTensor& t) { return t ? bits(*t) : nullptr; }
int32_t* ints(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

void need_dim(const char* name, const Tensor& t, int64_t dim, const char* what) {
  if (t.dim() != dim) refuse(std::string(name) + " must be " + what);
}

int32_t narrow(const char* name, int64_t v) {
  if (v > 0x7fffffff || v < -0x7fffffff) refuse(std::string(name) + " is out of range");
  return static_cast<int32_t>(v);
}

void add_rms_norm(const Tensor& x, const Tensor& weight, double eps, const OptTensor& residual,
                  const OptTensor& residual_out, const OptTensor& out, const OptTensor& out_fp8,
                  const OptTensor& scales, int64_t group) {
  need_dim("x", x, 2, "[tokens, hidden]");
  const int64_t T = x.size(0), H = x.size(1);
  Check c;
  const int64_t xs = c.rows("x", x, at::kBFloat16, {T, H});
  c.dense("weight", weight, at::kBFloat16, {H});
  if (out.has_value() == out_fp8.has_value()) refuse("give one of out and out_fp8");
  const int64_t ys = out ? c.rows("out", *out, at::kBFloat16, {T, H})
                         : c.rows("out_fp8", *out_fp8, at::kFloat8_e4m3fn, {T, H});
  const int64_t rs = residual ? c.rows("residual", *residual, at::kBFloat16, {T, H}) : 0;
  const int64_t ks = residual_out ? c.rows("residual_out", *residual_out, at::kBFloat16, {T, H}) : 0;
  if (out_fp8) {
    if (group < 0 || (group != 0 && (group % 32 != 0 || H % group != 0)))
      refuse("group_size must be 0 or a multiple of 32 that divides the hidden size");
    if (!scales) refuse("out_fp8 needs scales");
    c.dense("scales", *scales, at::kFloat, {T, group ? H / group : 1});
  } else if (scales || group != 0) {
    refuse("scales and group_size belong to out_fp8");
  }
  done("lm_add_rms_norm",
       lib.add_rms_norm(bits(x), xs, bits(residual), rs, bits(weight), static_cast<float>(eps), T,
                        narrow("hidden", H), bits(residual_out), ks, bits(out), ys,
                        out_fp8 ? static_cast<uint8_t*>(out_fp8->data_ptr()) : nullptr, ys,
                        scales ? static_cast<float*>(scales->data_ptr()) : nullptr,
                        static_cast<int32_t>(group), c.stream()));
}

void build_page_tables(const Tensor& cached, const Tensor& fresh, int64_t page_size, const Tensor& tables,
                       const Tensor& free_pages, const Tensor& free_count, const Tensor& seq_lens,
                       const Tensor& cu_q, const Tensor& positions, const Tensor& slots,
                       const OptTensor& free_count_out, const OptTensor& err_word) {
  need_dim("cached_lens", cached, 1, "a vector");
  need_dim("positions", positions, 1, "a vector");
  const int64_t B = cached.size(0), T = positions.size(0);
  const Tensor& left = free_count_out ? *free_count_out : free_count;
  Check c;
  c.dense("cached_lens", cached, at::kInt, {B});
  c.dense("new_lens", fresh, at::kInt, {B});
  c.dense("free_pages", free_pages, at::kInt, {-1});
  c.dense("free_count", free_count, at::kInt, {1});
  c.dense("free_count_out", left, at::kInt, {1});
  c.dense("seq_lens", seq_lens, at::kInt, {B});
  c.dense("cu_q", cu_q, at::kInt, {B + 1});
  c.dense("positions", positions, at::kInt, {T});
  c.dense("slot_mapping", slots, at::kLong, {T});
  const int64_t ts = c.table(tables, B);
  done("lm_build_page_tables",
       lib.build_page_tables(ints(cached), ints(fresh), narrow("requests", B), narrow("page_size", page_size),
                             ints(tables), ts, narrow("block_tables", tables.size(1)), ints(free_pages),
                             narrow("free_pages", free_pages.size(0)), ints(free_count), ints(left),
                             ints(seq_lens), ints(cu_q), ints(positions),
                             static_cast<int64_t*>(slots.data_ptr()), T, c.err(err_word), c.stream()));
}

void release_pages(const Tensor& rows, const Tensor& cached, int64_t page_size, const Tensor& tables,
                   const Tensor& free_pages, const Tensor& free_count, const OptTensor& err_word) {
  need_dim("block_tables", tables, 2, "a matrix");
  const int64_t B = tables.size(0);
  Check c;
  c.dense("rows", rows, at::kInt, {-1});
  c.dense("cached_lens", cached, at::kInt, {B});
  c.dense("free_pages", free_pages, at::kInt, {-1});
  c.dense("free_count", free_count, at::kInt, {1});
  const int64_t ts = c.table(tables, B);
  done("lm_release_pages",
       lib.release_pages(ints(rows), narrow("rows", rows.size(0)), ints(cached), narrow("requests", B),
                         narrow("page_size", page_size), ints(tables), ts,
                         narrow("block_tables", tables.size(1)), ints(free_pages),
                         narrow("free_pages", free_pages.size(0)), ints(free_count), c.err(err_word),
                         c.stream()));
}

void check_caches(Check& c, const Tensor& k, const Tensor& v) {
  need_dim("k_cache", k, 4, "[pages, page_size, kv_heads, head_dim]");
  c.heads("k_cache", k, k.sizes());
  c.heads("v_cache", v, k.sizes());
}

void rope_cache_write(const Tensor& qkv, const Tensor& positions, const Tensor& slots, const Tensor& cos_sin,
                      const Tensor& k, const Tensor& v, const Tensor& q_out, const OptTensor& q_weight,
                      const OptTensor& k_weight, double eps, bool interleaved, const OptTensor& err_word) {
  Check c;
  check_caches(c, k, v);
  need_dim("q_out", q_out, 3, "[tokens, heads, head_dim]");
  const int64_t T = q_out.size(0), Hq = q_out.size(1), Hkv = k.size(2), D = k.size(3);
  const int64_t qs = c.rows("qkv", qkv, at::kBFloat16, {T, (Hq + 2 * Hkv) * D});
  c.heads("q_out", q_out, {T, Hq, D});
  c.dense("positions", positions, at::kInt, {T});
  c.dense("slot_mapping", slots, at::kLong, {T});
  c.dense("cos_sin", cos_sin, at::kFloat, {-1, -1});
  if (q_weight) c.dense("q_norm_weight", *q_weight, at::kBFloat16, {D});
  if (k_weight) c.dense("k_norm_weight", *k_weight, at::kBFloat16, {D});
  done("lm_rope_cache_write",
       lib.rope_cache_write(bits(qkv), T == 1 ? 0 : qs, ints(positions), static_cast<const int64_t*>(slots.data_ptr()), T,
                            narrow("heads", Hq), narrow("heads", Hkv), narrow("head_dim", D),
                            static_cast<const float*>(cos_sin.data_ptr()), narrow("cos_sin", cos_sin.size(0)),
                            narrow("cos_sin", cos_sin.size(1)), interleaved ? 1 : 0, bits(q_weight),
                            bits(k_weight), static_cast<float>(eps), bits(q_out), stride(q_out, 0),
                            stride(q_out, 1), bits(k), stride(k, 0), stride(k, 1), stride(k, 2), bits(v),
                            stride(v, 0), stride(v, 1), stride(v, 2), k.size(0), narrow("page_size", k.size(1)),
                            c.err(err_word), c.stream()));
}

void paged_attention(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& tables,
                     const Tensor& seq_lens, const Tensor& cu_q, const Tensor& out, int64_t max_q_len,
                     const Tensor& workspace, std::optional<double> scale, int64_t window, const OptTensor& lse,
                     const OptTensor& err_word) {
  Check c;
  check_caches(c, k, v);
  need_dim("q", q, 3, "[tokens, heads, head_dim]");
  need_dim("block_tables", tables, 2, "a matrix");
  const int64_t T = q.size(0), Hq = q.size(1), D = k.size(3), B = tables.size(0);
  c.heads("q", q, {T, Hq, D});
  c.heads("out", out, {T, Hq, D});
  const int64_t ts = c.table(tables, B);
  c.dense("seq_lens", seq_lens, at::kInt, {B});
  c.dense("cu_q", cu_q, at::kInt, {B + 1});
  c.dense("workspace", workspace, at::kByte, {-1});
  if (lse) c.dense("lse", *lse, at::kFloat, {T, Hq});
  done("lm_paged_attention",
       lib.paged_attention(bits(q), stride(q, 0), stride(q, 1), bits(k), stride(k, 0), stride(k, 1),
                           stride(k, 2, D), bits(v), stride(v, 0), stride(v, 1), stride(v, 2, D), k.size(0),
                           narrow("page_size", k.size(1)), ints(tables), ts,
                           narrow("block_tables", tables.size(1)), ints(seq_lens), ints(cu_q),
                           narrow("requests", B), T, narrow("heads", Hq), narrow("heads", k.size(2)),
                           narrow("head_dim", D), narrow("max_q_len", max_q_len),
                           static_cast<float>(scale ? *scale : 1.0 / std::sqrt(static_cast<double>(D))),
                           narrow("window", window), bits(out), stride(out, 0), stride(out, 1),
                           lse ? static_cast<float*>(lse->data_ptr()) : nullptr, workspace.data_ptr(),
                           workspace.numel(), c.err(err_word), c.stream()));
}

}  // namespace

PYBIND11_MODULE(_decoder_ops, m) {
  m.attr("built_for") = LM_BUILT_FOR;
  m.def("bind", &bind);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("build_page_tables", &build_page_tables);
  m.def("release_pages", &release_pages);
  m.def("rope_cache_write", &rope_cache_write);
  m.def("paged_attention", &paged_attention);
}

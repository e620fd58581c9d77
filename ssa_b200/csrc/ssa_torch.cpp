// ssa_torch.cpp -- the block cache's operators for torch tensors, as a Python
// extension module (ssa_b200._ssa_torch). It checks the tensors, allocates
// results and workspace, and calls the C ABI (include/ssa_b200.h) on the
// current stream; ssa_b200/ops.py documents the operators.
//
// A decoding step makes a few launches of a few microseconds each for every
// layer, so the way from Python to the launch counts: through ctypes one such
// call took 14 to 24 us, through this module it takes 5 to 9, launch included.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <string>
#include <tuple>

#include "../../include/ssa_b200.h"

namespace {

using at::Tensor;
using c10::optional;

[[noreturn]] void raise(PyObject* type, const std::string& msg) {
  PyErr_SetString(type, msg.c_str());
  throw py::error_already_set();
}

// The exceptions of ssa_b200._lib.check.
void check(int rc, const char* what) {
  if (rc == SSA_OK) return;
  const std::string msg = std::string(what) + ": " + ssa_last_error();
  if (rc == SSA_ERR_INVALID || rc == SSA_ERR_WORKSPACE) raise(PyExc_ValueError, msg);
  if (rc == SSA_ERR_UNSUPPORTED) raise(PyExc_NotImplementedError, msg);
  raise(py::module_::import("ssa_b200._lib").attr("SSAError").ptr(), msg);
}

void need_cuda(const Tensor& t) {
  if (!t.is_cuda())
    raise(PyExc_RuntimeError, "ssa_b200 runs on CUDA tensors only (there is no CPU path); got a tensor on " + t.device().str());
}

void no_gradient(const Tensor& t, const char* what) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    raise(PyExc_RuntimeError, std::string(what) + " has no gradient: call it under torch.no_grad()");
  if (t._fw_grad(/*level=*/0).defined())  // a dual tensor: no_grad() does not end forward mode
    raise(PyExc_RuntimeError, std::string(what) + " has no gradient: its tensors may not have tangents (forward mode)");
}

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kFloat) return SSA_F32;
  if (t.scalar_type() == at::kBFloat16) return SSA_BF16;
  raise(PyExc_NotImplementedError,
        std::string("ssa_b200 kernels take float32 or bfloat16 tensors, got ") + toString(t.scalar_type()));
}

// Cache buffers are read and written where they lie: their type, shape,
// device and contiguity are checked, never mended by a copy.
void* buffer(const char* name, const Tensor& t, at::ScalarType type, at::IntArrayRef shape, const Tensor& like) {
  if (t.scalar_type() != type || t.sizes() != shape || t.device() != like.device() || !t.is_contiguous()) {
    std::ostringstream s;
    s << name << " must be a contiguous " << toString(type) << " tensor of shape " << shape << " on " << like.device()
      << ", got " << toString(t.scalar_type()) << " " << t.sizes() << (t.is_contiguous() ? "" : " (strided)") << " on "
      << t.device();
    raise(PyExc_ValueError, s.str());
  }
  return t.data_ptr();
}

// A (B, heads, n, d) tensor with rows the kernels can read: contiguous last
// axis, strides of whole vectors; copied only where it is not so.
Tensor rows(const Tensor& t) {
  if (t.dim() != 4) {
    std::ostringstream s;
    s << "expected a 4-D tensor, got shape " << t.sizes();
    raise(PyExc_ValueError, s.str());
  }
  const auto st = t.strides();
  bool ok = st[3] == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % (t.element_size() == 4 ? 16 : 8) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && st[i] % 4 == 0;
  return ok ? t : t.contiguous();
}

std::string shape_of(const Tensor& t) {
  std::ostringstream s;
  s << t.sizes();
  return s.str();
}

int32_t i32(int64_t v, const char* name) {
  if (v < 0 || v > INT32_MAX) raise(PyExc_ValueError, std::string(name) + " is out of range: " + std::to_string(v));
  return (int32_t)v;
}

struct Lens {
  const int32_t *table, *start, *lens;
};
Lens lens_of(const Tensor& table, const Tensor& start, const Tensor& lens, int64_t B, const Tensor& like) {
  if (table.dim() != 2 || table.size(0) != B)
    raise(PyExc_ValueError, "table (B, max_blocks) with B = " + std::to_string(B) + " expected, got " + shape_of(table));
  return {static_cast<int32_t*>(buffer("table", table, at::kInt, {B, table.size(1)}, like)),
          static_cast<int32_t*>(buffer("start", start, at::kInt, {B}, like)),
          static_cast<int32_t*>(buffer("lens", lens, at::kInt, {B}, like))};
}

// Uninitialised tensors on t's device, without the dispatcher's way there.
Tensor fresh(const Tensor& t, at::ScalarType type, at::IntArrayRef shape) {
  return at::detail::empty_cuda(shape, type, t.device(), c10::nullopt);
}
// (B, heads, n, d) as a view of (B, n, heads, d): the layout a projection reads.
Tensor fresh_heads(const Tensor& t, int64_t B, int64_t heads, int64_t n, int64_t d) {
  return at::detail::empty_strided_cuda({B, heads, n, d}, {n * heads * d, d, heads * d, 1}, t.scalar_type(), t.device());
}

void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

std::tuple<Tensor, Tensor, Tensor> cache_reserve(const Tensor& lens, const Tensor& new_lens, const Tensor& table,
                                                 const Tensor& free_pages, const Tensor& state, int64_t block_size,
                                                 const optional<std::tuple<Tensor, Tensor, Tensor>>& out) {
  need_cuda(lens);
  if (lens.dim() != 1 || table.dim() != 2 || free_pages.dim() != 1)
    raise(PyExc_ValueError, "cache_reserve: lens (B,), table (B, max_blocks) and free (num_pages,) expected");
  const int64_t B = lens.size(0), mb = table.size(1), P = free_pages.size(0);
  Tensor start, after, st;
  if (out) {
    std::tie(start, after, st) = *out;
  } else {
    start = fresh(lens, at::kInt, {B});
    after = fresh(lens, at::kInt, {B});
    st = fresh(lens, at::kInt, {2});
  }
  const auto p = [&](const char* name, const Tensor& t, at::IntArrayRef shape) {
    return static_cast<int32_t*>(buffer(name, t, at::kInt, shape, lens));
  };
  int32_t* pl = p("lens", lens, {B});
  int32_t* pn = p("new_lens", new_lens, {B});
  int32_t* pt = p("table", table, {B, mb});
  int32_t* pf = p("free", free_pages, {P});
  int32_t* ps = p("state", state, {2});
  int32_t* os = p("start (out)", start, {B});
  int32_t* ol = p("lens (out)", after, {B});
  int32_t* oc = p("state (out)", st, {2});
  const c10::cuda::OptionalCUDAGuard guard(lens.device());
  if (B)
    check(ssa_cache_reserve(i32(B, "B"), i32(mb, "max_blocks"), i32(block_size, "block_size"), i32(P, "num_pages"), pl, pn, pt,
                            pf, ps, os, ol, oc, stream_of(lens)),
          "ssa_cache_reserve");
  else if (!st.is_same(state))
    st.copy_(state);
  return {start, after, st};
}

optional<std::tuple<Tensor, Tensor>> cache_append(const Tensor& k_in, const Tensor& v_in, const Tensor& k_codes,
                                                  const Tensor& v_codes, const Tensor& amax, const Tensor& bounds,
                                                  const Tensor& tail, const Tensor& table, const Tensor& start,
                                                  const Tensor& lens, bool want_values) {
  need_cuda(k_in);
  need_cuda(v_in);
  no_gradient(k_in, "cache_append");
  no_gradient(v_in, "cache_append");
  if (k_in.scalar_type() != v_in.scalar_type() || k_in.sizes() != v_in.sizes() || k_in.device() != v_in.device())
    raise(PyExc_ValueError, "k " + shape_of(k_in) + " and v " + shape_of(v_in) + " differ in type, shape or device");
  const Tensor k = rows(k_in), v = rows(v_in);
  const int64_t B = k.size(0), n_kv = k.size(1), n = k.size(2), d = k.size(3);
  if (k_codes.dim() != 4) raise(PyExc_ValueError, "k_codes (num_pages, n_kv, block_size, d) expected, got " + shape_of(k_codes));
  const int64_t P = k_codes.size(0), bs = k_codes.size(2);
  const int dt = dtype_code(k);
  auto* pk = static_cast<int8_t*>(buffer("k_codes", k_codes, at::kChar, {P, n_kv, bs, d}, k));
  auto* pv = static_cast<int8_t*>(buffer("v_codes", v_codes, at::kChar, {P, n_kv, bs, d}, k));
  auto* pa = static_cast<float*>(buffer("amax", amax, at::kFloat, {P, n_kv, 2}, k));
  auto* pb = static_cast<int8_t*>(buffer("bounds", bounds, at::kChar, {P, n_kv, 2, d}, k));
  void* pt = buffer("tail", tail, k.scalar_type(), {B, n_kv, 2, bs, d}, k);
  const Lens ln = lens_of(table, start, lens, B, k);
  const c10::cuda::OptionalCUDAGuard guard(k.device());
  Tensor kv, vv;
  ssa_cache_params p = {};
  if (want_values) {
    kv = fresh_heads(k, B, n_kv, n, d);
    vv = fresh_heads(k, B, n_kv, n, d);
    p.o_sb = n * n_kv * d; p.o_sh = d; p.o_sn = n_kv * d;
  }
  if (B && n) {
    p.B = i32(B, "B"); p.H = p.n_kv = i32(n_kv, "n_kv"); p.n = i32(n, "n"); p.d = i32(d, "d");
    p.dtype = dt; p.block_size = i32(bs, "block_size"); p.max_blocks = i32(table.size(1), "max_blocks");
    p.num_pages = i32(P, "num_pages");
    p.k_sb = k.stride(0); p.k_sh = k.stride(1); p.k_sn = k.stride(2);
    p.v_sb = v.stride(0); p.v_sh = v.stride(1); p.v_sn = v.stride(2);
    check(ssa_cache_append(&p, k.data_ptr(), v.data_ptr(), pk, pv, pa, pb, pt, ln.table, ln.start, ln.lens,
                           want_values ? kv.data_ptr() : nullptr, want_values ? vv.data_ptr() : nullptr, stream_of(k)),
          "ssa_cache_append");
  }
  if (!want_values) return c10::nullopt;
  return std::make_tuple(kv, vv);
}

Tensor cache_select(const Tensor& q_in, const Tensor& bounds, const Tensor& amax, const Tensor& table, const Tensor& start,
                    const Tensor& lens, int64_t top, int64_t block_size, int64_t sink, int64_t local) {
  need_cuda(q_in);
  const Tensor q = rows(q_in);
  const int64_t B = q.size(0), H = q.size(1), n = q.size(2), d = q.size(3);
  if (bounds.dim() != 4) raise(PyExc_ValueError, "bounds (num_pages, n_kv, 2, d) expected, got " + shape_of(bounds));
  const int64_t P = bounds.size(0), n_kv = bounds.size(1);
  const int dt = dtype_code(q);
  auto* pb = static_cast<int8_t*>(buffer("bounds", bounds, at::kChar, {P, n_kv, 2, d}, q));
  auto* pa = static_cast<float*>(buffer("amax", amax, at::kFloat, {P, n_kv, 2}, q));
  const Lens ln = lens_of(table, start, lens, B, q);
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const Tensor out = fresh(q, at::kInt, {B, n, n_kv, i32(top, "top")});
  if (B && n) {
    ssa_cache_params p = {};
    p.B = i32(B, "B"); p.H = i32(H, "H"); p.n_kv = i32(n_kv, "n_kv"); p.n = i32(n, "n"); p.d = i32(d, "d");
    p.dtype = dt; p.block_size = i32(block_size, "block_size"); p.max_blocks = i32(table.size(1), "max_blocks");
    p.num_pages = i32(P, "num_pages");
    p.top = (int32_t)top; p.sink = i32(sink, "sink"); p.local = i32(local, "local"); p.causal = 1;
    p.q_sb = q.stride(0); p.q_sh = q.stride(1); p.q_sn = q.stride(2);
    check(ssa_cache_select(&p, q.data_ptr(), pb, pa, ln.table, ln.start, ln.lens, out.data_ptr<int32_t>(), stream_of(q)),
          "ssa_cache_select");
  }
  return out;
}

std::tuple<Tensor, optional<Tensor>> cache_attention(const Tensor& q_in, const Tensor& k_codes, const Tensor& v_codes,
                                                     const Tensor& amax, const Tensor& table, const Tensor& start,
                                                     const Tensor& lens, double scale, const optional<Tensor>& blocks,
                                                     bool causal, bool want_lse) {
  need_cuda(q_in);
  no_gradient(q_in, "cache_attention");
  const Tensor q = rows(q_in);
  const int64_t B = q.size(0), H = q.size(1), n = q.size(2), d = q.size(3);
  if (k_codes.dim() != 4) raise(PyExc_ValueError, "k_codes (num_pages, n_kv, block_size, d) expected, got " + shape_of(k_codes));
  const int64_t P = k_codes.size(0), n_kv = k_codes.size(1), bs = k_codes.size(2);
  ssa_cache_params p = {};
  p.dtype = dtype_code(q);
  auto* pk = static_cast<int8_t*>(buffer("k_codes", k_codes, at::kChar, {P, n_kv, bs, d}, q));
  auto* pv = static_cast<int8_t*>(buffer("v_codes", v_codes, at::kChar, {P, n_kv, bs, d}, q));
  auto* pa = static_cast<float*>(buffer("amax", amax, at::kFloat, {P, n_kv, 2}, q));
  const Lens ln = lens_of(table, start, lens, B, q);
  const int32_t* pl = nullptr;
  if (blocks) {
    if (blocks->dim() != 4) raise(PyExc_ValueError, "blocks (B, n, n_kv, top) expected, got " + shape_of(*blocks));
    p.top = i32(blocks->size(3), "top");
    pl = static_cast<int32_t*>(buffer("blocks", *blocks, at::kInt, {B, n, n_kv, blocks->size(3)}, q));
  }
  const c10::cuda::OptionalCUDAGuard guard(q.device());
  const Tensor out = fresh_heads(q, B, H, n, d);
  optional<Tensor> lse;
  if (want_lse) lse = fresh(q, at::kFloat, {B, H, n});
  if (B && n) {
    p.B = i32(B, "B"); p.H = i32(H, "H"); p.n_kv = i32(n_kv, "n_kv"); p.n = i32(n, "n"); p.d = i32(d, "d");
    p.block_size = i32(bs, "block_size"); p.max_blocks = i32(table.size(1), "max_blocks"); p.num_pages = i32(P, "num_pages");
    p.causal = causal; p.scale = (float)scale;
    p.q_sb = q.stride(0); p.q_sh = q.stride(1); p.q_sn = q.stride(2);
    p.o_sb = n * H * d; p.o_sh = d; p.o_sn = H * d;
    const size_t bytes = ssa_cache_attn_workspace_size(&p, pl != nullptr);
    const Tensor ws = fresh(q, at::kByte, {(int64_t)(bytes ? bytes : 1)});
    check(ssa_cache_attn(&p, q.data_ptr(), pk, pv, pa, ln.table, ln.start, ln.lens, pl, out.data_ptr(),
                         want_lse ? lse->data_ptr<float>() : nullptr, ws.data_ptr(), bytes, stream_of(q)),
          "ssa_cache_attn");
  }
  return {out, lse};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("cache_reserve", &cache_reserve);
  m.def("cache_append", &cache_append);
  m.def("cache_select", &cache_select);
  m.def("cache_attention", &cache_attention);
}

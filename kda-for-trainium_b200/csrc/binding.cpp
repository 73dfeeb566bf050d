// Python binding of the attention entry points (local, packed, 4-bit cache): argument checks, output
// and workspace allocation (torch's caching allocator), current stream, and
// the C ABI call in one native function per operator.  A decode step makes two
// of these calls per layer on kernels of a few microseconds; the same checks
// in Python and ctypes cost 23 to 29 us a call, here 5 to 7 (the backward
// passes, with two and three launches: 10 to 13).
// The semantics are those of the functions in kda/ops.py that call it.
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <string>
#include <tuple>

#include "kda.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = c10::optional<Tensor>;

namespace {

constexpr auto kBf16 = at::kBFloat16;
constexpr auto kF32 = at::kFloat;

[[noreturn]] void value_error(const std::string& what) { throw py::value_error(what); }

std::string shape_str(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + (s[i] < 0 ? std::string("*") : std::to_string(s[i]));
  return r + (s.size() == 1 ? ",)" : ")");
}

void check_kind(const Tensor& t, const char* name, at::ScalarType dtype, bool or_f32, const at::Device* dev) {
  if (!t.is_cuda()) value_error(std::string(name) + " must be a CUDA tensor");
  const auto st = t.scalar_type();
  if (st != dtype && !(or_f32 && st == kF32))
    value_error(std::string(name) + " must have dtype " + c10::toString(dtype) + (or_f32 ? " or Float" : "") + ", got " +
                c10::toString(st));
  if (dev && t.device() != *dev)
    value_error(std::string(name) + " is on " + t.device().str() + ", expected " + dev->str());
}

// want: -1 matches any size
void check_shape(const Tensor& t, const char* name, at::IntArrayRef want) {
  const auto got = t.sizes();
  bool ok = got.size() == want.size();
  for (size_t i = 0; ok && i < got.size(); ++i) ok = want[i] < 0 || want[i] == got[i];
  if (!ok) value_error(std::string(name) + " must have shape " + shape_str(want) + ", got " + shape_str(got));
}

void check_dense(const Tensor& t, const char* name, at::ScalarType dtype, at::IntArrayRef want, const at::Device& dev) {
  check_kind(t, name, dtype, false, &dev);
  check_shape(t, name, want);
  if (!t.is_contiguous()) value_error(std::string(name) + " must be contiguous");
}

struct Strides {
  int64_t s[3];
};

// A tensor of head rows that may be a view (a slice of a packed projection, a
// layer of a cache): the last axis contiguous, every row on 16 bytes, no
// expanded axis.  Returns its other strides; an axis of one entry counts as 0.
Strides check_rows(const Tensor& t, const char* name, at::ScalarType dtype, bool or_f32, at::IntArrayRef want,
                   const at::Device* dev = nullptr) {
  check_kind(t, name, dtype, or_f32, dev);
  check_shape(t, name, want);
  if (t.numel() == 0) value_error(std::string(name) + " must not be empty, got shape " + shape_str(t.sizes()));
  const int64_t per16 = 16 / t.element_size();
  const int n = static_cast<int>(t.dim()) - 1;
  bool ok = t.stride(n) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  Strides r{};
  for (int i = 0; i < n; ++i) {
    r.s[i] = t.size(i) > 1 ? t.stride(i) : 0;
    ok = ok && (t.size(i) == 1 || (r.s[i] > 0 && r.s[i] % per16 == 0));
  }
  if (!ok)
    value_error(std::string(name) +
                " must have a contiguous last axis, rows on 16-byte boundaries and no expanded axis, got strides " +
                shape_str(t.strides()));
  return r;
}

// From the caching allocator without the dispatcher: half of at::empty's time.
Tensor empty(at::IntArrayRef shape, at::ScalarType dtype, const at::Device& dev) {
  return Tensor(at::detail::empty_cuda(shape, dtype, dev, c10::nullopt));
}

Tensor out_or_empty(const OptTensor& out, const char* name, at::IntArrayRef shape, at::ScalarType dtype,
                    const at::Device& dev) {
  if (!out) return empty(shape, dtype, dev);
  check_dense(*out, name, dtype, shape, dev);
  return *out;
}

// The caller's workspace (on `dev`, at least n bytes, which lie together) or a fresh one.
Tensor workspace_or_empty(const OptTensor& ws, size_t n, const at::Device& dev) {
  if (!ws) return empty({static_cast<int64_t>(n > 0 ? n : 1)}, at::kByte, dev);
  if (ws->device() != dev)
    value_error("workspace is on " + ws->device().str() + ", the operands on " + dev.str());
  if (!ws->is_contiguous()) value_error("workspace must be contiguous");
  const size_t have = static_cast<size_t>(ws->numel()) * ws->element_size();
  if (have < n) value_error("workspace of " + std::to_string(n) + " bytes required, got " + std::to_string(have));
  return *ws;
}

void* stream(const at::Device& dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

void done(const char* fn, kda_status st) {
  if (st == KDA_OK) return;
  const std::string detail = kda_last_error();
  if (st == KDA_INVALID_ARG) value_error(std::string(fn) + ": " + detail);
  py::object cls = py::module_::import("kda._lib").attr("KdaError");
  PyErr_SetObject(cls.ptr(), cls(fn, static_cast<int>(st), detail).ptr());
  throw py::error_already_set();
}

template <typename T>
T* ptr(const Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
template <typename T>
T* ptr(const OptTensor& t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

// What the three norm entry points check alike.
struct NormArgs {
  Strides q, k;
  int64_t B, S, QH, KH, D, P;
  at::Device dev;
  at::ScalarType dtype;
};

NormArgs norm_args(const Tensor& q, const Tensor& k, const Tensor& gq, const Tensor& gk, const Tensor& table,
                   const OptTensor& positions, bool or_f32) {
  const Strides qs = check_rows(q, "q", kBf16, or_f32, {-1, -1, -1, -1});
  const int64_t B = q.size(0), S = q.size(1), D = q.size(3);
  if (D != 64 && D != 128 && D != 256) value_error("head_dim must be 64, 128 or 256, got " + std::to_string(D));
  const at::Device dev = q.device();
  const Strides ks = check_rows(k, "k", q.scalar_type(), false, {B, S, -1, D}, &dev);
  check_dense(gq, "gq", kF32, {D}, dev);
  check_dense(gk, "gk", kF32, {D}, dev);
  check_dense(table, "table", kF32, {-1, D / 2, 2}, dev);
  if (positions) check_dense(*positions, "positions", at::kInt, {B, S}, dev);
  return {qs, ks, B, S, q.size(2), k.size(2), D, table.size(0), dev, q.scalar_type()};
}

std::tuple<Tensor, Tensor> qk_norm_rope(const Tensor& q, const Tensor& k, const Tensor& gq, const Tensor& gk,
                                        const Tensor& table, const OptTensor& positions, double eps,
                                        const OptTensor& q_out, const OptTensor& k_out) {
  const NormArgs a = norm_args(q, k, gq, gk, table, positions, true);
  const c10::cuda::CUDAGuard guard(a.dev);
  Tensor qo = out_or_empty(q_out, "q_out", {a.B, a.S, a.QH, a.D}, a.dtype, a.dev);
  Tensor ko = out_or_empty(k_out, "k_out", {a.B, a.S, a.KH, a.D}, a.dtype, a.dev);
  done("kda_qk_norm_rope",
       kda_qk_norm_rope(q.data_ptr(), k.data_ptr(), ptr<float>(gq), ptr<float>(gk), ptr<float>(table), a.P,
                        ptr<int>(positions), static_cast<float>(eps), qo.data_ptr(), ko.data_ptr(), a.B, a.S, a.QH,
                        a.KH, a.D, a.q.s, a.k.s, a.dtype == kF32, stream(a.dev)));
  return {qo, ko};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> qk_norm_rope_backward(const Tensor& dq_out, const Tensor& dk_out,
                                                                 const Tensor& q, const Tensor& k, const Tensor& gq,
                                                                 const Tensor& gk, const Tensor& table,
                                                                 const OptTensor& positions, double eps,
                                                                 const OptTensor& workspace) {
  const NormArgs a = norm_args(q, k, gq, gk, table, positions, true);
  check_dense(dq_out, "dq_out", a.dtype, {a.B, a.S, a.QH, a.D}, a.dev);
  check_dense(dk_out, "dk_out", a.dtype, {a.B, a.S, a.KH, a.D}, a.dev);
  const c10::cuda::CUDAGuard guard(a.dev);
  Tensor dq = empty({a.B, a.S, a.QH, a.D}, a.dtype, a.dev), dk = empty({a.B, a.S, a.KH, a.D}, a.dtype, a.dev);
  Tensor dgq = empty({a.D}, kF32, a.dev), dgk = empty({a.D}, kF32, a.dev);
  const int f32 = a.dtype == kF32;
  const size_t nb = kda_qk_norm_rope_backward_workspace_size(a.B, a.S, a.QH, a.KH, a.D, f32);
  Tensor ws = workspace_or_empty(workspace, nb, a.dev);
  done("kda_qk_norm_rope_backward",
       kda_qk_norm_rope_backward(dq_out.data_ptr(), dk_out.data_ptr(), q.data_ptr(), k.data_ptr(), ptr<float>(gq),
                                 ptr<float>(gk), ptr<float>(table), a.P, ptr<int>(positions),
                                 static_cast<float>(eps), dq.data_ptr(), dk.data_ptr(), ptr<float>(dgq),
                                 ptr<float>(dgk), a.B, a.S, a.QH, a.KH, a.D, a.q.s, a.k.s, f32, ws.data_ptr(), nb,
                                 stream(a.dev)));
  return {dq, dk, dgq, dgk};
}

Tensor qk_norm_rope_append(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& gq, const Tensor& gk,
                           const Tensor& table, const Tensor& k_cache, const Tensor& v_cache, const Tensor& lengths,
                           double eps, const OptTensor& q_out) {
  const NormArgs a = norm_args(q, k, gq, gk, table, c10::nullopt, false);
  const Strides vs = check_rows(v, "v", kBf16, false, {a.B, a.S, a.KH, a.D}, &a.dev);
  const Strides kc = check_rows(k_cache, "k_cache", kBf16, false, {a.B, -1, a.KH, a.D}, &a.dev);
  const int64_t T = k_cache.size(1);
  const Strides vc = check_rows(v_cache, "v_cache", kBf16, false, {a.B, T, a.KH, a.D}, &a.dev);
  check_dense(lengths, "lengths", at::kInt, {a.B}, a.dev);
  const c10::cuda::CUDAGuard guard(a.dev);
  Tensor qo = out_or_empty(q_out, "q_out", {a.B, a.S, a.QH, a.D}, kBf16, a.dev);
  done("kda_qk_norm_rope_append_bf16",
       kda_qk_norm_rope_append_bf16(q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr<float>(gq), ptr<float>(gk),
                                    ptr<float>(table), a.P, ptr<int>(lengths), static_cast<float>(eps),
                                    qo.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), T, a.B, a.S, a.QH, a.KH,
                                    a.D, a.q.s, a.k.s, vs.s, kc.s, vc.s, stream(a.dev)));
  return qo;
}

struct WindowArgs {
  Strides q, k, v;
  int64_t B, S, QH, KH, D;
  at::Device dev;
};

void check_groups(int64_t QH, int64_t KH) {
  if (QH % KH)
    value_error("query heads " + std::to_string(QH) + " must be a multiple of kv heads " + std::to_string(KH));
}

WindowArgs window_args(const Tensor& q, const Tensor& k, const Tensor& v) {
  const Strides qs = check_rows(q, "q", kBf16, false, {-1, -1, -1, 128});
  const int64_t B = q.size(0), S = q.size(1);
  const at::Device dev = q.device();
  const Strides ks = check_rows(k, "k", kBf16, false, {B, S, -1, 128}, &dev);
  const Strides vs = check_rows(v, "v", kBf16, false, {B, S, k.size(2), 128}, &dev);
  check_groups(q.size(2), k.size(2));
  return {qs, ks, vs, B, S, q.size(2), k.size(2), 128, dev};
}

std::tuple<Tensor, OptTensor> gqa_window(const Tensor& q, const Tensor& k, const Tensor& v, int64_t window,
                                         int64_t sinks, const OptTensor& out, bool with_lse) {
  const WindowArgs a = window_args(q, k, v);
  const c10::cuda::CUDAGuard guard(a.dev);
  Tensor y = out_or_empty(out, "out", {a.B, a.S, a.QH, a.D}, kBf16, a.dev);
  OptTensor lse;
  if (with_lse) lse = empty({a.B, a.QH, a.S}, kF32, a.dev);
  done("kda_gqa_window_bf16",
       kda_gqa_window_bf16(q.data_ptr(), k.data_ptr(), v.data_ptr(), y.data_ptr(), ptr<float>(lse), a.B, a.S, a.QH,
                           a.KH, a.D, window, sinks, a.q.s, a.k.s, a.v.s, stream(a.dev)));
  return {y, lse};
}

std::tuple<Tensor, Tensor, Tensor> gqa_window_backward(const Tensor& dout, const Tensor& q, const Tensor& k,
                                                       const Tensor& v, const Tensor& out, const Tensor& lse,
                                                       int64_t window, int64_t sinks, const OptTensor& workspace) {
  const WindowArgs a = window_args(q, k, v);
  check_dense(dout, "dout", kBf16, {a.B, a.S, a.QH, a.D}, a.dev);
  check_dense(out, "out", kBf16, {a.B, a.S, a.QH, a.D}, a.dev);
  check_dense(lse, "lse", kF32, {a.B, a.QH, a.S}, a.dev);
  const c10::cuda::CUDAGuard guard(a.dev);
  Tensor dq = empty({a.B, a.S, a.QH, a.D}, kBf16, a.dev);
  Tensor dk = empty({a.B, a.S, a.KH, a.D}, kBf16, a.dev), dv = empty({a.B, a.S, a.KH, a.D}, kBf16, a.dev);
  const size_t nb = kda_gqa_window_backward_workspace_size(a.B, a.S, a.QH, a.KH, a.D, window, sinks);
  Tensor ws = workspace_or_empty(workspace, nb, a.dev);
  done("kda_gqa_window_backward_bf16",
       kda_gqa_window_backward_bf16(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                    ptr<float>(lse), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), a.B, a.S, a.QH,
                                    a.KH, a.D, window, sinks, a.q.s, a.k.s, a.v.s, ws.data_ptr(), nb,
                                    stream(a.dev)));
  return {dq, dk, dv};
}

Tensor gqa_window_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& lengths,
                         int64_t window, int64_t sinks, const OptTensor& out) {
  const Strides qs = check_rows(q, "q", kBf16, false, {-1, -1, 128});
  const int64_t B = q.size(0), QH = q.size(1), D = 128;
  const at::Device dev = q.device();
  const Strides ks = check_rows(k_cache, "k_cache", kBf16, false, {B, -1, -1, D}, &dev);
  const int64_t T = k_cache.size(1), KH = k_cache.size(2);
  const Strides vs = check_rows(v_cache, "v_cache", kBf16, false, {B, T, KH, D}, &dev);
  check_groups(QH, KH);
  check_dense(lengths, "lengths", at::kInt, {B}, dev);
  const c10::cuda::CUDAGuard guard(dev);
  Tensor y = out_or_empty(out, "out", {B, QH, D}, kBf16, dev);
  done("kda_gqa_window_decode_bf16",
       kda_gqa_window_decode_bf16(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ptr<int>(lengths),
                                  y.data_ptr(), B, T, QH, KH, D, window, sinks, qs.s, ks.s, vs.s, stream(dev)));
  return y;
}

// ------------------------------------------------ packed sequences, 4-bit caches
Tensor packed_plan(const Tensor& offsets, int64_t tokens, const OptTensor& out) {
  check_kind(offsets, "offsets", at::kInt, false, nullptr);
  check_shape(offsets, "offsets", {-1});
  if (!offsets.is_contiguous()) value_error("offsets must be contiguous");
  const at::Device dev = offsets.device();
  const int64_t n = offsets.size(0) - 1;
  if (n < 1) value_error("offsets must have two entries or more, got " + std::to_string(n + 1));
  if (tokens < 1) value_error("tokens must be positive, got " + std::to_string(tokens));
  const size_t nb = kda_packed_plan_size(tokens, n);
  if (nb == 0) value_error("too many tokens or sequences: " + std::to_string(tokens) + " and " + std::to_string(n));
  const c10::cuda::CUDAGuard guard(dev);
  Tensor plan = out_or_empty(out, "out", {static_cast<int64_t>(nb / 4)}, at::kInt, dev);
  done("kda_packed_plan", kda_packed_plan(ptr<int>(offsets), n, tokens, plan.data_ptr(), nb, stream(dev)));
  // a backward that still holds the plan from before raises, as after any change in place
  if (out && !plan.is_inference()) plan.unsafeGetTensorImpl()->bump_version();
  return plan;
}

struct PackedArgs {
  Strides q, k, v;
  int64_t T, QH, KH, D;
  at::Device dev;
  size_t plan;  // bytes
};

PackedArgs packed_args(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& plan) {
  const Strides qs = check_rows(q, "q", kBf16, false, {-1, -1, 128});
  const int64_t T = q.size(0);
  const at::Device dev = q.device();
  const Strides ks = check_rows(k, "k", kBf16, false, {T, -1, 128}, &dev);
  const Strides vs = check_rows(v, "v", kBf16, false, {T, k.size(1), 128}, &dev);
  check_groups(q.size(1), k.size(1));
  check_dense(plan, "plan", at::kInt, {-1}, dev);
  return {qs, ks, vs, T, q.size(1), k.size(1), 128, dev, static_cast<size_t>(plan.numel()) * 4};
}

std::tuple<Tensor, OptTensor> gqa_packed(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& plan,
                                         const OptTensor& out, bool with_lse) {
  const PackedArgs a = packed_args(q, k, v, plan);
  const c10::cuda::CUDAGuard guard(a.dev);
  Tensor y = out_or_empty(out, "out", {a.T, a.QH, a.D}, kBf16, a.dev);
  OptTensor lse;
  if (with_lse) lse = empty({a.QH, a.T}, kF32, a.dev);
  done("kda_gqa_packed_bf16",
       kda_gqa_packed_bf16(q.data_ptr(), k.data_ptr(), v.data_ptr(), plan.data_ptr(), a.plan, y.data_ptr(),
                           ptr<float>(lse), !out, a.T, a.QH, a.KH, a.D, a.q.s, a.k.s, a.v.s, stream(a.dev)));
  return {y, lse};
}

std::tuple<Tensor, Tensor, Tensor> gqa_packed_backward(const Tensor& dout, const Tensor& q, const Tensor& k,
                                                       const Tensor& v, const Tensor& out, const Tensor& lse,
                                                       const Tensor& plan, const OptTensor& workspace) {
  const PackedArgs a = packed_args(q, k, v, plan);
  check_dense(dout, "dout", kBf16, {a.T, a.QH, a.D}, a.dev);
  check_dense(out, "out", kBf16, {a.T, a.QH, a.D}, a.dev);
  check_dense(lse, "lse", kF32, {a.QH, a.T}, a.dev);
  const c10::cuda::CUDAGuard guard(a.dev);
  Tensor dq = empty({a.T, a.QH, a.D}, kBf16, a.dev);
  Tensor dk = empty({a.T, a.KH, a.D}, kBf16, a.dev), dv = empty({a.T, a.KH, a.D}, kBf16, a.dev);
  const size_t nb = kda_gqa_packed_backward_workspace_size(a.T, a.plan, a.QH, a.KH, a.D);
  Tensor ws = workspace_or_empty(workspace, nb, a.dev);
  done("kda_gqa_packed_backward_bf16",
       kda_gqa_packed_backward_bf16(dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                    ptr<float>(lse), plan.data_ptr(), a.plan, dq.data_ptr(), dk.data_ptr(),
                                    dv.data_ptr(), 1, a.T, a.QH, a.KH, a.D, a.q.s, a.k.s, a.v.s, ws.data_ptr(), nb,
                                    stream(a.dev)));
  return {dq, dk, dv};
}

// A 4-bit cache (B, KH, blocks, bytes): its last two axes lie together, blocks start on 16
// bytes, no expanded axis.  Returns the group its block size stands for.
int64_t check_q4(const Tensor& t, const char* name, at::IntArrayRef want, const at::Device* dev, int64_t (&strides)[2]) {
  check_kind(t, name, at::kByte, false, dev);
  check_shape(t, name, want);
  if (t.numel() == 0) value_error(std::string(name) + " must not be empty, got shape " + shape_str(t.sizes()));
  int64_t group = 0;
  for (const int64_t g : {32, 64, 128})
    if (static_cast<int64_t>(kda_q4_block_bytes(g)) == t.size(3)) group = g;
  if (group == 0)
    value_error(std::string(name) + " must have blocks of 1280, 1152 or 1088 bytes (groups of 32, 64 or 128), got " +
                std::to_string(t.size(3)));
  bool ok = t.stride(3) == 1 && (t.size(2) == 1 || t.stride(2) == t.size(3)) &&
            reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
    ok = ok && (t.size(i) == 1 || (strides[i] > 0 && strides[i] % 16 == 0));
  }
  if (!ok)
    value_error(std::string(name) +
                " must have contiguous blocks on 16-byte boundaries and no expanded axis, got strides " +
                shape_str(t.strides()));
  return group;
}

void kv_append_q4(const Tensor& k, const Tensor& v, const Tensor& k_cache, const Tensor& v_cache,
                  const Tensor& lengths, const OptTensor& offsets) {
  Strides ks, vs;
  int64_t B, KH, tokens;
  if (offsets) {
    ks = check_rows(k, "k", kBf16, false, {-1, -1, 128});
    tokens = k.size(0), KH = k.size(1);
  } else {
    ks = check_rows(k, "k", kBf16, false, {-1, -1, -1, 128});
    tokens = k.size(0) * k.size(1), KH = k.size(2);
  }
  const at::Device dev = k.device();
  vs = check_rows(v, "v", kBf16, false, k.sizes(), &dev);
  if (offsets) {  // strides of token and head
    ks = {{0, ks.s[0], ks.s[1]}};
    vs = {{0, vs.s[0], vs.s[1]}};
  }
  int64_t kc[2], vc[2];
  const int64_t group = check_q4(k_cache, "k_cache", {offsets ? -1 : k.size(0), KH, -1, -1}, &dev, kc);
  B = k_cache.size(0);
  check_q4(v_cache, "v_cache", k_cache.sizes(), &dev, vc);
  check_dense(lengths, "lengths", at::kInt, {B}, dev);
  if (offsets) check_dense(*offsets, "offsets", at::kInt, {B + 1}, dev);
  const c10::cuda::CUDAGuard guard(dev);
  done("kda_kv_append_q4",
       kda_kv_append_q4(k.data_ptr(), v.data_ptr(), ptr<int>(offsets), ptr<int>(lengths), k_cache.data_ptr(),
                        v_cache.data_ptr(), tokens, B, k_cache.size(2), KH, 128, group, ks.s, vs.s, kc, vc,
                        stream(dev)));
}

Tensor kv_read_q4(const Tensor& cache, const OptTensor& out) {
  int64_t cs[2];
  const int64_t group = check_q4(cache, "cache", {-1, -1, -1, -1}, nullptr, cs);
  const at::Device dev = cache.device();
  const int64_t B = cache.size(0), KH = cache.size(1), n = cache.size(2);
  const c10::cuda::CUDAGuard guard(dev);
  Tensor y = out_or_empty(out, "out", {B, 16 * n, KH, 128}, kBf16, dev);
  done("kda_kv_read_q4", kda_kv_read_q4(cache.data_ptr(), y.data_ptr(), B, n, KH, 128, group, cs, stream(dev)));
  return y;
}

Tensor gqa_decode_q4(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& lengths,
                     const c10::optional<int64_t>& window, int64_t sinks, const OptTensor& out,
                     const OptTensor& workspace) {
  const Strides qs = check_rows(q, "q", kBf16, false, {-1, -1, 128});
  const int64_t B = q.size(0), QH = q.size(1), D = 128;
  const at::Device dev = q.device();
  int64_t kc[2], vc[2];
  const int64_t group = check_q4(k_cache, "k_cache", {B, -1, -1, -1}, &dev, kc);
  check_q4(v_cache, "v_cache", k_cache.sizes(), &dev, vc);
  const int64_t KH = k_cache.size(1), n = k_cache.size(2);
  check_groups(QH, KH);
  check_dense(lengths, "lengths", at::kInt, {B}, dev);
  const c10::cuda::CUDAGuard guard(dev);
  Tensor y = out_or_empty(out, "out", {B, QH, D}, kBf16, dev);
  const size_t nb = kda_gqa_decode_q4_workspace_size(QH, KH);
  Tensor ws = workspace_or_empty(workspace, nb, dev);
  done("kda_gqa_decode_q4",
       kda_gqa_decode_q4(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), ptr<int>(lengths), y.data_ptr(), B, n,
                         QH, KH, D, group, window ? *window : 16 * n, sinks, qs.s, kc, vc, ws.data_ptr(), nb,
                         stream(dev)));
  return y;
}

}  // namespace

PYBIND11_MODULE(_binding, m) {
  m.doc() = "Native calls of the attention operators: local, packed, 4-bit cache (see kda.ops).";
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("qk_norm_rope_backward", &qk_norm_rope_backward);
  m.def("qk_norm_rope_append", &qk_norm_rope_append);
  m.def("gqa_window", &gqa_window);
  m.def("gqa_window_backward", &gqa_window_backward);
  m.def("gqa_window_decode", &gqa_window_decode);
  m.def("packed_plan", &packed_plan);
  m.def("gqa_packed", &gqa_packed);
  m.def("gqa_packed_backward", &gqa_packed_backward);
  m.def("kv_append_q4", &kv_append_q4);
  m.def("kv_read_q4", &kv_read_q4);
  m.def("gqa_decode_q4", &gqa_decode_q4);
}

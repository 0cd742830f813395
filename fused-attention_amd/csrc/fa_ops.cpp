// fa_ops.cpp - norm and rotation of queries and keys, the paged cache's append and the attention
// over it as torch operators over the C ABI of libfa.so: the checks of their arguments, the
// allocation of outputs and workspaces on the launch stream, and the autograd node of the first.
//
// The host time of these calls is most of a small one, so their checks are made here and not in
// Python.  Shapes, strides and ranges raise ValueError, types TypeError, as the Python layer's other
// entry points; a launch failure raises RuntimeError.
#include "fa_ops.h"

#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime_api.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/extension.h>

#include <cmath>
#include <optional>
#include <sstream>

#include "fa.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

template <typename... A>
std::string text(const A&... a) {
  std::ostringstream s;
  (void)std::initializer_list<int>{((s << a), 0)...};
  return s.str();
}

#define FA_VALUE(cond, ...) \
  if (!(cond)) throw pybind11::value_error(text(__VA_ARGS__))
#define FA_TYPE(cond, ...) \
  if (!(cond)) throw pybind11::type_error(text(__VA_ARGS__))

void* stream_of(const Tensor& t) {
  return static_cast<void*>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

int dtype_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? FA_BF16 : FA_F16; }

void check_status(int status, const char* entry) {
  if (status == FA_OK) return;
  const std::string msg = text(entry, ": ", fa_strerror(status), " (status ", status, ")");
  if (status == FA_ERR_DTYPE) throw pybind11::type_error(msg);
  if (status == FA_ERR_LAUNCH) throw std::runtime_error(msg);
  throw pybind11::value_error(msg);
}

void check_rows(const Tensor& x, const char* name, const char* heads) {
  FA_TYPE(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, name, " must be float16 or bfloat16, got ",
          x.scalar_type());
  FA_VALUE(x.dim() == 4, name, " must be [B, ", heads, ", N, D], got ", x.sizes());
  FA_VALUE(x.size(3) == 32 || x.size(3) == 64 || x.size(3) == 128, "head dim ", x.size(3), " of ", name,
           " not supported; allowed 32, 64, 128");
  FA_VALUE(x.numel() > 0, name, " must not be empty, got ", x.sizes());
  FA_VALUE(x.size(0) < (1 << 30) && x.size(1) < (1 << 30) && x.size(2) < (1 << 30), name, " is too large: ", x.sizes());
}

void check_device(const Tensor& x, const Tensor& like, const char* name) {
  FA_VALUE(x.is_cuda(), "fused kernels need GPU tensors; move ", name, " to the GPU first");
  FA_VALUE(x.device() == like.device(), name, " is on ", x.device(), ", the call's rows are on ", like.device());
}

// Rows that the kernels can read as they are (dims contiguous, 16-byte rows), or a copy that is.
Tensor readable(const Tensor& x) {
  bool ok = x.stride(3) == 1 && (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (x.size(i) == 1 || (x.stride(i) & 7) == 0);
  return ok ? x : x.clone(at::MemoryFormat::Contiguous);
}

// 16-byte aligned and contiguous, or a copy that is.
Tensor dense16(const Tensor& x) {
  return x.is_contiguous() && (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0 ? x
                                                                                   : x.clone(at::MemoryFormat::Contiguous);
}

fa_rows rows(const Tensor& x) {
  auto s = [&](int i) { return x.size(i) == 1 ? 0LL : (long long)x.stride(i); };
  return fa_rows{x.data_ptr(), s(0), s(1), s(2)};
}

// New rows of x's shape, laid out in memory as x is: by token (a packed projection's views) or by head.
Tensor rows_like(const Tensor& x) {
  const int64_t B = x.size(0), H = x.size(1), N = x.size(2), D = x.size(3);
  if (H > 1 && N > 1 && x.stride(1) < x.stride(2))
    return at::empty_strided({B, H, N, D}, {N * H * D, D, H * D, 1}, x.options());
  return at::empty({B, H, N, D}, x.options());
}

// The rotation of a call, and the tensors it points into.
struct Rotation {
  fa_rotation r{};
  Tensor table, positions, wq, wk;
};

void check_weight(const Tensor& w, const Tensor& like, const char* name) {
  FA_TYPE(w.scalar_type() == like.scalar_type() || w.scalar_type() == at::kFloat, name, " must be ", like.scalar_type(),
          " or float32, got ", w.scalar_type());
  FA_VALUE(w.dim() == 1 && w.size(0) == like.size(3), name, " must be [", like.size(3), "], got ", w.sizes());
}

// x: the rows (for B, N, D and the type); table_name: past tables the positions start at.
Rotation rotation_of(const Tensor& x, const OptTensor& wq, const OptTensor& wk, const OptTensor& table,
                     const OptTensor& positions, const std::optional<std::vector<int64_t>>& sections, double eps,
                     bool interleaved) {
  Rotation t;
  const int64_t B = x.size(0), N = x.size(2), D = x.size(3);
  if (wq) check_weight(*wq, x, "q_weight");
  if (wk) check_weight(*wk, x, "k_weight");
  if (wq && wk) FA_TYPE(wq->scalar_type() == wk->scalar_type(), "q_weight and k_weight must share one dtype");
  FA_VALUE(eps >= 0 && std::isfinite(eps), "eps must be finite and not negative, got ", eps);
  FA_VALUE(table || (!positions && !sections), "positions and sections need a table");
  if (table) {
    FA_TYPE(table->scalar_type() == at::kFloat, "table must be float32, got ", table->scalar_type());
    FA_VALUE(table->dim() == 2 && table->size(0) >= 1 && table->size(0) < (1LL << 31), "table must be [length, rotary_dim], got ",
             table->sizes());
    const int64_t R = table->size(1);
    FA_VALUE(R >= 16 && R <= D && R % 16 == 0, "rotary_dim ", R, " must be a multiple of 16 up to the head dim ", D);
    t.r.axes = 1;
    if (sections) {
      FA_VALUE(positions, "sections need positions");
      FA_VALUE(sections->size() >= 1 && sections->size() <= 3, "sections must name 1 to 3 axes, got ", sections->size());
      t.r.axes = (int)sections->size();
      int64_t end = 0;
      for (size_t i = 0; i < sections->size(); ++i) {
        FA_VALUE((*sections)[i] >= 0 && (*sections)[i] <= R, "section ", i, " is ", (*sections)[i]);
        end += (*sections)[i];
        if (i + 1 < sections->size()) t.r.section_end[i] = (int)std::min(end, R / 2);
      }
      FA_VALUE(end == R / 2, "sections must sum to rotary_dim / 2 = ", R / 2, ", got ", end);
    }
    if (positions) {
      const auto st = positions->scalar_type();
      FA_TYPE(st == at::kInt || st == at::kLong, "positions must be int32 or int64, got ", st);
      Tensor p = *positions;
      const bool by_axis = sections.has_value();
      FA_VALUE(by_axis ? p.dim() == 2 || p.dim() == 3 : p.dim() == 1 || p.dim() == 2, "positions must be ",
               by_axis ? "[axes, B, N] or [axes, N]" : "[B, N] or [N]", ", got ", p.sizes());
      if (!by_axis) p = p.unsqueeze(0);
      if (p.dim() == 2) p = p.unsqueeze(1);
      FA_VALUE(p.size(0) == t.r.axes && (p.size(1) == B || p.size(1) == 1) && p.size(2) == N, "positions must be ",
               by_axis ? "[axes, B, N] or [axes, N]" : "[B, N] or [N]", " with ", t.r.axes, " axes, B = ", B, ", N = ", N,
               ", got ", positions->sizes());
      t.positions = p;
    }
    t.table = *table;
  }
  if (wq) t.wq = *wq;
  if (wk) t.wk = *wk;
  t.r.eps = (float)eps;
  t.r.interleaved = interleaved;
  return t;
}

// Devices, then the pointers (after every other check, so a refusal does not depend on a GPU).
void place(Rotation& t, const Tensor& x) {
  if (t.wq.defined()) {
    check_device(t.wq, x, "q_weight");
    t.wq = dense16(t.wq);
    t.r.q_weight = t.wq.data_ptr();
  }
  if (t.wk.defined()) {
    check_device(t.wk, x, "k_weight");
    t.wk = dense16(t.wk);
    t.r.k_weight = t.wk.data_ptr();
  }
  const Tensor& w = t.wq.defined() ? t.wq : t.wk;
  if (w.defined()) t.r.weight_dtype = w.scalar_type() == at::kFloat ? FA_F32 : dtype_code(w);
  if (!t.table.defined()) return;
  check_device(t.table, x, "table");
  t.table = dense16(t.table);
  t.r.table = t.table.data_ptr<float>();
  t.r.table_len = (int)t.table.size(0);
  t.r.rotary_dim = (int)t.table.size(1);
  if (!t.positions.defined()) return;
  check_device(t.positions, x, "positions");
  Tensor p = t.positions;
  if (p.size(2) > 1 && p.stride(2) != 1) p = p.contiguous();
  t.positions = p;
  t.r.positions = p.data_ptr();
  t.r.positions_int64 = p.scalar_type() == at::kLong;
  t.r.pos_axis_stride = p.size(0) == 1 ? 0 : p.stride(0);
  t.r.pos_batch_stride = p.size(1) == 1 ? 0 : p.stride(1);
}

Rotation check_qk(const Tensor& q, const Tensor& k, const OptTensor& wq, const OptTensor& wk, const OptTensor& table,
                  const OptTensor& positions, const std::optional<std::vector<int64_t>>& sections, double eps,
                  bool interleaved) {
  check_rows(q, "q", "H");
  check_rows(k, "k", "H_kv");
  FA_TYPE(q.scalar_type() == k.scalar_type(), "q and k must share one dtype; got ", q.scalar_type(), ", ", k.scalar_type());
  FA_VALUE(q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(3) == k.size(3),
           "q and k must agree in B, N and D; got ", q.sizes(), ", ", k.sizes());
  FA_VALUE(wq.has_value() == wk.has_value(), "give both q_weight and k_weight, or neither");
  Rotation t = rotation_of(q, wq, wk, table, positions, sections, eps, interleaved);
  check_device(q, q, "q");
  check_device(k, q, "k");
  return t;
}

std::tuple<Tensor, Tensor> turn(const Tensor& q, const Tensor& k, Rotation& t) {
  Tensor oq = at::empty(q.sizes(), q.options()), ok = at::empty(k.sizes(), k.options());
  const fa_rows a = rows(q), b = rows(k), c = rows(oq), d = rows(ok);
  check_status(fa_qk_norm_rotary(&a, &b, &c, &d, &t.r, q.size(0), q.size(1), k.size(1), q.size(2), q.size(3),
                                 dtype_code(q), stream_of(q)),
               "fa_qk_norm_rotary");
  return {oq, ok};
}

using Sections = std::optional<std::vector<int64_t>>;

std::tuple<Tensor, Tensor> qk_norm_rotary(const Tensor& q_in, const Tensor& k_in, const OptTensor& wq, const OptTensor& wk,
                                          const OptTensor& table, const OptTensor& positions, const Sections& sections,
                                          double eps, bool interleaved) {
  Rotation t = check_qk(q_in, k_in, wq, wk, table, positions, sections, eps, interleaved);
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(q_in.device());
  place(t, q_in);
  return turn(readable(q_in), readable(k_in), t);
}

struct QkNormRotary : public torch::autograd::Function<QkNormRotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q_in,
                                                const Tensor& k_in, const OptTensor& wq, const OptTensor& wk,
                                                const OptTensor& table, const OptTensor& positions,
                                                const Sections& sections, double eps, bool interleaved) {
    Rotation t = rotation_of(q_in, wq, wk, table, positions, sections, eps, interleaved);
    const c10::DeviceGuard guard(q_in.device());
    place(t, q_in);
    const Tensor q = readable(q_in), k = readable(k_in);
    auto [oq, ok] = turn(q, k, t);
    ctx->save_for_backward({q, k, t.wq, t.wk, t.table, t.positions});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["sections"] = sections ? c10::IValue(*sections) : c10::IValue();
    return {oq, ok};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grad_out) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "fused_qk_norm_rotary_autograd has no second derivative (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1];
    auto opt = [&](int i) { return saved[i].defined() ? OptTensor(saved[i]) : OptTensor(); };
    const c10::IValue sec = ctx->saved_data["sections"];
    Sections sections;
    if (!sec.isNone()) sections = sec.toIntVector();
    const c10::DeviceGuard guard(q.device());
    // (positions are saved as [axes, B, N])
    OptTensor positions = opt(5);
    if (positions && !sections) positions = positions->squeeze(0);
    Rotation t = rotation_of(q, opt(2), opt(3), opt(4), positions, sections, ctx->saved_data["eps"].toDouble(),
                             ctx->saved_data["interleaved"].toBool());
    place(t, q);
    const Tensor gq = readable(grad_out[0].to(q.scalar_type())), gk = readable(grad_out[1].to(k.scalar_type()));
    Tensor dq = rows_like(q), dk = rows_like(k), dwq, dwk, ws;
    const int B = q.size(0), H = q.size(1), Hkv = k.size(1), N = q.size(2), D = q.size(3);
    size_t bytes = 0;
    if (t.wq.defined()) {
      dwq = at::empty({D}, t.wq.options()), dwk = at::empty({D}, t.wk.options());
      bytes = fa_qk_norm_rotary_workspace_size(B, H, Hkv, N, D);
      ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    }
    const fa_rows a = rows(q), b = rows(k), c = rows(gq), d = rows(gk), e = rows(dq), f = rows(dk);
    const int status = fa_qk_norm_rotary_bwd(&a, &b, &c, &d, &e, &f, bytes ? dwq.data_ptr() : nullptr,
                                             bytes ? dwk.data_ptr() : nullptr, &t.r, B, H, Hkv, N, D, dtype_code(q),
                                             bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q));
    TORCH_CHECK(status == FA_OK, "fa_qk_norm_rotary_bwd: ", fa_strerror(status), " (status ", status, ")");
    return {dq, dk, dwq, dwk, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

bool capturing(const Tensor& x) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  const hipStream_t stream = c10::hip::getCurrentHIPStream(x.device().index()).stream();
  return hipStreamIsCapturing(stream, &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}

// A gradient accumulator remembers the stream that was current when it was made, and lives as long as
// some graph of its leaf does.  A backward under capture would make that stream wait for the captured
// one, which the runtime answers by ending the process: refuse it while it is a Python error.
void check_capture(const Tensor& x, const char* name) {
  if (!x.defined() || !x.requires_grad() || !x.is_leaf()) return;
  const auto acc = torch::autograd::impl::try_get_grad_accumulator(x);
  if (!acc || !acc->stream()) return;
  if (*acc->stream() != c10::hip::getCurrentHIPStream(x.device().index()).unwrap())
    throw std::runtime_error(text("fused_qk_norm_rotary_autograd under graph capture: an earlier graph of ", name,
                                  " made on another stream is still alive; drop its outputs before capturing"));
}

std::tuple<Tensor, Tensor> qk_norm_rotary_autograd(const Tensor& q, const Tensor& k, const OptTensor& wq,
                                                   const OptTensor& wk, const OptTensor& table,
                                                   const OptTensor& positions, const Sections& sections, double eps,
                                                   bool interleaved) {
  {
    const Rotation t = check_qk(q, k, wq, wk, table, positions, sections, eps, interleaved);
    if (at::GradMode::is_enabled() && capturing(q)) {
      check_capture(q, "q");
      check_capture(k, "k");
      if (wq) check_capture(*wq, "q_weight");
      if (wk) check_capture(*wk, "k_weight");
    }
  }
  const auto out = QkNormRotary::apply(q, k, wq, wk, table, positions, sections, eps, interleaved);
  return {out[0], out[1]};
}

// ---- the paged cache

fa_paged_cache check_cache(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& table,
                           const Tensor& like) {
  FA_TYPE(kc.scalar_type() == at::kFloat8_e4m3fn && vc.scalar_type() == at::kFloat8_e4m3fn,
          "the cache's keys and values must be float8_e4m3fn, got ", kc.scalar_type(), ", ", vc.scalar_type());
  FA_TYPE(ks.scalar_type() == at::kFloat8_e8m0fnu && vs.scalar_type() == at::kFloat8_e8m0fnu,
          "the cache's scales must be float8_e8m0fnu, got ", ks.scalar_type(), ", ", vs.scalar_type());
  FA_VALUE(kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.numel() > 0,
           "the cache's keys and values must both be [num_pages, H_kv, page_size, D], got ", kc.sizes(), ", ", vc.sizes());
  FA_VALUE(ks.dim() == 2 && ks.size(0) == kc.size(0) && ks.size(1) == kc.size(1) && ks.sizes() == vs.sizes(),
           "the cache's scales must be [num_pages, H_kv], got ", ks.sizes(), ", ", vs.sizes());
  FA_VALUE(kc.size(3) == like.size(3), "head dim ", kc.size(3), " of the cache is not the rows' ", like.size(3));
  FA_VALUE(kc.size(2) == 16 || kc.size(2) == 32 || kc.size(2) == 64 || kc.size(2) == 128, "page size ", kc.size(2),
           " not supported; allowed 16, 32, 64, 128");
  FA_VALUE(kc.size(0) < (1LL << 31) && kc.size(1) < (1 << 30), "the cache is too large: ", kc.sizes());
  FA_VALUE(kc.is_contiguous() && vc.is_contiguous() && ks.is_contiguous() && vs.is_contiguous(),
           "the cache's tensors must be contiguous");
  FA_TYPE(table.scalar_type() == at::kInt, "block_table must be int32, got ", table.scalar_type());
  FA_VALUE(table.dim() == 2 && table.size(0) == like.size(0) && table.size(1) >= 1 && table.size(1) < (1LL << 31),
           "block_table must be [B, pages] with B = ", like.size(0), ", got ", table.sizes());
  fa_paged_cache c{};
  c.table_width = (int)table.size(1), c.num_pages = (int)kc.size(0), c.page_size = (int)kc.size(2), c.H_kv = (int)kc.size(1);
  return c;
}

Tensor place_cache(fa_paged_cache& c, const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs,
                   const Tensor& table, const Tensor& like) {
  check_device(kc, like, "the cache");
  check_device(vc, like, "the cache");
  check_device(ks, like, "the cache");
  check_device(vs, like, "the cache");
  check_device(table, like, "block_table");
  c.k = kc.data_ptr(), c.v = vc.data_ptr(), c.k_scale = ks.data_ptr(), c.v_scale = vs.data_ptr();
  Tensor t = table;
  if (t.size(1) > 1 && t.stride(1) != 1) t = t.contiguous();
  c.block_table = t.data_ptr<int>();
  c.table_stride = t.size(0) == 1 ? 0 : t.stride(0);
  return t;
}

void check_lens(const Tensor& x, const Tensor& like, const char* name) {
  FA_TYPE(x.scalar_type() == at::kInt, name, " must be int32, got ", x.scalar_type());
  FA_VALUE(x.dim() == 1 && x.size(0) == like.size(0), name, " must be [B] with B = ", like.size(0), ", got ", x.sizes());
}

void written(const Tensor& x) {
  if (!x.is_inference()) x.unsafeGetTensorImpl()->bump_version();
}

OptTensor append_paged_kv(const Tensor& kc, const Tensor& vc, const Tensor& ks, const Tensor& vs, const Tensor& k_in,
                          const Tensor& v_in, const Tensor& block_table, const Tensor& past, const OptTensor& fresh,
                          const OptTensor& q_in, const OptTensor& wq, const OptTensor& wk, const OptTensor& table,
                          const OptTensor& positions, const Sections& sections, double eps, bool interleaved) {
  check_rows(k_in, "k", "H_kv");
  check_rows(v_in, "v", "H_kv");
  FA_TYPE(k_in.scalar_type() == v_in.scalar_type(), "k and v must share one dtype; got ", k_in.scalar_type(), ", ",
          v_in.scalar_type());
  FA_VALUE(k_in.sizes() == v_in.sizes(), "k and v must both be [B, H_kv, N, D]; got ", k_in.sizes(), ", ", v_in.sizes());
  if (q_in) {
    check_rows(*q_in, "q", "H");
    FA_TYPE(q_in->scalar_type() == k_in.scalar_type(), "q, k, v must share one dtype; got ", q_in->scalar_type(), ", ",
            k_in.scalar_type());
    FA_VALUE(q_in->size(0) == k_in.size(0) && q_in->size(2) == k_in.size(2) && q_in->size(3) == k_in.size(3),
             "q and k must agree in B, N and D; got ", q_in->sizes(), ", ", k_in.sizes());
    FA_VALUE(wq.has_value() == wk.has_value(), "give both q_weight and k_weight, or neither");
  } else {
    FA_VALUE(!wq, "q_weight needs q");
  }
  fa_paged_cache c = check_cache(kc, vc, ks, vs, block_table, k_in);
  FA_VALUE(c.H_kv == k_in.size(1), "the cache holds ", c.H_kv, " heads, k has ", k_in.size(1));
  check_lens(past, k_in, "past_lens");
  if (fresh) check_lens(*fresh, k_in, "new_lens");
  Rotation t = rotation_of(k_in, wq, wk, table, positions, sections, eps, interleaved);
  check_device(k_in, k_in, "k");
  check_device(v_in, k_in, "v");
  if (q_in) check_device(*q_in, k_in, "q");
  check_device(past, k_in, "past_lens");
  if (fresh) check_device(*fresh, k_in, "new_lens");
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(k_in.device());
  place(t, k_in);
  const Tensor pages = place_cache(c, kc, vc, ks, vs, block_table, k_in);
  const Tensor k = readable(k_in), v = readable(v_in), p = past.contiguous();
  const Tensor f = fresh ? fresh->contiguous() : Tensor();
  Tensor q, oq;
  fa_rows rq{}, ro{};
  if (q_in) {
    q = readable(*q_in);
    oq = at::empty(q.sizes(), q.options());
    rq = rows(q), ro = rows(oq);
  }
  const fa_rows rk = rows(k), rv = rows(v);
  check_status(fa_paged_append(q_in ? &rq : nullptr, &rk, &rv, q_in ? &ro : nullptr, &c, p.data_ptr<int>(),
                               f.defined() ? f.data_ptr<int>() : nullptr, &t.r, k.size(0), q_in ? q.size(1) : c.H_kv,
                               k.size(2), k.size(3), dtype_code(k), stream_of(k)),
               "fa_paged_append");
  for (const Tensor* x : {&kc, &vc, &ks, &vs}) written(*x);
  return q_in ? OptTensor(oq) : OptTensor();
}

std::tuple<Tensor, OptTensor> paged_attention(const Tensor& q_in, const Tensor& kc, const Tensor& vc, const Tensor& ks,
                                              const Tensor& vs, const Tensor& block_table, const Tensor& past,
                                              const OptTensor& fresh, bool with_lse) {
  check_rows(q_in, "q", "H");
  fa_paged_cache c = check_cache(kc, vc, ks, vs, block_table, q_in);
  FA_VALUE(q_in.size(1) % c.H_kv == 0, "the cache's ", c.H_kv, " heads must divide q's ", q_in.size(1));
  check_lens(past, q_in, "past_lens");
  if (fresh) check_lens(*fresh, q_in, "new_lens");
  check_device(q_in, q_in, "q");
  check_device(past, q_in, "past_lens");
  if (fresh) check_device(*fresh, q_in, "new_lens");
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(q_in.device());
  const Tensor pages = place_cache(c, kc, vc, ks, vs, block_table, q_in);
  const Tensor q = readable(q_in), p = past.contiguous();
  const Tensor f = fresh ? fresh->contiguous() : Tensor();
  const int B = q.size(0), H = q.size(1), N = q.size(2), D = q.size(3);
  Tensor o = rows_like(q_in), ws;
  OptTensor lse;
  if (with_lse) lse = at::empty({B, H, N}, q.options().dtype(at::kFloat));
  const size_t bytes = fa_paged_attention_workspace_size(B, H, c.H_kv, N, D, (long long)c.table_width * c.page_size);
  if (bytes) ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
  const fa_rows rq = rows(q), ro = rows(o);
  check_status(fa_paged_attention(&rq, &c, p.data_ptr<int>(), f.defined() ? f.data_ptr<int>() : nullptr, &ro,
                                  with_lse ? lse->data_ptr<float>() : nullptr, B, H, N, D, dtype_code(q),
                                  static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(D))),
                                  bytes ? ws.data_ptr() : nullptr, bytes, stream_of(q)),
               "fa_paged_attention");
  return {o, lse};
}

}  // namespace

void fa_def_ops(pybind11::module_& m) {
  m.def("qk_norm_rotary", &qk_norm_rotary, "Norm and rotation of q and k; returns both");
  m.def("qk_norm_rotary_autograd", &qk_norm_rotary_autograd, "The same with a backward");
  m.def("append_paged_kv", &append_paged_kv, "Store k (normed, turned) and v in their pages; returns q turned");
  m.def("paged_attention", &paged_attention, "Attention of q over the pages; returns (o, lse or None)");
}

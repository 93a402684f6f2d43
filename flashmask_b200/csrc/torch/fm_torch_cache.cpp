// Native host of the operators around attention: norm and rotation of q and k with its autograd node, the 8-bit paged
// cache, attention over it.  Checks, allocations and calls into the C ABI; a decode step makes three such calls in a few
// microseconds each, which is what its kernels take.
#include "fm_torch.h"

#include <ATen/cuda/EmptyTensor.h>

#include <cmath>
#include <cstring>

namespace fm_host {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

namespace {

constexpr const char* kNoCpu = "flashmask_b200 runs on CUDA (sm_100a) tensors only; there is no CPU path";

// A new tensor on t's device, past the dispatcher: 1 us where at::empty takes 2, and a decode step makes eight.
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

bool aligned16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }

// t [B, S, H, D] as the kernels read it in 16-byte vectors: rows contiguous, every stride a multiple of 8, base aligned.
Tensor vec_rows(const Tensor& t) {
  if (t.numel() == 0) return t;
  bool ok = t.stride(-1) == 1 && aligned16(t);
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) == 1 || t.stride(i) % 8 == 0);
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
// (a dimension of one element may carry any stride)
void vec_strides(int64_t* out, const Tensor& t) { for (int i = 0; i < 3; ++i) out[i] = t.size(i) == 1 ? 0 : t.stride(i); }

// Whether a forward-mode derivative comes with t: requires_grad and GradMode say nothing of it.
bool has_tangent(const Tensor& t) { return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined(); }
bool has_tangent(const std::optional<Tensor>& t) { return t && has_tangent(*t); }

Tensor packed(const Tensor& t) {
  const Tensor c = t.contiguous();
  return c.numel() == 0 || aligned16(c) ? c : c.clone();
}

// ---------------------------------------------------------------------------- norm and rotation
fm_norm_rotary_args norm_args(const Tensor& q, const Tensor& k, const Tensor& qw, const Tensor& kw, const Tensor& cos,
                              const Tensor& sin, const Tensor& pos, double eps, bool interleaved) {
  fm_norm_rotary_args a;
  std::memset(&a, 0, sizeof(a));
  a.B = (int)q.size(0); a.S = (int)q.size(1); a.Hq = (int)q.size(2); a.Hk = (int)k.size(2); a.d = (int)q.size(3);
  a.rot = 2 * (int)cos.size(1);
  a.dtype = dtype_code(q);
  a.interleaved = interleaved;
  a.table = (int)cos.size(0);
  a.eps = (float)eps;
  a.q = q.data_ptr(); a.k = k.data_ptr();
  if (qw.defined()) { a.q_weight = qw.data_ptr(); a.weight_f32 = qw.scalar_type() == at::kFloat; }
  if (kw.defined()) { a.k_weight = kw.data_ptr(); a.weight_f32 = kw.scalar_type() == at::kFloat; }
  a.cos = cos.data_ptr<float>(); a.sin = sin.data_ptr<float>();
  if (pos.defined()) {
    a.positions = pos.data_ptr();
    a.positions_64 = pos.scalar_type() == at::kLong;
    a.positions_stride = pos.dim() == 2 && pos.size(0) > 1 ? pos.stride(0) : 0;
  }
  vec_strides(a.q_stride, q); vec_strides(a.k_stride, k);
  return a;
}

// The forward's outputs; `keep`: what the backward needs.
std::pair<Tensor, Tensor> norm_forward(const Tensor& q_in, const Tensor& k_in, const std::optional<Tensor>& qw_in,
                                       const std::optional<Tensor>& kw_in, const Tensor& cos_in, const Tensor& sin_in,
                                       const std::optional<Tensor>& pos_in, double eps, bool interleaved, variable_list* keep) {
  const c10::cuda::CUDAGuard guard(q_in.device());
  const Tensor q = vec_rows(q_in), k = vec_rows(k_in), cos = packed(cos_in), sin = packed(sin_in);
  const Tensor qw = qw_in ? packed(*qw_in) : Tensor(), kw = kw_in ? packed(*kw_in) : Tensor();
  const Tensor pos = pos_in ? (pos_in->stride(-1) == 1 ? *pos_in : pos_in->contiguous()) : Tensor();
  Tensor qo = fresh(q.sizes(), q.scalar_type(), q), ko = fresh(k.sizes(), k.scalar_type(), q);
  fm_norm_rotary_args a = norm_args(q, k, qw, kw, cos, sin, pos, eps, interleaved);
  a.q_out = qo.data_ptr(); a.k_out = ko.data_ptr();
  vec_strides(a.qo_stride, qo); vec_strides(a.ko_stride, ko);
  check(fm_norm_rotary_fwd(&a, stream_of(q)), "fm_norm_rotary_fwd");
  if (keep) *keep = {q, k, qw, kw, cos, sin, pos};
  return {qo, ko};
}

// A gradient that itself has none: with create_graph it is part of a graph that says so, and not a constant.
class FirstOrder : public torch::autograd::Function<FirstOrder> {
 public:
  static Variable forward(AutogradContext*, const Variable& grad, const Variable&) { return grad.view_as(grad); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK_NOT_IMPLEMENTED(false, "the gradients of qk_norm_rotary have no gradient");
    return {};
  }
};
Tensor first_order(const Tensor& grad) {
  if (!grad.defined() || !at::GradMode::is_enabled()) return grad;
  return FirstOrder::apply(grad, at::empty({0}, grad.options()).requires_grad_(true));
}

class NormRotary : public torch::autograd::Function<NormRotary> {
 public:
  static variable_list forward(AutogradContext* ctx, const Variable& q, const Variable& k, const std::optional<Tensor>& qw_in,
                               const std::optional<Tensor>& kw_in, const Tensor& cos, const Tensor& sin,
                               const std::optional<Tensor>& pos, double eps, bool interleaved) {
    variable_list keep;
    const auto [qo, ko] = norm_forward(q, k, qw_in, kw_in, cos, sin, pos, eps, interleaved, &keep);
    ctx->save_for_backward(keep);
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["dqw"] = qw_in && qw_in->requires_grad();
    ctx->saved_data["dkw"] = kw_in && kw_in->requires_grad();
    return {qo, ko};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const variable_list s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &qw = s[2], &kw = s[3];
    const c10::cuda::CUDAGuard guard(q.device());
    const Tensor gq = vec_rows(grads[0]), gk = vec_rows(grads[1]);
    fm_norm_rotary_args a = norm_args(q, k, qw, kw, s[4], s[5], s[6], ctx->saved_data["eps"].toDouble(), ctx->saved_data["interleaved"].toBool());
    Tensor dq = fresh(q.sizes(), q.scalar_type(), q), dk = fresh(k.sizes(), k.scalar_type(), q), dqw, dkw, ws;
    a.q_out = dq.data_ptr(); a.k_out = dk.data_ptr();
    a.d_q = gq.data_ptr(); a.d_k = gk.data_ptr();
    vec_strides(a.qo_stride, dq); vec_strides(a.ko_stride, dk); vec_strides(a.dq_stride, gq); vec_strides(a.dk_stride, gk);
    if (qw.defined() && ctx->saved_data["dqw"].toBool()) { dqw = fresh(qw.sizes(), qw.scalar_type(), q); a.dq_weight = dqw.data_ptr(); }
    if (kw.defined() && ctx->saved_data["dkw"].toBool()) { dkw = fresh(kw.sizes(), kw.scalar_type(), q); a.dk_weight = dkw.data_ptr(); }
    if (dqw.defined() || dkw.defined()) {
      a.workspace_bytes = fm_norm_rotary_bwd_workspace_bytes(&a);
      ws = fresh({(int64_t)a.workspace_bytes}, at::kByte, q);
      a.workspace = ws.data_ptr();
    }
    check(fm_norm_rotary_bwd(&a, stream_of(q)), "fm_norm_rotary_bwd");
    return {first_order(dq), first_order(dk), first_order(dqw), first_order(dkw), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

std::pair<Tensor, Tensor> norm_rotary(const Tensor& q, const Tensor& k, const std::optional<Tensor>& qw, const std::optional<Tensor>& kw,
                                      const Tensor& cos, const Tensor& sin, const std::optional<Tensor>& pos, double eps,
                                      bool interleaved) {
  TORCH_CHECK(q.is_cuda(), kNoCpu);
  require(q.dim() == 4 && k.dim() == 4, "query and key must be [B, S, H, D]");
  require(q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3), "key's shape does not match query");
  require(q.scalar_type() == k.scalar_type(), "query and key must share a dtype");
  require(q.device() == k.device() && q.device() == cos.device() && q.device() == sin.device(), "all tensors must be on the device of query");
  dtype_code(q);
  const int64_t d = q.size(3);
  require(cos.dim() == 2 && cos.sizes() == sin.sizes() && 2 * cos.size(1) <= d, "cos and sin must be [positions, n] with 2 n <= head dim");
  require(cos.scalar_type() == at::kFloat && sin.scalar_type() == at::kFloat, "cos and sin must be float32");
  require(!cos.requires_grad() && !sin.requires_grad() && !has_tangent(cos) && !has_tangent(sin), "cos and sin take no gradient");
  for (const auto* w : {&qw, &kw}) {
    if (!*w) continue;
    require((*w)->dim() == 1 && (*w)->size(0) == d, "weights must be [head dim]");
    require((*w)->device() == q.device(), "weights must be on the device of query");
    require((*w)->scalar_type() == at::kFloat || (*w)->scalar_type() == q.scalar_type(), "weights must be float32 or of query's dtype");
  }
  require(!qw || !kw || (*qw).scalar_type() == (*kw).scalar_type(), "weights must share a dtype");
  if (pos) {
    require(pos->device() == q.device(), "positions must be on the device of query");
    require(pos->scalar_type() == at::kInt || pos->scalar_type() == at::kLong, "positions must be int32 or int64");
    require((pos->dim() == 1 && pos->size(0) == q.size(1)) ||
            (pos->dim() == 2 && pos->size(1) == q.size(1) && (pos->size(0) == q.size(0) || pos->size(0) == 1)), "positions must be [B, S] or [S]");
  }
  pybind11::gil_scoped_release nogil;
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(q) || has_tangent(k) || has_tangent(qw) || has_tangent(kw)), "qk_norm_rotary has no forward-mode derivative");
  if (!at::GradMode::is_enabled() || !(q.requires_grad() || k.requires_grad() || (qw && qw->requires_grad()) || (kw && kw->requires_grad())))
    return norm_forward(q, k, qw, kw, cos, sin, pos, eps, interleaved, nullptr);
  const variable_list r = NormRotary::apply(q, k, qw, kw, cos, sin, pos, eps, interleaved);
  return {r[0], r[1]};
}

// ---------------------------------------------------------------------------- cache
void no_gradient(const Tensor& t, const char* what) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what, " has no gradient: call it under torch.no_grad()");
  TORCH_CHECK(!has_tangent(t), what, " has no gradient, and none in forward mode");
}

struct Cache { const Tensor &k, &v, &ks, &vs; };

fm_kv_cache cache_of(const Cache& c, const char* what) {
  fm_kv_cache r;
  for (const Tensor* t : {&c.k, &c.v, &c.ks, &c.vs}) no_gradient(*t, what);
  require(c.k.dim() == 4 && c.v.dim() == 4 && c.k.sizes().slice(0, 3) == c.v.sizes().slice(0, 3),
          "cache k and v must be [num_pages, Hkv, page_size, D]");
  require(c.k.scalar_type() == c.v.scalar_type() && (c.k.scalar_type() == at::kFloat8_e4m3fn || c.k.scalar_type() == at::kChar),
          "cache k and v must be float8_e4m3fn or int8");
  require(c.ks.scalar_type() == at::kFloat && c.vs.scalar_type() == at::kFloat && c.ks.sizes() == c.k.sizes().slice(0, 2) &&
          c.vs.sizes() == c.k.sizes().slice(0, 2), "cache scales must be float32 [num_pages, Hkv]");
  require(c.k.is_contiguous() && c.v.is_contiguous() && c.ks.is_contiguous() && c.vs.is_contiguous(), "cache tensors must be contiguous");
  require(c.k.device() == c.v.device() && c.k.device() == c.ks.device() && c.k.device() == c.vs.device(), "cache tensors must be on one device");
  TORCH_CHECK_NOT_IMPLEMENTED(c.k.size(0) <= INT_MAX && c.k.size(1) <= INT_MAX, "cache too large");
  r.k = c.k.data_ptr(); r.v = c.v.data_ptr(); r.k_scale = c.ks.data_ptr<float>(); r.v_scale = c.vs.data_ptr<float>();
  r.num_pages = (int)c.k.size(0); r.Hkv = (int)c.k.size(1); r.page_size = (int)c.k.size(2); r.d = (int)c.k.size(3); r.dv = (int)c.v.size(3);
  r.dtype = c.k.scalar_type() == at::kChar ? FM_CACHE_INT8 : FM_CACHE_E4M3;
  return r;
}

const int32_t* ints(const std::optional<Tensor>& t, int64_t B, const Tensor& like, const char* msg, Tensor* keep) {
  if (!t) return nullptr;
  require(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == B && t->device() == like.device(), msg);
  *keep = t->contiguous();
  return keep->data_ptr<int>();
}

fm_kv_args kv_args(const Cache& c, const Tensor& table, int64_t B, int64_t S, Tensor* keep) {
  fm_kv_args a;
  std::memset(&a, 0, sizeof(a));
  require(table.scalar_type() == at::kInt && table.dim() == 2 && table.size(0) == B && table.device() == c.k.device(),
          "page_table must be int32 [B, pages] on the cache's device");
  TORCH_CHECK_NOT_IMPLEMENTED(B <= 65535 && S <= INT_MAX - 65536 && table.size(1) <= INT_MAX, "too many sequences, rows or pages");
  *keep = table.stride(1) == 1 || table.size(1) <= 1 ? table : table.contiguous();
  if (table.size(0) > 1 && keep->stride(0) < table.size(1)) *keep = keep->contiguous();
  a.B = (int)B; a.S = (int)S;
  a.max_pages = (int)table.size(1);
  a.table_stride = keep->stride(0);
  a.page_table = keep->data_ptr<int>();
  return a;
}

void kv_write(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs, const Tensor& key_in, const Tensor& value_in,
              const Tensor& table, const Tensor& start, const std::optional<Tensor>& lengths) {
  const Cache c{ck, cv, cks, cvs};
  TORCH_CHECK(ck.is_cuda() && key_in.is_cuda(), kNoCpu);
  const fm_kv_cache f = cache_of(c, "kv_cache_write");
  require(key_in.dim() == 4 && value_in.dim() == 4 && key_in.sizes().slice(0, 3) == value_in.sizes().slice(0, 3) && key_in.size(2) == f.Hkv &&
          key_in.size(3) == f.d && value_in.size(3) == f.dv, "key and value must be [B, S, Hkv, D] of the cache's heads");
  require(key_in.scalar_type() == value_in.scalar_type(), "key and value must share a dtype");
  require(key_in.device() == ck.device() && value_in.device() == ck.device(), "key and value must be on the cache's device");
  no_gradient(key_in, "kv_cache_write");
  no_gradient(value_in, "kv_cache_write");
  const c10::cuda::CUDAGuard guard(ck.device());
  Tensor keep[3];
  fm_kv_args a = kv_args(c, table, key_in.size(0), key_in.size(1), &keep[0]);
  a.dtype = dtype_code(key_in);
  a.start = ints(start, a.B, ck, "start must be int32 [B] on the cache's device", &keep[1]);
  a.lengths = ints(lengths, a.B, ck, "lengths must be int32 [B] on the cache's device", &keep[2]);
  const Tensor key = vec_rows(key_in), value = vec_rows(value_in);
  a.k = key.data_ptr(); a.v = value.data_ptr();
  vec_strides(a.k_stride, key); vec_strides(a.v_stride, value);
  check(fm_kv_write(&f, &a, stream_of(ck)), "fm_kv_write");
}

std::pair<Tensor, Tensor> kv_read(const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs, const Tensor& table,
                                  const Tensor& start, const Tensor& seqlens, int64_t length, at::ScalarType dtype) {
  const Cache c{ck, cv, cks, cvs};
  TORCH_CHECK(ck.is_cuda(), kNoCpu);
  const fm_kv_cache f = cache_of(c, "kv_cache_read");
  require(length >= 0, "length must not be negative");
  const c10::cuda::CUDAGuard guard(ck.device());
  Tensor keep[3];
  fm_kv_args a = kv_args(c, table, table.size(0), length, &keep[0]);
  a.start = ints(start, a.B, ck, "start must be int32 [B] on the cache's device", &keep[1]);
  a.seqlens = ints(seqlens, a.B, ck, "seqlens must be int32 [B] on the cache's device", &keep[2]);
  Tensor k = fresh({a.B, length, f.Hkv, f.d}, dtype, ck), v = fresh({a.B, length, f.Hkv, f.dv}, dtype, ck);
  a.dtype = dtype_code(k);
  a.k_out = k.data_ptr(); a.v_out = v.data_ptr();
  check(fm_kv_read(&f, &a, stream_of(ck)), "fm_kv_read");
  return {k, v};
}

// Rows (queries x heads of a group) up to which the cache is read by the kernel for few rows.  Beyond, the tokens are
// read back once into dense 16-bit tensors and the dense forward, which feeds the tensor cores, takes the call.  Measured, 32 / 8
// heads, d = 128: 96 rows 40 us and 100 rows 52 us for 16384 keys, 69 and 80 us for 8 x 4096, 111 and 102 us for 64 x 512: the
// kernel's time goes with the number of 32-row tiles and the other's hardly with the rows.
// Head dims above 128: the dense forward does not deal a row block's K tiles to several CTAs, so its time does not depend on
// the rows while these leave SMs idle, and the kernel's goes with all rows of the call: the line is a number of rows of all kv heads together.  Kernel / dense
// forward, us with the launch (rows of each kv head):
//   d = 192 (5400)  1 head, 5200 rows of 2048 keys 51 / 63, of 16384 258 / 320, of 65536 942 / 1200;  2 heads, 2000 of 16384 201 / 332, past the line 4000 387 / 330;
//                   8 heads, 400 of 2048 37 / 57, of 16384 166 / 293, past 1000 of 2048 72 / 72, of 16384 387 / 389;  4 x 8 heads, 168 of 2048 55 / 65, past 400 104 / 65
//   d = 256 (900)   1 head, 900 of 2048 37 / 49, of 16384 172 / 186, past 1200 223 / 184;  4 heads, 224 of 2048 37 / 47, of 16384 172 / 195, past 480 346 / 197;
//                   8 heads, 100 of 2048 37 / 49, of 16384 162 / 215, past 224 328 / 215;  4 x 8 heads, past 128 of 2048 117 / 92
// A window shortens both sides: 1024 of 16384 keys, d = 192, 1 head, 5200 rows 59 / 53, 8 heads, 660 41 / 57, d = 256, 1 head, 896 31 / 43; window 64 43 / 39, 25 / 37, 20 / 35.
int64_t few_rows(int64_t d, int64_t kv_heads) { return std::max<int64_t>(96, d <= 128 ? 0 : (d <= 192 ? 5400 : 900) / std::max<int64_t>(kv_heads, 1)); }
// Without an upper bound of the lengths the dense tensors cover the whole page table, which may be far wider than the
// sequences are long: beyond this many bytes the kernel for few rows, which needs none, keeps the call.
constexpr int64_t kNoBound = (int64_t)1 << 40, kMostDense = (int64_t)2 << 30;

std::pair<Tensor, Tensor> kv_attention(const Tensor& query, const Tensor& ck, const Tensor& cv, const Tensor& cks, const Tensor& cvs,
                                       const Tensor& table, const Tensor& seqlens, const std::optional<Tensor>& lengths,
                                       const std::optional<Tensor>& sink, bool causal, int64_t window, std::optional<double> scale_in,
                                       int64_t max_seqlen) {
  const Cache c{ck, cv, cks, cvs};
  TORCH_CHECK(ck.is_cuda() && query.is_cuda(), kNoCpu);
  const fm_kv_cache f = cache_of(c, "kv_cache_attention");
  require(query.dim() == 4 && query.size(3) == f.d, "query must be [B, S, H, D] of the cache's head dim");
  require(f.Hkv > 0 && query.size(2) % f.Hkv == 0 && query.size(2) > 0, "num q heads must be a multiple of num kv heads");
  require(query.device() == ck.device(), "query must be on the cache's device");
  if (sink) require(sink->numel() == query.size(2), "sink must have one logit per q head");
  TORCH_CHECK_VALUE(window >= 0 && (causal || window == 0), "window_size needs causal=True and at least one token");
  no_gradient(query, "kv_cache_attention");
  if (sink) no_gradient(*sink, "kv_cache_attention");
  const c10::cuda::CUDAGuard guard(ck.device());
  Tensor keep[3];
  const int64_t B = query.size(0), S = query.size(1), Hq = query.size(2);
  fm_kv_args a = kv_args(c, table, B, S, &keep[0]);
  a.Hq = (int)Hq;
  a.dtype = dtype_code(query);
  a.seqlens = ints(seqlens, B, ck, "seqlens must be int32 [B] on the cache's device", &keep[1]);
  a.lengths = ints(lengths, B, ck, "q_lengths must be int32 [B] on the cache's device", &keep[2]);
  a.causal = causal;
  a.window = (int)std::min<int64_t>(window, INT_MAX);
  const double scale = scale_in ? *scale_in : 1.0 / std::sqrt((double)f.d);
  a.softmax_scale = (float)scale;
  void* stream = stream_of(ck);
  const Tensor sink32 = sink ? sink_fp32(*sink, query) : Tensor();
  // columns of the dense tensors (with rows that do not count the real ones stand up to S columns further left).  The last is the last
  // row's own position, so a window leaves S + window - 1 that a row can see: FM_FWD_MASK_DENSE holds with any window.
  int64_t cols = std::min<int64_t>(max_seqlen, (int64_t)a.max_pages * f.page_size);
  cols = std::max<int64_t>(lengths ? cols + S : cols, S);
  if (window > 0) cols = std::min(cols, S + std::min<int64_t>(window, INT_MAX) - 1);
  const bool dense = cols <= fm_fwd_max_keys(f.d, f.dv) && (max_seqlen < kNoBound || B * cols * f.Hkv * (f.d + f.dv) * 2 <= kMostDense);
  if (S * (Hq / f.Hkv) > few_rows(f.d, B * f.Hkv) && B > 0 && dense) {
    const Tensor shift = fresh({B}, at::kInt, ck), bounds = fresh({B, 1, cols, causal ? 1 : 2}, at::kInt, ck), marks = fresh({B, f.Hkv}, at::kInt, ck);
    a.marks = marks.data_ptr<int>();
    check(fm_kv_bounds(&f, &a, (int)cols, shift.data_ptr<int>(), bounds.data_ptr<int>(), stream), "fm_kv_bounds");
    const Tensor k = fresh({B, cols, f.Hkv, f.d}, query.scalar_type(), ck), v = fresh({B, cols, f.Hkv, f.dv}, query.scalar_type(), ck);
    fm_kv_args r = a;
    r.S = (int)cols; r.start = shift.data_ptr<int>(); r.k_out = k.data_ptr(); r.v_out = v.data_ptr();
    check(fm_kv_read(&f, &r, stream), "fm_kv_read");
    const Tensor q = rows(vec_rows(query)), out = fresh({B, S, Hq, f.dv}, q.scalar_type(), ck), lse = fresh({B, Hq, S}, at::kFloat, ck);
    int tm = 0, tn = 0;
    check(fm_fwd_tile_shape(f.d, f.dv, &tm, &tn), "fm_fwd_tile_shape");
    const Tensor minmax = scan_mask(bounds, (int)S, causal, tm, tn, stream);
    fm_attn_args x = base_args(q, k, v, out, lse, causal, scale, sink32);
    set_mask(&x, bounds, minmax, tm, tn);
    x.fwd_flags = FM_FWD_MASK_DENSE;
    Tensor ws;
    if ((x.workspace_bytes = fm_fwd_workspace_bytes(&x)) != 0) {
      ws = fresh({(int64_t)x.workspace_bytes}, at::kByte, ck);
      x.workspace = ws.data_ptr();
    }
    check(fm_fwd(&x, stream), "fm_fwd");
    a.o = out.data_ptr(); a.lse = lse.data_ptr<float>();
    check(fm_kv_nan_rows(&f, &a, stream), "fm_kv_nan_rows");
    return {out, lse};
  }
  const Tensor q = vec_rows(query);
  const Tensor out = fresh({B, S, Hq, f.dv}, q.scalar_type(), ck), lse = fresh({B, Hq, S}, at::kFloat, ck);
  a.workspace_bytes = fm_kv_attention_workspace_bytes(&f, &a);
  const Tensor ws = fresh({(int64_t)a.workspace_bytes}, at::kByte, ck);
  a.workspace = ws.data_ptr();
  a.q = q.data_ptr(); a.o = out.data_ptr(); a.lse = lse.data_ptr<float>();
  vec_strides(a.q_stride, q);
  if (sink32.defined()) a.sink = sink32.data_ptr<float>();
  check(fm_kv_attention(&f, &a, stream), "fm_kv_attention");
  return {out, lse};
}

}  // namespace

void register_cache(pybind11::module_& m) {
  m.def("norm_rotary", &norm_rotary);
  m.def("kv_write", &kv_write);
  m.def("kv_read", [](const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& table, const Tensor& start,
                      const Tensor& seqlens, int64_t length, bool fp16) {
    return kv_read(k, v, ks, vs, table, start, seqlens, length, fp16 ? at::kHalf : at::kBFloat16);
  });
  m.def("kv_attention", &kv_attention);
}

}  // namespace fm_host

// Native kernels of the torch ops over packed sequences and over a paged cache:
// farope::seq_fwd, seq_bwd, cache_append and cache_attn (defined in sequences.py,
// which also refuses CPU tensors).  As in torch_ops.cpp: argument checks,
// allocation and the C ABI call without the interpreter, and a native autograd
// node.  Nothing is read back from the device: sequence starts, lengths and page
// numbers are the kernels' to check.
#include "torch_util.h"

namespace {

using namespace farope_torch;
using Two = std::tuple<Tensor, Tensor>;
using Three = std::tuple<Tensor, Tensor, Tensor>;
using Opt = std::optional<Tensor>;

void check_heads(const Tensor& x, const char* name, const char* shape) {
  TORCH_CHECK_VALUE(x.dim() == 3, name, " must be ", shape, "; got shape ", shape_str(x));
}
void check_like(const Tensor& x, const char* name, const Tensor& q) {
  TORCH_CHECK_TYPE(x.scalar_type() == q.scalar_type(), "farope: ", name, " must share the other tensors' dtype; got ",
                   dtype_str(x), " and ", dtype_str(q));
  TORCH_CHECK(x.device() == q.device(), "farope: ", name, " must be on the other tensors' device");
}
void check_first(const Tensor& x) {
  TORCH_CHECK_TYPE(dtype_code(x.scalar_type()) >= 0, "farope: unsupported tensor dtype ", dtype_str(x));
  TORCH_CHECK(x.is_cuda(), "farope runs on ROCm GPUs only (hand-written gfx950 kernels); got a ", x.device(), " tensor");
}
void check_head_dim(int64_t D) {
  TORCH_CHECK_VALUE(D == 32 || D == 64 || D == 128 || D == 256, "farope: head_dim must be 32, 64, 128 or 256; got ", D);
}
void check_ints(const Tensor& x, const char* name, int64_t n, const Tensor& q) {
  TORCH_CHECK_TYPE(x.scalar_type() == at::kInt, "farope: ", name, " must be int32; got ", dtype_str(x));
  TORCH_CHECK_VALUE(x.dim() == 1 && (n < 0 || x.size(0) == n) && x.is_contiguous(), "farope: ", name,
                    " must be contiguous with ", n < 0 ? std::string("one dimension") : std::to_string(n) + " elements",
                    "; got shape ", shape_str(x));
  TORCH_CHECK(x.device() == q.device(), "farope: ", name, " must be on the other tensors' device");
}
void check_cu(const Tensor& cu, const Tensor& q) {
  check_ints(cu, "cu_seqlens", -1, q);
  TORCH_CHECK_VALUE(cu.size(0) >= 2, "farope: cu_seqlens must hold at least one sequence (2 elements)");
}
void check_tables(const Tensor& c, const Tensor& s, int64_t D, const Tensor& q) {
  TORCH_CHECK_VALUE(c.scalar_type() == at::kFloat && s.scalar_type() == at::kFloat && c.dim() == 2 && c.sizes() == s.sizes() &&
                        c.size(0) >= 1 && c.size(1) == D / 2 && c.is_contiguous() && s.is_contiguous(),
                    "farope: RoPE tables must be contiguous fp32 [n_pos, ", D / 2, "]; got ", dtype_str(c), " ", shape_str(c),
                    " and ", dtype_str(s), " ", shape_str(s));
  TORCH_CHECK(c.device() == q.device() && s.device() == q.device(), "farope: RoPE tables on ", c.device(), ", tensors on ",
              q.device());
}
const int32_t* ints(const Opt& x) { return x && x->defined() ? x->data_ptr<int32_t>() : nullptr; }
int32_t to32(int64_t x) {
  TORCH_CHECK_VALUE(x >= 0 && x <= INT32_MAX, "farope: sizes must fit 32 bits");
  return (int32_t)x;
}

farope_seq_desc make_desc(int64_t tokens, int64_t seqs, int64_t heads, int64_t kv_heads, const Tensor& x, const Tensor& cosp,
                          bool causal, bool has_cls, double scale) {
  farope_seq_desc d;
  d.tokens = to32(tokens);
  d.seqs = to32(seqs);
  d.heads = to32(heads);
  d.kv_heads = to32(kv_heads);
  d.head_dim = to32(x.size(-1));
  d.n_pos = to32(cosp.size(0));
  d.has_cls = has_cls;
  d.causal = causal;
  d.dtype = dtype_code(x.scalar_type());
  d.softmax_scale = (float)scale;
  return d;
}

void check_seq(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cosp, const Tensor& sinp, const Tensor& cu,
               const Opt& positions) {
  check_heads(q, "Q", "[T, H, D]");
  check_heads(k, "K", "[T, Hkv, D]");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "K and V must have the same shape; got ", shape_str(k), " and ", shape_str(v));
  TORCH_CHECK_VALUE(k.size(0) == q.size(0) && k.size(2) == q.size(2), "Q and K must agree in tokens and head_dim; got ",
                    shape_str(q), " and ", shape_str(k));
  TORCH_CHECK_VALUE(k.size(1) >= 1 && q.size(1) >= 1 && q.size(1) % k.size(1) == 0,
                    "farope: query heads must be a multiple of key heads; got ", q.size(1), " and ", k.size(1));
  check_head_dim(q.size(2));
  check_first(q);
  check_like(k, "K", q);
  check_like(v, "V", q);
  check_tables(cosp, sinp, q.size(2), q);
  check_cu(cu, q);
  if (positions) check_ints(*positions, "positions", q.size(0), q);
}

Two seq_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cosp, const Tensor& sinp, const Tensor& cu,
            const Opt& positions, bool causal, bool has_cls, double scale) {
  check_seq(q, k, v, cosp, sinp, cu, positions);
  const c10::DeviceGuard guard(q.device());
  const farope_seq_desc d = make_desc(q.size(0), cu.size(0) - 1, q.size(1), k.size(1), q, cosp, causal, has_cls, scale);
  const Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  const Tensor lse = at::empty({q.size(1), q.size(0)}, q.options().dtype(at::kFloat));
  if (d.tokens == 0) return {o, lse};
  const Tensor ws = workspace(q, farope_seq_workspace_elems(&d, 0, farope_seq_streams(&d, v.data_ptr(), strides(v)), 1));
  check_rc(farope_seq_fwd(&d, q.data_ptr(), strides(q), k.data_ptr(), strides(k), v.data_ptr(), strides(v), floats(cosp),
                          floats(sinp), ints(positions), cu.data_ptr<int32_t>(), o.data_ptr(), lse.data_ptr<float>(),
                          floats(ws), ws.defined() ? ws.numel() : 0, stream_of(q)),
           "farope_seq_fwd");
  return {o, lse};
}

Three seq_bwd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse,
              const Tensor& cosp, const Tensor& sinp, const Tensor& cu, const Opt& positions, bool causal, bool has_cls,
              double scale) {
  check_seq(q, k, v, cosp, sinp, cu, positions);
  TORCH_CHECK_VALUE(dout.sizes() == q.sizes() && o.sizes() == q.sizes() && o.is_contiguous(),
                    "farope: dO and O must have Q's shape, O contiguous");
  TORCH_CHECK(dout.device() == q.device(), "farope: dO must be on Q's device");
  check_like(o, "O", q);
  TORCH_CHECK_VALUE(lse.scalar_type() == at::kFloat && lse.dim() == 2 && lse.size(0) == q.size(1) && lse.size(1) == q.size(0) &&
                        lse.is_contiguous(),
                    "farope: LSE must be contiguous fp32 [H, T]");
  TORCH_CHECK(lse.device() == q.device(), "farope: LSE must be on Q's device");
  const c10::DeviceGuard guard(q.device());
  const Tensor g = dout.scalar_type() == q.scalar_type() ? dout : dout.to(q.scalar_type());
  const farope_seq_desc d = make_desc(q.size(0), cu.size(0) - 1, q.size(1), k.size(1), q, cosp, causal, has_cls, scale);
  const auto dense = [](const Tensor& t) { return at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)); };
  const Tensor dq = dense(q), dk = dense(k), dv = dense(v);
  if (d.tokens == 0) return {dq, dk, dv};
  const Tensor ws = workspace(q, farope_seq_workspace_elems(&d, 1, farope_seq_streams(&d, v.data_ptr(), strides(v)),
                                                            farope_seq_streams(&d, g.data_ptr(), strides(g))));
  check_rc(farope_seq_bwd(&d, q.data_ptr(), strides(q), k.data_ptr(), strides(k), v.data_ptr(), strides(v), o.data_ptr(),
                          g.data_ptr(), strides(g), lse.data_ptr<float>(), floats(cosp), floats(sinp), ints(positions),
                          cu.data_ptr<int32_t>(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), floats(ws),
                          ws.defined() ? ws.numel() : 0, stream_of(q)),
           "farope_seq_bwd");
  return {dq, dk, dv};
}

farope_cache_desc check_cache(const Tensor& kc, const Tensor& vc, const Tensor& pages, const Tensor& lengths, int64_t kv_heads,
                              const Tensor& x) {
  TORCH_CHECK_VALUE(kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.size(2) == kv_heads && kc.size(3) == x.size(2),
                    "farope: the caches must be [pages, page_rows, Hkv, D] with Hkv=", kv_heads, ", D=", x.size(2), "; got ",
                    shape_str(kc), " and ", shape_str(vc));
  TORCH_CHECK_VALUE(kc.size(0) >= 1 && kc.size(1) >= 1, "farope: the caches have no rows: ", shape_str(kc));
  check_like(kc, "the key cache", x);
  check_like(vc, "the value cache", x);
  for (const Tensor* t : {&kc, &vc}) {
    bool ok = t->stride(3) == 1 && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0;
    for (int i = 0; i < 3; ++i) ok = ok && t->stride(i) * (int64_t)t->element_size() % 16 == 0;
    TORCH_CHECK_VALUE(ok, "farope: cache rows must have contiguous channels and be 16-byte aligned");
  }
  TORCH_CHECK_TYPE(pages.scalar_type() == at::kInt, "farope: page_table must be int32; got ", dtype_str(pages));
  TORCH_CHECK_VALUE(pages.dim() == 2 && pages.size(1) >= 1 && (pages.size(1) == 1 || pages.stride(1) == 1),
                    "farope: page_table must be [B, max_pages], its rows contiguous; got shape ", shape_str(pages));
  TORCH_CHECK(pages.device() == x.device(), "farope: page_table must be on the other tensors' device");
  check_ints(lengths, "lengths", pages.size(0), x);
  farope_cache_desc c;
  c.k = kc.data_ptr();
  c.v = vc.data_ptr();
  for (int i = 0; i < 3; ++i) {
    c.k_stride[i] = kc.stride(i);
    c.v_stride[i] = vc.stride(i);
  }
  c.pages = to32(kc.size(0));
  c.page_rows = to32(kc.size(1));
  c.max_pages = to32(pages.size(1));
  c.table_stride = pages.stride(0);
  return c;
}

void cache_append(const Tensor& k, const Tensor& v, const Tensor& cosp, const Tensor& sinp, Tensor kc, Tensor vc,
                  const Tensor& pages, const Tensor& lengths, const Opt& cu, const Opt& positions, bool has_cls) {
  check_heads(k, "K", "[T, Hkv, D]");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(1) >= 1, "K and V must have the same shape; got ", shape_str(k), " and ",
                    shape_str(v));
  check_head_dim(k.size(2));
  check_first(k);
  check_like(v, "V", k);
  check_tables(cosp, sinp, k.size(2), k);
  const farope_cache_desc c = check_cache(kc, vc, pages, lengths, k.size(1), k);
  if (cu) {
    check_cu(*cu, k);
    TORCH_CHECK_VALUE(cu->size(0) == pages.size(0) + 1, "farope: cu_seqlens must hold the page table's ", pages.size(0),
                      " sequences; got ", cu->size(0), " elements");
  } else {
    TORCH_CHECK_VALUE(k.size(0) == pages.size(0), "farope: without cu_seqlens every sequence gets one token; got ", k.size(0),
                      " for ", pages.size(0), " sequences");
  }
  if (positions) check_ints(*positions, "positions", k.size(0), k);
  if (k.size(0) == 0) return;
  const c10::DeviceGuard guard(k.device());
  const farope_seq_desc d = make_desc(k.size(0), pages.size(0), k.size(1), k.size(1), k, cosp, true, has_cls, 1.0);
  check_rc(farope_cache_append(&d, k.data_ptr(), strides(k), v.data_ptr(), strides(v), floats(cosp), floats(sinp),
                               ints(positions), &c, pages.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), ints(cu),
                               stream_of(k)),
           "farope_cache_append");
}

Tensor cache_attn(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& cosp, const Tensor& sinp,
                  const Tensor& pages, const Tensor& lengths, const Opt& positions, bool has_cls, double scale) {
  check_heads(q, "Q", "[B, H, D]");
  check_head_dim(q.size(2));
  check_first(q);
  TORCH_CHECK_VALUE(kc.dim() == 4 && kc.size(2) >= 1 && q.size(1) >= 1 && q.size(1) % kc.size(2) == 0,
                    "farope: query heads must be a multiple of the cache's key heads; got ", shape_str(q), " and ", shape_str(kc));
  check_tables(cosp, sinp, q.size(2), q);
  const farope_cache_desc c = check_cache(kc, vc, pages, lengths, kc.size(2), q);
  TORCH_CHECK_VALUE(q.size(0) == pages.size(0), "farope: one query per sequence: got ", q.size(0), " for ", pages.size(0),
                    " sequences");
  if (positions) check_ints(*positions, "positions", q.size(0), q);
  const c10::DeviceGuard guard(q.device());
  const Tensor o = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  if (q.size(0) == 0) return o;
  const farope_seq_desc d = make_desc(q.size(0), q.size(0), q.size(1), kc.size(2), q, cosp, true, has_cls, scale);
  const Tensor ws = workspace(q, farope_decode_workspace_elems(&d, &c));
  check_rc(farope_decode(&d, q.data_ptr(), strides(q), floats(cosp), floats(sinp), ints(positions), &c,
                         pages.data_ptr<int32_t>(), lengths.data_ptr<int32_t>(), o.data_ptr(), floats(ws),
                         ws.defined() ? ws.numel() : 0, stream_of(q)),
           "farope_decode");
  return o;
}

// ---------------------------------------------------------------------------
// Autograd
// ---------------------------------------------------------------------------
using FwdSig = Two(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Opt&, bool,
                   bool, double);
using BwdSig = Three(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                     const Tensor&, const Tensor&, const Opt&, bool, bool, double);
using AppendSig = void(const Tensor&, const Tensor&, const Tensor&, const Tensor&, Tensor, Tensor, const Tensor&, const Tensor&,
                       const Opt&, const Opt&, bool);
using AttnSig = Tensor(const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                       const Opt&, bool, double);
template <typename Sig> c10::TypedOperatorHandle<Sig> find(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Sig>();
}
const c10::TypedOperatorHandle<FwdSig>& fwd_op() {
  static const auto op = find<FwdSig>("farope::seq_fwd");
  return op;
}
const c10::TypedOperatorHandle<BwdSig>& bwd_op() {
  static const auto op = find<BwdSig>("farope::seq_bwd");
  return op;
}
const c10::TypedOperatorHandle<AppendSig>& append_op() {
  static const auto op = find<AppendSig>("farope::cache_append");
  return op;
}
const c10::TypedOperatorHandle<AttnSig>& attn_op() {
  static const auto op = find<AttnSig>("farope::cache_attn");
  return op;
}

struct SeqFwdNode : torch::autograd::Function<SeqFwdNode> {
  static variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                               const Tensor& cosp, const Tensor& sinp, const Tensor& cu, const Opt& positions, bool causal,
                               bool has_cls, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Two r = fwd_op().call(q, k, v, cosp, sinp, cu, positions, causal, has_cls, scale);
    const auto& [o, lse] = r;
    ctx->mark_non_differentiable({lse});
    ctx->set_materialize_grads(false);   // (LSE's gradient is never used)
    ctx->save_for_backward({q, k, v, o, lse, cosp, sinp, cu, positions ? *positions : Tensor()});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["has_cls"] = has_cls;
    ctx->saved_data["scale"] = scale;
    return {o, lse};
  }
  static variable_list backward(torch::autograd::AutogradContext* ctx, variable_list grads) {
    variable_list out(10);
    if (!grads[0].defined()) return out;   // O received no gradient
    const variable_list s = ctx->get_saved_variables();
    std::tie(out[0], out[1], out[2]) =
        bwd_op().call(grads[0], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], s[8].defined() ? Opt(s[8]) : Opt(),
                      ctx->saved_data["causal"].toBool(), ctx->saved_data["has_cls"].toBool(), ctx->saved_data["scale"].toDouble());
    return out;
  }
};
Two seq_fwd_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cosp, const Tensor& sinp, const Tensor& cu,
                     const Opt& positions, bool causal, bool has_cls, double scale) {
  refuse_tangents("seq_fwd", {&q, &k, &v, &cosp, &sinp});
  if (at::GradMode::is_enabled() && any_requires_grad({&q, &k, &v})) {
    const variable_list r = SeqFwdNode::apply(q, k, v, cosp, sinp, cu, positions, causal, has_cls, scale);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return fwd_op().call(q, k, v, cosp, sinp, cu, positions, causal, has_cls, scale);
}

// The gradients are not differentiable again.
struct SeqBwdNode : torch::autograd::Function<SeqBwdNode> {
  static variable_list forward(torch::autograd::AutogradContext*, const Tensor& dout, const Tensor& q, const Tensor& k,
                               const Tensor& v, const Tensor& o, const Tensor& lse, const Tensor& cosp, const Tensor& sinp,
                               const Tensor& cu, const Opt& positions, bool causal, bool has_cls, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Three r = bwd_op().call(dout, q, k, v, o, lse, cosp, sinp, cu, positions, causal, has_cls, scale);
    return {std::get<0>(r), std::get<1>(r), std::get<2>(r)};
  }
  static variable_list backward(torch::autograd::AutogradContext*, variable_list) {
    TORCH_CHECK(false,
                "Trying to backward through farope.seq_bwd.default but no autograd formula was registered "
                "(the attention's gradients are not differentiable again).");
  }
};
Three seq_bwd_autograd(const Tensor& dout, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& lse,
                       const Tensor& cosp, const Tensor& sinp, const Tensor& cu, const Opt& positions, bool causal, bool has_cls,
                       double scale) {
  refuse_tangents("seq_bwd", {&dout, &q, &k, &v, &o, &lse, &cosp, &sinp});
  if (at::GradMode::is_enabled() && any_requires_grad({&dout, &q, &k, &v, &o, &lse})) {
    const variable_list r = SeqBwdNode::apply(dout, q, k, v, o, lse, cosp, sinp, cu, positions, causal, has_cls, scale);
    return {r[0], r[1], r[2]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  return bwd_op().call(dout, q, k, v, o, lse, cosp, sinp, cu, positions, causal, has_cls, scale);
}

// A cache is no part of an autograd graph.
void cache_append_autograd(const Tensor& k, const Tensor& v, const Tensor& cosp, const Tensor& sinp, Tensor kc, Tensor vc,
                           const Tensor& pages, const Tensor& lengths, const Opt& cu, const Opt& positions, bool has_cls) {
  refuse_tangents("cache_append", {&k, &v, &kc, &vc, &cosp, &sinp});
  TORCH_CHECK(!at::GradMode::is_enabled() || !any_requires_grad({&k, &v, &kc, &vc}),
              "farope: appending to a cache is not differentiable; call it under torch.no_grad() or with detached tensors");
  {
    at::AutoDispatchBelowADInplaceOrView below;
    append_op().call(k, v, cosp, sinp, kc, vc, pages, lengths, cu, positions, has_cls);
  }
  for (Tensor* t : {&kc, &vc})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

struct CacheAttnNode : torch::autograd::Function<CacheAttnNode> {
  static Tensor forward(torch::autograd::AutogradContext*, const Tensor& q, const Tensor& kc, const Tensor& vc,
                        const Tensor& cosp, const Tensor& sinp, const Tensor& pages, const Tensor& lengths, const Opt& positions,
                        bool has_cls, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    return attn_op().call(q, kc, vc, cosp, sinp, pages, lengths, positions, has_cls, scale);
  }
  static variable_list backward(torch::autograd::AutogradContext*, variable_list) {
    TORCH_CHECK(false, "Trying to backward through farope.cache_attn.default but no autograd formula was registered "
                       "(attention over a cache has no gradients).");
  }
};
Tensor cache_attn_autograd(const Tensor& q, const Tensor& kc, const Tensor& vc, const Tensor& cosp, const Tensor& sinp,
                           const Tensor& pages, const Tensor& lengths, const Opt& positions, bool has_cls, double scale) {
  refuse_tangents("cache_attn", {&q, &kc, &vc, &cosp, &sinp});
  if (at::GradMode::is_enabled() && any_requires_grad({&q, &kc, &vc}))
    return CacheAttnNode::apply(q, kc, vc, cosp, sinp, pages, lengths, positions, has_cls, scale);
  at::AutoDispatchBelowADInplaceOrView below;
  return attn_op().call(q, kc, vc, cosp, sinp, pages, lengths, positions, has_cls, scale);
}

}  // namespace

TORCH_LIBRARY_IMPL(farope, CUDA, m) {
  m.impl("seq_fwd", seq_fwd);
  m.impl("seq_bwd", seq_bwd);
  m.impl("cache_append", cache_append);
  m.impl("cache_attn", cache_attn);
}

TORCH_LIBRARY_IMPL(farope, AutogradCUDA, m) {
  m.impl("seq_fwd", seq_fwd_autograd);
  m.impl("seq_bwd", seq_bwd_autograd);
  m.impl("cache_append", cache_append_autograd);
  m.impl("cache_attn", cache_attn_autograd);
}

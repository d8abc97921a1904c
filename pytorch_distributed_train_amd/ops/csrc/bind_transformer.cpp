// Python binding of the transformer-training operators: AdamW,
// query/key norm with rotation, attention with recomputed probabilities.
// Arguments are checked here, before a launch: a kernel's bounds rest on them.
#include <torch/extension.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>

#include <hip/hip_runtime_api.h>

#include <cmath>
#include <vector>

extern "C" {
void pdta_adamw(float*, const float*, void*, void*, float*, float*, long,
                long*, float, const float*, double, double, float, float,
                const unsigned char*, float, unsigned, void*, hipStream_t);
int pdta_qknorm_rows(long, int, int);
void pdta_qknorm(const void* const*, const long*, const void* const*,
                 const long*, const float* const*, void* const*, const long*,
                 const int*,
                 const float*, const float*, const void*, int, int, int, int,
                 long, long, float, int, int, int, float*, float*, float*,
                 int, hipStream_t);
void pdta_attn_recompute(const void*, const void*, const void*, const void*,
                         const long*, void*, float*, void*, void*, void*,
                         const void*, const void*, int, int, int, int,
                         int, int, int, float, int, int, float*, int,
                         hipStream_t);
long pdta_attn_recompute_ws(long, long, long, long, long, long, int, int,
                            int);
}

namespace {

// the current stream of the current device (call under a DeviceGuard)
hipStream_t cur_stream() {
  return (hipStream_t)at::hip::getCurrentHIPStreamMasqueradingAsCUDA()
      .stream();
}

void launched(const char* what) {
  hipError_t e = hipGetLastError();
  TORCH_CHECK(e == hipSuccess, what, ": launch failed: ",
              hipGetErrorString(e));
}

// a flat array on `like`'s device that the 16-byte accesses may walk
void check_flat(const char* name, const at::Tensor& t, const at::Tensor& like,
                at::ScalarType dtype, long numel) {
  TORCH_CHECK(t.device() == like.device(), name, " must be on ",
              like.device(), ", is on ", t.device());
  TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", is ",
              t.scalar_type());
  TORCH_CHECK(t.is_contiguous() && t.numel() == numel, name,
              " must be contiguous with ", numel, " elements");
  TORCH_CHECK((uintptr_t)t.data_ptr() % 16 == 0, name,
              " must start at a multiple of 16 bytes");
}

int dt_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK(false, "unsupported dtype ", t.scalar_type());
  }
}

void adamw_step(at::Tensor p, at::Tensor g, at::Tensor m, at::Tensor v,
                at::Tensor step, double lr, c10::optional<at::Tensor> lr_dev,
                double beta1, double beta2, double eps, double weight_decay,
                c10::optional<at::Tensor> decay, double grad_scale,
                c10::optional<at::Tensor> m_scale,
                c10::optional<at::Tensor> v_scale, int64_t seed) {
  TORCH_CHECK(p.is_cuda(), "p must be on GPU");
  c10::DeviceGuard guard(p.device());
  long n = p.numel();
  TORCH_CHECK(n % 64 == 0, "p must have a multiple of 64 elements, has ", n);
  check_flat("p", p, p, at::kFloat, n);
  check_flat("g", g, p, at::kFloat, n);
  bool eight = m_scale.has_value();
  TORCH_CHECK(eight == v_scale.has_value(),
              "m_scale and v_scale come together");
  auto st = eight ? at::kFloat8_e4m3fn : at::kFloat;
  check_flat("m", m, p, st, n);
  check_flat("v", v, p, st, n);
  if (eight) {
    check_flat("m_scale", *m_scale, p, at::kFloat, n / 64);
    check_flat("v_scale", *v_scale, p, at::kFloat, n / 64);
  }
  if (decay.has_value()) check_flat("decay", *decay, p, at::kByte, n / 64);
  TORCH_CHECK(step.device() == p.device() &&
                  step.scalar_type() == at::kLong && step.numel() == 1,
              "step must be one int64 on ", p.device());
  if (lr_dev.has_value())
    TORCH_CHECK(lr_dev->device() == p.device() &&
                    lr_dev->scalar_type() == at::kFloat &&
                    lr_dev->numel() == 1,
                "lr must be one float32 on ", p.device());
  auto hyp = at::empty({4}, p.options());
  pdta_adamw(p.data_ptr<float>(), g.data_ptr<float>(), m.data_ptr(),
             v.data_ptr(), eight ? m_scale->data_ptr<float>() : nullptr,
             eight ? v_scale->data_ptr<float>() : nullptr, n,
             (long*)step.data_ptr<int64_t>(), (float)lr,
             lr_dev.has_value() ? lr_dev->data_ptr<float>() : nullptr, beta1,
             beta2, (float)eps, (float)weight_decay,
             decay.has_value() ? decay->data_ptr<uint8_t>() : nullptr,
             (float)grad_scale, (unsigned)seed, hyp.data_ptr(),
             cur_stream());
  launched("adamw_step");
}

// ---- query/key norm and rotation -----------------------------------------
// q [b, s, h, hd], k [b, s, hk, hd]; a dimension of one element has no
// stride to speak of
bool rows8(const at::Tensor& t) {
  if ((uintptr_t)t.data_ptr() % 16) return false;
  for (int d = 0; d < 3; ++d)
    if (t.size(d) > 1 && t.stride(d) % 8) return false;
  return true;
}

// dq, dk undefined: forward -> {q', k'}; else backward -> {dx_q, dx_k,
// dw_q, dw_k} (the last two empty without weights). outs: where the results
// go instead of new tensors, in the same order.
using Outs = std::vector<at::Tensor>;
std::vector<at::Tensor> qk_norm_rope(
    at::Tensor q, at::Tensor k, c10::optional<at::Tensor> wq,
    c10::optional<at::Tensor> wk, c10::optional<at::Tensor> cos,
    c10::optional<at::Tensor> sin, c10::optional<at::Tensor> positions,
    double eps, bool interleaved, c10::optional<at::Tensor> dq,
    c10::optional<at::Tensor> dk, const Outs& outs = {}) {
  TORCH_CHECK(q.is_cuda(), "q must be on GPU");
  c10::DeviceGuard guard(q.device());
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) &&
                  q.size(1) == k.size(1) && q.size(3) == k.size(3),
              "q and k must be [b, s, heads, hd], alike but for the heads");
  long b = q.size(0), s = q.size(1), hd = q.size(3);
  TORCH_CHECK(hd >= 1 && hd <= 256, "head size must be 1 to 256, is ", hd);
  // the forward has a wave a token; a grid holds 2^32 threads
  TORCH_CHECK(b * s < (1l << 26) - 4 && q.size(2) + k.size(2) < 65536,
              "too many rows");
  bool bwd = dq.has_value();
  TORCH_CHECK(bwd == dk.has_value(), "dq and dk come together");
  bool norm = wq.has_value();
  TORCH_CHECK(norm == wk.has_value(), "q_weight and k_weight come together");
  at::Tensor t[2] = {q, k}, d[2];
  if (bwd) d[0] = *dq, d[1] = *dk;
  bool vec = hd % 8 == 0;
  const void *x[2], *dy[2] = {nullptr, nullptr};
  long xs[6], gs[6] = {0, 0, 0, 0, 0, 0};
  const float* w[2] = {nullptr, nullptr};
  int heads[2];
  for (int i = 0; i < 2; ++i) {
    TORCH_CHECK(t[i].device() == q.device() &&
                    t[i].scalar_type() == q.scalar_type(),
                "q and k must have one device and dtype");
    TORCH_CHECK(hd == 1 || t[i].numel() == 0 || t[i].stride(3) == 1,
                "heads must be contiguous in memory");
    vec = vec && rows8(t[i]);
    x[i] = t[i].data_ptr();
    heads[i] = t[i].size(2);
    for (int j = 0; j < 3; ++j) xs[3 * i + j] = t[i].stride(j);
    if (bwd) {
      TORCH_CHECK(d[i].device() == q.device() &&
                      d[i].scalar_type() == q.scalar_type() &&
                      d[i].sizes() == t[i].sizes() &&
                      (hd == 1 || d[i].numel() == 0 || d[i].stride(3) == 1),
                  "a gradient must be like its output");
      vec = vec && rows8(d[i]);
      dy[i] = d[i].data_ptr();
      for (int j = 0; j < 3; ++j) gs[3 * i + j] = d[i].stride(j);
    }
    if (norm) {
      const at::Tensor& wt = i ? *wk : *wq;
      TORCH_CHECK(wt.device() == q.device() &&
                      wt.scalar_type() == at::kFloat && wt.numel() == hd &&
                      wt.is_contiguous(),
                  "weights must be contiguous float32 [", hd, "] on ",
                  q.device());
      vec = vec && (uintptr_t)wt.data_ptr() % 16 == 0;
      w[i] = wt.data_ptr<float>();
    }
  }
  long rot = 0, npos = 0;
  bool pos32 = false;
  TORCH_CHECK(cos.has_value() == sin.has_value(),
              "cos and sin come together");
  TORCH_CHECK(cos.has_value() || norm, "neither weights nor tables");
  if (cos.has_value()) {
    TORCH_CHECK(cos->dim() == 2 && cos->sizes() == sin->sizes() &&
                    cos->device() == q.device() &&
                    sin->device() == q.device() &&
                    cos->scalar_type() == at::kFloat &&
                    sin->scalar_type() == at::kFloat &&
                    cos->is_contiguous() && sin->is_contiguous(),
                "cos and sin must be contiguous float32 [positions, rot/2] "
                "on ",
                q.device());
    npos = cos->size(0);
    rot = 2 * cos->size(1);
    TORCH_CHECK(rot >= 2 && rot <= hd, "tables for ", rot,
                " elements, heads have ", hd);
    TORCH_CHECK(npos < (1l << 31), "too many positions");
    TORCH_CHECK(positions.has_value() || s <= npos, "tables for ", npos,
                " positions, sequences of ", s);
    vec = vec && rot % (interleaved ? 8 : 16) == 0 &&
          (uintptr_t)cos->data_ptr() % 16 == 0 &&
          (uintptr_t)sin->data_ptr() % 16 == 0;
  }
  if (positions.has_value()) {
    TORCH_CHECK(positions->device() == q.device() &&
                    positions->is_contiguous() &&
                    positions->numel() == b * s,
                "positions must be contiguous [b, s] on ", q.device());
    pos32 = positions->scalar_type() == at::kInt;
    TORCH_CHECK(pos32 || positions->scalar_type() == at::kLong,
                "positions must be int32 or int64");
  }
  at::Tensor y[2], dw[2];
  void* yp[2];
  long ys[6];
  auto f32 = q.options().dtype(at::kFloat);
  bool dws = bwd && norm;
  TORCH_CHECK(outs.empty() || outs.size() == (dws ? 4 : 2),
              "outs must be all results");
  for (int i = 0; i < 2; ++i) {
    if (outs.empty()) {
      y[i] = at::empty({b, s, heads[i], hd}, q.options());
      if (dws) dw[i] = at::empty({hd}, f32);
    } else {
      y[i] = outs[i];
      TORCH_CHECK(y[i].device() == q.device() &&
                      y[i].scalar_type() == q.scalar_type() &&
                      y[i].sizes() == t[i].sizes() &&
                      (y[i].numel() == 0 || y[i].stride(3) == 1),
                  "a result must be like its input");
      if (dws) {
        dw[i] = outs[2 + i];
        check_flat("a weight's gradient", dw[i], q, at::kFloat, hd);
      }
    }
    vec = vec && rows8(y[i]);
    yp[i] = y[i].data_ptr();
    for (int j = 0; j < 3; ++j) ys[3 * i + j] = y[i].stride(j);
  }
  at::Tensor part;
  if (dws) {
    int rows = pdta_qknorm_rows(b * s, heads[0] + heads[1], vec);
    if (rows == 0) return {y[0], y[1], dw[0].zero_(), dw[1].zero_()};
    part = at::empty({rows, 2 * hd}, f32);
  }
  pdta_qknorm(x, xs, dy, gs, w, yp, ys, heads,
              rot ? cos->data_ptr<float>() : nullptr,
              rot ? sin->data_ptr<float>() : nullptr,
              positions.has_value() ? positions->data_ptr() : nullptr, pos32,
              npos, rot, hd, b, s, (float)eps, interleaved, vec, bwd,
              dws ? part.data_ptr<float>() : nullptr,
              dws ? dw[0].data_ptr<float>() : nullptr,
              dws ? dw[1].data_ptr<float>() : nullptr, dt_of(q),
              cur_stream());
  launched("qk_norm_rope");
  if (!bwd) return {y[0], y[1]};
  if (!norm) return {y[0], y[1], at::Tensor(), at::Tensor()};
  return {y[0], y[1], dw[0], dw[1]};
}

// ---- attention with recomputed probabilities -----------------------------
struct AttnShape {
  long b, sq, sk, h, hk, hd;
};

AttnShape attn_check(const at::Tensor& q, const at::Tensor& k,
                     const at::Tensor& v,
                     const c10::optional<at::Tensor>& q_lens,
                     const c10::optional<at::Tensor>& kv_lens, double scale) {
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
              "q, k and v must be [b, s, heads, hd]");
  AttnShape n = {q.size(0), q.size(1), k.size(1),
                 q.size(2), k.size(2), q.size(3)};
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == n.b &&
                  k.size(3) == n.hd,
              "k and v must be [", n.b, ", sk, hk, ", n.hd, "]");
  TORCH_CHECK(n.hd >= 8 && n.hd <= 128 && n.hd % 8 == 0,
              "head size must be a multiple of 8 up to 128, is ", n.hd);
  TORCH_CHECK(n.hk > 0 ? n.h % n.hk == 0 : n.h == 0, "heads of q (", n.h,
              ") must be a multiple of those of k (", n.hk, ")");
  TORCH_CHECK(q.scalar_type() == at::kBFloat16 ||
                  q.scalar_type() == at::kHalf,
              "q must be bfloat16 or float16 on GPU, is ", q.scalar_type());
  for (const at::Tensor* t : {&q, &k, &v}) {
    TORCH_CHECK(t->device() == q.device() &&
                    t->scalar_type() == q.scalar_type(),
                "q, k and v must have one device and dtype");
    TORCH_CHECK(t->numel() == 0 || (t->stride(3) == 1 && rows8(*t)),
                "rows must be contiguous, 16-byte aligned, strides "
                "multiples of 8");
  }
  long g = n.hk ? n.h / n.hk : 1;
  // blocks of 256 threads for 128 rows or keys; a grid holds 2^32 threads
  TORCH_CHECK((n.sq + n.sk + 1024) * g < (1l << 31) &&
                  n.b * n.hk * ((n.sq * g + n.sk) / 128 + 2) < (1l << 24),
              "attention: too many rows");
  for (const auto* l : {&q_lens, &kv_lens})
    if (l->has_value()) {
      const at::Tensor& t = **l;
      TORCH_CHECK(t.device() == q.device() && t.is_contiguous() &&
                      t.numel() == n.b &&
                      (t.scalar_type() == at::kInt ||
                       t.scalar_type() == at::kLong),
                  "lengths must be contiguous int32 or int64 [", n.b, "] on ",
                  q.device());
    }
  if (q_lens.has_value() && kv_lens.has_value())
    TORCH_CHECK(q_lens->scalar_type() == kv_lens->scalar_type(),
                "q_lens and kv_lens must have one dtype");
  TORCH_CHECK(scale > 0.0 && std::isfinite((float)scale) &&
                  (float)scale > 0.f,
              "scale must be positive, is ", scale);
  return n;
}

void attn_strides(const at::Tensor& t, long* st) {
  // a dimension of one element is never stepped along
  for (int d = 0; d < 3; ++d) st[d] = t.size(d) > 1 ? t.stride(d) : 0;
}

const void* len_ptr(const c10::optional<at::Tensor>& t) {
  return t.has_value() ? t->data_ptr() : nullptr;
}

bool lens_wide(const c10::optional<at::Tensor>& a,
               const c10::optional<at::Tensor>& b) {
  const auto& t = a.has_value() ? a : b;
  return t.has_value() && t->scalar_type() == at::kLong;
}

// {out [b, sq, h, hd], lse [b, hk, sq * h / hk] (empty unless want_lse)}
std::vector<at::Tensor> attn_recompute_fwd(
    at::Tensor q, at::Tensor k, at::Tensor v,
    c10::optional<at::Tensor> q_lens, c10::optional<at::Tensor> kv_lens,
    double scale, bool causal, bool want_lse) {
  TORCH_CHECK(q.is_cuda(), "q must be on GPU");
  c10::DeviceGuard guard(q.device());
  AttnShape n = attn_check(q, k, v, q_lens, kv_lens, scale);
  long g = n.hk ? n.h / n.hk : 1;
  auto out = at::empty({n.b, n.sq, n.h, n.hd}, q.options());
  auto lse = at::empty({want_lse ? n.b * n.hk * n.sq * g : 0},
                       q.options().dtype(at::kFloat));
  long st[15] = {0};
  attn_strides(q, st);
  attn_strides(k, st + 3);
  attn_strides(v, st + 6);
  if (out.numel()) {
    bool lens = q_lens.has_value() || kv_lens.has_value();
    long need = pdta_attn_recompute_ws(n.b, n.sq, n.sk, n.hk, g, n.hd, causal,
                                       lens, 0);
    at::Tensor ws;
    if (need) ws = at::empty({need}, lse.options());
    pdta_attn_recompute(q.data_ptr(), k.data_ptr(), v.data_ptr(), nullptr,
                        st, out.data_ptr(),
                        want_lse ? lse.data_ptr<float>() : nullptr, nullptr,
                        nullptr, nullptr, len_ptr(q_lens),
                        len_ptr(kv_lens), lens_wide(q_lens, kv_lens), n.b,
                        n.sq, n.sk, n.hk, g, n.hd, (float)scale, causal, 0,
                        need ? ws.data_ptr<float>() : nullptr, dt_of(q),
                        cur_stream());
    launched("attn_recompute_fwd");
  }
  return {out, lse};
}

// {dq, dk, dv}, contiguous; dv_out: where dv goes instead, with strides
std::vector<at::Tensor> attn_recompute_bwd(
    at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor out, at::Tensor lse,
    at::Tensor dout, c10::optional<at::Tensor> q_lens,
    c10::optional<at::Tensor> kv_lens, double scale, bool causal,
    c10::optional<at::Tensor> dv_out = c10::nullopt) {
  TORCH_CHECK(q.is_cuda(), "q must be on GPU");
  c10::DeviceGuard guard(q.device());
  AttnShape n = attn_check(q, k, v, q_lens, kv_lens, scale);
  long g = n.hk ? n.h / n.hk : 1;
  for (const at::Tensor* t : {&out, &dout})
    TORCH_CHECK(t->device() == q.device() &&
                    t->scalar_type() == q.scalar_type() &&
                    t->sizes() == q.sizes(),
                "out and its gradient must be like q");
  TORCH_CHECK(out.is_contiguous() &&
                  (dout.numel() == 0 || (dout.stride(3) == 1 && rows8(dout))),
              "out must be contiguous, its gradient have aligned rows");
  TORCH_CHECK(lse.device() == q.device() &&
                  lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
                  lse.numel() == n.b * n.hk * n.sq * g,
              "lse must be the forward's");
  auto dq = at::empty({n.b, n.sq, n.h, n.hd}, q.options());
  auto dk = at::empty({n.b, n.sk, n.hk, n.hd}, q.options());
  at::Tensor dv = dv_out.has_value() ? *dv_out : at::empty_like(dk);
  TORCH_CHECK(dv.device() == q.device() &&
                  dv.scalar_type() == q.scalar_type() &&
                  dv.sizes() == dk.sizes() &&
                  (dv.numel() == 0 || (dv.stride(3) == 1 && rows8(dv))),
              "dv_out must be like v, with aligned rows");
  bool lens = q_lens.has_value() || kv_lens.has_value();
  long need = pdta_attn_recompute_ws(n.b, n.sq, n.sk, n.hk, g, n.hd, causal,
                                     lens, 1);
  at::Tensor ws;
  if (need) ws = at::empty({need}, lse.options());
  long st[15];
  attn_strides(q, st);
  attn_strides(k, st + 3);
  attn_strides(v, st + 6);
  attn_strides(dout, st + 9);
  attn_strides(dv, st + 12);
  if (dq.numel() || dk.numel()) {
    pdta_attn_recompute(q.data_ptr(), k.data_ptr(), v.data_ptr(),
                        dout.data_ptr(), st, out.data_ptr(),
                        lse.data_ptr<float>(), dq.data_ptr(), dk.data_ptr(),
                        dv.data_ptr(), len_ptr(q_lens), len_ptr(kv_lens),
                        lens_wide(q_lens, kv_lens), n.b, n.sq, n.sk, n.hk, g,
                        n.hd, (float)scale, causal, 1,
                        need ? ws.data_ptr<float>() : nullptr, dt_of(q),
                        cur_stream());
    launched("attn_recompute_bwd");
  }
  return {dq, dk, dv};
}

// ---- autograd -----------------------------------------------------------
// The GPU path's autograd nodes are C++: the engine's device thread then runs
// backward without taking the GIL. 4 x 65 tokens of 3 heads, forward and
// backward: 92 us with Python nodes, 68 with these; now 64, 18 of it kernels.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

c10::optional<at::Tensor> maybe(const at::Tensor& t) {
  return t.defined() ? c10::optional<at::Tensor>(t) : c10::nullopt;
}
at::Tensor plain(const c10::optional<at::Tensor>& t) {
  return t.has_value() ? *t : at::Tensor();
}
void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what,
              ": a gradient of the gradient is not supported");
}

// A leaf keeps one node that gathers its gradient, with the stream that was
// current when the node was made, for as long as any graph holds it. If that
// is the default stream and a backward pass is captured on another, autograd
// makes the default stream wait for the capture, which ends the process. A
// forward that would lead there is refused.
void capture_check(const std::vector<at::Tensor>& leaves) {
  if (!at::GradMode::is_enabled()) return;
  hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(cur_stream(), &st) != hipSuccess ||
      st == hipStreamCaptureStatusNone)
    return;
  for (const at::Tensor& t : leaves) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
    auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) continue;
    auto s = node->stream();
    TORCH_CHECK(!s.has_value() || s->id() != 0,
                "captured with a gradient: another graph of the same leaf, "
                "made on the default stream, is alive; delete it first");
  }
}

// t itself if 16-byte accesses can walk its rows
at::Tensor walkable(const at::Tensor& t) {
  return t.dim() == 4 && t.stride(3) == 1 && rows8(t) ? t : t.contiguous();
}

struct AttentionRecompute
    : public torch::autograd::Function<AttentionRecompute> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q0,
                            const at::Tensor& k0, const at::Tensor& v0,
                            const c10::optional<at::Tensor>& q_lens,
                            const c10::optional<at::Tensor>& kv_lens,
                            double scale, bool causal) {
    at::Tensor q = walkable(q0), k = walkable(k0), v = walkable(v0);
    auto r = attn_recompute_fwd(q, k, v, q_lens, kv_lens, scale, causal,
                                true);
    ctx->save_for_backward(
        {q, k, v, r[0], r[1], plain(q_lens), plain(kv_lens)});
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["causal"] = causal;
    return r[0];
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("attention_recompute");
    auto s = ctx->get_saved_variables();
    auto r = attn_recompute_bwd(s[0], s[1], s[2], s[3], s[4], walkable(g[0]),
                                maybe(s[5]), maybe(s[6]),
                                ctx->saved_data["scale"].toDouble(),
                                ctx->saved_data["causal"].toBool());
    return {r[0], r[1], r[2], at::Tensor(), at::Tensor(), at::Tensor(),
            at::Tensor()};
  }
};

at::Tensor attention_recompute(at::Tensor q, at::Tensor k, at::Tensor v,
                               c10::optional<at::Tensor> q_lens,
                               c10::optional<at::Tensor> kv_lens,
                               double scale, bool causal) {
  c10::OptionalDeviceGuard guard(at::device_of(q));
  capture_check({q, k, v});
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return AttentionRecompute::apply(q, k, v, q_lens, kv_lens, scale, causal);
  return attn_recompute_fwd(walkable(q), walkable(k), walkable(v), q_lens,
                            kv_lens, scale, causal, false)[0];
}

at::Tensor inner1(const at::Tensor& t) {
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

struct QKNormRope : public torch::autograd::Function<QKNormRope> {
  using Opt = c10::optional<at::Tensor>;
  static variable_list forward(AutogradContext* ctx, const at::Tensor& q0,
                               const at::Tensor& k0, const Opt& wq,
                               const Opt& wk, const Opt& cos, const Opt& sin,
                               const Opt& pos, double eps,
                               bool interleaved) {
    at::Tensor q = inner1(q0), k = inner1(k0);
    auto r = qk_norm_rope(q, k, wq, wk, cos, sin, pos, eps, interleaved,
                          c10::nullopt, c10::nullopt);
    ctx->save_for_backward(
        {q, k, plain(wq), plain(wk), plain(cos), plain(sin), plain(pos)});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once("qk_norm_rope");
    auto s = ctx->get_saved_variables();
    for (int i = 0; i < 2; ++i)
      if (!g[i].defined()) g[i] = at::zeros_like(s[i]);
    auto r = qk_norm_rope(s[0], s[1], maybe(s[2]), maybe(s[3]), maybe(s[4]),
                          maybe(s[5]), maybe(s[6]),
                          ctx->saved_data["eps"].toDouble(),
                          ctx->saved_data["interleaved"].toBool(),
                          inner1(g[0]), inner1(g[1]));
    r.resize(9);
    return r;
  }
};

std::vector<at::Tensor> qk_norm_rope_grad(
    at::Tensor q, at::Tensor k, c10::optional<at::Tensor> wq,
    c10::optional<at::Tensor> wk, c10::optional<at::Tensor> cos,
    c10::optional<at::Tensor> sin, c10::optional<at::Tensor> pos, double eps,
    bool interleaved) {
  c10::OptionalDeviceGuard guard(at::device_of(q));
  capture_check({q, k, plain(wq), plain(wk)});
  bool w = wq.has_value() && wk.has_value() &&
           (wq->requires_grad() || wk->requires_grad());
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || w))
    return QKNormRope::apply(q, k, wq, wk, cos, sin, pos, eps, interleaved);
  return qk_norm_rope(inner1(q), inner1(k), wq, wk, cos, sin, pos, eps,
                      interleaved, c10::nullopt, c10::nullopt);
}

}  // namespace

void bind_transformer(pybind11::module_& m) {
  m.def("adamw_step", &adamw_step, py::arg("p"), py::arg("g"), py::arg("m"),
        py::arg("v"), py::arg("step"), py::arg("lr"), py::arg("lr_dev"),
        py::arg("beta1"), py::arg("beta2"), py::arg("eps"),
        py::arg("weight_decay"), py::arg("decay"), py::arg("grad_scale"),
        py::arg("m_scale"), py::arg("v_scale"), py::arg("seed"));
  m.def("qk_norm_rope", &qk_norm_rope, py::arg("q"), py::arg("k"),
        py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"),
        py::arg("sin"), py::arg("positions"), py::arg("eps"),
        py::arg("interleaved"), py::arg("dq") = py::none(),
        py::arg("dk") = py::none(), py::arg("outs") = Outs());
  m.def("attn_recompute_fwd", &attn_recompute_fwd, py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("q_lens"), py::arg("kv_lens"),
        py::arg("scale"), py::arg("causal"), py::arg("want_lse"));
  m.def("attn_recompute_bwd", &attn_recompute_bwd, py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("out"), py::arg("lse"),
        py::arg("dout"), py::arg("q_lens"), py::arg("kv_lens"),
        py::arg("scale"), py::arg("causal"),
        py::arg("dv_out") = py::none());
  m.def("capture_check", &capture_check);
  // differentiable forms
  m.def("attention_recompute", &attention_recompute, py::arg("q"),
        py::arg("k"), py::arg("v"), py::arg("q_lens"), py::arg("kv_lens"),
        py::arg("scale"), py::arg("causal"),
        py::call_guard<py::gil_scoped_release>());
  m.def("qk_norm_rope_grad", &qk_norm_rope_grad, py::arg("q"), py::arg("k"),
        py::arg("q_weight"), py::arg("k_weight"), py::arg("cos"),
        py::arg("sin"), py::arg("positions"), py::arg("eps"),
        py::arg("interleaved"), py::call_guard<py::gil_scoped_release>());
}

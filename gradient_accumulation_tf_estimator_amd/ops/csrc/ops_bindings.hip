// PyTorch bindings of the norm, clipping and relative-attention kernels: checks
// of shapes, types and alignment, allocation of outputs, launches on the
// current stream of the operands' device.

#include <algorithm>
#include <cstdint>
#include <vector>

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/extension.h>

#include "ga_ops.h"

namespace {

typedef c10::optional<at::Tensor> MaybeTensor;

int type_of(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return GA_FP32;
    case at::kBFloat16: return GA_BF16;
    case at::kHalf: return GA_FP16;
    default: TORCH_CHECK(false, name, " must be fp32, bf16 or fp16, got ", t.scalar_type());
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

hipStream_t stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

void check_launch(hipError_t e, const char* what) {
  TORCH_CHECK(e == hipSuccess, what, " launch failed: ", hipGetErrorString(e));
}

// ---------------- root-mean-square norm ----------------

const int kMaxNormWidth = 8192;

// rows [R, H] with neighbouring columns and any row stride; whether 16-byte
// accesses may be used
bool check_rows(const at::Tensor& t, const char* name, const at::Tensor& like) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the GPU that holds x");
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have x's dtype");
  TORCH_CHECK(t.dim() == 2 && t.size(0) == like.size(0) && t.size(1) == like.size(1),
              name, " must be [rows, hidden] like x");
  TORCH_CHECK(t.numel() == 0 || t.size(1) == 1 || t.stride(1) == 1, name, "'s columns must be contiguous");
  return aligned16(t.data_ptr()) && (t.size(0) <= 1 || t.stride(0) % 8 == 0);
}

RmsArgs norm_args(const at::Tensor& x, const at::Tensor& w, double eps, bool& vec) {
  TORCH_CHECK(x.dim() == 2, "x must be [rows, hidden]");
  type_of(x, "x");
  const int64_t H = x.size(1);
  TORCH_CHECK(H >= 1 && H <= kMaxNormWidth, "RMS norm width must be 1..", kMaxNormWidth, ", got ", H);
  vec = check_rows(x, "x", x) && H % 8 == 0;
  TORCH_CHECK(w.is_cuda() && w.device() == x.device() && w.scalar_type() == x.scalar_type() &&
              w.dim() == 1 && w.numel() == H && w.is_contiguous(),
              "weight must be a contiguous [hidden] tensor of x's dtype and device");
  vec = vec && aligned16(w.data_ptr());
  TORCH_CHECK(eps >= 0, "eps must not be negative");
  RmsArgs a = {};
  a.x = x.data_ptr();
  a.x_stride = x.stride(0);
  a.w = w.data_ptr();
  a.R = x.size(0);
  a.H = (int)H;
  a.eps = (float)eps;
  return a;
}

// x, res: rows; the outputs have the caller's shape, so that none is a view
std::vector<at::Tensor> rms_norm_fwd(at::Tensor x, MaybeTensor res, at::Tensor w, double eps, at::IntArrayRef shape) {
  bool vec;
  RmsArgs a = norm_args(x, w, eps, vec);
  const c10::OptionalDeviceGuard guard(x.device());
  auto y = at::empty(shape, x.options());
  auto h = res ? at::empty(shape, x.options()) : x;
  auto rstd = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  if (res) {
    vec = check_rows(*res, "residual", x) && vec;
    a.res = res->data_ptr();
    a.res_stride = res->stride(0);
    a.h = h.data_ptr();
  }
  if (a.R == 0) return {y, h, rstd};
  a.y = y.data_ptr();
  a.rstd = rstd.data_ptr<float>();
  check_launch(rms_forward(type_of(x, "x"), vec, a, stream_of(x)), "rms_norm_fwd");
  return {y, h, rstd};
}

// dw_acc: an fp32 slice that dw is added to; the second result is then empty
std::vector<at::Tensor> rms_norm_bwd(at::Tensor dy, MaybeTensor dh, at::Tensor h, at::Tensor w,
                                     at::Tensor rstd, MaybeTensor dw_acc, at::IntArrayRef shape) {
  bool vec;
  RmsArgs a = norm_args(h, w, 0.0, vec);
  const c10::OptionalDeviceGuard guard(h.device());
  vec = check_rows(dy, "dy", h) && vec;
  TORCH_CHECK(rstd.device() == h.device() && rstd.scalar_type() == at::kFloat && rstd.is_contiguous() &&
              rstd.numel() == h.size(0), "rstd must be the forward's");
  if (dh) {
    vec = check_rows(*dh, "dh", h) && vec;
    a.dh = dh->data_ptr();
    a.dh_stride = dh->stride(0);
  }
  if (dw_acc)
    TORCH_CHECK(dw_acc->device() == h.device() && dw_acc->scalar_type() == at::kFloat &&
                dw_acc->is_contiguous() && dw_acc->numel() == a.H, "dw_acc must be an fp32 [hidden] slice");
  auto dx = at::empty(shape, h.options());
  auto dw = dw_acc ? at::Tensor() : at::empty({a.H}, w.options());
  if (a.R == 0) {
    if (dw.defined()) dw.zero_();
    return {dx, dw};
  }
  auto slabs = at::empty({rms_slabs(a.R, a.H), a.H}, h.options().dtype(at::kFloat));
  a.dy = dy.data_ptr();
  a.dy_stride = dy.stride(0);
  a.rstd = rstd.data_ptr<float>();
  a.y = dx.data_ptr();
  a.slabs = slabs.data_ptr<float>();
  check_launch(rms_backward(type_of(h, "h"), vec, a, dw.defined() ? dw.data_ptr() : nullptr,
                            dw_acc ? dw_acc->data_ptr<float>() : nullptr, stream_of(h)), "rms_norm_bwd");
  return {dx, dw};
}

// [rows, hidden] with neighbouring columns; a copy only where needed
at::Tensor as_rows(const at::Tensor& t) {
  auto r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}
MaybeTensor as_rows(const MaybeTensor& t) { return t ? MaybeTensor(as_rows(*t)) : t; }
MaybeTensor maybe(const at::Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

// gradients of gradients would be lost without a word
void once() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "this operator has no second derivative: call it without create_graph");
}

// whether a forward-mode derivative comes with the tensor (there is one level)
bool has_tangent(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }

// The autograd node lives here: in Python its forward and backward cost more
// than the kernels on a small batch. `dw_acc`: an fp32 slice that the weight's
// gradient is added to instead of being returned.
struct AddRmsNorm : public torch::autograd::Function<AddRmsNorm> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, at::Tensor x, MaybeTensor res,
                                                at::Tensor w, double eps, MaybeTensor dw_acc) {
    w = w.contiguous();
    auto r = rms_norm_fwd(as_rows(x), as_rows(res), w, eps, x.sizes());
    ctx->save_for_backward({r[1], w, r[2]});
    ctx->set_materialize_grads(false);
    ctx->saved_data["res"] = res.has_value();
    if (dw_acc) ctx->saved_data["acc"] = *dw_acc;
    return {r[0], res ? r[1] : x};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    once();
    const auto saved = ctx->get_saved_variables();
    const auto dy = grads[0], dh = grads[1];
    at::Tensor dx = dh, dw;
    if (dy.defined()) {  // y was used
      const auto acc = ctx->saved_data.find("acc");
      auto r = rms_norm_bwd(as_rows(dy), as_rows(maybe(dh)), as_rows(saved[0]), saved[1], saved[2],
                            acc == ctx->saved_data.end() ? MaybeTensor() : MaybeTensor(acc->second.toTensor()), dy.sizes());
      dx = r[0];
      dw = r[1];
    }
    return {dx, ctx->saved_data["res"].toBool() ? dx : at::Tensor(), dw, at::Tensor(), at::Tensor()};
  }
};

std::vector<at::Tensor> add_rms_norm(at::Tensor x, MaybeTensor res, at::Tensor w, double eps, MaybeTensor dw_acc) {
  return AddRmsNorm::apply(x, res, w, eps, dw_acc);
}

std::vector<at::Tensor> rms_norm_fp8(at::Tensor x, MaybeTensor res, at::Tensor w, double eps, int64_t group) {
  bool vec;
  TORCH_CHECK(!has_tangent(x) && !(res && has_tangent(*res)) && !has_tangent(w),
              "rms_norm_fp8 has no gradient, forward-mode ones included");
  auto shape = x.sizes().vec();  // the outputs have the caller's shape
  const auto given = x;
  x = as_rows(x);
  res = as_rows(res);
  w = w.contiguous();
  RmsArgs a = norm_args(x, w, eps, vec);
  const c10::OptionalDeviceGuard guard(x.device());
  TORCH_CHECK(group == 0 || group == 32 || group == 64 || group == 128, "group must be 0 (a row), 32, 64 or 128");
  TORCH_CHECK(group == 0 || a.H % group == 0, "hidden must be a multiple of the group");
  const int64_t groups = group ? a.H / group : 1;
  auto q = at::empty(shape, x.options().dtype(at::kFloat8_e4m3fn));
  auto h = res ? at::empty(shape, x.options()) : given;
  shape.back() = groups;
  auto scales = at::empty(shape, x.options().dtype(at::kFloat));
  if (res) {
    vec = check_rows(*res, "residual", x) && vec;
    a.res = res->data_ptr();
    a.res_stride = res->stride(0);
    a.h = h.data_ptr();
  }
  if (a.R == 0) return {q, scales, h};
  a.q = (unsigned char*)q.data_ptr();
  a.scales = scales.data_ptr<float>();
  a.group = (int)group;
  check_launch(rms_fp8(type_of(x, "x"), vec, a, stream_of(x)), "rms_norm_fp8");
  return {q, scales, h};
}

// ---------------- global norm and clipping ----------------

// No output may lie over another output or over another tensor's input: the
// blocks that read and write them run in no order. out[i] == in[i] is in place.
void check_apart(const std::vector<at::Tensor>& ins, const std::vector<at::Tensor>& outs) {
  struct Span { uintptr_t lo, hi; bool out; };
  std::vector<Span> spans;
  for (size_t i = 0; i < ins.size(); ++i) {
    if (ins[i].numel() == 0) continue;
    const uintptr_t a = (uintptr_t)ins[i].data_ptr(), b = (uintptr_t)outs[i].data_ptr();
    spans.push_back({b, b + outs[i].nbytes(), true});
    if (a != b) spans.push_back({a, a + ins[i].nbytes(), false});
  }
  std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.lo < y.lo; });
  uintptr_t out_end = 0, any_end = 0;
  for (const Span& s : spans) {
    TORCH_CHECK(s.lo >= (s.out ? any_end : out_end),
                "an output shares memory with another tensor of the list (is one listed twice?)");
    any_end = std::max(any_end, s.hi);
    if (s.out) out_end = std::max(out_end, s.hi);
  }
}

// -> norm of all tensors, and with `write` outs[i] = ins[i] * min(1, clip / norm)
// (new tensors where outs is empty). Tensors are taken as their memory,
// whatever the order of their dimensions; an output has to have its input's
// strides.
std::tuple<at::Tensor, std::vector<at::Tensor>> global_norm(std::vector<at::Tensor> ins, std::vector<at::Tensor> outs,
                                                            bool write, double clip) {
  TORCH_CHECK_VALUE(!ins.empty(), "global_norm needs at least one tensor");
  TORCH_CHECK_VALUE(!write || clip > 0, "clip_norm must be positive");
  const auto dev = ins[0].device();
  TORCH_CHECK_VALUE(ins[0].is_cuda(), "tensors must be on a GPU");
  const c10::OptionalDeviceGuard guard(dev);
  long long total = 0;
  for (size_t i = 0; i < ins.size(); ++i) {
    TORCH_CHECK_VALUE(ins[i].device() == dev, "tensors must be on one device");
    const auto t = ins[i].scalar_type();
    TORCH_CHECK_VALUE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "tensors must be fp32, bf16 or fp16, got ", t);
    TORCH_CHECK(ins[i].is_non_overlapping_and_dense(), "tensor ", i,
                " has gaps or overlaps in memory: pass a contiguous copy");
    total += ins[i].numel();
  }
  if (write && outs.empty()) {
    for (const auto& t : ins) outs.push_back(at::empty_like(t));
  } else if (write) {
    TORCH_CHECK_VALUE(outs.size() == ins.size(), "one output for each tensor");
    for (size_t i = 0; i < ins.size(); ++i)
      TORCH_CHECK(outs[i].device() == dev && outs[i].scalar_type() == ins[i].scalar_type() &&
                  outs[i].sizes() == ins[i].sizes() && outs[i].strides() == ins[i].strides(),
                  "output ", i, " must have its tensor's device, dtype, shape and strides");
    check_apart(ins, outs);
    for (auto& t : outs)
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // written behind autograd's back
  }
  // about 4096 blocks for large sets, at least 8192 elements a block
  long long chunk = (total / 4096 + 2047) / 2048 * 2048;
  if (chunk < 8192) chunk = 8192;
  TORCH_CHECK(chunk <= (1ll << 30), "too many elements");
  std::vector<ClipArgs> launches;
  long long blocks = 0;
  for (size_t i = 0; i < ins.size(); ++i) {
    const long long n = ins[i].numel();
    if (n == 0) continue;
    if (launches.empty() || launches.back().count == GA_CLIP_TENSORS) {
      launches.emplace_back();
      launches.back().count = 0;
      launches.back().first[0] = 0;
      launches.back().chunk = (int)chunk;
    }
    ClipArgs& a = launches.back();
    const int t = a.count++;
    a.in[t] = ins[i].data_ptr();
    a.out[t] = write ? outs[i].data_ptr() : nullptr;
    a.n[t] = n;
    a.type[t] = (unsigned char)type_of(ins[i], "tensor");
    a.vec[t] = aligned16(a.in[t]) && aligned16(a.out[t]);
    a.first[t + 1] = a.first[t] + (int)((n + chunk - 1) / chunk);
    blocks += (n + chunk - 1) / chunk;
  }
  auto sums = at::empty({blocks}, ins[0].options().dtype(at::kDouble));
  auto result = at::empty({2}, ins[0].options().dtype(at::kFloat));  // norm, factor
  hipStream_t s = stream_of(ins[0]);
  long long at_block = 0;
  for (const auto& a : launches) {
    check_launch(clip_sums(a, sums.data_ptr<double>() + at_block, s), "global_norm");
    at_block += a.first[a.count];
  }
  float* r = result.data_ptr<float>();
  check_launch(clip_finish(blocks ? sums.data_ptr<double>() : nullptr, (int)blocks, clip, r, write ? r + 1 : nullptr, s),
               "global_norm");
  if (write)
    for (size_t i = launches.size(); i-- > 0;) check_launch(clip_scale(launches[i], r + 1, s), "clip_by_global_norm");
  return {result.select(0, 0), outs};
}

// ---------------- attention with a relative position bias ----------------

void check_bias(const at::Tensor& table, const at::Tensor& map, const at::Tensor& like, int64_t NH) {
  TORCH_CHECK(table.device() == like.device() && table.scalar_type() == at::kBFloat16 && table.is_contiguous() &&
              table.dim() == 2 && table.size(1) == NH, "the bias table must be a contiguous bf16 [buckets, heads] tensor");
  TORCH_CHECK(table.size(0) >= 1 && table.size(0) <= GA_REL_MAX_BUCKETS, "buckets must be 1..", GA_REL_MAX_BUCKETS);
  TORCH_CHECK(map.device() == like.device() && map.scalar_type() == at::kInt && map.is_contiguous() && map.dim() == 1 &&
              map.numel() % 2 == 1 && map.numel() >= 3 && map.numel() <= 2 * GA_REL_MAX_DISTANCE + 1,
              "the bucket map must be an int32 [2 * max_distance + 1] tensor, max_distance 1..", GA_REL_MAX_DISTANCE);
}

void check_heads(int64_t NH, int64_t NKV, int64_t D) {
  TORCH_CHECK(D == 64 || D == 128, "head size must be 64 or 128, got ", D);
  TORCH_CHECK(NH >= 1 && NKV >= 1 && NH % NKV == 0, "query heads must be a multiple of key/value heads");
}

// The kernels hold scale and bias / scale in 32 bits; table values are below
// 2^29, and beyond these bounds one of the two would be zero or infinite.
void check_scale(double scale) {
  TORCH_CHECK_VALUE(scale >= 0x1p-96 && scale <= 0x1p96, "scale must be within 2^-96 .. 2^96 on a GPU, got ", scale);
}

RelArgs rel_args(const at::Tensor& qkv, int64_t NH, int64_t NKV, const at::Tensor& table, const at::Tensor& map,
                 const MaybeTensor& mask, bool causal, double scale) {
  TORCH_CHECK(qkv.is_cuda() && qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 3 && qkv.is_contiguous() &&
              aligned16(qkv.data_ptr()), "qkv must be a contiguous, 16-byte aligned bf16 [B, S, (NH + 2 NKV) D] GPU tensor");
  TORCH_CHECK(NH >= 1 && NKV >= 1 && qkv.size(2) % (NH + 2 * NKV) == 0, "qkv's last dimension must be (NH + 2 NKV) * D");
  const int64_t B = qkv.size(0), S = qkv.size(1), D = qkv.size(2) / (NH + 2 * NKV);
  check_heads(NH, NKV, D);
  check_bias(table, map, qkv, NH);
  check_scale(scale);
  // a launch has fewer than 2^32 threads, 512 for each 128 rows of a head; a chunk of 64 rows is addressed by 32 bits from its start
  TORCH_CHECK(qkv.size(2) <= (1 << 23), "too many heads");
  TORCH_CHECK(S < (1ll << 24) && B * NH * (S / 128 + 1) < (1ll << 22), "too many rows");
  if (mask)
    TORCH_CHECK(mask->device() == qkv.device() && mask->scalar_type() == at::kByte && mask->is_contiguous() &&
                mask->dim() == 2 && mask->size(0) == B && mask->size(1) == S, "mask must be a contiguous u8 [B, S] tensor");
  RelArgs a = {};
  a.qkv = (const __bf16*)qkv.data_ptr();
  a.width = (int)qkv.size(2);
  a.table = (const __bf16*)table.data_ptr();
  a.map = map.data_ptr<int>();
  a.mask = mask ? mask->data_ptr<unsigned char>() : nullptr;
  a.B = (int)B;
  a.S = (int)S;
  a.NH = (int)NH;
  a.NKV = (int)NKV;
  a.D = (int)D;
  a.buckets = (int)table.size(0);
  a.far = (int)(map.numel() / 2);
  a.causal = causal;
  a.scale = (float)scale;
  return a;
}

// -> out [B, S, NH * D], lse [2, B, NH, S] (empty unless wanted)
std::vector<at::Tensor> rel_attn_fwd(at::Tensor qkv, int64_t NH, int64_t NKV, at::Tensor table, at::Tensor map,
                                     MaybeTensor mask, bool causal, double scale, bool want_lse) {
  RelArgs a = rel_args(qkv, NH, NKV, table, map, mask, causal, scale);
  const c10::OptionalDeviceGuard guard(qkv.device());
  auto out = at::empty({a.B, a.S, NH * a.D}, qkv.options());
  auto lse = want_lse ? at::empty({2, a.B, NH, a.S}, qkv.options().dtype(at::kFloat)) : at::Tensor();
  if (out.numel() == 0) return {out, lse};
  a.out = (__bf16*)out.data_ptr();
  a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
  a.spans = rel_spans(a.B, a.S, a.NH);
  at::Tensor split;
  if (a.spans > 1) {
    split = at::empty({(int64_t)a.spans * a.B * NH * a.S * (a.D + 2)}, qkv.options().dtype(at::kFloat));
    a.split = split.data_ptr<float>();
  }
  check_launch(rel_forward(a, stream_of(qkv)), "rel_attn_fwd");
  return {out, lse};
}

// -> dqkv like qkv, dtable like table
std::vector<at::Tensor> rel_attn_bwd(at::Tensor dout, at::Tensor qkv, at::Tensor out, at::Tensor lse, int64_t NH,
                                     int64_t NKV, at::Tensor table, at::Tensor map, MaybeTensor mask, bool causal,
                                     double scale) {
  RelArgs a = rel_args(qkv, NH, NKV, table, map, mask, causal, scale);
  const c10::OptionalDeviceGuard guard(qkv.device());
  for (const auto& t : {dout, out})
    TORCH_CHECK(t.device() == qkv.device() && t.scalar_type() == at::kBFloat16 && t.is_contiguous() &&
                t.numel() == (int64_t)a.B * a.S * NH * a.D && aligned16(t.data_ptr()),
                "dout and out must be contiguous, 16-byte aligned bf16 [B, S, NH * D] tensors");
  TORCH_CHECK(lse.device() == qkv.device() && lse.scalar_type() == at::kFloat && lse.is_contiguous() &&
              lse.numel() == 2 * (int64_t)a.B * NH * a.S, "lse must be the forward's");
  auto dqkv = at::empty_like(qkv);
  auto dtable = at::empty_like(table);
  if (dqkv.numel() == 0) {
    dtable.zero_();
    return {dqkv, dtable};
  }
  auto dsum = at::empty({a.B, NH, a.S}, lse.options());
  a.q_spans = rel_spans(a.B, a.S, a.NH);
  auto doff = at::empty({(int64_t)a.B * NH * rel_doff_rows(a.S, a.q_spans), 2 * a.far + 1}, lse.options());
  at::Tensor dq;
  if (a.q_spans > 1) {
    dq = at::empty({(int64_t)a.q_spans * a.B * NH * a.S * (a.D + 4)}, lse.options());
    a.dq = dq.data_ptr<float>();
  }
  rel_parts(a.B, a.S, a.NH, a.NKV, a.D, &a.parts, &a.spans);
  at::Tensor dkv;
  if (a.parts > 1) {
    dkv = at::empty({(int64_t)a.parts * a.B * NKV * a.S, 2 * a.D}, lse.options());
    a.dkv = dkv.data_ptr<float>();
  }
  a.out = (__bf16*)out.data_ptr();
  a.lse = lse.data_ptr<float>();
  a.dout = (const __bf16*)dout.data_ptr();
  a.dsum = dsum.data_ptr<float>();
  a.doff = doff.data_ptr<float>();
  a.dtable = (__bf16*)dtable.data_ptr();
  a.dqkv = (__bf16*)dqkv.data_ptr();
  check_launch(rel_backward(a, stream_of(qkv)), "rel_attn_bwd");
  return {dqkv, dtable};
}

at::Tensor aligned(const at::Tensor& t) {
  const auto c = t.contiguous();
  return aligned16(c.data_ptr()) ? c : c.clone();
}

struct RelAttention : public torch::autograd::Function<RelAttention> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, at::Tensor qkv, at::Tensor table, at::Tensor map,
                            MaybeTensor mask, int64_t NH, int64_t NKV, bool causal, double scale) {
    qkv = aligned(qkv);
    table = table.contiguous();
    auto r = rel_attn_fwd(qkv, NH, NKV, table, map, mask, causal, scale, true);
    ctx->save_for_backward({qkv, table, map, mask ? *mask : at::Tensor(), r[0], r[1]});
    ctx->saved_data["NH"] = NH;
    ctx->saved_data["NKV"] = NKV;
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    once();
    const auto s = ctx->get_saved_variables();
    auto r = rel_attn_bwd(aligned(grads[0]), s[0], s[4], s[5], ctx->saved_data["NH"].toInt(), ctx->saved_data["NKV"].toInt(),
                          s[1], s[2], maybe(s[3]), ctx->saved_data["causal"].toBool(), ctx->saved_data["scale"].toDouble());
    at::Tensor none;
    return {r[0], r[1], none, none, none, none, none, none};
  }
};

// with gradients recorded, the forward keeps what the backward needs
at::Tensor rel_attention(at::Tensor qkv, at::Tensor table, at::Tensor map, MaybeTensor mask, int64_t NH, int64_t NKV,
                         bool causal, double scale) {
  TORCH_CHECK(!has_tangent(qkv) && !has_tangent(table), "relative attention has no forward-mode derivative on a GPU");
  if (at::GradMode::is_enabled() && (qkv.requires_grad() || table.requires_grad()))
    return RelAttention::apply(qkv, table, map, mask, NH, NKV, causal, scale);
  return rel_attn_fwd(aligned(qkv), NH, NKV, table.contiguous(), map, mask, causal, scale, false)[0];
}

// q [B, Sq, NH, D], caches [B, S, NKV, D] of any strides with contiguous, 16-byte aligned rows
at::Tensor rel_attn_token(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor table, at::Tensor map,
                          at::Tensor lengths, double scale) {
  for (const auto& t : {q, k, v, table})
    TORCH_CHECK(!has_tangent(t), "relative_attention_decode has no gradient, forward-mode ones included");
  TORCH_CHECK(q.is_cuda() && q.dim() == 4 && k.dim() == 4 && v.dim() == 4, "q, k and v must be 4-dimensional GPU tensors");
  const int64_t B = q.size(0), Sq = q.size(1), NH = q.size(2), D = q.size(3), S = k.size(1), NKV = k.size(2);
  check_heads(NH, NKV, D);
  TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == B && k.size(3) == D, "caches must be [B, S, NKV, D] with q's B and D");
  for (const auto& t : {q, k, v}) {
    TORCH_CHECK(t.device() == q.device() && t.scalar_type() == at::kBFloat16, "q, k and v must be bf16 on one GPU");
    TORCH_CHECK(t.numel() == 0 || (t.stride(3) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
                t.stride(2) % 8 == 0 && aligned16(t.data_ptr())),
                "q, k and v need contiguous heads that start on 16 bytes");
  }
  check_bias(table, map, q, NH);
  TORCH_CHECK(lengths.device() == q.device() && lengths.scalar_type() == at::kInt && lengths.is_contiguous() &&
              lengths.dim() == 1 && lengths.numel() == B, "lengths must be an int32 [B] tensor on the same GPU");
  check_scale(scale);
  TORCH_CHECK(NH / NKV <= 32, "at most 32 query heads a key/value head");
  // fewer than 2^32 threads here too
  TORCH_CHECK(S < (1ll << 31) - 64 && B * NH * Sq < (1ll << 22), "too many rows");
  const c10::OptionalDeviceGuard guard(q.device());
  auto out = at::empty({B, Sq, NH, D}, q.options());
  if (out.numel() == 0) return out;
  if (S == 0) return out.zero_();
  RelTokenArgs a = {};
  a.q = (const __bf16*)q.data_ptr();
  a.k = (const __bf16*)k.data_ptr();
  a.v = (const __bf16*)v.data_ptr();
  a.q_b = q.stride(0); a.q_s = q.stride(1); a.q_h = q.stride(2);
  a.k_b = k.stride(0); a.k_s = k.stride(1); a.k_h = k.stride(2);
  a.v_b = v.stride(0); a.v_s = v.stride(1); a.v_h = v.stride(2);
  a.table = (const __bf16*)table.data_ptr();
  a.map = map.data_ptr<int>();
  a.lengths = lengths.data_ptr<int>();
  a.out = (__bf16*)out.data_ptr();
  a.B = (int)B; a.Sq = (int)Sq; a.S = (int)S; a.NH = (int)NH; a.NKV = (int)NKV; a.D = (int)D;
  a.buckets = (int)table.size(0);
  a.far = (int)(map.numel() / 2);
  a.scale = (float)scale;
  a.splits = rel_token_splits(a.B, a.Sq, a.S, a.NH, a.NKV);
  at::Tensor parts;
  if (a.splits > 1) {
    const int64_t tiles = (NH / NKV * Sq + 31) / 32;
    parts = at::empty({B * NKV * tiles * a.splits, 32, D + 2}, q.options().dtype(at::kFloat));
    a.parts = parts.data_ptr<float>();
  }
  check_launch(rel_token(a, stream_of(q)), "rel_attn_token");
  return out;
}

}  // namespace

void register_ops(pybind11::module_& mod) {
  mod.def("add_rms_norm", &add_rms_norm, "x (+ residual) -> y, h, with gradients");
  mod.def("rms_norm_fp8", &rms_norm_fp8, "x (+ residual) -> e4m3 values, scales, h");
  mod.def("rel_attention", &rel_attention, "attention over packed qkv with a bucket bias, with gradients");
  mod.def("rel_attn_token", &rel_attn_token, "new tokens over a K/V cache with a bucket bias");
  mod.def("global_norm", &global_norm, "norm over many tensors; with outputs, clipped copies");
}

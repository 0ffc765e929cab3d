// Native host binding of the router's autograd Function (torch C++ extension `moe_mi355._moe_torch`).
//
// The router step is short on the GPU (C2: ~85 us of kernels for fwd + bwd), so its host work shows: the
// Python Function, eight output allocations through Python, the zeroed-workspace lookup and the ctypes
// conversion of ~25 arguments per call add up to more than the kernels on a slow host.  This file does the
// same work in C++: a torch::autograd::Function whose forward allocates the outputs with ATen, takes the
// current HIP stream from c10 and calls moe_router_fwd, and whose backward (run by the autograd engine
// without returning to Python) calls moe_router_bwd.  It calls the same C ABI entry points
// (include/moe_mi355.h) as the ctypes path and launches the same kernels; argument validation with the
// Python error types stays in moe_mi355/router.py.
//
// The operations that a layer's pass is made of (op_* below) are bound the same way: with few tokens their kernels are
// shorter than the Python that allocates their outputs and converts up to 38 ctypes arguments.  Host work of a pass,
// measured through Python and ctypes -> here: routing 16 bf16 tokens (H 4096, E 8) 24 -> 14 us, a small layer's inference
// 150 -> 122, norm + router with its backward 169 -> 64, dispatch and combine with their backward 169 -> 65, a small
// training step 420 -> 238.
#include <torch/extension.h>

// In torch's ROCm build GPU tensors carry the device type `cuda`; the HIP guard and stream types that accept
// it are the ones "masquerading as CUDA".
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <hip/hip_runtime_api.h>

#include <map>
#include <mutex>
#include <optional>
#include <string>
#include <tuple>
#include <utility>
#include <vector>

#include "../../include/moe_mi355.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

[[noreturn]] void raise_rc(int rc, const char* what) {
  char buf[512];
  buf[0] = 0;
  moe_last_error(buf, sizeof buf);
  if (rc < 0) throw pybind11::value_error(std::string(what) + ": " + buf + " (code " + std::to_string(rc) + ")");
  throw std::runtime_error(std::string(what) + ": " + buf + " (hip error " + std::to_string(rc) + ")");
}

int code_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? MOE_BF16 : MOE_F32; }

// The forward's workspace holds a ticket counter that must be zero when a launch starts and that the kernels
// leave at zero: one zero-initialised buffer per (device, stream), reused by every call on that stream.  A call
// may launch several kernels that hand data on through it (the packed gate, the per-block partials), so stream
// order keeps calls apart only if no other thread's launches come between one call's: FwdWorkspace holds the
// buffer's lock until the call's last launch is queued (no call of this file holds the GIL meanwhile, so a
// waiting thread stops no other).
// Under graph capture each capture takes a fresh slice of a per-device arena instead,
// zeroed and synchronised once outside any capture (on the first eager call): the kernels leave the counter at
// zero after every replay, so that slice serves every replay of its graph, and the graph holds no fill node.
// Captures past the arena's end fall back to a zeroed buffer made inside the capture (a captured fill kernel).
struct StreamBuffer {
  std::mutex mu;
  at::Tensor buf;
};
std::mutex g_ws_mu;  // the two maps and the arenas; never held while a StreamBuffer's lock is waited for
std::map<std::pair<int, hipStream_t>, StreamBuffer> g_ws;  // entries stay where they are (a map's nodes)
constexpr int64_t kArenaBytes = 32 << 20;
struct CaptureArena {
  at::Tensor buf;
  int64_t used = 0;
};
std::map<int, CaptureArena> g_arena;

class FwdWorkspace {
 public:
  FwdWorkspace(size_t nbytes, const at::Device& dev, hipStream_t s) {
    const int64_t n = std::max<int64_t>((int64_t)nbytes, 1);
    const auto opts = at::TensorOptions().dtype(at::kByte).device(dev);
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(s, &st) != hipSuccess) {
      (void)hipGetLastError();
      throw std::runtime_error("moe_router_fwd: hipStreamIsCapturing failed");
    }
    StreamBuffer* sb = nullptr;
    {
      std::lock_guard<std::mutex> lk(g_ws_mu);
      CaptureArena& ar = g_arena[(int)dev.index()];
      if (st != hipStreamCaptureStatusNone) {
        const int64_t n256 = (n + 255) / 256 * 256;
        if (ar.buf.defined() && ar.used + n256 <= kArenaBytes) {
          buf_ = ar.buf.narrow(0, ar.used, n);
          ar.used += n256;
        } else {
          buf_ = at::zeros({n}, opts);
        }
        return;
      }
      if (!ar.buf.defined()) {
        ar.buf = at::zeros({kArenaBytes}, opts);
        if (hipStreamSynchronize(s) != hipSuccess) {  // once: later captures may replay on any stream
          (void)hipGetLastError();
          throw std::runtime_error("moe_router_fwd: hipStreamSynchronize failed");
        }
      }
      sb = &g_ws[{(int)dev.index(), s}];
    }
    lock_ = std::unique_lock<std::mutex>(sb->mu);
    if (!sb->buf.defined() || sb->buf.numel() < n) sb->buf = at::zeros({n}, opts);
    buf_ = sb->buf;
  }
  void* data_ptr() const { return buf_.data_ptr(); }

 private:
  at::Tensor buf_;
  std::unique_lock<std::mutex> lock_;
};

struct RouterFn : public torch::autograd::Function<RouterFn> {
  // link_x: x is also returned, as an eighth output, for the layer's expert path to consume.  Its gradient
  // (the expert path's gradient of x) then arrives here as an upstream gradient and is added inside the dx
  // kernel, instead of autograd summing the two contributions to x's gradient in a separate addition.
  static variable_list forward(AutogradContext* ctx, const Variable& x_in, const Variable& gw_in, int64_t k,
                               double aux_coef, double z_coef, const std::optional<Variable>& bias_in, bool link_x,
                               bool diff_logits) {
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
    const at::Tensor x = x_in.contiguous();
    const at::Tensor gw = gw_in.contiguous();
    const int64_t N = x.size(0), H = x.size(1), E = gw.size(1);
    at::Tensor bias;
    if (bias_in.has_value() && bias_in->defined()) bias = bias_in->detach().to(at::kFloat).contiguous();
    const auto dev = x.device();
    const auto f32 = at::TensorOptions().dtype(at::kFloat).device(dev);
    const auto i64 = at::TensorOptions().dtype(at::kLong).device(dev);
    at::Tensor idx = at::empty({N, k}, i64);
    at::Tensor w = at::empty({N, k}, x.options());
    at::Tensor logits = at::empty({N, E}, f32);
    at::Tensor lse = at::empty({N}, f32);
    at::Tensor cnt = at::empty({E}, i64);
    at::Tensor stats = at::empty({MOE_STATS_HEAD + E}, f32);
    at::Tensor aux = at::empty({}, f32);
    at::Tensor z = at::empty({}, f32);
    if (N == 0) {
      cnt.zero_();
      stats.zero_();
      aux.zero_();
      z.zero_();
    } else {
      const hipStream_t s = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
      const int xdt = code_of(x), wdt = code_of(gw);
      const size_t nbytes = moe_router_fwd_workspace(N, H, E, k, xdt, wdt);
      const FwdWorkspace ws(nbytes, dev, s);
      const int rc = moe_router_fwd(x.data_ptr(), xdt, gw.data_ptr(), wdt,
                                    bias.defined() ? bias.data_ptr<float>() : nullptr, N, H, E, k,
                                    idx.data_ptr<int64_t>(), w.data_ptr(), xdt, logits.data_ptr<float>(),
                                    lse.data_ptr<float>(), cnt.data_ptr<int64_t>(), stats.data_ptr<float>(),
                                    (float)aux_coef, (float)z_coef, aux.data_ptr<float>(), z.data_ptr<float>(),
                                    ws.data_ptr(), nbytes, s);
      if (rc != 0) raise_rc(rc, "moe_router_fwd");
    }
    ctx->save_for_backward({x, gw, logits, idx, cnt});
    ctx->saved_data["aux_coef"] = aux_coef;
    ctx->saved_data["z_coef"] = z_coef;
    ctx->set_materialize_grads(false);
    // diff_logits: a loss of the caller's formed on the logits sends its gradient back through them
    if (diff_logits) ctx->mark_non_differentiable({idx, cnt, stats});
    else ctx->mark_non_differentiable({idx, logits, cnt, stats});
    if (link_x) return {idx, w, aux, z, logits, cnt, stats, x_in};
    return {idx, w, aux, z, logits, cnt, stats};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    variable_list out(8);
    if (!(need_x || need_w)) return out;
    const auto saved = ctx->get_saved_variables();
    const at::Tensor& x = saved[0];
    const at::Tensor& gw = saved[1];
    const at::Tensor& logits = saved[2];
    const at::Tensor& idx = saved[3];
    const at::Tensor& cnt = saved[4];
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    at::Tensor g_w = grads[1];
    at::Tensor g_aux = grads[2];
    at::Tensor g_z = grads[3];
    // the linked x output's gradient (the expert path's gradient of x), if any
    at::Tensor dx_add;
    if (need_x && grads.size() > 7 && grads[7].defined()) dx_add = grads[7].to(x.scalar_type()).contiguous();
    at::Tensor g_logits;  // undefined unless the forward left the logits differentiable
    if (grads[4].defined()) g_logits = grads[4].to(at::kFloat).contiguous();
    const float aux_coef = g_aux.defined() ? (float)ctx->saved_data["aux_coef"].toDouble() : 0.f;
    const float z_coef = g_z.defined() ? (float)ctx->saved_data["z_coef"].toDouble() : 0.f;
    int gdt = MOE_F32;
    if (g_w.defined()) {
      g_w = g_w.contiguous();
      if (g_w.scalar_type() != at::kFloat && g_w.scalar_type() != at::kBFloat16) g_w = g_w.to(at::kFloat);
      gdt = code_of(g_w);
    }
    if (g_aux.defined()) g_aux = g_aux.detach().to(at::kFloat).reshape({1}).contiguous();
    if (g_z.defined()) g_z = g_z.detach().to(at::kFloat).reshape({1}).contiguous();
    const int64_t N = x.size(0), H = x.size(1), E = gw.size(1), K = idx.size(1);
    at::Tensor dx = at::empty({N, H}, x.options());
    at::Tensor dw;
    if (N == 0) {
      dw = at::zeros({H, E}, gw.options());
      dx.zero_();
    } else {
      dw = at::empty({H, E}, gw.options());
      const int xdt = code_of(x), wdt = code_of(gw);
      const size_t nbytes = moe_router_bwd_workspace(N, H, E, K, xdt, wdt);
      const at::Tensor ws = at::empty({std::max<int64_t>((int64_t)nbytes, 1)}, x.options().dtype(at::kByte));
      const hipStream_t s = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(x.device().index()).stream();
      const int rc = moe_router_bwd_logits(x.data_ptr(), xdt, gw.data_ptr(), wdt, logits.data_ptr<float>(),
                                           idx.data_ptr<int64_t>(), g_w.defined() ? g_w.data_ptr() : nullptr, gdt,
                                           cnt.data_ptr<int64_t>(), g_aux.defined() ? g_aux.data_ptr<float>() : nullptr,
                                           g_z.defined() ? g_z.data_ptr<float>() : nullptr, aux_coef, z_coef,
                                           g_logits.defined() ? g_logits.data_ptr<float>() : nullptr, N, H, E, K,
                                           dx_add.defined() ? dx_add.data_ptr() : nullptr, dx.data_ptr(), dw.data_ptr(),
                                           ws.data_ptr(), nbytes, s);
      if (rc != 0) raise_rc(rc, "moe_router_bwd");
    }
    if (need_x) out[0] = dx;
    if (need_w) out[1] = dw;
    return out;
  }
};

variable_list router_core(const at::Tensor& x, const at::Tensor& gate_w, int64_t k, double aux_coef,
                          double z_coef, const std::optional<at::Tensor>& bias, bool link_x, bool diff_logits) {
  return RouterFn::apply(x, gate_w, k, aux_coef, z_coef, bias, link_x, diff_logits);
}

// ---- the operations of moe_mi355/ops.py: outputs from ATen, one C ABI call, no autograd.  ops.py has checked device,
// types and shapes; tensors arrive as its callers passed them and are made contiguous here where it made them so. ----

using OptTensor = std::optional<at::Tensor>;

hipStream_t stream_of(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
const void* ptr(const OptTensor& t) { return t.has_value() && t->defined() ? t->data_ptr() : nullptr; }
at::Tensor scratch(size_t n, const at::Tensor& like) {
  return at::empty({std::max<int64_t>((int64_t)n, 1)}, like.options().dtype(at::kByte));
}
void check_rc(int rc, const char* what) {
  if (rc != 0) raise_rc(rc, what);
}

std::vector<at::Tensor> op_router_forward(const at::Tensor& x_in, const at::Tensor& gw_in, int64_t k, const OptTensor& bias,
                                          bool w_bf16, double aux_coef, double z_coef) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
  const at::Tensor x = x_in.contiguous(), gw = gw_in.contiguous();
  const int64_t N = x.size(0), H = x.size(1), E = gw.size(1);
  const auto f32 = x.options().dtype(at::kFloat);
  const auto i64 = x.options().dtype(at::kLong);
  at::Tensor idx = at::empty({N, k}, i64), w = at::empty({N, k}, x.options().dtype(w_bf16 ? at::kBFloat16 : at::kFloat));
  at::Tensor logits = at::empty({N, E}, f32), lse = at::empty({N}, f32), cnt = at::empty({E}, i64);
  at::Tensor stats = at::empty({MOE_STATS_HEAD + E}, f32), aux = at::empty({}, f32), z = at::empty({}, f32);
  const hipStream_t s = stream_of(x);
  const int xdt = code_of(x), wdt = code_of(gw);
  const size_t nbytes = moe_router_fwd_workspace(N, H, E, k, xdt, wdt);
  const FwdWorkspace ws(nbytes, x.device(), s);
  check_rc(moe_router_fwd(x.data_ptr(), xdt, gw.data_ptr(), wdt, static_cast<const float*>(ptr(bias)), N, H, E, k,
                          idx.data_ptr<int64_t>(), w.data_ptr(), w_bf16 ? MOE_BF16 : MOE_F32, logits.data_ptr<float>(),
                          lse.data_ptr<float>(), cnt.data_ptr<int64_t>(), stats.data_ptr<float>(), (float)aux_coef,
                          (float)z_coef, aux.data_ptr<float>(), z.data_ptr<float>(), ws.data_ptr(), nbytes, s),
           "moe_router_fwd");
  return {idx, w, logits, lse, cnt, stats, aux, z};
}

std::vector<at::Tensor> op_rmsnorm_router_forward(const at::Tensor& x_in, const at::Tensor& weight_in, double eps,
                                                  const at::Tensor& gw_in, int64_t k, const OptTensor& bias,
                                                  double aux_coef, double z_coef) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
  const at::Tensor x = x_in.contiguous(), weight = weight_in.contiguous(), gw = gw_in.contiguous();
  const int64_t N = x.size(0), H = x.size(1), E = gw.size(1);
  const auto f32 = x.options().dtype(at::kFloat);
  const auto i64 = x.options().dtype(at::kLong);
  at::Tensor xn = at::empty_like(x), rstd = at::empty({N}, f32), idx = at::empty({N, k}, i64);
  at::Tensor w = at::empty({N, k}, x.options()), logits = at::empty({N, E}, f32), lse = at::empty({N}, f32);
  at::Tensor cnt = at::empty({E}, i64), stats = at::empty({MOE_STATS_HEAD + E}, f32);
  at::Tensor aux = at::empty({}, f32), z = at::empty({}, f32);
  const hipStream_t s = stream_of(x);
  const int xdt = code_of(x), wdt = code_of(gw);
  const size_t nbytes = moe_rmsnorm_router_fwd_workspace(N, H, E, k, xdt, wdt);
  const FwdWorkspace ws(nbytes, x.device(), s);
  check_rc(moe_rmsnorm_router_fwd(x.data_ptr(), xdt, weight.data_ptr(), code_of(weight), (float)eps, gw.data_ptr(), wdt,
                                  static_cast<const float*>(ptr(bias)), N, H, E, k, xn.data_ptr(), rstd.data_ptr<float>(),
                                  idx.data_ptr<int64_t>(), w.data_ptr(), xdt, logits.data_ptr<float>(),
                                  lse.data_ptr<float>(), cnt.data_ptr<int64_t>(), stats.data_ptr<float>(),
                                  (float)aux_coef, (float)z_coef, aux.data_ptr<float>(), z.data_ptr<float>(),
                                  ws.data_ptr(), nbytes, s),
           "moe_rmsnorm_router_fwd");
  return {xn, rstd, idx, w, logits, lse, cnt, stats, aux, z};
}

std::vector<at::Tensor> op_rmsnorm_router_backward(const at::Tensor& x_in, const at::Tensor& weight_in,
                                                   const at::Tensor& rstd, const at::Tensor& xn_in, const at::Tensor& gw_in,
                                                   const at::Tensor& logits_in, const at::Tensor& idx_in,
                                                   const OptTensor& grad_w, const OptTensor& dxn, const OptTensor& cnt,
                                                   const OptTensor& grad_aux, const OptTensor& grad_z, double aux_coef,
                                                   double z_coef, const OptTensor& grad_logits) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
  const at::Tensor x = x_in.contiguous(), weight = weight_in.contiguous(), xn = xn_in.contiguous();
  const at::Tensor gw = gw_in.contiguous(), logits = logits_in.contiguous(), idx = idx_in.contiguous();
  const int64_t N = x.size(0), H = x.size(1), E = gw.size(1), K = idx.size(1);
  at::Tensor dx = at::empty_like(x), dweight = at::empty_like(weight), dgate = at::empty({H, E}, gw.options());
  const int xdt = code_of(x), wdt = code_of(gw);
  const size_t nbytes = moe_rmsnorm_router_bwd_workspace(N, H, E, K, xdt, wdt);
  const at::Tensor ws = scratch(nbytes, x);
  check_rc(moe_rmsnorm_router_bwd_logits(
               x.data_ptr(), xdt, weight.data_ptr(), code_of(weight), rstd.data_ptr<float>(), xn.data_ptr(), gw.data_ptr(),
               wdt, logits.data_ptr<float>(), idx.data_ptr<int64_t>(), ptr(grad_w),
               grad_w.has_value() && grad_w->defined() ? code_of(*grad_w) : MOE_F32, static_cast<const int64_t*>(ptr(cnt)),
               static_cast<const float*>(ptr(grad_aux)), static_cast<const float*>(ptr(grad_z)), (float)aux_coef,
               (float)z_coef, static_cast<const float*>(ptr(grad_logits)), ptr(dxn), N, H, E, K, dx.data_ptr(), dweight.data_ptr(), dgate.data_ptr(), ws.data_ptr(),
               nbytes, stream_of(x)),
           "moe_rmsnorm_router_bwd");
  return {dx, dweight, dgate};
}

std::tuple<OptTensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> op_plan(const at::Tensor& idx_in, int64_t E,
                                                                               int64_t capacity, int64_t layout) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(idx_in.device());
  at::Tensor idx = idx_in.contiguous();
  if (idx.scalar_type() != at::kLong) idx = idx.to(at::kLong);
  const int64_t N = idx.size(0), K = idx.size(1), M = N * K;
  const auto i32 = idx.options().dtype(at::kInt);
  OptTensor drop;
  if (capacity >= 0) drop = at::empty({N, K}, idx.options().dtype(at::kBool));
  at::Tensor row_slot = at::empty({M}, i32), slot_row = at::empty({M}, i32), offsets = at::empty({E + 1}, i32);
  at::Tensor ndrop = at::empty({1}, i32);
  const size_t nbytes = moe_plan_workspace(N, K, E);
  const at::Tensor ws = scratch(nbytes, idx);
  check_rc(moe_plan(idx.data_ptr<int64_t>(), N, K, E, capacity, (int)layout,
                    static_cast<uint8_t*>(const_cast<void*>(ptr(drop))), row_slot.data_ptr<int>(),
                    slot_row.data_ptr<int>(), offsets.data_ptr<int>(), ndrop.data_ptr<int>(), ws.data_ptr(), nbytes,
                    stream_of(idx)),
           "moe_plan");
  return {drop, row_slot, slot_row, offsets, ndrop};
}

at::Tensor op_permute(const at::Tensor& x_in, const at::Tensor& slot_row, const at::Tensor& offsets, int64_t N, int64_t K,
                      int64_t E) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
  const at::Tensor x = x_in.contiguous();
  const int64_t H = x.size(1);
  at::Tensor xp = at::empty({N * K, H}, x.options());
  check_rc(moe_permute(x.data_ptr(), H * x.element_size(), slot_row.data_ptr<int>(), offsets.data_ptr<int>(), N, K, E,
                       xp.data_ptr(), stream_of(x)),
           "moe_permute");
  return xp;
}

at::Tensor op_combine(const at::Tensor& y_in, const at::Tensor& w_in, const OptTensor& drop, const at::Tensor& slot_row,
                      const at::Tensor& offsets, int64_t N, int64_t K, int64_t E) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(y_in.device());
  const at::Tensor y = y_in.contiguous(), w = w_in.contiguous();
  const int64_t H = y.size(1);
  at::Tensor out = at::empty({N, H}, y.options());
  check_rc(moe_combine(y.data_ptr(), code_of(y), w.data_ptr(), code_of(w), static_cast<const uint8_t*>(ptr(drop)),
                       slot_row.data_ptr<int>(), offsets.data_ptr<int>(), N, K, H, E, out.data_ptr(), stream_of(y)),
           "moe_combine");
  return out;
}

std::tuple<at::Tensor, OptTensor> op_combine_backward(const at::Tensor& dout_in, const at::Tensor& y, const at::Tensor& w_in,
                                                      const OptTensor& drop, const at::Tensor& slot_row,
                                                      const at::Tensor& offsets, int64_t N, int64_t K, int64_t E,
                                                      bool need_dw, bool zero_tail) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(y.device());
  const at::Tensor dout = dout_in.contiguous(), w = w_in.contiguous();
  const int64_t H = y.size(1);
  at::Tensor dy = at::empty_like(y);
  OptTensor dw;
  if (need_dw) dw = at::empty({N, K}, w.options());
  const hipStream_t s = stream_of(y);
  check_rc(moe_combine_bwd(dout.data_ptr(), y.data_ptr(), code_of(y), w.data_ptr(), code_of(w),
                           static_cast<const uint8_t*>(ptr(drop)), slot_row.data_ptr<int>(), offsets.data_ptr<int>(), N, K,
                           H, E, dy.data_ptr(), const_cast<void*>(ptr(dw)), s),
           "moe_combine_bwd");
  if (zero_tail)
    check_rc(moe_zero_tail(dy.data_ptr(), H * dy.element_size(), offsets.data_ptr<int>(), E, dy.size(0), s),
             "moe_zero_tail");
  return {dy, dw};
}

at::Tensor op_unpermute_sum(const at::Tensor& dxp_in, const OptTensor& addend_in, const at::Tensor& slot_row,
                            const at::Tensor& offsets, int64_t N, int64_t K, int64_t E) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dxp_in.device());
  const at::Tensor dxp = dxp_in.contiguous();
  OptTensor addend;
  if (addend_in.has_value() && addend_in->defined()) addend = addend_in->contiguous();
  const int64_t H = dxp.size(1);
  at::Tensor dx = at::empty({N, H}, dxp.options());
  check_rc(moe_unpermute_sum(dxp.data_ptr(), ptr(addend), code_of(dxp), slot_row.data_ptr<int>(), offsets.data_ptr<int>(),
                             N, K, H, E, dx.data_ptr(), stream_of(dxp)),
           "moe_unpermute_sum");
  return dx;
}

// Bytes of the grouped GEMM's tile tables and of the partial tiles of products split over k.
size_t gemm_workspace(bool f32, bool fwd, int64_t R, int64_t H, int64_t F, int64_t E) {
  if (f32)
    return moe_swiglu_f32_workspace(E) +
           (fwd ? moe_swiglu_fwd_f32_split_workspace(R, H, F, E) : moe_swiglu_f32_split_workspace(R, H, F, E));
  return moe_swiglu_workspace(E) +
         (fwd ? moe_swiglu_fwd_split_workspace(R, H, F, E) : moe_swiglu_split_workspace(R, H, F, E));
}

std::tuple<at::Tensor, OptTensor, at::Tensor> op_swiglu_forward(const at::Tensor& xp, const at::Tensor& wg,
                                                                const at::Tensor& wu, const at::Tensor& wd,
                                                                const at::Tensor& offsets, bool keep_preact) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(xp.device());
  const bool f32 = xp.scalar_type() == at::kFloat;
  const int64_t R = xp.size(0), H = xp.size(1), E = wg.size(0), F = wg.size(1);
  at::Tensor act = at::empty({R, F}, xp.options()), y = at::empty({R, H}, xp.options());
  OptTensor hgu;
  if (keep_preact) hgu = at::empty({R, 2 * F}, xp.options());
  const size_t nbytes = gemm_workspace(f32, true, R, H, F, E);
  const at::Tensor ws = scratch(nbytes, xp);
  const hipStream_t s = stream_of(xp);
  void* const h = const_cast<void*>(ptr(hgu));
  if (f32)
    check_rc(moe_swiglu_fwd_f32(xp.data_ptr<float>(), wg.data_ptr<float>(), wu.data_ptr<float>(), wd.data_ptr<float>(),
                                offsets.data_ptr<int>(), R, H, F, E, act.data_ptr<float>(), static_cast<float*>(h),
                                y.data_ptr<float>(), ws.data_ptr(), nbytes, s),
             "moe_swiglu_fwd_f32");
  else
    check_rc(moe_swiglu_fwd(xp.data_ptr(), wg.data_ptr(), wu.data_ptr(), wd.data_ptr(), offsets.data_ptr<int>(), R, H, F, E,
                            act.data_ptr(), h, y.data_ptr(), ws.data_ptr(), nbytes, s),
             "moe_swiglu_fwd");
  return {act, hgu, y};
}

std::vector<at::Tensor> op_swiglu_backward(const at::Tensor& dy, const at::Tensor& xp, const at::Tensor& act,
                                           const at::Tensor& hgu, const at::Tensor& wg, const at::Tensor& wu,
                                           const at::Tensor& wd, const at::Tensor& offsets) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(xp.device());
  const bool f32 = xp.scalar_type() == at::kFloat;
  const int64_t R = xp.size(0), H = xp.size(1), E = wg.size(0), F = wg.size(1);
  at::Tensor dh = at::empty({R, 2 * F}, xp.options()), dxp = at::empty({R, H}, xp.options());
  at::Tensor dwg = at::empty_like(wg), dwu = at::empty_like(wu), dwd = at::empty_like(wd);
  const size_t nbytes = gemm_workspace(f32, false, R, H, F, E);
  const at::Tensor ws = scratch(nbytes, xp);
  const hipStream_t s = stream_of(xp);
  if (f32)
    check_rc(moe_swiglu_bwd_f32(dy.data_ptr<float>(), xp.data_ptr<float>(), act.data_ptr<float>(), hgu.data_ptr<float>(),
                                wg.data_ptr<float>(), wu.data_ptr<float>(), wd.data_ptr<float>(), offsets.data_ptr<int>(), R,
                                H, F, E, dh.data_ptr<float>(), dxp.data_ptr<float>(), dwg.data_ptr<float>(),
                                dwu.data_ptr<float>(), dwd.data_ptr<float>(), ws.data_ptr(), nbytes, s),
             "moe_swiglu_bwd_f32");
  else
    check_rc(moe_swiglu_bwd(dy.data_ptr(), xp.data_ptr(), act.data_ptr(), hgu.data_ptr(), wg.data_ptr(), wu.data_ptr(),
                            wd.data_ptr(), offsets.data_ptr<int>(), R, H, F, E, dh.data_ptr(), dxp.data_ptr(),
                            dwg.data_ptr(), dwu.data_ptr(), dwd.data_ptr(), ws.data_ptr(), nbytes, s),
             "moe_swiglu_bwd");
  return {dxp, dwg, dwu, dwd};
}

// ---- MXFP4 experts ----

std::tuple<at::Tensor, at::Tensor> op_quant_mxfp4(const at::Tensor& t_in) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(t_in.device());
  const at::Tensor t = t_in.contiguous();
  std::vector<int64_t> qs = t.sizes().vec(), ss = qs;
  const int64_t cols = qs.back(), rows = t.numel() / cols;
  qs.back() = cols / 2;
  ss.back() = cols / 32;
  const auto u8 = t.options().dtype(at::kByte);
  at::Tensor q = at::empty(qs, u8), sc = at::empty(ss, u8);
  check_rc(moe_quant_mxfp4(t.data_ptr(), code_of(t), rows, cols, q.data_ptr(), sc.data_ptr(), stream_of(t)),
           "moe_quant_mxfp4");
  return {q, sc};
}

at::Tensor op_dequant_mxfp4(const at::Tensor& q_in, const at::Tensor& sc_in, bool bf16) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q_in.device());
  const at::Tensor q = q_in.contiguous(), sc = sc_in.contiguous();
  std::vector<int64_t> vs = q.sizes().vec();
  vs.back() *= 2;
  at::Tensor v = at::empty(vs, q.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
  const int64_t cols = vs.back(), rows = v.numel() / cols;
  check_rc(moe_dequant_mxfp4(q.data_ptr(), sc.data_ptr(), rows, cols, v.data_ptr(), bf16 ? MOE_BF16 : MOE_F32, stream_of(q)),
           "moe_dequant_mxfp4");
  return v;
}

// wq, ws: the quantized gate [E, F, H], up [E, F, H] and down [E, H, F] matrices and their scales, contiguous.
std::tuple<OptTensor, at::Tensor> op_swiglu_forward_mxfp4(const at::Tensor& xp_in, const std::vector<at::Tensor>& wq,
                                                          const std::vector<at::Tensor>& ws, const at::Tensor& offsets,
                                                          bool keep_preact) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(xp_in.device());
  const at::Tensor xp = xp_in.contiguous();
  const int64_t R = xp.size(0), H = xp.size(1), E = wq[0].size(0), F = wq[0].size(1);
  at::Tensor y = at::empty({R, H}, xp.options());
  OptTensor hgu;
  if (keep_preact) hgu = at::empty({R, 2 * F}, xp.options());
  const size_t nbytes = moe_swiglu_fwd_mxfp4_workspace(R, H, F, E);
  const at::Tensor w = scratch(nbytes, xp);
  check_rc(moe_swiglu_fwd_mxfp4(xp.data_ptr(), wq[0].data_ptr(), ws[0].data_ptr(), wq[1].data_ptr(), ws[1].data_ptr(),
                                wq[2].data_ptr(), ws[2].data_ptr(), offsets.data_ptr<int>(), R, H, F, E,
                                const_cast<void*>(ptr(hgu)), y.data_ptr(), w.data_ptr(), nbytes, stream_of(xp)),
           "moe_swiglu_fwd_mxfp4");
  return {hgu, y};
}

at::Tensor op_swiglu_backward_mxfp4(const at::Tensor& dy_in, const at::Tensor& hgu_in, const std::vector<at::Tensor>& wq,
                                    const std::vector<at::Tensor>& ws, const at::Tensor& offsets) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(dy_in.device());
  const at::Tensor dy = dy_in.contiguous(), hgu = hgu_in.contiguous();
  const int64_t R = dy.size(0), H = dy.size(1), E = wq[0].size(0), F = wq[0].size(1);
  at::Tensor dxp = at::empty({R, H}, dy.options());
  const size_t nbytes = moe_swiglu_bwd_mxfp4_workspace(R, H, F, E);
  const at::Tensor w = scratch(nbytes, dy);
  check_rc(moe_swiglu_bwd_mxfp4(dy.data_ptr(), hgu.data_ptr(), wq[0].data_ptr(), ws[0].data_ptr(), wq[1].data_ptr(),
                                ws[1].data_ptr(), wq[2].data_ptr(), ws[2].data_ptr(), offsets.data_ptr<int>(), R, H, F, E,
                                dxp.data_ptr(), w.data_ptr(), nbytes, stream_of(dy)),
           "moe_swiglu_bwd_mxfp4");
  return dxp;
}

// ---- rows in 8 bits, the norm that gives them, int8 products ----
// With one decoded token these calls' kernels are a few microseconds, so their arguments are checked here.

// All given tensors on one GPU (the messages of _lib.require_device).
void one_gpu(std::initializer_list<const at::Tensor*> ts) {
  const at::Tensor* first = nullptr;
  for (const at::Tensor* t : ts) {
    if (t == nullptr || !t->defined()) continue;
    if (!t->is_cuda())
      throw std::runtime_error("moe_mi355 runs on an AMD Instinct GPU (gfx950) only; got a tensor on " + t->device().str() +
                               ". Move the module and inputs to the GPU.");
    if (first == nullptr) first = t;
    else if (t->device() != first->device())
      throw std::runtime_error("moe_mi355: tensors on different devices (" + first->device().str() + " vs " +
                               t->device().str() + ")");
  }
}
const at::Tensor* opt(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }

std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}
void need(bool ok, const char* what, const std::string& msg) {
  if (!ok) throw pybind11::value_error(std::string(what) + ": " + msg);
}
void need_type(bool ok, const char* what, const std::string& msg) {
  if (!ok) throw pybind11::type_error(std::string(what) + ": " + msg);
}
bool is_float(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }
void need_shape(const at::Tensor& t, at::IntArrayRef want, const char* what, const char* name) {
  if (t.sizes() == want) return;
  std::string s = "[";
  for (size_t i = 0; i < want.size(); ++i) s += (i ? ", " : "") + std::to_string(want[i]);
  throw pybind11::value_error(std::string(what) + ": " + name + " must be " + s + "], got " + shape_of(t));
}

std::tuple<at::Tensor, at::Tensor> op_quant_rows_int8(const at::Tensor& t_in) {
  const char* const what = "quant_rows_int8";
  one_gpu({&t_in});
  need_type(is_float(t_in), what, "rows are float32 or bfloat16");
  need(t_in.dim() >= 1 && t_in.size(-1) >= 16 && t_in.size(-1) % 16 == 0, what,
       "the last dim must be a positive multiple of 16, got " + shape_of(t_in));
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(t_in.device());
  const at::Tensor t = t_in.contiguous();
  const int64_t cols = t.size(-1), rows = t.numel() / cols;
  at::Tensor q = at::empty(t.sizes(), t.options().dtype(at::kChar));
  at::Tensor sc = at::empty(t.sizes().slice(0, t.dim() - 1), t.options().dtype(at::kFloat));
  check_rc(moe_quant_rows_int8(t.data_ptr(), code_of(t), rows, cols, cols, q.data_ptr(), sc.data_ptr<float>(), stream_of(t)),
           "moe_quant_rows_int8");
  return {q, sc};
}

at::Tensor op_dequant_rows(const at::Tensor& q_in, const at::Tensor& sc_in, bool bf16) {
  const char* const what = "dequant_rows";
  one_gpu({&q_in, &sc_in});
  need_type(q_in.scalar_type() == at::kChar || q_in.scalar_type() == at::kByte, what, "q is int8, or uint8 (e4m3 bytes)");
  need_type(sc_in.scalar_type() == at::kFloat, what, "scale is float32");
  need(q_in.dim() >= 1 && q_in.size(-1) >= 16 && q_in.size(-1) % 16 == 0, what,
       "the last dim must be a positive multiple of 16, got " + shape_of(q_in));
  need_shape(sc_in, q_in.sizes().slice(0, q_in.dim() - 1), what, "scale");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q_in.device());
  const at::Tensor q = q_in.contiguous(), sc = sc_in.contiguous();
  at::Tensor v = at::empty(q.sizes(), q.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
  const int64_t cols = q.size(-1);
  check_rc(moe_dequant_rows(q.data_ptr(), q.scalar_type() == at::kChar ? MOE_INT8 : MOE_E4M3, sc.data_ptr<float>(),
                            q.numel() / cols, cols, v.data_ptr(), code_of(v), stream_of(q)),
           "moe_dequant_rows");
  return v;
}

void need_rows_int8(const at::Tensor& q, const at::Tensor& sc, const char* what) {
  need_type(q.scalar_type() == at::kChar && sc.scalar_type() == at::kFloat, what, "rows are int8 and their scales float32");
  need(q.dim() >= 1, what, "rows must have a dim to sum over");
  need_shape(sc, q.sizes().slice(0, q.dim() - 1), what, "the rows' scales");
}
void need_weight_int8(const at::Tensor& w, const at::Tensor& sw, const char* what) {
  need_type(w.scalar_type() == at::kChar && sw.scalar_type() == at::kFloat, what,
            "weights are int8 and their scales float32");
  need(w.is_contiguous() && sw.is_contiguous(), what, "weights and their scales must be contiguous");
}
void need_offsets(const at::Tensor& o, int64_t E, const char* what) {
  need(o.scalar_type() == at::kInt && o.dim() == 1 && o.size(0) == E + 1 && o.is_contiguous(), what,
       "offsets must be contiguous int32 [" + std::to_string(E + 1) + "]");
}

at::Tensor op_matmul_int8(const at::Tensor& q_in, const at::Tensor& sc_in, const at::Tensor& wq, const at::Tensor& wsc,
                          const OptTensor& offsets, bool bf16) {
  const char* const what = "matmul_int8";
  one_gpu({&q_in, &sc_in, &wq, &wsc, opt(offsets)});
  need_rows_int8(q_in, sc_in, what);
  need_weight_int8(wq, wsc, what);
  const bool grouped = offsets.has_value();
  need(wq.dim() == (grouped ? 3 : 2), what,
       std::string("wq must be ") + (grouped ? "[E, N, K] with offsets" : "[N, K] without offsets") + ", got " + shape_of(wq));
  need_shape(wsc, wq.sizes().slice(0, wq.dim() - 1), what, "wscale");
  const int64_t K = wq.size(-1), N = wq.size(-2), E = grouped ? wq.size(0) : 1;
  need(q_in.size(-1) == K && (!grouped || q_in.dim() == 2), what,
       "rows " + shape_of(q_in) + " do not go with weights " + shape_of(wq));
  if (grouped) need_offsets(*offsets, E, what);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q_in.device());
  const at::Tensor q = q_in.contiguous(), sc = sc_in.contiguous();
  std::vector<int64_t> ys = q.sizes().vec();
  ys.back() = N;
  at::Tensor y = at::empty(ys, q.options().dtype(bf16 ? at::kBFloat16 : at::kFloat));
  const size_t nbytes = moe_matmul_int8_workspace(sc.numel(), K, N, E);
  at::Tensor ws;
  if (nbytes > 0) ws = scratch(nbytes, q);
  check_rc(moe_matmul_int8(q.data_ptr(), sc.data_ptr<float>(), wq.data_ptr(), wsc.data_ptr<float>(),
                           static_cast<const int*>(ptr(offsets)), sc.numel(), K, N, E, y.data_ptr(), code_of(y),
                           nbytes > 0 ? ws.data_ptr() : nullptr, nbytes, stream_of(q)),
           "moe_matmul_int8");
  return y;
}

at::Tensor op_swiglu_forward_int8(const at::Tensor& xq_in, const at::Tensor& sx_in, const std::vector<at::Tensor>& wq,
                                  const std::vector<at::Tensor>& ws, const at::Tensor& offsets, const OptTensor& row_slot,
                                  int64_t top_k) {
  const char* const what = "swiglu_forward_int8";
  need(wq.size() == 3 && ws.size() == 3, what, "wq and wscale are (gate, up, down)");
  one_gpu({&xq_in, &sx_in, &wq[0], &wq[1], &wq[2], &ws[0], &ws[1], &ws[2], &offsets, opt(row_slot)});
  need_rows_int8(xq_in, sx_in, what);
  for (int i = 0; i < 3; ++i) need_weight_int8(wq[i], ws[i], what);
  need(xq_in.dim() == 2 && wq[0].dim() == 3, what, "rows are [T, H] and weights of rank 3");
  const int64_t T = xq_in.size(0), H = xq_in.size(1), E = wq[0].size(0), F = wq[0].size(1);
  need_shape(wq[0], {E, F, H}, what, "gate");
  need_shape(wq[1], {E, F, H}, what, "up");
  need_shape(wq[2], {E, H, F}, what, "down");
  need_shape(ws[0], {E, F}, what, "gate scale");
  need_shape(ws[1], {E, F}, what, "up scale");
  need_shape(ws[2], {E, H}, what, "down scale");
  need_offsets(offsets, E, what);
  int64_t R = T;
  if (row_slot.has_value()) {
    need(row_slot->scalar_type() == at::kInt && row_slot->dim() == 1 && row_slot->is_contiguous() && top_k >= 1, what,
         "row_slot must be contiguous int32 [R], with top_k >= 1");
    R = row_slot->size(0);
  }
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(xq_in.device());
  const at::Tensor xq = xq_in.contiguous(), sx = sx_in.contiguous();
  at::Tensor y = at::empty({R, H}, xq.options().dtype(at::kBFloat16));
  if (R == 0) return y;
  const size_t nbytes = moe_swiglu_fwd_int8_workspace(R, H, F, E);
  const at::Tensor w = scratch(nbytes, xq);
  check_rc(moe_swiglu_fwd_int8(xq.data_ptr(), sx.data_ptr<float>(), T, static_cast<const int*>(ptr(row_slot)), top_k,
                               wq[0].data_ptr(), ws[0].data_ptr<float>(), wq[1].data_ptr(), ws[1].data_ptr<float>(),
                               wq[2].data_ptr(), ws[2].data_ptr<float>(), offsets.data_ptr<int>(), R, H, F, E, y.data_ptr(),
                               w.data_ptr(), nbytes, stream_of(xq)),
           "moe_swiglu_fwd_int8");
  return y;
}

void need_norm(const at::Tensor& x, const at::Tensor& weight, const char* what) {
  need_type(is_float(x) && is_float(weight), what, "tensors are float32 or bfloat16");
  need(x.dim() == 2 && weight.dim() == 1 && weight.size(0) == x.size(1), what,
       "x must be [N, H] and weight [H], got " + shape_of(x) + " and " + shape_of(weight));
}
void need_like(const at::Tensor& t, const at::Tensor& x, const char* what, const char* name) {
  need_type(t.scalar_type() == x.scalar_type(), what, std::string(name) + " must have x's dtype");
  need_shape(t, x.sizes(), what, name);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> op_rmsnorm_residual_forward(const at::Tensor& x_in, const at::Tensor& r_in,
                                                                           const at::Tensor& weight_in, double eps) {
  const char* const what = "rmsnorm_residual_forward";
  one_gpu({&x_in, &r_in, &weight_in});
  need_norm(x_in, weight_in, what);
  need_like(r_in, x_in, what, "residual");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
  const at::Tensor x = x_in.contiguous(), r = r_in.contiguous(), weight = weight_in.contiguous();
  at::Tensor xn = at::empty(x.sizes(), x.options()), h = at::empty(x.sizes(), x.options());
  at::Tensor rstd = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  check_rc(moe_rmsnorm_residual_fwd(x.data_ptr(), r.data_ptr(), code_of(x), weight.data_ptr(), code_of(weight), (float)eps,
                                    x.size(0), x.size(1), h.data_ptr(), xn.data_ptr(), rstd.data_ptr<float>(), stream_of(x)),
           "moe_rmsnorm_residual_fwd");
  return {xn, h, rstd};
}

std::tuple<at::Tensor, at::Tensor> op_rmsnorm_residual_backward(const at::Tensor& h_in, const at::Tensor& weight_in,
                                                                const at::Tensor& rstd_in, const OptTensor& dxn_in,
                                                                const OptTensor& dh_in) {
  const char* const what = "rmsnorm_residual_backward";
  one_gpu({&h_in, &weight_in, &rstd_in, opt(dxn_in), opt(dh_in)});
  need_norm(h_in, weight_in, what);
  need(rstd_in.scalar_type() == at::kFloat && rstd_in.dim() == 1 && rstd_in.size(0) == h_in.size(0), what,
       "rstd must be float32 [" + std::to_string(h_in.size(0)) + "]");
  need(dxn_in.has_value() || dh_in.has_value(), what, "needs a gradient of xn or of h");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(h_in.device());
  const at::Tensor h = h_in.contiguous(), weight = weight_in.contiguous(), rstd = rstd_in.contiguous();
  OptTensor dxn, dh;
  if (dxn_in.has_value()) {
    need_like(*dxn_in, h, what, "dxn");
    dxn = dxn_in->contiguous();
  }
  if (dh_in.has_value()) {
    need_like(*dh_in, h, what, "dh");
    dh = dh_in->contiguous();
  }
  at::Tensor d = at::empty(h.sizes(), h.options()), dw = at::empty(weight.sizes(), weight.options());
  const size_t nbytes = moe_rmsnorm_residual_bwd_workspace(h.size(0), h.size(1));
  const at::Tensor ws = scratch(nbytes, h);
  check_rc(moe_rmsnorm_residual_bwd(h.data_ptr(), code_of(h), weight.data_ptr(), code_of(weight), rstd.data_ptr<float>(),
                                    ptr(dxn), ptr(dh), h.size(0), h.size(1), d.data_ptr(), dw.data_ptr(), ws.data_ptr(), nbytes,
                                    stream_of(h)),
           "moe_rmsnorm_residual_bwd");
  return {d, dw};
}

std::tuple<at::Tensor, at::Tensor, OptTensor, OptTensor> op_rmsnorm_quant(const at::Tensor& x_in, const at::Tensor& weight_in,
                                                                          double eps, const OptTensor& r_in, bool e4m3,
                                                                          bool keep_norm) {
  const char* const what = "rmsnorm_quant";
  one_gpu({&x_in, &weight_in, opt(r_in)});
  need_norm(x_in, weight_in, what);
  if (r_in.has_value()) need_like(*r_in, x_in, what, "residual");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x_in.device());
  const at::Tensor x = x_in.contiguous(), weight = weight_in.contiguous();
  OptTensor r, xn, h;
  if (r_in.has_value()) {
    r = r_in->contiguous();
    h = at::empty(x.sizes(), x.options());
  }
  if (keep_norm) xn = at::empty(x.sizes(), x.options());
  at::Tensor q = at::empty(x.sizes(), x.options().dtype(e4m3 ? at::kByte : at::kChar));
  at::Tensor sc = at::empty({x.size(0)}, x.options().dtype(at::kFloat));
  check_rc(moe_rmsnorm_quant(x.data_ptr(), ptr(r), code_of(x), weight.data_ptr(), code_of(weight), (float)eps, x.size(0),
                             x.size(1), e4m3 ? MOE_E4M3 : MOE_INT8, q.data_ptr(), sc.data_ptr<float>(),
                             const_cast<void*>(ptr(h)), const_cast<void*>(ptr(xn)), stream_of(x)),
           "moe_rmsnorm_quant");
  return {q, sc, xn, h};
}

// ---- the balance loss of sequences ----

std::vector<at::Tensor> op_balance_forward(const at::Tensor& logits_in, const at::Tensor& idx_in, const OptTensor& off_in,
                                           const OptTensor& mask_in, double balance_coef, double z_coef) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(logits_in.device());
  const at::Tensor logits = logits_in.contiguous(), idx = idx_in.contiguous();
  OptTensor off, mask;
  if (off_in.has_value()) off = off_in->to(at::kLong).contiguous();
  if (mask_in.has_value()) mask = mask_in->contiguous();
  const int64_t N = logits.size(0), E = logits.size(1), K = idx.size(1), S = off.has_value() ? off->size(0) - 1 : 1;
  const auto f32 = logits.options();
  const auto i64 = logits.options().dtype(at::kLong);
  at::Tensor balance = at::empty({}, f32), z = at::empty({}, f32), counts = at::empty({S, E}, i64);
  at::Tensor tokens = at::empty({S + 2}, i64), mean_prob = at::empty({S, E}, f32);
  const size_t nbytes = moe_balance_fwd_workspace(N, E, S);
  const at::Tensor ws = scratch(nbytes, logits);
  check_rc(moe_balance_fwd(logits.data_ptr<float>(), idx.data_ptr<int64_t>(), static_cast<const int64_t*>(ptr(off)),
                           static_cast<const uint8_t*>(ptr(mask)), N, E, K, S, (float)balance_coef, (float)z_coef,
                           balance.data_ptr<float>(), z.data_ptr<float>(), counts.data_ptr<int64_t>(),
                           tokens.data_ptr<int64_t>(), mean_prob.data_ptr<float>(), ws.data_ptr(), nbytes, stream_of(logits)),
           "moe_balance_fwd");
  return {balance, z, counts, tokens, mean_prob};
}

at::Tensor op_balance_backward(const at::Tensor& logits_in, const at::Tensor& counts_in, const at::Tensor& tokens_in,
                               int64_t K, const OptTensor& off_in, const OptTensor& mask_in, const OptTensor& grad_b,
                               const OptTensor& grad_z, double balance_coef, double z_coef) {
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(logits_in.device());
  const at::Tensor logits = logits_in.contiguous(), counts = counts_in.contiguous(), tokens = tokens_in.contiguous();
  OptTensor off, mask;
  if (off_in.has_value()) off = off_in->to(at::kLong).contiguous();
  if (mask_in.has_value()) mask = mask_in->contiguous();
  const int64_t N = logits.size(0), E = logits.size(1), S = counts.size(0);
  at::Tensor d = at::empty_like(logits);
  check_rc(moe_balance_bwd(logits.data_ptr<float>(), counts.data_ptr<int64_t>(), tokens.data_ptr<int64_t>(),
                           static_cast<const int64_t*>(ptr(off)), static_cast<const uint8_t*>(ptr(mask)),
                           static_cast<const float*>(ptr(grad_b)), static_cast<const float*>(ptr(grad_z)), N, E, K, S,
                           (float)balance_coef, (float)z_coef, d.data_ptr<float>(), stream_of(logits)),
           "moe_balance_bwd");
  return d;
}

}  // namespace

PYBIND11_MODULE(_moe_torch, m) {
  m.doc() = "Native autograd binding of the fused HIP router (forward and backward over the moe_mi355 C ABI).";
  // No call holds the GIL: none touches a Python object, and one that waits (for the allocator, a full queue or the
  // workspace lock) holds up no other thread.
  const pybind11::call_guard<pybind11::gil_scoped_release> nogil;
  m.def("router_core", &router_core, "(x, gate_w, k, aux_coef, z_coef, bias) -> (idx, w, aux, z, logits, cnt, stats)",
        pybind11::arg("x"), pybind11::arg("gate_w"), pybind11::arg("k"), pybind11::arg("aux_coef"),
        pybind11::arg("z_coef"), pybind11::arg("bias") = pybind11::none(), pybind11::arg("link_x") = false,
        pybind11::arg("diff_logits") = false, nogil);
  m.def("router_forward", &op_router_forward, nogil);
  m.def("rmsnorm_router_forward", &op_rmsnorm_router_forward, nogil);
  m.def("rmsnorm_router_backward", &op_rmsnorm_router_backward, nogil);
  m.def("plan", &op_plan, nogil);
  m.def("permute", &op_permute, nogil);
  m.def("combine", &op_combine, nogil);
  m.def("combine_backward", &op_combine_backward, nogil);
  m.def("unpermute_sum", &op_unpermute_sum, nogil);
  m.def("swiglu_forward", &op_swiglu_forward, nogil);
  m.def("swiglu_backward", &op_swiglu_backward, nogil);
  m.def("quant_mxfp4", &op_quant_mxfp4, nogil);
  m.def("dequant_mxfp4", &op_dequant_mxfp4, nogil);
  m.def("swiglu_forward_mxfp4", &op_swiglu_forward_mxfp4, nogil);
  m.def("swiglu_backward_mxfp4", &op_swiglu_backward_mxfp4, nogil);
  m.def("quant_rows_int8", &op_quant_rows_int8, nogil);
  m.def("dequant_rows", &op_dequant_rows, nogil);
  m.def("matmul_int8", &op_matmul_int8, nogil);
  m.def("swiglu_forward_int8", &op_swiglu_forward_int8, nogil);
  m.def("rmsnorm_residual_forward", &op_rmsnorm_residual_forward, nogil);
  m.def("rmsnorm_residual_backward", &op_rmsnorm_residual_backward, nogil);
  m.def("rmsnorm_quant", &op_rmsnorm_quant, nogil);
  m.def("balance_forward", &op_balance_forward, nogil);
  m.def("balance_backward", &op_balance_backward, nogil);
}

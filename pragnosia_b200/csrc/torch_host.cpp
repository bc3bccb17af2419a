// The host half of the operators whose kernels are shorter than the Python around them: argument checks, output allocation, the
// library call and the autograd nodes, in C++. A call of a few microseconds on the GPU spent 15 us in Python, a training pass of
// the scan (B16 T512 D704: 104 us of kernels) 160, most of it in the autograd functions' Python frames. The C ABI stays what the
// kernels are reached by; this file only prepares its arguments, and ops.py / scan_kernel.py / assoc_kernel.py call it.
#include <ATen/TracerMode.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/extension.h>

#include "../../include/pragnosia_b200.h"

namespace {
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int CHUNK = 64;
// Bytes of per-chunk states the fp32 plain prefill takes at most: more chains or chunks than that go one group after the other. Without
// a limit 768 chains of 4096 tokens took 805 MB for 3.41 ms; 3.49 at 256 MiB, 3.66 at 64, 5.2 at 16.
constexpr long long FP32_SCRATCH = 256LL << 20;

void check(int status, const char *what) {
    if (status == PGB_OK) return;
    std::string msg = std::string(what) + ": " + pgb_status_string(status);
    if (status == PGB_ERR_CUDA) msg += std::string(" [") + pgb_last_cuda_error() + "]";
    throw std::runtime_error(msg);
}
void need_cuda(const Tensor &t) {
    if (t.defined() && !t.is_cuda()) throw std::runtime_error("pragnosia_b200 ops run on CUDA tensors only (there is no CPU path)");
}
template <typename... P> void need_cuda(const Tensor &t, const P &...rest) { need_cuda(t); need_cuda(rest...); }

// an absent tensor is an undefined one from here on
Tensor opt(const OptTensor &t) { return t.has_value() ? *t : Tensor(); }
OptTensor some(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor f32c(const Tensor &t) {
    if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
    return t.to(at::kFloat).contiguous();
}
Tensor as(const Tensor &t, at::ScalarType dt) { return !t.defined() || t.scalar_type() == dt ? t : t.to(dt); }
Tensor like(const Tensor &t, at::ScalarType dt) { return as(t, dt).contiguous(); }
float *fp(const Tensor &t) { return t.defined() ? static_cast<float *>(t.data_ptr()) : nullptr; }
void *vp(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
int code(const Tensor &t) { return t.scalar_type() == at::kFloat ? PGB_F32 : PGB_BF16; }
bool io_type(at::ScalarType t) { return t == at::kFloat || t == at::kBFloat16; }
Tensor alloc(const Tensor &ref, at::IntArrayRef shape, at::ScalarType dt) { return at::empty(shape, ref.options().dtype(dt).requires_grad(false)); }
Tensor bytes(const Tensor &ref, long long n) { return alloc(ref, {n}, at::kByte); }

// the library reads CUDA's current device and is handed that device's current stream
struct OnDevice {
    c10::cuda::CUDAGuard guard;
    void *stream;
    explicit OnDevice(const Tensor &t) : guard(t.device()), stream(c10::cuda::getCurrentCUDAStream(t.device().index()).stream()) {}
};

// ------------------------------------------------------------------------------------------------ lambda scan
// The angle as fp32 with unit stride over D and either zero (batch, time) strides -- one angle per channel, read as such -- or
// the dense strides.
struct Angle { Tensor t; long long sb, st; };
Angle angle_view(const Tensor &ang, int64_t B, int64_t T, int64_t D) {
    Tensor a = as(ang, at::kFloat);
    if (a.dim() == 1) a = a.expand({B, T, D});
    TORCH_CHECK_VALUE(a.sizes() == at::IntArrayRef({B, T, D}), "lambda_scan: u, logmag, ang must share the shape (B,T,D)");
    if (D > 1 && a.stride(2) != 1) a = a.contiguous();
    long long sb = B > 1 ? a.stride(0) : 0, st = T > 1 ? a.stride(1) : 0;
    if (!(sb == 0 && st == 0) && !(st == D && sb == T * D)) { a = a.contiguous(); sb = T * D; st = D; }
    return {a, sb, st};
}

struct LambdaOut { Tensor y, hr, hi, hia; };
LambdaOut lambda_fwd(const Tensor &u, const Tensor &lm, const Tensor &ang, const Tensor &h0r_, const Tensor &h0i_, int segments, bool keep) {
    need_cuda(u, lm, ang, h0r_, h0i_);
    TORCH_CHECK_VALUE(u.dim() == 3 && lm.sizes() == u.sizes(), "lambda_scan: u, logmag, ang must share the shape (B,T,D)");
    const int64_t B = u.size(0), T = u.size(1), D = u.size(2);
    OnDevice dev(u);
    const Tensor u32 = f32c(u), lm32 = f32c(lm), h0r = f32c(h0r_), h0i = f32c(h0i_);
    const Angle a = angle_view(ang, B, T, D);
    LambdaOut r{alloc(u, {B, T, D}, at::kFloat), alloc(u, {B, D}, at::kFloat), alloc(u, {B, D}, at::kFloat), Tensor()};
    if (keep) {
        r.hia = alloc(u, {B, T, D}, at::kFloat);
        check(pgb_lambda_scan_fwd_train(fp(u32), fp(lm32), fp(a.t), a.sb, a.st, fp(h0r), fp(h0i), fp(r.y), fp(r.hia), fp(r.hr), fp(r.hi), B, T, D,
                                        dev.stream), "pgb_lambda_scan_fwd_train");
    } else {
        check(pgb_lambda_scan_fwd_ex(fp(u32), fp(lm32), fp(a.t), a.sb, a.st, fp(h0r), fp(h0i), fp(r.y), fp(r.hr), fp(r.hi), B, T, D, segments,
                                     dev.stream), "pgb_lambda_scan_fwd");
    }
    return r;
}
struct LambdaGrads { Tensor du, dlm, dan, d0r, d0i; };
LambdaGrads lambda_bwd(const Tensor &g_, const Tensor &u_, const Tensor &lm_, const Tensor &ang, const Tensor &hr_, const Tensor &hi_, const Tensor &gli_,
                       bool want_dh0) {
    need_cuda(g_, u_, lm_, ang, hr_, hi_);
    const int64_t B = u_.size(0), T = u_.size(1), D = u_.size(2);
    OnDevice dev(u_);
    const Tensor g = f32c(g_), u = f32c(u_), lm = f32c(lm_), hr = f32c(hr_), hi = f32c(hi_), gli = f32c(gli_);
    const Angle a = angle_view(ang, B, T, D);
    LambdaGrads r{alloc(u, {B, T, D}, at::kFloat), alloc(u, {B, T, D}, at::kFloat), alloc(u, {B, T, D}, at::kFloat), Tensor(), Tensor()};
    if (want_dh0) { r.d0r = alloc(u, {B, D}, at::kFloat); r.d0i = alloc(u, {B, D}, at::kFloat); }
    check(pgb_lambda_scan_bwd(fp(g), fp(u), fp(lm), fp(a.t), a.sb, a.st, fp(hr), fp(hi), fp(gli), fp(r.du), fp(r.dlm), fp(r.dan), fp(r.d0r), fp(r.d0i),
                              B, T, D, dev.stream), "pgb_lambda_scan_bwd");
    return r;
}

// Differentiable scan (the reference's _Scan, src/scan_kernel.py:105-140): the forward keeps Im h for the adjoint.
struct LambdaScan : torch::autograd::Function<LambdaScan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &u, const Tensor &lm, const Tensor &ang, const OptTensor &h0r, const OptTensor &h0i) {
        LambdaOut r = lambda_fwd(u, lm, ang, opt(h0r), opt(h0i), 0, true);
        ctx->save_for_backward({u, lm, ang, r.y, r.hia});
        ctx->set_materialize_grads(false);                            // no gradient arrived: undefined, not a tensor of zeros to add
        ctx->saved_data["dh0"] = h0r.has_value();
        return {r.y, r.hr, r.hi};
    }
    static variable_list backward(AutogradContext *ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();
        Tensor g = grads[0].defined() ? as(grads[0], at::kFloat) : at::zeros_like(s[3]);
        if (grads[1].defined()) {
            g = g.clone();
            g.select(1, g.size(1) - 1).add_(as(grads[1], at::kFloat));
        }
        LambdaGrads r = lambda_bwd(g, s[0], s[1], s[2], s[3], s[4], grads[2], ctx->saved_data["dh0"].toBool());
        return {r.du, r.dlm, r.dan, r.d0r, r.d0i};
    }
};

bool wants_grad(const Tensor &t) { return t.defined() && t.requires_grad(); }

// (Re h, Re h_T, Im h_T) in u's type; differentiable where a gradient is wanted
std::tuple<Tensor, Tensor, Tensor> scan(const Tensor &u, const Tensor &lm, const Tensor &ang, const OptTensor &h0r, const OptTensor &h0i) {
    const at::ScalarType dt = u.scalar_type();
    if (at::GradMode::is_enabled() && (wants_grad(u) || wants_grad(lm) || wants_grad(ang) || wants_grad(opt(h0r)) || wants_grad(opt(h0i)))) {
        need_cuda(u, lm, ang, opt(h0r), opt(h0i));
        variable_list r = LambdaScan::apply(as(u, at::kFloat), as(lm, at::kFloat), as(ang, at::kFloat), some(as(opt(h0r), at::kFloat)),
                                            some(as(opt(h0i), at::kFloat)));
        return {as(r[0], dt), as(r[1], dt), as(r[2], dt)};
    }
    LambdaOut r = lambda_fwd(u, lm, ang, opt(h0r), opt(h0i), 0, false);
    return {as(r.y, dt), as(r.hr, dt), as(r.hi, dt)};
}

// ------------------------------------------------------------------------------------------------ prep
struct PrepIn { Tensor q, k, v, gate, theta, pos; long long gsb, gst; };
PrepIn prep_in(const Tensor &qp_, const Tensor &kp_, const Tensor &vp_, const Tensor &gl_, const Tensor &theta, const Tensor &pos) {
    need_cuda(qp_, kp_, vp_, theta, pos);
    TORCH_CHECK_VALUE(qp_.dim() == 4 && kp_.sizes() == qp_.sizes() && vp_.sizes() == qp_.sizes(), "prep: qp, kp, vp must share the shape (B,T,H,D)");
    const at::ScalarType dt = io_type(qp_.scalar_type()) ? qp_.scalar_type() : at::kFloat;
    const int64_t per = std::max<int64_t>(1, qp_.size(3) / 32);       // channels a lane moves in one access: strides must keep it aligned
    auto strided = [&](Tensor t) {
        t = as(t, dt);
        const bool ok = t.stride(3) == 1 && t.stride(0) % per == 0 && t.stride(1) % per == 0 && t.stride(2) % per == 0;
        return ok ? t : t.contiguous();
    };
    PrepIn p{strided(qp_), strided(kp_), strided(vp_), as(gl_, dt), f32c(theta), as(pos, at::kLong).contiguous(), 0, 0};
    if (p.k.strides() != p.q.strides() || p.v.strides() != p.q.strides()) { p.q = p.q.contiguous(); p.k = p.k.contiguous(); p.v = p.v.contiguous(); }
    if (p.gate.defined()) {
        if (p.gate.stride(2) != 1) p.gate = p.gate.contiguous();
        p.gsb = p.gate.stride(0); p.gst = p.gate.stride(1);
    }
    return p;
}
std::tuple<Tensor, Tensor, Tensor> prep_fwd(const Tensor &qp, const Tensor &kp, const Tensor &vp_, const OptTensor &gl, const Tensor &theta, const Tensor &pos,
                                            bool out_bf16) {
    const PrepIn p = prep_in(qp, kp, vp_, opt(gl), theta, pos);
    const int64_t B = p.q.size(0), T = p.q.size(1), H = p.q.size(2), D = p.q.size(3);
    OnDevice dev(p.q);
    const at::ScalarType dt = out_bf16 ? at::kBFloat16 : at::kFloat;
    Tensor q = alloc(p.q, {B, H, T, D}, dt), k = alloc(p.q, {B, H, T, D}, dt), v = alloc(p.q, {B, H, T, D}, dt);
    check(pgb_aspin_prep_fwd(vp(p.q), vp(p.k), vp(p.v), code(p.q), p.q.stride(0), p.q.stride(1), p.q.stride(2), vp(p.gate), p.gsb, p.gst, fp(p.theta),
                             static_cast<const long long *>(vp(p.pos)), vp(q), vp(k), vp(v), code(q), B, T, H, D, dev.stream), "pgb_aspin_prep_fwd");
    return {q, k, v};
}
using PrepGrads = std::tuple<Tensor, Tensor, Tensor, OptTensor, OptTensor>;
PrepGrads prep_bwd(const Tensor &qp, const Tensor &kp, const Tensor &vp_, const OptTensor &gl, const Tensor &theta, const Tensor &pos, const Tensor &dq_,
                   const Tensor &dk_, const Tensor &dv_, bool want_theta) {
    need_cuda(dq_, dk_, dv_);
    const PrepIn p = prep_in(qp, kp, vp_, opt(gl), theta, pos);
    const int64_t B = p.q.size(0), T = p.q.size(1), H = p.q.size(2), D = p.q.size(3);
    OnDevice dev(p.q);
    const at::ScalarType gt = io_type(dq_.scalar_type()) ? dq_.scalar_type() : at::kFloat, dt = p.q.scalar_type();
    const Tensor dq = like(dq_, gt), dk = like(dk_, gt), dv = like(dv_, gt);
    Tensor dqp = alloc(p.q, {B, T, H, D}, dt), dkp = alloc(p.q, {B, T, H, D}, dt), dvp = alloc(p.q, {B, T, H, D}, dt), dgl, part;
    if (p.gate.defined()) dgl = alloc(p.q, {B, T, H}, at::kFloat);
    if (want_theta) part = alloc(p.q, {B * pgb_aspin_prep_bwd_tiles(T), H, D / 2}, at::kFloat);
    check(pgb_aspin_prep_bwd(vp(p.q), vp(p.k), vp(p.v), code(p.q), p.q.stride(0), p.q.stride(1), p.q.stride(2), vp(p.gate), p.gsb, p.gst, fp(p.theta),
                             static_cast<const long long *>(vp(p.pos)), vp(dq), vp(dk), vp(dv), code(dq), vp(dqp), vp(dkp), vp(dvp), fp(dgl), fp(part), B, T, H,
                             D, dev.stream), "pgb_aspin_prep_bwd");
    return {dqp, dkp, dvp, some(dgl), want_theta ? OptTensor(part.sum(0)) : OptTensor()};
}

// The backward kernels have no derivative of their own: with create_graph a second differentiation through `grads` raises instead of
// leaving its share out.
variable_list once(const char *what, const variable_list &saved, variable_list grads, const variable_list &incoming) {
    auto wants = [](const variable_list &l) { return std::any_of(l.begin(), l.end(), wants_grad); };
    if (!at::GradMode::is_enabled() || !(wants(saved) || wants(incoming))) return grads;
    const auto node = std::make_shared<torch::autograd::Error>(std::string("Trying to backward through the gradient of ") + what + ": it has no derivative",
                                                               torch::autograd::collect_next_edges(saved, incoming));
    for (Tensor &g : grads)
        if (g.defined()) torch::autograd::set_history(g, node);
    return grads;
}

// prep with its backward kernel
struct Prep : torch::autograd::Function<Prep> {
    static variable_list forward(AutogradContext *ctx, const Tensor &qp, const Tensor &kp, const Tensor &vp_, const OptTensor &gl, const Tensor &theta,
                                 const Tensor &pos) {
        ctx->save_for_backward({qp, kp, vp_, opt(gl), theta, pos});
        ctx->saved_data["theta"] = theta.requires_grad();
        auto [q, k, v] = prep_fwd(qp, kp, vp_, gl, theta, pos, true);
        return {q, k, v};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        auto [dq, dk, dv, dgl, dth] = prep_bwd(s[0], s[1], s[2], some(s[3]), s[4], s[5], g[0], g[1], g[2], ctx->saved_data["theta"].toBool());
        return once("pragnosia_b200 prep", s, {as(dq, s[0].scalar_type()), as(dk, s[1].scalar_type()), as(dv, s[2].scalar_type()),
                    dgl ? as(*dgl, s[3].scalar_type()) : Tensor(), dth ? as(*dth, s[4].scalar_type()) : Tensor(), Tensor()}, g);
    }
};
using Three = std::optional<std::tuple<Tensor, Tensor, Tensor>>;
// nullopt: a tracer, a torch_dispatch mode (fake tensors, make_fx, selective checkpointing), a functorch transform or a tensor subclass
// wants to see the registered operators
template <typename... P> bool plain(const P &...ts) {
    using c10::DispatchKey;
    const c10::DispatchKeySet special{DispatchKey::Python, DispatchKey::FuncTorchBatched, DispatchKey::FuncTorchGradWrapper};
    return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::tracer::impl::is_dispatch_enabled() &&
           !c10::impl::tls_is_dispatch_key_included(DispatchKey::FuncTorchDynamicLayerFrontMode) &&
           (... && (!ts.defined() || !ts.key_set().has_any(special)));
}
Three prep_diff(const Tensor &qp, const Tensor &kp, const Tensor &vp_, const OptTensor &gl, const Tensor &theta, const Tensor &pos) {
    if (!plain(qp, kp, vp_, opt(gl), theta, pos)) return std::nullopt;
    variable_list r = Prep::apply(qp, kp, vp_, gl, theta, pos);
    return std::make_tuple(r[0], r[1], r[2]);
}

// ------------------------------------------------------------------------------------------------ associative scan
// the tensor the final state is written to: a new one, or the caller's (which may be the S0 it passed: every (sequence, head)
// reads its entering state before it writes its final one)
Tensor state_out(const OptTensor &S_out, const Tensor &ref, int64_t B, int64_t H, int64_t D) {
    if (!S_out.has_value()) return alloc(ref, {B, H, D, D}, at::kFloat);
    TORCH_CHECK_VALUE(S_out->scalar_type() == at::kFloat && S_out->is_contiguous() && S_out->sizes() == at::IntArrayRef({B, H, D, D}),
                      "S_out must be a contiguous fp32 (B,H,D,D) tensor");
    return *S_out;
}
// The plain rule in fp32 with the chunks of a sequence side by side (prefill_fp32_chunk.cu), in groups whose scratch is bounded: whole
// batch rows, or some heads of one, or (a chain that is too long by itself) one chain piece by piece with its state handed on. False:
// the scratch could not be had, nothing was launched.
bool prefill_fp32_grouped(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &la, const Tensor &S0, const Tensor &theta, const Tensor &shift,
                          double shift_host, const Tensor &o, const Tensor &S, const Tensor &sent, void *stream) {
    const long long B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3), NC = (T + CHUNK - 1) / CHUNK;
    const long long chunk = pgb_aspin_prefill_fp32_scratch_bytes(1, 1, CHUNK, D), chain = pgb_aspin_prefill_fp32_scratch_bytes(1, 1, T, D);
    const long long chains = std::min(B * H, std::max(1LL, FP32_SCRATCH / chain)), piece = chain <= FP32_SCRATCH ? T : FP32_SCRATCH / chunk * CHUNK;
    const long long nb = std::max(1LL, chains / H), nh = std::min(chains, H);
    const long long n = pgb_aspin_prefill_fp32_scratch_bytes(nb, nh, std::min(piece, T), D);
    Tensor scratch;
    try {
        scratch = bytes(q, n);
    } catch (const c10::OutOfMemoryError &) {
        return false;
    }
    char *out = static_cast<char *>(vp(o));
    for (long long b = 0; b < B; b += nb)
        for (long long h = 0; h < H; h += nh)
            for (long long t = 0; t < T; t += piece) {
                const long long c = b * H + h, Bn = std::min(nb, B - b), Hn = std::min(nh, H - h), Tn = std::min(piece, T - t), row = c * T + t;
                const float *first = t > 0 ? fp(S) + c * D * D : S0.defined() ? fp(S0) + c * D * D : nullptr;
                check(pgb_aspin_prefill_fp32_fwd(fp(q) + row * D, fp(k) + row * D, fp(v) + row * D, fp(la) + row, first,
                                                 t == 0 && theta.defined() ? fp(theta) + h * (D / 2) : nullptr, fp(shift), shift_host,
                                                 out + row * D * o.element_size(), code(o), fp(S) + c * D * D,
                                                 sent.defined() ? static_cast<char *>(vp(sent)) + (c * NC + t / CHUNK) * D * D * 2 : nullptr, vp(scratch), n,
                                                 Bn, Hn, Tn, D, stream), "pgb_aspin_prefill_fp32_fwd");
            }
    return true;
}
using ScanOut = std::tuple<Tensor, Tensor, OptTensor>;
// out_type: -1 = q's (fp32 where q is neither fp32 nor bf16), else a dtype code
ScanOut prefill(const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &la_, const OptTensor &beta_, const OptTensor &S0_, const OptTensor &theta_,
                const OptTensor &shift_dev_, double shift_host, bool want_sent, int precision, int out_type, const OptTensor &S_out) {
    need_cuda(q_, k_, v_, la_, opt(shift_dev_));
    const int64_t B = q_.size(0), H = q_.size(1), T = q_.size(2), D = q_.size(3);
    OnDevice dev(q_);
    const at::ScalarType dt = io_type(q_.scalar_type()) ? q_.scalar_type() : at::kFloat;
    const Tensor q = like(q_, dt), k = like(k_, dt), v = like(v_, dt), la = f32c(la_), beta = f32c(opt(beta_)), S0 = f32c(opt(S0_)), theta = opt(theta_),
                 shift = opt(shift_dev_);
    const at::ScalarType ot = out_type < 0 ? dt : out_type == PGB_F32 ? at::kFloat : at::kBFloat16;
    Tensor o = alloc(q, {B, H, T, D}, ot), S = state_out(S_out, q, B, H, D), sent;
    if (want_sent) sent = alloc(q, {B, H, (T + CHUNK - 1) / CHUNK, D, D}, at::kBFloat16);
    const int oc = code(o);
    if (beta.defined() && dt == at::kBFloat16 && precision != PGB_PREFILL_FP32 && B * H <= 65535) {
        // delta rule on the tensor cores: the chunk inverses go through a scratch buffer
        long long n = want_sent ? pgb_aspin_delta_scratch_bytes(B, H, T) : pgb_aspin_delta_prefill_scratch_bytes(B, H, T, D);
        Tensor scratch;
        try {
            scratch = bytes(q, n);
        } catch (const c10::OutOfMemoryError &) {                     // without the segments' share, then
            const long long least = pgb_aspin_delta_scratch_bytes(B, H, T);
            if (n == least) throw;
            scratch = bytes(q, n = least);
        }
        check(pgb_aspin_delta_prefill_fwd(vp(q), vp(k), vp(v), fp(la), fp(beta), fp(S0), fp(theta), fp(shift), shift_host, vp(o), oc, fp(S), vp(sent),
                                          vp(scratch), n, B, H, T, D, dev.stream), "pgb_aspin_delta_prefill_fwd");
        return {o, S, some(sent)};
    }
    if (!beta.defined() && dt == at::kBFloat16 && precision != PGB_PREFILL_FP32 && D == 64 && !(S0.defined() && S0.is_same_size(S) && S0.data_ptr() == S.data_ptr())) {
        const long long n = pgb_aspin_prefill_segments_scratch_bytes(B, H, T, D); // few long chains, or few in the last round: their segments side by side
        if (n > 0) {
            const Tensor scratch = bytes(q, n);
            check(pgb_aspin_prefill_segments_fwd(vp(q), vp(k), vp(v), fp(la), fp(S0), fp(theta), fp(shift), shift_host, vp(o), oc, fp(S), vp(sent),
                                                 vp(scratch), n, B, H, T, D, dev.stream), "pgb_aspin_prefill_segments_fwd");
            return {o, S, some(sent)};
        }
    }
    // fp32 plain rule: the chunks side by side, also where the chains alone fill the GPU (1024 chains of 8 chunks: 616 us against the
    // walk's 776; 24 of 64: 134 against 1258). A single chunk a chain at D = 64 is the walk's: 96 .. 1024 chains 31 .. 121 us against 32 .. 130.
    if (!beta.defined() && dt == at::kFloat && precision != PGB_PREFILL_TENSOR && B > 0 && H > 0 && T > 0 && B * H <= 65535 && (D == 64 || D == 128) &&
        !(D == 64 && T <= CHUNK && 2 * B * H > at::cuda::getCurrentDeviceProperties()->multiProcessorCount) &&
        prefill_fp32_grouped(q, k, v, la, S0, theta, shift, shift_host, o, S, sent, dev.stream))
        return {o, S, some(sent)};
    check(pgb_aspin_prefill_fwd(vp(q), vp(k), vp(v), code(q), fp(la), fp(beta), fp(S0), fp(theta), fp(shift), shift_host, vp(o), oc, fp(S), vp(sent), B, H, T,
                                D, precision, dev.stream), "pgb_aspin_prefill_fwd");
    return {o, S, some(sent)};
}

// The scan with what its backward reads: (o, S, sent, W, X); bf16 q, k, v, fp32 la, beta, all contiguous; W and X with the delta rule.
struct TrainOut { Tensor o, S, sent, W, X; };
TrainOut train_fwd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &la, const Tensor &beta, const Tensor &S0) {
    need_cuda(q, k, v, la, beta, S0);
    const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
    OnDevice dev(q);
    if (!beta.defined()) {
        const long long n = pgb_aspin_prefill_segments_scratch_bytes(B, H, T, D);
        TrainOut r{alloc(q, {B, H, T, D}, at::kBFloat16), alloc(q, {B, H, D, D}, at::kFloat), alloc(q, {B, H, (T + CHUNK - 1) / CHUNK, D, D}, at::kBFloat16),
                   Tensor(), Tensor()};
        const Tensor scratch = n > 0 ? bytes(q, n) : Tensor();
        check(pgb_aspin_prefill_train_fwd(vp(q), vp(k), vp(v), fp(la), fp(S0), vp(r.o), fp(r.S), vp(r.sent), vp(scratch), n, B, H, T, D, dev.stream),
              "pgb_aspin_prefill_train_fwd");
        return r;
    }
    const long long n = pgb_aspin_delta_scratch_bytes(B, H, T);
    TrainOut r{alloc(q, {B, H, T, D}, at::kBFloat16), alloc(q, {B, H, D, D}, at::kFloat), alloc(q, {B, H, (T + CHUNK - 1) / CHUNK, D, D}, at::kBFloat16),
               alloc(q, {B, H, T, D}, at::kBFloat16), bytes(q, n)};
    check(pgb_aspin_delta_prefill_train_fwd(vp(q), vp(k), vp(v), fp(la), fp(beta), fp(S0), vp(r.o), fp(r.S), vp(r.sent), vp(r.W), vp(r.X), n, B, H, T, D,
                                            dev.stream), "pgb_aspin_delta_prefill_train_fwd");
    return r;
}
struct TrainGrads { Tensor dq, dk, dv, dla, dbe, dS0; };
TrainGrads train_bwd(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &la, const Tensor &beta, const Tensor &sent, const Tensor &W, const Tensor &X,
                     const Tensor &dout_, const Tensor &dsent_, const Tensor &dS_, bool want_dS0) {
    need_cuda(q, k, v, la, beta, sent, dout_);
    const int64_t B = q.size(0), H = q.size(1), T = q.size(2), D = q.size(3);
    OnDevice dev(q);
    const Tensor dout = like(dout_, at::kBFloat16), dsent = f32c(dsent_), dS = f32c(dS_);
    TrainGrads r{alloc(q, {B, H, T, D}, at::kBFloat16), alloc(q, {B, H, T, D}, at::kBFloat16), alloc(q, {B, H, T, D}, at::kBFloat16),
                 alloc(q, {B, H, T}, at::kFloat), Tensor(), Tensor()};
    if (beta.defined()) r.dbe = alloc(q, {B, H, T}, at::kFloat);
    if (want_dS0) r.dS0 = alloc(q, {B, H, D, D}, at::kFloat);
    const long long n = pgb_aspin_train_scratch_bytes(B, H, T, D, beta.defined());
    const Tensor scratch = bytes(q, n);
    check(pgb_aspin_train_bwd(vp(q), vp(k), vp(v), fp(la), fp(beta), vp(sent), vp(W), vp(X), vp(dout), fp(dsent), fp(dS), vp(r.dq), vp(r.dk), vp(r.dv),
                              fp(r.dla), fp(r.dbe), fp(r.dS0), vp(scratch), n, B, H, T, D, dev.stream), "pgb_aspin_train_bwd");
    return r;
}

// The scan of bf16 operands with all its gradients as one library call each way (train_chunk.cu): (o, final state, state entering
// each chunk), each of them differentiable. No beta: the plain rule.
struct Scan : torch::autograd::Function<Scan> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q_, const Tensor &k_, const Tensor &v_, const Tensor &la, const OptTensor &beta,
                                 const OptTensor &S0) {
        const Tensor q = q_.contiguous(), k = k_.contiguous(), v = v_.contiguous(), la32 = f32c(la), be32 = f32c(opt(beta));
        TrainOut r = train_fwd(q, k, v, la32, be32, f32c(opt(S0)));
        ctx->save_for_backward({q, k, v, la32, be32, r.sent, r.W, r.X});
        ctx->set_materialize_grads(false);
        auto &d = ctx->saved_data;
        d["la"] = static_cast<int64_t>(la.scalar_type());
        if (beta) d["beta"] = static_cast<int64_t>(beta->scalar_type());
        if (S0) d["S0"] = static_cast<int64_t>(S0->scalar_type());
        d["dS0"] = S0.has_value() && S0->requires_grad();
        return {r.o, r.S, r.sent};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        const variable_list s = ctx->get_saved_variables();
        auto &d = ctx->saved_data;
        auto type = [&](const char *n) { return static_cast<at::ScalarType>(d[n].toInt()); };
        TrainGrads r = train_bwd(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], g[0].defined() ? g[0] : at::zeros_like(s[0]), g[2], g[1], d["dS0"].toBool());
        return once("pragnosia_b200 scan", s, {r.dq, r.dk, r.dv, as(r.dla, type("la")), r.dbe.defined() ? as(r.dbe, type("beta")) : Tensor(),
                    r.dS0.defined() ? as(r.dS0, type("S0")) : Tensor()}, g);
    }
};
Three scan_diff(const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &la, const OptTensor &beta, const OptTensor &S0) {
    if (!plain(q, k, v, la, opt(beta), opt(S0))) return std::nullopt;
    variable_list r = Scan::apply(q, k, v, la, beta, S0);
    return std::make_tuple(r[0], r[1], r[2]);
}

// ------------------------------------------------------------------------------------------------ losses over the vocabulary
enum { REDUCE_NONE = 0, REDUCE_SUM = 1, REDUCE_MEAN = 2 };
constexpr int64_t MOST_WORDS = 1 << 30;                               // the entry points' V is an int
const char *const XENT = "linear_cross_entropy", *const DISTILL = "linear_distill", *const EMBED = "embedding";
void same_device(const char *what, const Tensor &a, const Tensor &b) {
    TORCH_CHECK_VALUE(a.device() == b.device(), what, ": its tensors are on ", a.device(), " and ", b.device());
}
Tensor whole_numbers(const char *what, const Tensor &t) {
    TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, what, ": ids are int64 or int32, got ", t.scalar_type());
    return like(t, at::kLong);
}
// h as [N][d], W as it is: both contiguous, of one of the two types, 16-byte aligned (a view into a larger tensor need not be)
struct HeadIn { Tensor h, w; int64_t N, V, d; };
Tensor head_operand(const Tensor &t) {
    const Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
HeadIn head_in(const char *what, const Tensor &h, const Tensor &w) {
    need_cuda(h, w);
    same_device(what, h, w);
    TORCH_CHECK_VALUE(w.dim() == 2 && h.dim() >= 1 && h.size(-1) == w.size(1), what, ": h is (..., d) and the weight (V, d), got ", h.sizes(), " and ", w.sizes());
    TORCH_CHECK_TYPE(h.scalar_type() == w.scalar_type() && io_type(h.scalar_type()), what, ": h and the weight are both float32 or both bfloat16, got ",
                     h.scalar_type(), " and ", w.scalar_type());
    const int64_t d = w.size(1);
    TORCH_CHECK_VALUE(w.size(0) >= 1 && w.size(0) <= MOST_WORDS && d >= 8 && d <= 65536 && d % 8 == 0, what,
                      ": the weight is (V, d) with V from 1 to 2^30 and d a multiple of 8 up to 65536, got ", w.sizes());
    return {head_operand(h.dim() == 2 ? h : h.reshape({-1, d})), head_operand(w), h.numel() / d, w.size(0), d};
}
// What a row is held to: a word each (target), or a teacher's entries (lists, marks, ent; kept: their logits).
struct HeadWant { Tensor target; int64_t ignore; Tensor lists, marks, ent, kept; double tau; };
struct HeadOut { Tensor loss, L, stats; };                            // loss: [N] or 0-d; stats: rows that count, whether one that does not is no number
// keep: for a gradient. Without one, L and stats lie behind the scratch: few rows are scored in the time of this call (11.4 us with two allocations more, 8.9 now).
HeadOut head_fwd(const char *what, const HeadIn &x, const HeadWant &t, int reduction, bool keep = true) {
    OnDevice dev(x.h);
    HeadOut r{alloc(x.h, reduction == REDUCE_NONE ? at::IntArrayRef({x.N}) : at::IntArrayRef(), at::kFloat)};
    if (keep) { r.L = alloc(x.h, {x.N, 2}, at::kFloat); r.stats = alloc(x.h, {2}, at::kFloat); }
    if (x.N == 0) {                                                    // nothing to add up: 0, and 0 / 0 as the mean
        if (reduction == REDUCE_SUM) r.loss.zero_();
        if (reduction == REDUCE_MEAN) r.loss.fill_(std::numeric_limits<float>::quiet_NaN());
        if (keep) r.stats.zero_();
        return r;
    }
    const bool list = t.lists.defined();
    const int k = list ? t.lists.size(1) : 0;
    const long long n = pgb_head_loss_fwd_scratch_bytes(x.N, x.V, x.d, code(x.h));
    const long long behind = (n + 255) / 256 * 256;
    const Tensor scratch = bytes(x.h, keep ? n : behind + 8 * (x.N + 1));
    float *const L = keep ? fp(r.L) : reinterpret_cast<float *>(static_cast<char *>(vp(scratch)) + behind), *const stats = keep ? fp(r.stats) : L + 2 * x.N;
    float *row = reduction == REDUCE_NONE ? fp(r.loss) : nullptr, *loss = reduction == REDUCE_NONE ? nullptr : fp(r.loss);
    if (list)
        check(pgb_linear_distill_fwd(vp(x.h), vp(x.w), code(x.h), static_cast<int *>(vp(t.lists)), static_cast<unsigned *>(vp(t.marks)), fp(t.ent), fp(t.kept), k, t.tau, row, loss, stats, L,
                                     vp(scratch), n, reduction, x.N, x.V, x.d, dev.stream), what);
    else
        check(pgb_linear_xent_fwd(vp(x.h), vp(x.w), code(x.h), static_cast<long long *>(vp(t.target)), t.ignore, row, loss, stats, L, vp(scratch),
                                  n, reduction, x.N, x.V, x.d, dev.stream), what);
    return r;
}
// what the forward pass left, as a registered operator's caller hands it over
void head_state(const char *what, const HeadIn &x, const Tensor &t, at::IntArrayRef sizes, at::ScalarType type) {
    TORCH_CHECK_VALUE(t.device() == x.h.device() && t.scalar_type() == type && t.sizes() == sizes && t.is_contiguous(), what, ": a tensor of the forward pass is ", type,
                      sizes, ", contiguous, got ", t.scalar_type(), t.sizes(), " on ", t.device());
}
void head_state(const char *what, const HeadIn &x, const Tensor &L, const Tensor &stats, const Tensor &grad, int reduction) {
    head_state(what, x, L, {x.N, 2}, at::kFloat);
    head_state(what, x, stats, {2}, at::kFloat);
    TORCH_CHECK_VALUE(grad.device() == x.h.device() && grad.numel() == (reduction == REDUCE_NONE ? x.N : 1), what, ": a gradient per loss, got ", grad.sizes());
}
void head_lists(const HeadIn &x, const Tensor &lists, const Tensor &ent) {
    TORCH_CHECK_VALUE(lists.dim() == 3 && lists.size(1) >= 1, DISTILL, ": lists are (N, k, 2), got ", lists.sizes());
    head_state(DISTILL, x, lists, {x.N, lists.size(1), 2}, at::kInt);
    head_state(DISTILL, x, ent, {x.N}, at::kFloat);
}
std::tuple<Tensor, Tensor> head_bwd(const char *what, const HeadIn &x, const HeadWant &t, const Tensor &L, const Tensor &stats, const Tensor &grad_, int reduction,
                                    bool want_dh, bool want_dw) {
    OnDevice dev(x.h);
    Tensor dh, dw;
    if (want_dh) dh = alloc(x.h, {x.N, x.d}, x.h.scalar_type());
    if (want_dw) dw = alloc(x.h, {x.V, x.d}, x.h.scalar_type());
    if (x.N == 0) {
        if (want_dw) dw.zero_();
        return {dh, dw};
    }
    const Tensor grad = f32c(grad_);
    const long long n = pgb_head_loss_bwd_scratch_bytes(x.N, x.V, x.d, code(x.h), want_dh, want_dw);
    const Tensor scratch = bytes(x.h, n);
    if (t.lists.defined())
        check(pgb_linear_distill_bwd(vp(x.h), vp(x.w), code(x.h), static_cast<int *>(vp(t.lists)), fp(t.ent), fp(t.kept), t.lists.size(1), t.tau, fp(L), fp(stats),
                                     fp(grad), vp(dh), vp(dw), vp(scratch), n, reduction, x.N, x.V, x.d, dev.stream), what);
    else
        check(pgb_linear_xent_bwd(vp(x.h), vp(x.w), code(x.h), static_cast<long long *>(vp(t.target)), t.ignore, fp(L), fp(stats), fp(grad), vp(dh), vp(dw),
                                  vp(scratch), n, reduction, x.N, x.V, x.d, dev.stream), what);
    return {dh, dw};
}
HeadWant xent_want(const HeadIn &x, const Tensor &h, const Tensor &target, int64_t ignore) {
    need_cuda(target);
    same_device(XENT, h, target);
    TORCH_CHECK_VALUE(target.sizes() == h.sizes().slice(0, h.dim() - 1), XENT, ": a target per row of h, got ", target.sizes(), " for ", h.sizes());
    const Tensor t = whole_numbers(XENT, target);
    return {t.dim() == 1 ? t : t.reshape({x.N}), ignore, Tensor(), Tensor(), Tensor(), Tensor(), 1.0};
}
std::tuple<Tensor, Tensor, Tensor> teacher_lists(const Tensor &ids_, const Tensor &logits_, double tau, int64_t V) {
    need_cuda(ids_, logits_);
    same_device(DISTILL, ids_, logits_);
    TORCH_CHECK_VALUE(ids_.dim() >= 1 && ids_.sizes() == logits_.sizes(), DISTILL, ": a teacher's ids and logits share their shape, got ", ids_.sizes(), " and ",
                      logits_.sizes());
    TORCH_CHECK_VALUE(tau >= 1e-37 && tau <= 3e38, DISTILL, ": the temperature is positive (1e-37 to 3e38), got ", tau);
    const int64_t k = ids_.size(-1);
    TORCH_CHECK_VALUE(V >= 1 && V <= MOST_WORDS, DISTILL, ": 1 to 2^30 words, got ", V);
    TORCH_CHECK_VALUE(k >= 1 && k <= 1024, DISTILL, ": 1 to 1024 teacher entries a row, got ", k);
    const int64_t N = ids_.numel() / k;
    OnDevice dev(ids_);
    const Tensor ids = whole_numbers(DISTILL, ids_).reshape({N, k}), logits = f32c(logits_).reshape({N, k});
    Tensor lists = alloc(ids, {N, k, 2}, at::kInt), marks = alloc(ids, {N, (V + 63) / 64, 4}, at::kInt), ent = alloc(ids, {N}, at::kFloat);
    if (N > 0)
        check(pgb_teacher_lists(static_cast<long long *>(vp(ids)), fp(logits), tau, static_cast<int *>(vp(lists)), static_cast<unsigned *>(vp(marks)), fp(ent), N, V,
                                k, dev.stream), "pgb_teacher_lists");
    return {lists, marks, ent};
}
HeadWant distill_want(const HeadIn &x, const Tensor &h, const Tensor &ids, const Tensor &logits, double tau) {
    same_device(DISTILL, h, ids);
    TORCH_CHECK_VALUE(ids.dim() == h.dim() && ids.sizes().slice(0, ids.dim() - 1) == h.sizes().slice(0, h.dim() - 1), DISTILL, ": k teacher entries per row of h, got ",
                      ids.sizes(), " for ", h.sizes());
    auto [lists, marks, ent] = teacher_lists(ids, logits, tau, x.V);
    return {Tensor(), 0, lists, marks, ent, alloc(x.h, {x.N, lists.size(1)}, at::kFloat), tau};
}

// Either loss with its gradients: what the backward pass reads is h, W, the targets and two numbers a row.
struct HeadLoss : torch::autograd::Function<HeadLoss> {
    static variable_list forward(AutogradContext *ctx, const Tensor &h_, const Tensor &w_, const OptTensor &target, int64_t ignore, const OptTensor &ids,
                                 const OptTensor &logits, double tau, int64_t reduction) {
        const char *what = target ? XENT : DISTILL;
        const HeadIn x = head_in(what, h_, w_);
        const HeadWant t = target ? xent_want(x, h_, *target, ignore) : distill_want(x, h_, *ids, *logits, tau);
        HeadOut r = head_fwd(what, x, t, reduction);
        ctx->save_for_backward({x.h, x.w, t.target, t.lists, t.ent, t.kept, r.L, r.stats});    // not marks: N V / 4 bytes that only the forward pass reads
        auto &d = ctx->saved_data;
        d["ignore"] = ignore; d["tau"] = tau; d["reduction"] = reduction; d["shape"] = h_.sizes().vec();
        ctx->set_materialize_grads(false);
        if (reduction != REDUCE_NONE) return {r.loss};
        return {r.loss.view(h_.sizes().slice(0, h_.dim() - 1))};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        variable_list none(8);
        if (!g[0].defined()) return none;
        const variable_list s = ctx->get_saved_variables();
        auto &d = ctx->saved_data;
        const HeadIn x{s[0], s[1], s[0].size(0), s[1].size(0), s[1].size(1)};
        const HeadWant t{s[2], d["ignore"].toInt(), s[3], Tensor(), s[4], s[5], d["tau"].toDouble()};
        const bool list = t.lists.defined();
        auto [dh, dw] = head_bwd(list ? DISTILL : XENT, x, t, s[6], s[7], g[0].reshape({-1}), d["reduction"].toInt(), ctx->needs_input_grad(0), ctx->needs_input_grad(1));
        none[0] = dh.defined() ? dh.view(d["shape"].toIntVector()) : dh;
        none[1] = dw;
        return once(list ? "pragnosia_b200 linear_distill" : "pragnosia_b200 linear_cross_entropy", s, none, g);
    }
};
// A backward pass captured into a graph hands its gradient to the leaf's accumulation node on the stream that node was made on. One that
// lives on from an eager pass of another stream is outside of the capture, and torch ends the process: refused here, before anything is launched.
void capture_alone(const char *what, const Tensor &leaf) {
    if (!wants_grad(leaf) || !leaf.is_leaf() || !leaf.is_cuda()) return;
    const c10::cuda::CUDAStream here = c10::cuda::getCurrentCUDAStream(leaf.device().index());
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(here.stream(), &status) != cudaSuccess || status == cudaStreamCaptureStatusNone) return;
    const std::shared_ptr<torch::autograd::Node> node = torch::autograd::impl::try_get_grad_accumulator(leaf);
    const std::optional<c10::Stream> made = node ? node->stream() : std::nullopt;
    if (made && *made != here.unwrap())
        throw std::runtime_error(std::string(what) + ": a backward pass of this weight or input from another stream is still alive (its loss is referenced), which a "
                                 "capture cannot take in: drop it before capturing, or capture on the stream it ran on");
}
// nullopt: something wants to see the registered operators (see plain)
OptTensor linear_xent(const Tensor &h, const Tensor &w, const Tensor &target, int64_t ignore, int64_t reduction) {
    if (!plain(h, w, target)) return std::nullopt;
    if (at::GradMode::is_enabled() && (wants_grad(h) || wants_grad(w))) {
        capture_alone(XENT, h); capture_alone(XENT, w);
        return HeadLoss::apply(h, w, OptTensor(target), ignore, OptTensor(), OptTensor(), 1.0, reduction)[0];
    }
    const HeadIn x = head_in(XENT, h, w);
    const Tensor loss = head_fwd(XENT, x, xent_want(x, h, target, ignore), reduction, false).loss;
    return reduction == REDUCE_NONE ? loss.view(target.sizes()) : loss;
}
OptTensor linear_distill(const Tensor &h, const Tensor &w, const Tensor &ids, const Tensor &logits, double tau, int64_t reduction) {
    if (!plain(h, w, ids, logits)) return std::nullopt;
    if (at::GradMode::is_enabled() && (wants_grad(h) || wants_grad(w))) {
        capture_alone(DISTILL, h); capture_alone(DISTILL, w);
        return HeadLoss::apply(h, w, OptTensor(), 0, OptTensor(ids), OptTensor(logits.detach()), tau, reduction)[0];
    }
    const HeadIn x = head_in(DISTILL, h, w);
    const Tensor loss = head_fwd(DISTILL, x, distill_want(x, h, ids, logits, tau), reduction, false).loss;
    return reduction == REDUCE_NONE ? loss.view(h.sizes().slice(0, h.dim() - 1)) : loss;
}

// ------------------------------------------------------------------------------------------------ embedding
Tensor embed_weight(const Tensor &w) {
    TORCH_CHECK_TYPE(io_type(w.scalar_type()), EMBED, ": the weight is float32 or bfloat16, got ", w.scalar_type());
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(0) >= 1 && w.size(0) <= MOST_WORDS && w.size(1) >= 1 && w.size(1) <= 65536, EMBED,
                      ": the weight is (V, d), V up to 2^30 and d up to 65536, got ", w.sizes());
    return w.contiguous();
}
Tensor embed_fwd(const Tensor &ids_, const Tensor &w_, double scale) {
    need_cuda(ids_, w_);
    same_device(EMBED, ids_, w_);
    OnDevice dev(w_);
    const Tensor w = embed_weight(w_), ids = whole_numbers(EMBED, ids_);
    std::vector<int64_t> shape = ids_.sizes().vec();
    shape.push_back(w.size(1));
    Tensor y = alloc(w, shape, w.scalar_type());
    if (ids.numel() > 0)
        check(pgb_embedding_fwd(static_cast<long long *>(vp(ids)), vp(w), code(w), scale, vp(y), ids.numel(), w.size(0), w.size(1), dev.stream),
              "pgb_embedding_fwd");
    return y;
}
Tensor embed_bwd(const Tensor &ids_, const Tensor &g_, double scale, int64_t padding, int64_t V) {
    need_cuda(ids_, g_);
    same_device(EMBED, ids_, g_);
    OnDevice dev(g_);
    TORCH_CHECK_TYPE(io_type(g_.scalar_type()), EMBED, ": the gradient is float32 or bfloat16, got ", g_.scalar_type());
    const Tensor g = g_.contiguous(), ids = whole_numbers(EMBED, ids_);
    const int64_t d = g.size(-1), N = ids.numel();
    TORCH_CHECK_VALUE(g.numel() == N * d && d >= 1 && d <= 65536 && V >= 1 && V <= MOST_WORDS, EMBED, ": a row of gradient per id, got ", g.sizes(), " for ", ids.sizes());
    Tensor dw = alloc(g, {V, d}, g.scalar_type());
    if (N == 0) return dw.zero_();
    const long long n = pgb_embedding_bwd_scratch_bytes(N, V, d);
    const Tensor scratch = n > 0 ? bytes(g, n) : Tensor();
    check(pgb_embedding_bwd(static_cast<long long *>(vp(ids)), vp(g), code(g), scale, padding, vp(dw), vp(scratch), n, N, V, d, dev.stream), "pgb_embedding_bwd");
    return dw;
}
struct Embed : torch::autograd::Function<Embed> {
    static variable_list forward(AutogradContext *ctx, const Tensor &ids, const Tensor &w, double scale, int64_t padding) {
        ctx->save_for_backward({ids});
        auto &d = ctx->saved_data;
        d["scale"] = scale; d["padding"] = padding; d["V"] = w.size(0);
        ctx->set_materialize_grads(false);
        return {embed_fwd(ids, w, scale)};
    }
    static variable_list backward(AutogradContext *ctx, variable_list g) {
        if (!g[0].defined()) return variable_list(4);
        const variable_list s = ctx->get_saved_variables();
        auto &d = ctx->saved_data;
        return once("pragnosia_b200 embedding", s, {Tensor(), embed_bwd(s[0], g[0], d["scale"].toDouble(), d["padding"].toInt(), d["V"].toInt()), Tensor(), Tensor()}, g);
    }
};
OptTensor embedding(const Tensor &ids, const Tensor &w, double scale, int64_t padding) {
    if (!plain(ids, w)) return std::nullopt;
    if (at::GradMode::is_enabled() && wants_grad(w)) {
        need_cuda(ids, w);
        embed_weight(w);
        capture_alone(EMBED, w);
        return Embed::apply(ids, w, scale, padding)[0];
    }
    return embed_fwd(ids, w, scale);
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    using nogil_t = pybind11::call_guard<pybind11::gil_scoped_release>;             // as a ctypes call would: other threads run meanwhile
    const nogil_t nogil;
    m.def("lambda_scan", [](const Tensor &u, const Tensor &lm, const Tensor &ang, const OptTensor &h0r, const OptTensor &h0i, int segments, bool keep) {
        LambdaOut r = lambda_fwd(u, lm, ang, opt(h0r), opt(h0i), segments, keep);
        return std::make_tuple(r.y, r.hr, r.hi, some(r.hia));
    }, nogil);
    m.def("lambda_scan_bwd", [](const Tensor &g, const Tensor &u, const Tensor &lm, const Tensor &ang, const Tensor &hr, const Tensor &hi, const OptTensor &gli,
                                bool want_dh0) {
        LambdaGrads r = lambda_bwd(g, u, lm, ang, hr, hi, opt(gli), want_dh0);
        return std::make_tuple(r.du, r.dlm, r.dan, some(r.d0r), some(r.d0i));
    }, nogil);
    m.def("scan", &scan, nogil);
    m.def("prep", &prep_fwd, nogil);
    m.def("prep_bwd", &prep_bwd, nogil);
    m.def("prep_diff", &prep_diff, nogil);
    m.def("prefill", &prefill, nogil);
    m.def("scan_train_fwd", [](const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &la, const OptTensor &beta, const OptTensor &S0) {
        TrainOut r = train_fwd(q, k, v, la, opt(beta), opt(S0));
        return std::make_tuple(r.o, r.S, r.sent, some(r.W), some(r.X));
    }, nogil);
    m.def("scan_train_bwd", [](const Tensor &q, const Tensor &k, const Tensor &v, const Tensor &la, const OptTensor &beta, const Tensor &sent, const OptTensor &W,
                               const OptTensor &X, const Tensor &dout, const OptTensor &dsent, const OptTensor &dS, bool want_dS0) {
        TrainGrads r = train_bwd(q, k, v, la, opt(beta), sent, opt(W), opt(X), dout, opt(dsent), opt(dS), want_dS0);
        return std::make_tuple(r.dq, r.dk, r.dv, r.dla, some(r.dbe), some(r.dS0));
    }, nogil);
    m.def("scan_diff", &scan_diff, nogil);
    m.def("capture_alone", [](const std::string &what, const Tensor &leaf) { capture_alone(what.c_str(), leaf); }, nogil);
    m.def("linear_xent", &linear_xent, nogil);
    m.def("linear_xent_fwd", [](const Tensor &h, const Tensor &w, const Tensor &target, int64_t ignore, int reduction) {
        const HeadIn x = head_in(XENT, h, w);
        HeadOut r = head_fwd(XENT, x, xent_want(x, h, target, ignore), reduction);
        return std::make_tuple(r.loss, r.L, r.stats);
    }, nogil);
    m.def("linear_xent_bwd", [](const Tensor &h, const Tensor &w, const Tensor &target, int64_t ignore, const Tensor &L, const Tensor &stats, const Tensor &grad,
                                int reduction, bool want_dh, bool want_dw) {
        const HeadIn x = head_in(XENT, h, w);
        head_state(XENT, x, L, stats, grad, reduction);
        auto [dh, dw] = head_bwd(XENT, x, xent_want(x, h, target, ignore), L, stats, grad, reduction, want_dh, want_dw);
        return std::make_tuple(some(dh), some(dw));
    }, nogil);
    m.def("teacher_lists", &teacher_lists, nogil);
    m.def("linear_distill", &linear_distill, nogil);
    m.def("linear_distill_fwd", [](const Tensor &h, const Tensor &w, const Tensor &lists, const Tensor &marks, const Tensor &ent, double tau, int reduction) {
        const HeadIn x = head_in(DISTILL, h, w);
        head_lists(x, lists, ent);
        head_state(DISTILL, x, marks, {x.N, (x.V + 63) / 64, 4}, at::kInt);
        const Tensor kept = alloc(x.h, {x.N, lists.size(1)}, at::kFloat);
        HeadOut r = head_fwd(DISTILL, x, {Tensor(), 0, lists, marks, ent, kept, tau}, reduction);
        return std::make_tuple(r.loss, r.L, r.stats, kept);
    }, nogil);
    m.def("linear_distill_bwd", [](const Tensor &h, const Tensor &w, const Tensor &lists, const Tensor &ent, const Tensor &kept, double tau,
                                   const Tensor &L, const Tensor &stats, const Tensor &grad, int reduction, bool want_dh, bool want_dw) {
        const HeadIn x = head_in(DISTILL, h, w);
        head_lists(x, lists, ent);
        head_state(DISTILL, x, kept, {x.N, lists.size(1)}, at::kFloat);
        head_state(DISTILL, x, L, stats, grad, reduction);
        auto [dh, dw] = head_bwd(DISTILL, x, {Tensor(), 0, lists, Tensor(), ent, kept, tau}, L, stats, grad, reduction, want_dh, want_dw);
        return std::make_tuple(some(dh), some(dw));
    }, nogil);
    m.def("embedding", &embedding, nogil);
    m.def("embedding_fwd", &embed_fwd, nogil);
    m.def("embedding_bwd", &embed_bwd, nogil);
}

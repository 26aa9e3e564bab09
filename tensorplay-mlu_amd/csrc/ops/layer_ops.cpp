// What stands between a language model's matrix products: dropout whose mask
// is never stored (kernels/seeded_dropout.hip), the join of a block to its
// residual stream with the norms on both sides of it
// (kernels/residual_norm.hip), and the log probabilities of given tokens
// (kernels/token_log_probs.hip), forward and backward.  The reference has no
// counterpart; entries follow the attention layer's conventions: device float
// tensors of one dtype or the call is declined, shapes that contradict each
// other are errors, operands are read where they lie and copied only when the
// kernels cannot address them.

#include <algorithm>
#include <cmath>

#include "../kernels/layers.h"
#include "entries.h"
#include "tp_amd_ops.h"

using namespace tp_amd;

namespace {

// ---- dropout ------------------------------------------------------------------

// Checks p and the seed; the threshold and scale of 0 < p < 1.
DropArgs drop_args(const char* op, double p, uint64_t seed, const tp_amd_tensor* seed_tensor, uint64_t offset, int device) {
    TP_AMD_CHECK(p >= 0.0 && p <= 1.0, op, ": p has to lie between 0 and 1");
    DropArgs d{seed, nullptr, offset, keep_threshold(p), p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0f};
    if (seed_tensor != nullptr) {
        check_view(*seed_tensor, "seed");
        if (!on_device(*seed_tensor) || seed_tensor->device != device || seed_tensor->dtype != TP_AMD_INT64) {
            TP_AMD_DECLINE("a seed in memory is one int64 on the operands' device");
        }
        TP_AMD_CHECK(numel(*seed_tensor) == 1, op, ": a seed in memory is one number, not ", numel(*seed_tensor));
        d.seed_at = static_cast<const int64_t*>(seed_tensor->data);
    }
    return d;
}

int dropout(const char* op, const tp_amd_tensor* input, double p, uint64_t seed, const tp_amd_tensor* seed_tensor, uint64_t offset,
            tp_amd_tensor* result) {
    return guarded_result(result, [&] {
        const TensorRef& in = deref(input, "input");
        check_view(in, "input");
        if (!on_device(in) || !is_native_float(in.dtype)) TP_AMD_DECLINE("seeded_dropout runs on the device for float tensors");
        const DropArgs drop = drop_args(op, p, seed, seed_tensor, offset, in.device);
        const MaybeOwned x = contiguous_on_device(in);
        Owned out = empty_on(sizes_of(in), in.dtype, in.device);
        launch_seeded_dropout(in.dtype, numel(in), x.ref.data, drop, out.ref().data, in.device);
        return out;
    });
}

// ---- the join of a block to its residual stream ------------------------------------

// [tokens..., D] as rows: copied when its token axes do not merge or its last
// axis is not dense.
Rows rows_of(const TensorRef& t, MaybeOwned& hold) {
    auto in_place = [](const TensorRef& x, Rows& r) {
        r.data = x.data;
        return (x.sizes[x.ndim - 1] == 1 || x.strides[x.ndim - 1] == 1) && axes_merge(x, x.ndim - 1, r.step);
    };
    Rows r{};
    if (in_place(t, r)) return r;
    hold = contiguous_on_device(t);
    TP_AMD_CHECK(in_place(hold.ref, r), "internal: a dense copy that is no rows");
    return r;
}

int64_t rows_in(const TensorRef& t) {
    int64_t n = 1;
    for (int d = 0; d + 1 < t.ndim; ++d) n *= t.sizes[d];
    return n;
}

Sizes token_shape(const TensorRef& t) { return Sizes(t.sizes, t.sizes + t.ndim - 1); }

// What forward and backward share: checks and the arguments they make.
struct ResidualNorm {
    ResidualNormArgs args{};
    MaybeOwned hold_x, hold_y, hold_gate, hold_w[2];

    ResidualNorm(const TensorRef& x, const tp_amd_tensor* y, const tp_amd_tensor* gate, const tp_amd_tensor* w1, const tp_amd_tensor* w2,
                 bool norm1, bool norm2, double a, double b, double p, uint64_t seed, const tp_amd_tensor* seed_tensor, uint64_t offset) {
        check_view(x, "residual");
        if (!on_device(x) || !is_native_float(x.dtype) || x.ndim < 1) {
            TP_AMD_DECLINE("residual_norm runs on the device for rows of a float dtype");
        }
        const int64_t dim = x.sizes[x.ndim - 1];
        TP_AMD_CHECK(dim > 0, "residual_norm: rows of no elements");
        if (dim > kResidualNormMaxDim) TP_AMD_DECLINE("residual_norm: rows wider than the device kernels take");
        TP_AMD_CHECK(y != nullptr || norm2, "residual_norm: neither a branch nor a norm");
        TP_AMD_CHECK(y != nullptr || (gate == nullptr && !norm1 && a == 1.0 && b == 1.0 && p == 0.0),
                     "residual_norm: without a branch there is no gate, no norm of it, no dropout and no scale");
        TP_AMD_CHECK(w1 == nullptr || norm1, "residual_norm: a weight for a norm that is not taken of the branch");
        TP_AMD_CHECK(w2 == nullptr || norm2, "residual_norm: a weight for a norm that is not taken");
        args.a = static_cast<float>(a);
        args.b = static_cast<float>(b);
        TP_AMD_CHECK(std::isfinite(args.a) && std::isfinite(args.b), "residual_norm: the scales have to be finite");
        args.drop = drop_args("residual_norm", p, seed, seed_tensor, offset, x.device);
        args.drops = p > 0.0;
        if (y != nullptr) {
            check_view(*y, "branch");
            if (!same_kind(*y, x)) TP_AMD_DECLINE("residual_norm: a branch of another dtype or device");
            TP_AMD_CHECK(sizes_of(*y) == sizes_of(x), "residual_norm: a branch of another shape than the residual's");
        }
        const tp_amd_tensor* weights[2] = {w1, w2};
        for (const tp_amd_tensor* w : weights) {
            if (w == nullptr) continue;
            check_view(*w, "weight");
            if (!same_kind(*w, x)) TP_AMD_DECLINE("residual_norm: a weight of another dtype or device");
            TP_AMD_CHECK(w->ndim == 1 && w->sizes[0] == dim, "residual_norm: a weight is one row of ", dim);
        }
        args.rows = rows_in(x);
        TP_AMD_CHECK(args.rows < kMaxRows, "residual_norm: ", args.rows, " rows");
        args.dim = static_cast<int>(dim);
        args.norm1 = norm1;
        args.norm2 = norm2;
        args.rows_per_gate = std::max<int64_t>(args.rows, 1);
        if (gate != nullptr) set_gate(x, *gate);
        args.x = rows_of(x, hold_x);
        if (y != nullptr) args.y = rows_of(*y, hold_y);
        for (int i = 0; i < 2; ++i) {
            if (weights[i] == nullptr) continue;
            hold_w[i] = contiguous_on_device(*weights[i]);
            (i ? args.w2 : args.w1) = hold_w[i].ref.data;
        }
    }

    // A gate has the residual's size on its first token axes and 1 on the
    // others, or those left out; its last axis is D or 1.
    void set_gate(const TensorRef& x, const TensorRef& gate) {
        check_view(gate, "gate");
        if (!same_kind(gate, x)) TP_AMD_DECLINE("residual_norm: a gate of another dtype or device");
        TP_AMD_CHECK(gate.ndim <= x.ndim, "residual_norm: a gate of more axes than the residual");
        const int lead = x.ndim - gate.ndim, tokens = x.ndim - 1;
        bool prefix = true;
        int64_t groups = 1;
        for (int d = 0; d < x.ndim; ++d) {
            const int64_t n = d < lead ? 1 : gate.sizes[d - lead];
            TP_AMD_CHECK(n == x.sizes[d] || n == 1, "residual_norm: a gate of ", n, " does not expand to ", x.sizes[d]);
            if (d == tokens || x.sizes[d] == 1) continue;
            if (n == 1) prefix = false;
            else if (!prefix) TP_AMD_DECLINE("residual_norm: a gate that repeats over an axis before one it has");
            else groups *= n;
        }
        args.gate_one = gate.ndim == 0 || (gate.sizes[gate.ndim - 1] == 1 && args.dim != 1);
        args.rows_per_gate = groups > 0 ? std::max<int64_t>(args.rows / groups, 1) : 1;
        const bool lies = gate.ndim == 0 || ((gate.sizes[gate.ndim - 1] == 1 || gate.strides[gate.ndim - 1] == 1) &&
                                             axes_merge(gate, gate.ndim - 1, args.gate.step));
        if (!lies) hold_gate = contiguous_on_device(gate);
        args.gate = Rows{lies ? gate.data : hold_gate.ref.data, lies ? args.gate.step : gate.sizes[gate.ndim - 1]};
        if (gate.ndim == 0) args.gate.step = 0;
    }
};

float eps_of(double eps) {
    TP_AMD_CHECK(!std::isnan(eps), "residual_norm: eps is not a number");
    return static_cast<float>(eps);
}

// A row of float32 statistics per token.
void statistics(const tp_amd_tensor* t, const TensorRef& x, MaybeOwned& hold, float*& data) {
    if (t == nullptr) return;
    check_view(*t, "statistics");
    if (!on_device(*t) || t->device != x.device || t->dtype != TP_AMD_FLOAT32) {
        TP_AMD_DECLINE("residual_norm_backward: float32 statistics on the operands' device");
    }
    TP_AMD_CHECK(sizes_of(*t) == token_shape(x), "residual_norm_backward: statistics of another shape");
    hold = contiguous_on_device(*t);
    data = static_cast<float*>(hold.ref.data);
}

// ---- log probabilities of tokens -------------------------------------------------------

// What forward and backward share.
struct TokenProbs {
    TokenProbsArgs args{};
    MaybeOwned hold_x, hold_t;

    TokenProbs(const TensorRef& x, const tp_amd_tensor* targets, double scale, int64_t ignore_index) {
        check_view(x, "logits");
        if (!on_device(x) || !is_native_float(x.dtype) || x.ndim < 1) {
            TP_AMD_DECLINE("token_log_probs runs on the device for rows of logits of a float dtype");
        }
        args.scale = static_cast<float>(scale);
        // (also times log2 e, as the kernels' powers of two have it)
        TP_AMD_CHECK(args.scale > 0.0f && args.scale < 2.3e38f, "token_log_probs: the scale has to be positive and finite");
        args.rows = rows_in(x);
        args.vocab = x.sizes[x.ndim - 1];
        TP_AMD_CHECK(args.vocab > 0 || args.rows == 0, "token_log_probs: rows of no logits");
        TP_AMD_CHECK(args.rows < kMaxRows && args.vocab < (int64_t{1} << 31), "token_log_probs: ", args.rows, " rows of ", args.vocab, " logits");
        args.ignore = ignore_index;
        if (targets != nullptr) {
            check_view(*targets, "targets");
            if (!index_tensor(*targets, x.device)) TP_AMD_DECLINE("token_log_probs: targets are integers on the logits' device");
            TP_AMD_CHECK(sizes_of(*targets) == token_shape(x), "token_log_probs: targets are one a row of logits");
            hold_t = contiguous_on_device(*targets);
            args.target = hold_t.ref.data;
            args.wide_target = targets->dtype == TP_AMD_INT64;
        }
        args.logits = rows_of(x, hold_x);
    }
};

}  // namespace

extern "C" {

int tp_amd_seeded_dropout(const tp_amd_tensor* input, double p, uint64_t seed, const tp_amd_tensor* seed_tensor, uint64_t offset,
                          tp_amd_tensor* result) {
    return dropout("seeded_dropout", input, p, seed, seed_tensor, offset, result);
}

int tp_amd_seeded_dropout_backward(const tp_amd_tensor* grad_output, double p, uint64_t seed, const tp_amd_tensor* seed_tensor,
                                   uint64_t offset, tp_amd_tensor* result) {
    return dropout("seeded_dropout_backward", grad_output, p, seed, seed_tensor, offset, result);
}

int tp_amd_residual_norm(const tp_amd_tensor* residual, const tp_amd_tensor* branch, const tp_amd_tensor* gate,
                         const tp_amd_tensor* branch_weight, const tp_amd_tensor* weight, double residual_scale, double branch_scale,
                         double branch_eps, double eps, double p, uint64_t seed, const tp_amd_tensor* seed_tensor, uint64_t offset,
                         tp_amd_tensor* sum, tp_amd_tensor* normed, tp_amd_tensor* branch_rstd, tp_amd_tensor* rstd) {
    return guarded_results({sum, normed, branch_rstd, rstd}, [&] {
        const TensorRef& x = deref(residual, "residual");
        const float eps1 = eps_of(branch_eps), eps2 = eps_of(eps);
        const bool norm1 = branch_eps >= 0.0, norm2 = eps >= 0.0;
        ResidualNorm n(x, branch, gate, branch_weight, weight, norm1, norm2, residual_scale, branch_scale, p, seed, seed_tensor, offset);
        n.args.eps1 = eps1;
        n.args.eps2 = eps2;
        Owned z, h, r1, r2;
        if (branch != nullptr) {
            z = empty_on(sizes_of(x), x.dtype, x.device);
            n.args.z = z.ref().data;
        }
        if (norm1) {
            r1 = empty_on(token_shape(x), TP_AMD_FLOAT32, x.device);
            n.args.r1 = static_cast<float*>(r1.ref().data);
        }
        if (norm2) {
            h = empty_on(sizes_of(x), x.dtype, x.device);
            r2 = empty_on(token_shape(x), TP_AMD_FLOAT32, x.device);
            n.args.h = h.ref().data;
            n.args.r2 = static_cast<float*>(r2.ref().data);
        }
        launch_residual_norm(x.dtype, n.args, x.device);
        if (branch != nullptr) *sum = z.release(); else set_undefined(sum);
        if (norm2) *normed = h.release(); else set_undefined(normed);
        if (norm1) *branch_rstd = r1.release(); else set_undefined(branch_rstd);
        if (norm2) *rstd = r2.release(); else set_undefined(rstd);
    });
}

int tp_amd_residual_norm_backward(const tp_amd_tensor* grad_sum, const tp_amd_tensor* grad_normed, const tp_amd_tensor* residual,
                                  const tp_amd_tensor* branch, const tp_amd_tensor* branch_rstd, const tp_amd_tensor* rstd,
                                  const tp_amd_tensor* gate, const tp_amd_tensor* branch_weight, const tp_amd_tensor* weight,
                                  double residual_scale, double branch_scale, double p, uint64_t seed, const tp_amd_tensor* seed_tensor,
                                  uint64_t offset, const int* output_mask, tp_amd_tensor* dresidual, tp_amd_tensor* dbranch,
                                  tp_amd_tensor* dgate, tp_amd_tensor* dbranch_weight, tp_amd_tensor* dweight) {
    return guarded_results({dresidual, dbranch, dgate, dbranch_weight, dweight}, [&] {
        const TensorRef& x = deref(residual, "residual");
        TP_AMD_CHECK(grad_sum != nullptr || grad_normed != nullptr, "residual_norm_backward: no gradient of either result");
        TP_AMD_CHECK(grad_normed == nullptr || rstd != nullptr, "residual_norm_backward: a gradient of a norm without its statistics");
        ResidualNorm n(x, branch, gate, branch_weight, weight, branch_rstd != nullptr, rstd != nullptr || branch == nullptr, residual_scale,
                       branch_scale, p, seed, seed_tensor, offset);
        const tp_amd_tensor* grads[2] = {grad_sum, grad_normed};
        for (const tp_amd_tensor* g : grads) {
            if (g == nullptr) continue;
            check_view(*g, "gradient");
            if (!same_kind(*g, x)) TP_AMD_DECLINE("residual_norm_backward: gradients of the operands' dtype on their device");
            TP_AMD_CHECK(sizes_of(*g) == sizes_of(x), "residual_norm_backward: a gradient of another shape");
        }
        MaybeOwned hold_r[2], hold_g[2];
        statistics(branch_rstd, x, hold_r[0], n.args.r1);
        statistics(rstd, x, hold_r[1], n.args.r2);
        if (grad_sum != nullptr) n.args.dz = rows_of(*grad_sum, hold_g[0]);
        if (grad_normed != nullptr) n.args.dh = rows_of(*grad_normed, hold_g[1]);
        n.args.norm2 = grad_normed != nullptr;  // no gradient comes through it otherwise
        auto want = [&](int i) { return output_mask == nullptr || output_mask[i] != 0; };
        const bool wants[5] = {want(0), want(1) && branch != nullptr, want(2) && gate != nullptr, want(3) && branch_weight != nullptr,
                               want(4) && weight != nullptr};
        Owned out[5];
        void** data[5] = {&n.args.dx, &n.args.dy, &n.args.dgate, &n.args.dw1, &n.args.dw2};
        const tp_amd_tensor* like[5] = {&x, branch, gate, branch_weight, weight};
        bool any = false;
        for (int i = 0; i < 5; ++i) {
            if (!wants[i]) continue;
            any = true;
            out[i] = empty_on(sizes_of(*like[i]), x.dtype, x.device);
            *data[i] = out[i].ref().data;
            // no row adds to it, or no gradient reaches it
            if (i > 1 && numel(out[i].ref()) > 0 && (n.args.rows == 0 || (i == 4 && grad_normed == nullptr))) {
                fill(out[i].ref(), scalar_of(0.0));
                *data[i] = nullptr;
            }
        }
        if (any) launch_residual_norm_backward(x.dtype, n.args, x.device);
        tp_amd_tensor* slots[5] = {dresidual, dbranch, dgate, dbranch_weight, dweight};
        for (int i = 0; i < 5; ++i) {
            if (wants[i]) *slots[i] = out[i].release();
            else set_undefined(slots[i]);
        }
    });
}

int tp_amd_token_log_probs(const tp_amd_tensor* logits, const tp_amd_tensor* targets, double scale, int64_t top, int want_entropy,
                           int64_t ignore_index, tp_amd_tensor* logprob, tp_amd_tensor* entropy, tp_amd_tensor* stats,
                           tp_amd_tensor* top_logprobs, tp_amd_tensor* top_indices) {
    return guarded_results({logprob, entropy, stats, top_logprobs, top_indices}, [&] {
        const TensorRef& x = deref(logits, "logits");
        TokenProbs t(x, targets, scale, ignore_index);
        TP_AMD_CHECK(top >= 0, "token_log_probs: a negative number of alternatives");
        if (top > kTokenProbsMaxTop) TP_AMD_DECLINE("token_log_probs: more alternatives than the device kernels take");
        TP_AMD_CHECK(top <= t.args.vocab || t.args.rows == 0, "token_log_probs: ", top, " alternatives of ", t.args.vocab, " tokens");
        const Sizes rows = token_shape(x);
        auto with = [&](int64_t n) {
            Sizes s = rows;
            s.push_back(n);
            return s;
        };
        Owned lp, h, st = empty_on(with(2), TP_AMD_FLOAT32, x.device), values, indices;
        t.args.stats = static_cast<float*>(st.ref().data);
        if (targets != nullptr) {
            lp = empty_on(rows, TP_AMD_FLOAT32, x.device);
            t.args.logprob = static_cast<float*>(lp.ref().data);
        }
        if (want_entropy) {
            h = empty_on(rows, TP_AMD_FLOAT32, x.device);
            t.args.entropy = static_cast<float*>(h.ref().data);
        }
        if (top > 0) {
            values = empty_on(with(top), TP_AMD_FLOAT32, x.device);
            indices = empty_on(with(top), TP_AMD_INT64, x.device);
            t.args.top_values = static_cast<float*>(values.ref().data);
            t.args.top_index = static_cast<int64_t*>(indices.ref().data);
        }
        t.args.top = static_cast<int>(top);
        launch_token_log_probs(x.dtype, t.args, x.device);
        if (targets != nullptr) *logprob = lp.release(); else set_undefined(logprob);
        if (want_entropy) *entropy = h.release(); else set_undefined(entropy);
        *stats = st.release();
        if (top > 0) *top_logprobs = values.release(); else set_undefined(top_logprobs);
        if (top > 0) *top_indices = indices.release(); else set_undefined(top_indices);
    });
}

int tp_amd_token_log_probs_backward(const tp_amd_tensor* grad_logprob, const tp_amd_tensor* grad_entropy, const tp_amd_tensor* logits,
                                    const tp_amd_tensor* targets, const tp_amd_tensor* stats, const tp_amd_tensor* entropy, double scale,
                                    int64_t ignore_index, tp_amd_tensor* result) {
    return guarded_result(result, [&] {
        const TensorRef &x = deref(logits, "logits"), &st = deref(stats, "stats");
        TP_AMD_CHECK(grad_logprob != nullptr || grad_entropy != nullptr, "token_log_probs_backward: no gradient of either result");
        TP_AMD_CHECK(grad_logprob == nullptr || targets != nullptr, "token_log_probs_backward: a gradient of log probabilities without their tokens");
        TP_AMD_CHECK(grad_entropy == nullptr || entropy != nullptr, "token_log_probs_backward: a gradient of the entropy without the entropy");
        TokenProbs t(x, targets, scale, ignore_index);
        Sizes stat_shape = token_shape(x);
        auto take = [&](const tp_amd_tensor* g, const Sizes& shape, MaybeOwned& hold) -> const float* {
            if (g == nullptr) return nullptr;
            check_view(*g, "gradient or statistics");
            if (!on_device(*g) || g->device != x.device || g->dtype != TP_AMD_FLOAT32) {
                TP_AMD_DECLINE("token_log_probs_backward: float32 gradients and statistics on the logits' device");
            }
            TP_AMD_CHECK(sizes_of(*g) == shape, "token_log_probs_backward: gradients or statistics of another shape");
            hold = contiguous_on_device(*g);
            return static_cast<const float*>(hold.ref.data);
        };
        MaybeOwned hold[4];
        t.args.da = take(grad_logprob, stat_shape, hold[0]);
        t.args.db = take(grad_entropy, stat_shape, hold[1]);
        if (grad_entropy != nullptr) t.args.entropy = const_cast<float*>(take(entropy, stat_shape, hold[2]));
        stat_shape.push_back(2);
        t.args.stats = const_cast<float*>(take(&st, stat_shape, hold[3]));
        Owned out = empty_on(sizes_of(x), x.dtype, x.device);
        t.args.dlogits = out.ref().data;
        launch_token_log_probs_backward(x.dtype, t.args, x.device);
        return out;
    });
}

}  // extern "C"

// The attention layer's operators: the norm and position rotation of each
// head's query and key (kernels/head_norm.hip), and causal attention with a
// sliding window and first tokens that stay visible (kernels/attention.hip,
// kernels/attention_backward.hip), forward and backward.  The reference has no
// counterpart; entries follow the neural-network layers' conventions: device
// float tensors of one dtype or the call is declined, shapes that contradict
// each other are errors, operands are read where they lie and copied only when
// the kernels cannot address them.

#include "../kernels/attention.h"
#include "entries.h"
#include "tp_amd_ops.h"

using namespace tp_amd;

namespace {

// ---- norm and rotation of heads -------------------------------------------------

// Token axes as two: the last one, and the ones before it as one.
struct Tokens {
    Sizes shape;
    int64_t outer = 1, inner = 1;
    Tokens() = default;
    explicit Tokens(const TensorRef& t) {
        for (int d = 0; d + 2 < t.ndim; ++d) shape.push_back(t.sizes[d]);
        for (size_t d = 0; d + 1 < shape.size(); ++d) outer *= shape[d];
        if (!shape.empty()) inner = shape.back();
    }
    int64_t count() const { return outer * inner; }
    bool split(const TensorRef& t, int64_t& outer_step, int64_t& inner_step) const {
        const int n = static_cast<int>(shape.size());
        inner_step = n > 0 ? t.strides[n - 1] : 0;
        outer_step = 0;
        return n < 2 || axes_merge(t, n - 1, outer_step);
    }
};

// [tokens..., heads, D] as the kernels read it; copied when they cannot.
HeadRows head_rows(const TensorRef& t, const Tokens& tokens, MaybeOwned& hold) {
    auto in_place = [&](const TensorRef& x, HeadRows& r) {
        r.data = x.data;
        r.head = x.strides[x.ndim - 2];
        return (x.sizes[x.ndim - 1] == 1 || x.strides[x.ndim - 1] == 1) && tokens.split(x, r.outer, r.inner);
    };
    HeadRows r{};
    if (in_place(t, r)) return r;
    hold = contiguous_on_device(t);
    TP_AMD_CHECK(in_place(hold.ref, r), "qk_norm_rope: internal: a dense copy that cannot be addressed");
    return r;
}

// What forward and backward share: checks, the table, positions and weights.
struct HeadNorm {
    HeadNormArgs args{};
    Tokens tokens;
    MaybeOwned hold_q, hold_k, hold_table, hold_pos, hold_w[2];

    HeadNorm(const TensorRef& q, const TensorRef& k, const TensorRef& table, const TensorRef& positions,
             const tp_amd_tensor* qw, const tp_amd_tensor* kw, int interleaved) {
        check_view(q, "query");
        check_view(k, "key");
        check_view(table, "table");
        check_view(positions, "positions");
        if (!on_device(q) || !is_native_float(q.dtype) || !same_kind(k, q) || q.ndim < 2 || k.ndim < 2 || !on_device(table) ||
            table.device != q.device || table.dtype != TP_AMD_FLOAT32 || table.ndim != 2 || !index_tensor(positions, q.device)) {
            TP_AMD_DECLINE("qk_norm_rope runs on the device for queries and keys of one float dtype, a 2-D float32 table and integer positions");
        }
        const int64_t dim = q.sizes[q.ndim - 1], rotary = table.sizes[1];
        if (dim > kHeadNormMaxDim) TP_AMD_DECLINE("qk_norm_rope: heads wider than the device kernels take");
        tokens = Tokens(q);
        const Tokens key_tokens(k);
        TP_AMD_CHECK(k.sizes[k.ndim - 1] == dim && key_tokens.shape == tokens.shape,
                     "qk_norm_rope: queries and keys differ in their tokens or head size");
        TP_AMD_CHECK(dim > 0 && rotary % 2 == 0 && rotary <= dim, "qk_norm_rope: a table row rotates ", rotary,
                     " elements of heads of ", dim);
        const tp_amd_tensor* weights[2] = {qw, kw};
        const int64_t heads[2] = {q.sizes[q.ndim - 2], k.sizes[k.ndim - 2]};
        for (int s = 0; s < 2; ++s) {
            TP_AMD_CHECK(heads[s] < (int64_t{1} << 30), "qk_norm_rope: too many heads");
            args.side[s].heads = static_cast<int>(heads[s]);
            if (weights[s] == nullptr) continue;
            check_view(*weights[s], "weight");
            if (!same_kind(*weights[s], q)) TP_AMD_DECLINE("qk_norm_rope: a weight of another dtype or device");
            TP_AMD_CHECK(weights[s]->ndim == 1 && weights[s]->sizes[0] == dim, "qk_norm_rope: a weight is one row of ", dim);
        }
        TensorRef pos = expand_to(positions, tokens.shape);
        args.side[0].x = head_rows(q, tokens, hold_q);
        args.side[1].x = head_rows(k, tokens, hold_k);
        for (int s = 0; s < 2; ++s) {
            if (weights[s] == nullptr) continue;
            hold_w[s] = contiguous_on_device(*weights[s]);
            args.side[s].weight = hold_w[s].ref.data;
        }
        args.outer = tokens.outer;
        args.inner = tokens.inner;
        args.dim = static_cast<int>(dim);
        args.rotary = static_cast<int>(rotary);
        args.interleaved = interleaved != 0;
        hold_table = contiguous_on_device(table);
        args.table = static_cast<const float*>(hold_table.ref.data);
        args.table_rows = table.sizes[0];
        if (!tokens.split(pos, args.pos_outer, args.pos_inner)) {
            hold_pos = contiguous_on_device(pos);
            pos = hold_pos.ref;
            TP_AMD_CHECK(tokens.split(pos, args.pos_outer, args.pos_inner), "qk_norm_rope: internal: positions");
        }
        args.positions = pos.data;
        args.wide_positions = positions.dtype == TP_AMD_INT64;
    }
    Sizes stat_shape(const TensorRef& t) const {
        Sizes s = sizes_of(t);
        s.pop_back();
        return s;
    }
};

// ---- attention --------------------------------------------------------------------

// [B, T, H, D] as the kernels read it: rows of whole 16-byte packets on
// 16-byte boundaries, 128 tokens within the reach of one buffer resource.
// Anything else is copied, a D that is no whole number of packets padded with
// zeros.
struct TokenTensor {
    TokenRows rows{};
    MaybeOwned hold;

    static bool addressable(const TensorRef& t, TokenRows& r) {
        const int64_t e = element_size(t.dtype), v = 16 / e;
        r = TokenRows{t.data, t.strides[0], t.strides[1], t.strides[2]};
        auto step_fits = [&](int d) { return t.sizes[d] <= 1 || t.strides[d] % v == 0; };
        // (a token axis of one element may have any stride)
        if (t.sizes[1] <= 1) r.token = 0;
        return (t.sizes[3] <= 1 || t.strides[3] == 1) && t.sizes[3] % v == 0 && reinterpret_cast<uintptr_t>(t.data) % 16 == 0 &&
               step_fits(0) && step_fits(1) && step_fits(2) && r.token >= 0 && r.token * e < (int64_t{1} << 24);
    }

    explicit TokenTensor(const TensorRef& t, int64_t dim) {
        if (addressable(t, rows)) return;
        if (dim == t.sizes[3]) {
            hold.hold = empty_on(sizes_of(t), t.dtype, t.device);
            strided_copy(hold.hold.ref(), t);
        } else {
            hold.hold = empty_on({t.sizes[0], t.sizes[1], t.sizes[2], dim}, t.dtype, t.device);
            if (numel(hold.hold.ref()) > 0) fill(hold.hold.ref(), scalar_of(0.0));
            TensorRef part = hold.hold.ref();
            part.sizes[3] = t.sizes[3];
            strided_copy(part, t);
        }
        TP_AMD_CHECK(addressable(hold.hold.ref(), rows) || numel(t) == 0, "sliding_window_attention: internal: a copy that cannot be addressed");
    }
};

// A result [B, T, H, D]: written with rows of ``dim``, handed back with D.
struct TokenResult {
    Owned wide;
    int64_t want;
    TokenResult(const TensorRef& like, int64_t dim) : want(like.sizes[3]) {
        wide = empty_on({like.sizes[0], like.sizes[1], like.sizes[2], dim}, like.dtype, like.device);
    }
    void* data() { return wide.ref().data; }
    TensorRef release() {
        if (wide.ref().sizes[3] == want) return wide.release();
        TensorRef part = wide.ref();
        part.sizes[3] = want;
        Owned narrow = empty_on(sizes_of(part), part.dtype, part.device);
        strided_copy(narrow.ref(), part);
        return narrow.release();
    }
};

// The checks forward and backward share, and the arguments they make.
struct Attention {
    AttentionArgs args{};
    int64_t dim;  // D in whole packets

    Attention(const TensorRef& q, const TensorRef& k, const TensorRef& v, int64_t window, int64_t sinks, double scale,
              const tp_amd_tensor* lengths, const tp_amd_tensor* starts) {
        check_view(q, "query");
        check_view(k, "key");
        check_view(v, "value");
        if (!on_device(q) || !is_native_float(q.dtype) || !same_kind(k, q) || !same_kind(v, q) || q.ndim != 4 || k.ndim != 4 ||
            v.ndim != 4) {
            TP_AMD_DECLINE("sliding_window_attention runs on the device for 4-D queries, keys and values of one float dtype");
        }
        const int64_t b = q.sizes[0], d = q.sizes[3];
        if (d > kAttentionMaxDim) TP_AMD_DECLINE("sliding_window_attention: heads wider than the device kernels take");
        TP_AMD_CHECK(sizes_of(k) == sizes_of(v), "sliding_window_attention: keys and values differ in shape");
        TP_AMD_CHECK(k.sizes[0] == b && k.sizes[3] == d && d > 0, "sliding_window_attention: queries of ", b, " sequences with heads of ",
                     d, ", keys of ", k.sizes[0], " with ", k.sizes[3]);
        TP_AMD_CHECK(k.sizes[2] > 0 && q.sizes[2] % k.sizes[2] == 0, "sliding_window_attention: ", q.sizes[2],
                     " query heads cannot share ", k.sizes[2], " key heads");
        TP_AMD_CHECK(sinks >= 0, "sliding_window_attention: negative sinks");
        const float s = static_cast<float>(scale);
        // (also times log2 e, as the kernels' powers of two have it)
        TP_AMD_CHECK(s > 0.0f && s < 2.3e38f, "sliding_window_attention: the scale has to be positive and finite");
        TP_AMD_CHECK(q.sizes[1] + k.sizes[1] < (int64_t{1} << 30) && b < (int64_t{1} << 30) && q.sizes[2] < (int64_t{1} << 30),
                     "sliding_window_attention: sizes past 2^30");
        per_sequence(lengths, "lengths", b, q.device, args.lengths, args.wide_lengths, args.lengths_step);
        per_sequence(starts, "starts", b, q.device, args.starts, args.wide_starts, args.starts_step);
        const int64_t v16 = 16 / element_size(q.dtype);
        dim = (d + v16 - 1) / v16 * v16;
        args.batch = static_cast<int>(b);
        args.queries = static_cast<int>(q.sizes[1]);
        args.keys = static_cast<int>(k.sizes[1]);
        args.heads = static_cast<int>(q.sizes[2]);
        args.kv_heads = static_cast<int>(k.sizes[2]);
        args.dim = static_cast<int>(dim);
        args.window = window;
        args.sinks = sinks;
        args.scale = s;
    }

    static void per_sequence(const tp_amd_tensor* t, const char* what, int64_t batch, int device, const void*& data, bool& wide,
                             int64_t& step) {
        data = nullptr;
        if (t == nullptr) return;
        check_view(*t, what);
        if (!index_tensor(*t, device)) TP_AMD_DECLINE("sliding_window_attention: lengths and starts are integers on the operands' device");
        TP_AMD_CHECK(t->ndim == 1 && t->sizes[0] == batch, "sliding_window_attention: ", what, " are one number a sequence");
        data = t->data;
        wide = t->dtype == TP_AMD_INT64;
        step = t->strides[0];
    }
};

Sizes lse_shape(const TensorRef& q) { return {q.sizes[0], q.sizes[2], q.sizes[1]}; }

}  // namespace

extern "C" {

int tp_amd_qk_norm_rope(const tp_amd_tensor* query, const tp_amd_tensor* key, const tp_amd_tensor* table,
                        const tp_amd_tensor* positions, const tp_amd_tensor* query_weight,
                        const tp_amd_tensor* key_weight, double eps, int interleaved, tp_amd_tensor* query_out,
                        tp_amd_tensor* key_out, tp_amd_tensor* query_rstd, tp_amd_tensor* key_rstd) {
    return guarded_results({query_out, key_out, query_rstd, key_rstd}, [&] {
        const TensorRef &q = deref(query, "query"), &k = deref(key, "key");
        HeadNorm norm(q, k, deref(table, "table"), deref(positions, "positions"), query_weight, key_weight, interleaved);
        norm.args.eps = static_cast<float>(eps);
        Owned out[2], rstd[2];
        const TensorRef* in[2] = {&q, &k};
        for (int s = 0; s < 2; ++s) {
            out[s] = empty_on(sizes_of(*in[s]), q.dtype, q.device);
            rstd[s] = empty_on(norm.stat_shape(*in[s]), TP_AMD_FLOAT32, q.device);
            norm.args.side[s].out = out[s].ref().data;
            norm.args.side[s].rstd = static_cast<float*>(rstd[s].ref().data);
        }
        if (numel(q) + numel(k) > 0) launch_head_norm(q.dtype, norm.args, q.device);
        *query_out = out[0].release();
        *key_out = out[1].release();
        *query_rstd = rstd[0].release();
        *key_rstd = rstd[1].release();
    });
}

int tp_amd_qk_norm_rope_backward(const tp_amd_tensor* grad_query, const tp_amd_tensor* grad_key,
                                 const tp_amd_tensor* query, const tp_amd_tensor* key, const tp_amd_tensor* table,
                                 const tp_amd_tensor* positions, const tp_amd_tensor* query_rstd,
                                 const tp_amd_tensor* key_rstd, const tp_amd_tensor* query_weight,
                                 const tp_amd_tensor* key_weight, int interleaved, const int* output_mask,
                                 tp_amd_tensor* dquery, tp_amd_tensor* dkey, tp_amd_tensor* dquery_weight,
                                 tp_amd_tensor* dkey_weight) {
    return guarded_results({dquery, dkey, dquery_weight, dkey_weight}, [&] {
        const TensorRef &q = deref(query, "query"), &k = deref(key, "key");
        const TensorRef *grad[2] = {&deref(grad_query, "grad_query"), &deref(grad_key, "grad_key")};
        const TensorRef *stat[2] = {&deref(query_rstd, "query_rstd"), &deref(key_rstd, "key_rstd")};
        const TensorRef* in[2] = {&q, &k};
        HeadNorm norm(q, k, deref(table, "table"), deref(positions, "positions"), query_weight, key_weight, interleaved);
        auto want = [&](int i) { return output_mask == nullptr || output_mask[i] != 0; };
        MaybeOwned hold_grad[2], hold_stat[2];
        Owned dx[2], dw[2];
        for (int s = 0; s < 2; ++s) {
            check_view(*grad[s], "gradient");
            check_view(*stat[s], "statistics");
            if (!same_kind(*grad[s], q) || !on_device(*stat[s]) || stat[s]->device != q.device || stat[s]->dtype != TP_AMD_FLOAT32) {
                TP_AMD_DECLINE("qk_norm_rope_backward: gradients of the operands' dtype and float32 statistics on their device");
            }
            TP_AMD_CHECK(sizes_of(*grad[s]) == sizes_of(*in[s]), "qk_norm_rope_backward: a gradient of another shape");
            TP_AMD_CHECK(sizes_of(*stat[s]) == norm.stat_shape(*in[s]), "qk_norm_rope_backward: statistics of another shape");
            HeadNormSide& side = norm.args.side[s];
            side.dy = head_rows(*grad[s], norm.tokens, hold_grad[s]);
            hold_stat[s] = contiguous_on_device(*stat[s]);
            side.rstd = static_cast<float*>(hold_stat[s].ref.data);
            if (want(s)) {
                dx[s] = empty_on(sizes_of(*in[s]), q.dtype, q.device);
                side.out = dx[s].ref().data;
            }
            if (want(2 + s)) {
                dw[s] = empty_on({in[s]->sizes[in[s]->ndim - 1]}, q.dtype, q.device);
                side.dweight = dw[s].ref().data;
            }
        }
        if (want(0) || want(1) || want(2) || want(3)) launch_head_norm_backward(q.dtype, norm.args, q.device);
        tp_amd_tensor* slots[4] = {dquery, dkey, dquery_weight, dkey_weight};
        for (int s = 0; s < 4; ++s) {
            if (want(s)) *slots[s] = (s < 2 ? dx[s] : dw[s - 2]).release();
            else set_undefined(slots[s]);
        }
    });
}

int tp_amd_sliding_window_attention(const tp_amd_tensor* query, const tp_amd_tensor* key, const tp_amd_tensor* value,
                                    int64_t window, int64_t sinks, double scale, const tp_amd_tensor* lengths,
                                    const tp_amd_tensor* starts, tp_amd_tensor* out, tp_amd_tensor* lse) {
    return guarded_results({out, lse}, [&] {
        const TensorRef &q = deref(query, "query"), &k = deref(key, "key"), &v = deref(value, "value");
        Attention a(q, k, v, window, sinks, scale, lengths, starts);
        const TokenTensor tq(q, a.dim), tk(k, a.dim), tv(v, a.dim);
        TokenResult o(q, a.dim);
        Owned l = empty_on(lse_shape(q), TP_AMD_FLOAT32, q.device);
        a.args.q = tq.rows;
        a.args.k = tk.rows;
        a.args.v = tv.rows;
        a.args.out = o.data();
        a.args.lse = static_cast<float*>(l.ref().data);
        if (numel(q) > 0) launch_attention(q.dtype, a.args, q.device);
        Owned narrow(o.release());
        *out = narrow.release();
        *lse = l.release();
    });
}

int tp_amd_sliding_window_attention_backward(const tp_amd_tensor* grad_out, const tp_amd_tensor* query, const tp_amd_tensor* key,
                                             const tp_amd_tensor* value, const tp_amd_tensor* out, const tp_amd_tensor* lse,
                                             int64_t window, int64_t sinks, double scale, const tp_amd_tensor* lengths,
                                             const tp_amd_tensor* starts, tp_amd_tensor* dquery, tp_amd_tensor* dkey,
                                             tp_amd_tensor* dvalue) {
    return guarded_results({dquery, dkey, dvalue}, [&] {
        const TensorRef &q = deref(query, "query"), &k = deref(key, "key"), &v = deref(value, "value");
        const TensorRef &g = deref(grad_out, "grad_out"), &o = deref(out, "out"), &l = deref(lse, "lse");
        Attention a(q, k, v, window, sinks, scale, lengths, starts);
        check_view(g, "grad_out");
        check_view(o, "out");
        check_view(l, "lse");
        if (!same_kind(g, q) || !same_kind(o, q) || !on_device(l) || l.device != q.device || l.dtype != TP_AMD_FLOAT32) {
            TP_AMD_DECLINE("sliding_window_attention_backward: out and its gradient of the operands' dtype, float32 lse");
        }
        TP_AMD_CHECK(sizes_of(g) == sizes_of(q) && sizes_of(o) == sizes_of(q), "sliding_window_attention_backward: out and its gradient have the queries' shape");
        TP_AMD_CHECK(sizes_of(l) == lse_shape(q), "sliding_window_attention_backward: lse of another shape");
        const TokenTensor tq(q, a.dim), tk(k, a.dim), tv(v, a.dim), tg(g, a.dim), to(o, a.dim);
        const MaybeOwned tl = contiguous_on_device(l);
        TokenResult dq(q, a.dim), dk(k, a.dim), dv(v, a.dim);
        a.args.q = tq.rows;
        a.args.k = tk.rows;
        a.args.v = tv.rows;
        a.args.dout = tg.rows;
        a.args.o = to.rows;
        a.args.lse = static_cast<float*>(tl.ref.data);
        a.args.dq = dq.data();
        a.args.dk = dk.data();
        a.args.dv = dv.data();
        if (a.args.batch > 0 && a.args.heads > 0) {
            launch_attention_backward(q.dtype, a.args, q.device);
        } else {
            for (TokenResult* r : {&dk, &dv}) {
                if (numel(r->wide.ref()) > 0) fill(r->wide.ref(), scalar_of(0.0));
            }
        }
        Owned oq(dq.release()), ok(dk.release()), ov(dv.release());
        *dquery = oq.release();
        *dkey = ok.release();
        *dvalue = ov.release();
    });
}

}  // extern "C"

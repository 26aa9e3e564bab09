// Gradients of causal attention with a sliding window and first tokens that
// stay visible.
//
// From the forward's l (the logarithm of a row's sum): P_ij = e^(s_ij - l_i),
// D_i = sum_d do_i o_i, dS_ij = P_ij (do_i . v_j - D_i), and
// dq_i = scale sum_j dS_ij k_j, dk_j = scale sum_i dS_ij q_i,
// dv_j = sum_i P_ij do_i, a key head's gradients over all its query heads.
//
// Two kernels form P and dS again, each for the sums it owns, so that nothing
// is added by atomics and the same call gives the same bits: one walks the keys
// that a block's queries see (dq, and D for the other), one the queries that
// see a block's keys, all heads of the group in turn (dk, dv).  Together 14
// flops a visible pair and element where a single pass with atomics would need
// 10.  Blocks own 128 rows in four waves, or 32 in one where there is little
// work.  Keys that stay visible to every later query have many more of them
// than the others: their walks are cut into parts of about the others' length,
// and with few blocks all walks are, the parts' float32 sums joined in order by
// a third kernel.  P and dS are rounded to the operands' type for the matrix
// instruction; sums are float32.  float16 does not hold every dS: it has the
// gradients' size, 1 / scale times what dq needs and 1 / keys of it.  So there
// dS is rounded at a power of two times its size that each sum keeps for itself
// (ColumnScale), and P at 2^12 times.
//
// Bound by the instructions that share a wave's issue: matrix products, and
// beside them an exponential, two products and two roundings an element and
// the reads from LDS (no bank conflicts).  bf16, 2 x 4096 tokens, 32 heads of
// 128 on 8 key heads, window 1024, medians (and best): dq 222 us (213), 815
// Tflop/s, its matrix cores busy 49 % of the cycles; dk and dv 368 us (354), 655
// Tflop/s, 36 %: two accumulators of 32 x 128 and the fragments of keys and values
// leave a wave no registers to read a tile ahead of its products, and 17 of them
// pass through scratch memory in every tile; the join 5 us.  float32, a sixteenth
// of bf16's rate: 1001 tokens, 12 heads of 64, window 256, 79 us in all, of which
// dq takes 40 with 384 waves on 1024 SIMDs, each on a walk of up to 11 tiles that
// only the other kernel cuts.

#include <algorithm>

#include "attention_tiles.h"
#include "../allocator.h"
#include "../common.h"
#include "../runtime.h"

namespace tp_amd {

namespace attention {

namespace {

struct Backward {
    Shape s;
    TokenRows q, k, v, o, dout;
    const float* lse;
    // what the first kernel finds of every query for the second one: -l log2 e
    // (and the bits P is scaled by) and D, [batch][heads][queries] each
    float *bias, *delta;
    void *dq, *dk, *dv;
    float scale, scale2;  // scale2: times log2 e
    int blocks;           // of 32 W queries (dq) or keys (dk, dv) a head
    int pairs;            // batch x key heads
    // dk, dv: the first sink_blocks blocks of a head walk in sink_parts parts,
    // the others in near_parts; parts of more than one leave float32 sums, the
    // first tokens' before the others'.
    int sink_blocks, sink_parts, near_parts;
    float* part;  // [head][part that leaves sums][2][rows][dim]
    __host__ __device__ int sink_slots() const { return sink_blocks * sink_parts; }
    __host__ __device__ int near_slots() const { return (blocks - sink_blocks) * near_parts; }
    __host__ __device__ int sums_of_sinks() const { return sink_parts > 1 ? sink_slots() : 0; }
    __host__ __device__ int sums() const { return sums_of_sinks() + (near_parts > 1 ? near_slots() : 0); }
};

// P is rounded at this power of two times its size.  float16 is full down to
// 2^-14 and steps by 2^-24 below, less than the P of 2^14 keys and more; P itself
// is at most 1 but for the rounding of s - l, which has 2^4 left.
template <typename T>
constexpr int kProbabilityBits = std::is_same_v<T, f16_t> ? 12 : 0;

// The power of two that the dS of a lane's column are multiplied with before
// float16 rounds them: the first that are not 0, and any that would pass 2^15,
// are brought to 2^7 .. 2^8, and the column's sums with them.  So an element is off
// by its half step or by 2^-32 of the column's largest so far.  (Other types have
// float32's exponents and leave dS as it is.)  The maximum and the products are
// 3 % of forward and backward of 2 x 4096 tokens, 32 heads of 128 under a window
// of 1024 (706 us without, 728 with), 11 % of 64 heads x 512 (68 and 75).
template <typename T>
struct ColumnScale {
    static constexpr bool kOn = std::is_same_v<T, f16_t>;
    float up = 0x1p60f;

    template <int DT>
    __device__ __forceinline__ void apply(f32x16& ds, f32x16 (&sums)[DT]) {
        if constexpr (kOn) {
            float top = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(ds[e]));
            top = both_halves(top, MaxOf{});
            const bool past = top * up > 0x1p15f;
            if (__any(past)) {
                // 2^(7 - exponent of top), for an infinite one too
                const float next = past ? __uint_as_float((261u << 23) - (__float_as_uint(top) & 0x7f800000u)) : up;
                const float turn = next * down();
                up = next;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sums[d][e] *= turn;
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) ds[e] *= up;
        }
    }
    // What the sums are multiplied with in the end.
    __device__ __forceinline__ float down() const { return kOn ? __uint_as_float((254u << 23) - __float_as_uint(up)) : 1.0f; }
};

// Rows of dq that hold a NaN and are `bad`, each lane's its own (query i at
// position `row`, with its bias and D): see "sums again".
template <typename T>
__device__ __attribute__((noinline)) void queries_again(const Backward* launched, int b_, int h_, int p0, int p1, bool bad, int i, int row,
                                                        float bias, float delta) {
    const Backward& p = as_launched(launched);
    const int b = shared_by_lanes(b_), h = shared_by_lanes(h_), hk = h / p.s.group;
    const S_<T>* kh = static_cast<const S_<T>*>(p.k.data) + b * p.k.batch + hk * p.k.head;
    const S_<T>* vh = static_cast<const S_<T>*>(p.v.data) + b * p.v.batch + hk * p.v.head;
    for_each_question(only_beside<T>(p.s, kh, p.k.token, shared_by_lanes(p0), shared_by_lanes(p1), bad, row), [&](int lane) __attribute__((always_inline)) {
        const int iu = __builtin_amdgcn_readlane(i, lane);
        const float bu = from_lane(bias, lane), du = from_lane(delta, lane);
        const S_<T>* q = static_cast<const S_<T>*>(p.q.data) + b * p.q.batch + h * p.q.head + iu * p.q.token;
        const S_<T>* g = static_cast<const S_<T>*>(p.dout.data) + b * p.dout.batch + h * p.dout.head + iu * p.dout.token;
        Two o{0.0f, 0.0f};
        for_seen(p.s.rule, __builtin_amdgcn_readlane(row, lane), [&](int j0, uint64_t seen) __attribute__((always_inline)) {
            const int mine = threadIdx.x % kWave;
            float ds = 0.0f;
            if (seen >> mine & 1) {
                const float s = row_product<T>(q, kh + (j0 + mine) * p.k.token, p.s.dim);
                ds = __builtin_amdgcn_exp2f(fmaf(s, p.scale2, bu)) * (row_product<T>(g, vh + (j0 + mine) * p.v.token, p.s.dim) - du);
            }
            add_rows<T>(o, ds, kh + j0 * p.k.token, p.k.token, seen, p.s.dim);
        });
        S_<T>* out = static_cast<S_<T>*>(p.dq) + ((static_cast<int64_t>(b) * p.s.queries + iu) * p.s.heads + h) * p.s.dim;
        store_two<T>(out, p.s.dim, Two{o.x * p.scale, o.y * p.scale});
        return i == iu;
    });
}

// What a block of dk and dv walks: keys kb RB .. last of a sequence, tiles
// from .. to - 1 of BQ queries, per_query_head of them from tile t0 on of every
// query head of the group.
template <int BQ, int RB>
struct KeyWalk {
    int bh, hk, b, kb, parts;
    int64_t at_part;  // of the parts' sums
    Sequence seq;
    int last, t0, per_query_head, from, to;
    __device__ __forceinline__ explicit KeyWalk(const Backward& p) {
        bh = blockIdx.x % p.pairs;
        const int slot = blockIdx.x / p.pairs;
        hk = bh % p.s.kv_heads, b = bh / p.s.kv_heads;
        const bool sink = slot < p.sink_slots();
        parts = sink ? p.sink_parts : p.near_parts;
        const int local = sink ? slot : slot - p.sink_slots(), part = local % parts;
        kb = (sink ? 0 : p.sink_blocks) + local / parts;
        at_part = static_cast<int64_t>(bh) * p.sums() + local + (sink ? 0 : p.sums_of_sinks());
        seq = sequence_of(p.s, b);
        last = min(kb * RB + RB, seq.length) - 1;
        // queries that see a key of the block: from the block's first key on, to
        // the window's end behind its last one or, of first tokens, to the end
        const int64_t reach = kb * RB < p.s.rule.sinks ? int64_t{kNoWindow} : int64_t{last} + p.s.rule.window - 1;
        const int i0 = max(kb * RB - seq.start, seq.first);
        const int i1 = static_cast<int>(min(reach - seq.start, static_cast<int64_t>(seq.end) - 1));
        t0 = i0 / BQ;
        per_query_head = last >= kb * RB && i0 <= i1 ? i1 / BQ - t0 + 1 : 0;
        const int64_t all = static_cast<int64_t>(per_query_head) * p.s.group;
        from = static_cast<int>(all * part / parts), to = static_cast<int>(all * (part + 1) / parts);
    }
};

// Rows of dk and dv (or of a part's sums) that hold a NaN, where `bad`, each
// lane's its own key: see "sums again".  A query without a sum counts as unseen,
// whatever it holds.
template <typename T, int BQ, int W>
__device__ __attribute__((noinline)) void keys_again(const Backward* launched, bool bad) {
    constexpr int RB = 32 * W;
    const Backward& p = as_launched(launched);
    const KeyWalk<BQ, RB> walk(p);
    const int b = walk.b, hk = walk.hk, last = walk.last, from = walk.from, to = walk.to;
    const Sequence& seq = walk.seq;
    const int mine = walk.kb * RB + static_cast<int>(threadIdx.x / kWave * 32 + threadIdx.x % 32);
    const S_<T>* kh = static_cast<const S_<T>*>(p.k.data) + b * p.k.batch + hk * p.k.head;
    const S_<T>* vh = static_cast<const S_<T>*>(p.v.data) + b * p.v.batch + hk * p.v.head;
    const S_<T>* qb = static_cast<const S_<T>*>(p.q.data) + b * p.q.batch;
    const S_<T>* db = static_cast<const S_<T>*>(p.dout.data) + b * p.dout.batch;
    const int lane_id = threadIdx.x % kWave;
    // of tile `it`, f(query head, its statistics, its rows)
    auto tile = [&](int it, const auto& f) __attribute__((always_inline)) {
        const int h = hk * p.s.group + it / walk.per_query_head, r0 = (walk.t0 + it % walk.per_query_head) * BQ;
        f(h, (static_cast<int64_t>(b) * p.s.heads + h) * p.s.queries, max(r0, seq.first), min(r0 + BQ, seq.end));
    };
    // Elements of dk and dv that rows the key sees, and others, make no number
    // (a row's P makes all of them, its D those of dk).
    const Elements all = all_elements(p.s.dim);
    Elements own_k{0, 0}, own_v{0, 0}, beside_k{0, 0}, beside_v{0, 0};
    for (int it = from; it < to && __any(bad && !(all.all_in(own_k) && all.all_in(own_v))); ++it) {
        tile(it, [&](int h, int64_t stat, int i0, int i1) __attribute__((always_inline)) {
            const S_<T>*q = qb + h * p.q.head, *g = db + h * p.dout.head;
            const int i = i0 + lane_id;
            bool odd = false, odd_p = false, odd_d = false, none = false;
            if (i < i1) {
                const float bias = p.bias[stat + i];
                none = bias == -INFINITY;
                odd_p = bias != bias;
                odd_d = !finite(p.delta[stat + i]);
                odd = odd_p || odd_d || !row_is_finite<T>(q + i * p.q.token, p.s.dim) || !row_is_finite<T>(g + i * p.dout.token, p.s.dim);
            }
            const uint64_t without = __ballot(none), by_p = __ballot(odd_p), by_d = __ballot(odd_d);
            for (uint64_t found = __ballot(odd); found != 0; found &= found - 1) {
                const int at = __ffsll(static_cast<unsigned long long>(found)) - 1;
                const bool sees = mine <= last && !(without >> at & 1) && p.s.rule.sees(seq.start + i0 + at, mine);
                const Elements in_q = odd_elements<T>(q + (i0 + at) * p.q.token, p.s.dim);
                const Elements in_g = odd_elements<T>(g + (i0 + at) * p.dout.token, p.s.dim);
                beside_k.add(in_q, !sees);
                beside_v.add(in_g, !sees);
                own_k.add((by_p | by_d) >> at & 1 ? all : in_q, sees);
                own_v.add(by_p >> at & 1 ? all : in_g, sees);
            }
        });
    }
    bad = bad && !(beside_k.all_in(own_k) && beside_v.all_in(own_v));
    for_each_question(bad, [&](int lane) __attribute__((always_inline)) {
        const int key = __builtin_amdgcn_readlane(mine, lane);
        const S_<T>*k = kh + key * p.k.token, *v = vh + key * p.v.token;
        Two dk{0.0f, 0.0f}, dv{0.0f, 0.0f};
        for (int it = from; it < to && key <= last; ++it) {
            tile(it, [&](int h, int64_t stat, int i0, int i1) __attribute__((always_inline)) {
                const int i = i0 + lane_id;
                const S_<T>*q = qb + h * p.q.head + i0 * p.q.token, *g = db + h * p.dout.head + i0 * p.dout.token;
                float pr = 0.0f, ds = 0.0f;
                const float bias = i < i1 ? p.bias[stat + i] : -INFINITY;
                const bool sees = bias != -INFINITY && p.s.rule.sees(seq.start + i, key);
                const uint64_t seen = __ballot(sees);
                if (seen == 0) return;
                if (sees) {
                    pr = __builtin_amdgcn_exp2f(fmaf(row_product<T>(q + lane_id * p.q.token, k, p.s.dim), p.scale2, bias - kProbabilityBits<T>));
                    ds = pr * (row_product<T>(g + lane_id * p.dout.token, v, p.s.dim) - p.delta[stat + i]);
                }
                add_rows<T>(dk, ds, q, p.q.token, seen, p.s.dim);
                add_rows<T>(dv, pr, g, p.dout.token, seen, p.s.dim);
            });
        }
        if (walk.parts > 1) {
            float* at = p.part + (walk.at_part * 2 * RB + key - walk.kb * RB) * p.s.dim;
            store_two<float>(at, p.s.dim, dk);
            store_two<float>(at + RB * p.s.dim, p.s.dim, dv);
        } else {
            const int64_t row = ((static_cast<int64_t>(b) * p.s.keys + key) * p.s.kv_heads + hk) * p.s.dim;
            store_two<T>(static_cast<S_<T>*>(p.dk) + row, p.s.dim, Two{dk.x * p.scale, dk.y * p.scale});
            store_two<T>(static_cast<S_<T>*>(p.dv) + row, p.s.dim, dv);
        }
        return mine == key;
    });
}

template <typename T, int DT, int BK, int W>
__global__ __launch_bounds__(W* kWave, W == 1 || (sizeof(S_<T>) == 4 && DT == 4) ? 1 : 2) void attention_dq_kernel(Backward p) {
    using S = S_<T>;
    constexpr int NS = BK / 32, RB = 32 * W;
    using Keys = Tile<T, DT, BK, W>;
    __shared__ __attribute__((aligned(1024))) char k0s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v0s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char k1s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v1s[Keys::kBytes];

    // as in the forward: long walks first, batch and key heads innermost
    const int bh = blockIdx.x % p.pairs, rest = blockIdx.x / p.pairs;
    const int g = rest % p.s.group, qb = p.blocks - 1 - rest / p.s.group;
    const int hk = bh % p.s.kv_heads, b = bh / p.s.kv_heads;
    const int h = hk * p.s.group + g;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, l32 = lane % 32, half = lane / 32;
    const Sequence seq = sequence_of(p.s, b);

    const int mine = qb * RB + wave * 32 + l32;
    const bool alive = mine >= seq.first && mine < seq.end;
    const int row = seq.start + mine;
    const int b0 = max(qb * RB, seq.first), b1 = min(qb * RB + RB, seq.end) - 1;
    const int w0 = seq.start + max(qb * RB + wave * 32, seq.first);
    const int w1 = seq.start + min(qb * RB + wave * 32 + 32, seq.end) - 1;

    f32x16 dq[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) dq[d] = zeros();
    ColumnScale<T> scaled;
    float bias = 0.0f, delta = 0.0f;
    if (b0 <= b1) {
        const int p0 = seq.start + b0, p1 = seq.start + b1;
        const KeyTiles tiles(p.s.rule, p0, p1, BK);
        const S* kh = static_cast<const S*>(p.k.data) + b * p.k.batch + hk * p.k.head;
        const S* vh = static_cast<const S*>(p.v.data) + b * p.v.batch + hk * p.v.head;
        const KeysSeen keep(p.s.rule, tiles, p1);
        typename Keys::Loads k_loads, v_loads;
        k_loads.init(kh, p.k.token, p.s.dim, wave, lane);
        v_loads.init(vh, p.v.token, p.s.dim, wave, lane);
        auto issue = [&](int i, char* kt, char* vt) __attribute__((always_inline)) {
            const int r0 = tiles.at(i) * BK;
            const bool whole = keep.all(r0, r0 + BK - 1);
            k_loads.issue(kt, r0, wave, whole, keep);
            v_loads.issue(vt, r0, wave, whole, keep);
        };
        if (tiles.count > 0) issue(0, k0s, v0s);
        uint4 qf[Keys::kSteps], df[Keys::kSteps];
        {
            auto rows_of = [&](const TokenRows& t) {
                const S* at = static_cast<const S*>(t.data) + b * t.batch + h * t.head + static_cast<int64_t>(qb * RB) * t.token;
                return buffer_over(at, static_cast<uint32_t>(((RB - 1) * t.token + p.s.dim) * sizeof(S)));
            };
            auto row_bytes = [&](const TokenRows& t) { return static_cast<uint32_t>((wave * 32 + l32) * t.token * sizeof(S)); };
            const Rsrc rq = rows_of(p.q), rd = rows_of(p.dout), ro = rows_of(p.o);
#pragma unroll
            for (int s = 0; s < Keys::kSteps; ++s) {
                qf[s] = load_fragment<T>(rq, alive, row_bytes(p.q), s, half, p.s.dim);
                df[s] = load_fragment<T>(rd, alive, row_bytes(p.dout), s, half, p.s.dim);
                const uint4 of = load_fragment<T>(ro, alive, row_bytes(p.o), s, half, p.s.dim);
                float x[Packet<T>::N], y[Packet<T>::N];
                unpack<T>(df[s], x);
                unpack<T>(of, y);
#pragma unroll
                for (int j = 0; j < Packet<T>::N; ++j) delta = fmaf(x[j], y[j], delta);
            }
        }
        delta = both_halves(delta, SumOf{});
        const int64_t stat = (static_cast<int64_t>(b) * p.s.heads + h) * p.s.queries + mine;
        if (alive) {
            // (a row whose sum is 0 has no probabilities, whatever its scores:
            // dk and dv have them as powers of -inf, and D as 0)
            const float l = p.lse[stat];
            bias = l == -INFINITY ? -INFINITY : -l * kLog2E;
        }
        typename Keys::ByRows rows;
        typename Keys::Transposed cols;
        rows.init(lane);
        cols.init(lane);
        // `sums` false: only D, as the sum of P dP, into `exact`
        float exact = 0.0f;
        auto step = [&](auto sums_, int i, const char* kt, const char* vt, char* kn, char* vn) __attribute__((always_inline)) {
            constexpr bool sums = decltype(sums_)::value;
            meet();
            if (i + 1 < tiles.count) issue(i + 1, kn, vn);
            const int j0 = tiles.at(i) * BK;
            if (!p.s.rule.any_sees(w0, w1, j0, j0 + BK - 1)) return;
            const bool whole = p.s.rule.all_see(w0, w1, j0, j0 + BK - 1);
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                f32x16 s = zeros(), ds = zeros();
#pragma unroll
                for (int f = 0; f < Keys::kSteps; ++f) {
                    s = mma<T>(rows.read(kt, u, f), qf[f], s);
                    ds = mma<T>(rows.read(vt, u, f), df[f], ds);
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) ds[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.scale2, bias)) * (sums ? ds[e] - delta : ds[e]);
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        if (!p.s.rule.sees(row, j0 + 32 * u + row_of(e, half))) ds[e] = 0.0f;
                    }
                }
                if constexpr (!sums) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) exact += ds[e];
                    continue;
                }
                scaled.apply(ds, dq);
#pragma unroll
                for (int f = 0; f < kFragsOf32<T>; ++f) {
                    const uint4 sf = pack_rows<T>(ds, f);
#pragma unroll
                    for (int d = 0; d < DT; ++d) dq[d] = mma<T>(cols.read(kt, d, u, f), sf, dq[d]);
                }
            }
        };
        auto walk = [&](auto sums) __attribute__((always_inline)) {
            for (int i = 0; i < tiles.count; i += 2) {
                step(sums, i, k0s, v0s, k1s, v1s);
                if (i + 1 >= tiles.count) break;
                step(sums, i + 1, k1s, v1s, k0s, v0s);
            }
        };
        // Rows of few keys have the largest gradients, and the rounding of
        // their out in D is as large there as that of dS: the D of rows that see
        // at most 128 keys, and of others in their block, which come behind them,
        // is summed up from P and dP, in a walk of its own: a
        // tenth of forward and backward (8192 tokens, 32 heads of 128 under a
        // window of 128 273 us, 242 without) where all rows are such.
        if (sizeof(S) == 2 && p.s.rule.count_seen(p0) <= 128) {
            walk(std::false_type{});
            delta = both_halves(exact, SumOf{});
            meet();
            if (tiles.count > 0) issue(0, k0s, v0s);
        }
        if (alive && half == 0) {
            p.bias[stat] = bias + kProbabilityBits<T>;
            p.delta[stat] = bias == -INFINITY ? 0.0f : delta;
        }
        walk(std::true_type{});
    }
    // A row that is outside its sequence or has no sum, beside keys and values
    // that may be infinite: zeros by selection.
    const bool any = alive && bias != -INFINITY;
    if (mine < p.s.queries) {
        S* out = static_cast<S*>(p.dq) + ((static_cast<int64_t>(b) * p.s.queries + mine) * p.s.heads + h) * p.s.dim;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int at = 32 * d + row_of(e, half);
                if (at >= p.s.dim) continue;
                const auto value = [&](int j) { return any ? dq[d][e + j] * scaled.down() * p.scale : 0.0f; };
                store4<T>(out + at, value(0), value(1), value(2), value(3));
            }
    }
    const bool bad = any && holds_nan(dq) && finite(bias) && finite(delta);
    if (__any(bad)) queries_again<T>(launched_with<Backward>(), b, h, seq.start + b0, seq.start + b1, bad, mine, row, bias, delta);
}

template <typename T, int DT, int BQ, int W>
__global__ __launch_bounds__(W* kWave, W == 1 || sizeof(S_<T>) == 4 ? 1 : 2) void attention_dkv_kernel(Backward p) {
    using S = S_<T>;
    constexpr int NS = BQ / 32, RB = 32 * W;
    // A lone wave has the registers to read all fragments of 32 rows before
    // their products, and the transposed ones between these, where a CU's other
    // waves do not hide the reads: 64 heads of 128 x 512, whole backward, 6 us
    // less (float32, whose products take longer, does not gain).
    constexpr bool kAhead = W == 1 && sizeof(S) == 2;
    using Rows = Tile<T, DT, BQ, W>;
    __shared__ __attribute__((aligned(1024))) char q0s[Rows::kBytes];
    __shared__ __attribute__((aligned(1024))) char d0s[Rows::kBytes];
    __shared__ __attribute__((aligned(1024))) char q1s[Rows::kBytes];
    __shared__ __attribute__((aligned(1024))) char d1s[Rows::kBytes];
    // bias and D of the tiles' rows (64 of each, whatever BQ)
    __shared__ __attribute__((aligned(1024))) float l0s[2 * kWave];
    __shared__ __attribute__((aligned(1024))) float l1s[2 * kWave];

    const KeyWalk<BQ, RB> walk(p);
    const int b = walk.b, hk = walk.hk, kb = walk.kb, last = walk.last, t0 = walk.t0, per_query_head = walk.per_query_head;
    const int from = walk.from, to = walk.to;
    const Sequence& seq = walk.seq;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, l32 = lane % 32, half = lane / 32;
    const int mine = kb * RB + wave * 32 + l32;  // this lane's key
    const int w0 = kb * RB + wave * 32, w1 = min(w0 + 32, seq.length) - 1;

    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) dk[d] = dv[d] = zeros();
    ColumnScale<T> scaled;
    if (from < to) {
        auto keep = [&](int i) { return i >= seq.first && i < seq.end; };
        typename Rows::Loads q_loads, d_loads;
        q_loads.init(static_cast<const S*>(p.q.data) + b * p.q.batch, p.q.token, p.s.dim, wave, lane);
        d_loads.init(static_cast<const S*>(p.dout.data) + b * p.dout.batch, p.dout.token, p.s.dim, wave, lane);
        const S* const q_all = q_loads.head;
        const S* const d_all = d_loads.head;
        // the walk's next tile to load: query head and first row
        int next_h = hk * p.s.group + from / per_query_head, next_row = (t0 + from % per_query_head) * BQ;
        const int end_row = (t0 + per_query_head) * BQ;
        auto issue = [&](char* qt, char* dt, float* lt) __attribute__((always_inline)) {
            const int h = next_h, r0 = next_row;
            next_row += BQ;
            if (next_row == end_row) {
                next_row = t0 * BQ;
                ++next_h;
            }
            q_loads.head = q_all + h * p.q.head;
            d_loads.head = d_all + h * p.dout.head;
            const bool whole = r0 >= seq.first && r0 + BQ <= seq.end;
            q_loads.issue(qt, r0, wave, whole, keep);
            d_loads.issue(dt, r0, wave, whole, keep);
            auto load_stat = [&](int w) {
                const float* at = (w == 0 ? p.bias : p.delta) + (static_cast<int64_t>(b) * p.s.heads + h) * p.s.queries + r0;
                const uint32_t off = lane < BQ && keep(r0 + lane) ? lane * sizeof(float) : kOutOfRange;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_over(at, BQ * sizeof(float)), (LdsPtr)(lt + w * kWave), 4, off, 0, 0, 0);
            };
            if (W > 1) {
                if (wave < 2) load_stat(wave);
            } else {
                load_stat(0);
                load_stat(1);
            }
        };
        int row0 = next_row;  // of the tile at hand
        issue(q0s, d0s, l0s);
        uint4 kf[Rows::kSteps], vf[Rows::kSteps];
        {
            auto rows_of = [&](const TokenRows& t) {
                const S* at = static_cast<const S*>(t.data) + b * t.batch + hk * t.head + static_cast<int64_t>(kb * RB) * t.token;
                return buffer_over(at, static_cast<uint32_t>(((RB - 1) * t.token + p.s.dim) * sizeof(S)));
            };
            auto row_bytes = [&](const TokenRows& t) { return static_cast<uint32_t>((wave * 32 + l32) * t.token * sizeof(S)); };
            const Rsrc rk = rows_of(p.k), rv = rows_of(p.v);
#pragma unroll
            for (int s = 0; s < Rows::kSteps; ++s) {
                kf[s] = load_fragment<T>(rk, mine <= last, row_bytes(p.k), s, half, p.s.dim);
                vf[s] = load_fragment<T>(rv, mine <= last, row_bytes(p.v), s, half, p.s.dim);
            }
        }
        typename Rows::ByRows rows;
        typename Rows::Transposed cols;
        rows.init(lane);
        cols.init(lane);
        // how far this lane's key is seen; a first token to the end
        const int reach_of_mine = mine < p.s.rule.sinks ? kNoWindow : p.s.rule.window;
        auto step = [&](int it, const char* qt, const char* dt, const float* lt, char* qn, char* dn, float* ln) __attribute__((always_inline)) {
            meet();
            const int r0 = row0;
            row0 = next_row;
            if (it + 1 < to) issue(qn, dn, ln);
            const int p0 = seq.start + max(r0, seq.first), p1 = seq.start + min(r0 + BQ, seq.end) - 1;
            if (w0 > w1 || !p.s.rule.any_sees(p0, p1, w0, w1)) return;
            // (rows outside the sequence are zeros here, whose scores with an
            // infinite key are no number: they are masked too)
            const bool whole = p1 - p0 == BQ - 1 && p.s.rule.all_see(p0, p1, w0, w1) && w1 == w0 + 31;
            const unsigned limit = max(min(reach_of_mine, p1 - mine + 1), 0);
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                f32x16 s = zeros(), ds = zeros();
                uint4 qc[kAhead ? Rows::kSteps : 1], dc[kAhead ? Rows::kSteps : 1];
                if constexpr (kAhead) {
                    uint4 qr[Rows::kSteps], dr[Rows::kSteps];
#pragma unroll
                    for (int f = 0; f < Rows::kSteps; ++f) {
                        qr[f] = rows.read(qt, u, f);
                        dr[f] = rows.read(dt, u, f);
                    }
#pragma unroll
                    for (int f = 0; f < Rows::kSteps; ++f) {
                        __builtin_amdgcn_sched_barrier(0);
                        s = mma<T>(qr[f], kf[f], s);
                        ds = mma<T>(dr[f], vf[f], ds);
                        qc[f] = cols.read(qt, f % DT, u, f / DT);
                        dc[f] = cols.read(dt, f % DT, u, f / DT);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                } else {
#pragma unroll
                    for (int f = 0; f < Rows::kSteps; ++f) {
                        s = mma<T>(rows.read(qt, u, f), kf[f], s);
                        ds = mma<T>(rows.read(dt, u, f), vf[f], ds);
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    const int r = 32 * u + row_of(e, half);
                    const float4 l = *reinterpret_cast<const float4*>(lt + r);
                    const float4 d = *reinterpret_cast<const float4*>(lt + kWave + r);
                    const float ls[4] = {l.x, l.y, l.z, l.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[e + j] = __builtin_amdgcn_exp2f(fmaf(s[e + j], p.scale2, ls[j]));
                        ds[e + j] = s[e + j] * (ds[e + j] - dd[j]);
                    }
                }
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        // (unsigned: rows before the key are out of reach too)
                        const unsigned behind = seq.start + r0 + 32 * u + row_of(e, half) - mine;
                        if (behind >= limit) s[e] = ds[e] = 0.0f;
                    }
                }
                scaled.apply(ds, dk);
#pragma unroll
                for (int f = 0; f < kFragsOf32<T>; ++f) {
                    const uint4 pf = pack_rows<T>(s, f), sf = pack_rows<T>(ds, f);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        dv[d] = mma<T>(kAhead ? dc[f * DT + d] : cols.read(dt, d, u, f), pf, dv[d]);
                        dk[d] = mma<T>(kAhead ? qc[f * DT + d] : cols.read(qt, d, u, f), sf, dk[d]);
                    }
                }
            }
        };
        for (int it = from; it < to; it += 2) {
            step(it, q0s, d0s, l0s, q1s, d1s, l1s);
            if (it + 1 >= to) break;
            step(it + 1, q1s, d1s, l1s, q0s, d0s, l0s);
        }
    }
    const bool bad = mine < p.s.keys && (holds_nan(dk) || holds_nan(dv));
    if constexpr (ColumnScale<T>::kOn) {
        constexpr float kDown = 1.0f / (1 << kProbabilityBits<T>);
        const float down = scaled.down() * kDown;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                dk[d][e] *= down;
                dv[d][e] *= kDown;
            }
    }
    if (mine < p.s.keys) {
        const int64_t at_row = ((static_cast<int64_t>(b) * p.s.keys + mine) * p.s.kv_heads + hk) * p.s.dim;
        float* const sums = p.part + (walk.at_part * 2 * RB + wave * 32 + l32) * p.s.dim;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int at = 32 * d + row_of(e, half);
                if (at >= p.s.dim) continue;
                if (walk.parts > 1) {
                    store4<float>(sums + at, dk[d][e], dk[d][e + 1], dk[d][e + 2], dk[d][e + 3]);
                    store4<float>(sums + RB * p.s.dim + at, dv[d][e], dv[d][e + 1], dv[d][e + 2], dv[d][e + 3]);
                } else {
                    store4<T>(static_cast<S*>(p.dk) + at_row + at, dk[d][e] * p.scale, dk[d][e + 1] * p.scale, dk[d][e + 2] * p.scale,
                              dk[d][e + 3] * p.scale);
                    store4<T>(static_cast<S*>(p.dv) + at_row + at, dv[d][e], dv[d][e + 1], dv[d][e + 2], dv[d][e + 3]);
                }
            }
    }
    if (__any(bad)) keys_again<T, BQ, W>(launched_with<Backward>(), bad);
}

// The parts of a block's sums in order, four elements a thread: blockIdx.x
// over a block's rows, y over the blocks of a head that were cut (from
// `first` on), z over batch x key heads.
constexpr int kJoin = 256;

template <typename T, int RB>
__global__ __launch_bounds__(kJoin) void attention_join_kernel(Backward p, int first) {
    const int kb = first + blockIdx.y, bh = blockIdx.z;
    const int hk = bh % p.s.kv_heads, b = bh / p.s.kv_heads;
    const bool sink = kb < p.sink_blocks;
    const int parts = sink ? p.sink_parts : p.near_parts;
    const int slot = sink ? kb * p.sink_parts : p.sums_of_sinks() + (kb - p.sink_blocks) * p.near_parts;
    const int quads = p.s.dim / 4, at = blockIdx.x * kJoin + threadIdx.x;
    const int which = at / (RB * quads), row = at / quads % RB, d = at % quads * 4;
    if (which > 1 || kb * RB + row >= p.s.keys) return;
    const float* from = p.part + (((static_cast<int64_t>(bh) * p.sums() + slot) * 2 + which) * RB + row) * p.s.dim + d;
    float4 t = *reinterpret_cast<const float4*>(from);
#pragma unroll 4
    for (int i = 1; i < parts; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(from + static_cast<int64_t>(i) * 2 * RB * p.s.dim);
        t.x += x.x;
        t.y += x.y;
        t.z += x.z;
        t.w += x.w;
    }
    const float f = which == 0 ? p.scale : 1.0f;
    S_<T>* out = static_cast<S_<T>*>(which == 0 ? p.dk : p.dv) +
                 ((static_cast<int64_t>(b) * p.s.keys + kb * RB + row) * p.s.kv_heads + hk) * p.s.dim + d;
    store4<T>(out, t.x * f, t.y * f, t.z * f, t.w * f);
}

template <typename T, int DT, int R, int W>
void dq_blocks(Backward p, const AttentionArgs& a, hipStream_t on) {
    p.blocks = (a.queries + 32 * W - 1) / (32 * W);
    const int64_t items = static_cast<int64_t>(a.batch) * a.heads * p.blocks;
    const unsigned grid = grid_of(items, W * kWave, "sliding_window_attention_backward");
    attention_dq_kernel<T, DT, R, W><<<grid, W * kWave, 0, on>>>(p);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

template <typename T, int DT, int R, int W>
void dkv_blocks(Backward p, const AttentionArgs& a, int device, hipStream_t on) {
    constexpr int RB = 32 * W;
    const int64_t pairs = p.pairs;
    p.blocks = (a.keys + RB - 1) / RB;
    // Tiles a walk has at most: of one near block, of one that stays visible.
    const int64_t group = p.s.group, tiles = (a.queries + R - 1) / R;
    const int64_t near = group * std::min<int64_t>(tiles, (RB + int64_t{p.s.rule.window} + R - 2) / R + 1), sink = group * tiles;
    TP_AMD_CHECK(sink < (int64_t{1} << 31), "sliding_window_attention_backward: too many queries of one key head");
    p.sink_blocks = std::min(p.blocks, (p.s.rule.sinks + RB - 1) / RB);
    const int64_t want = (W == kWide ? 2 : 4) * cu_count(device);  // blocks that fill the device once
    const int64_t near_blocks = pairs * (p.blocks - p.sink_blocks);
    p.near_parts = near_blocks == 0 ? 1 : static_cast<int>(std::max<int64_t>(1, std::min(want / near_blocks, near / 4)));
    // Parts as long as the other walks, and no more than four rounds of them:
    // each leaves 2 RB rows of sums (4 heads of 128 x 8192 under 4096 first
    // tokens and a window of 1: 160 MB, where parts of 4 tiles took 1.1 GB).
    const int64_t even = sink * pairs * p.sink_blocks / want;
    const int64_t piece = std::max({int64_t{4}, even / 4, near_blocks == 0 ? even : near / p.near_parts});
    p.sink_parts = p.sink_blocks == 0 ? 1 : static_cast<int>(std::max<int64_t>(1, (sink + piece - 1) / piece));
    const int64_t items = pairs * (p.sink_slots() + p.near_slots());
    const unsigned grid = grid_of(items, W * kWave, "sliding_window_attention_backward");
    const bool cut = p.sums() > 0;
    const Workspace part(static_cast<size_t>(pairs * p.sums()) * 2 * RB * a.dim * sizeof(float), device);
    p.part = static_cast<float*>(part.get());
    attention_dkv_kernel<T, DT, R, W><<<grid, W * kWave, 0, on>>>(p);
    TP_AMD_HIP_CHECK(hipGetLastError());
    if (!cut) return;
    const int first = p.sink_parts > 1 ? 0 : p.sink_blocks, end = p.near_parts > 1 ? p.blocks : p.sink_blocks;
    const unsigned wide = static_cast<unsigned>((2 * RB * (a.dim / 4) + kJoin - 1) / kJoin);
    // (walks are cut only where blocks are few: both are far below 2^16)
    attention_join_kernel<T, RB><<<dim3(wide, static_cast<unsigned>(end - first), static_cast<unsigned>(pairs)), kJoin, 0, on>>>(p, first);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

template <typename T, int DT>
void backward_tiles(const AttentionArgs& a, int device) {
    constexpr int R = sizeof(S_<T>) == 2 ? 64 : 32;
    Backward p;
    p.s = shape_of(a);
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.o = a.o;
    p.dout = a.dout;
    p.lse = a.lse;
    p.dq = a.dq;
    p.dk = a.dk;
    p.dv = a.dv;
    p.scale = a.scale;
    p.scale2 = a.scale * kLog2E;
    const int64_t pairs = static_cast<int64_t>(a.batch) * a.kv_heads;
    TP_AMD_CHECK(pairs < (int64_t{1} << 31), "sliding_window_attention_backward: too many heads");
    p.pairs = static_cast<int>(pairs);
    const size_t stats = static_cast<size_t>(a.batch) * a.heads * std::max(a.queries, 1);
    const Workspace found(2 * stats * sizeof(float), device);
    p.bias = static_cast<float*>(found.get());
    p.delta = p.bias + stats;
    const hipStream_t on = stream(device);
    const int64_t cus = cu_count(device), group = p.s.group;
    if (a.queries > 0) {
        // float32, bound by its products, fills more CUs with blocks of one
        // wave: 2 x 1000 queries, 12 heads of 64 (192 wide blocks) 9 us less.
        // 16-bit does not gain: 32 heads x 512 (128) 2.5 us more, x 1024 8 more.
        if (sizeof(S_<T>) == 2 || wide_blocks(a.batch, a.heads, a.queries) >= cus) dq_blocks<T, DT, R, kWide>(p, a, on);
        else if constexpr (sizeof(S_<T>) == 4) dq_blocks<T, DT, 32, 1>(p, a, on);
    }
    if (a.keys == 0) return;
    // Few key blocks: their walks are cut by query heads and rows, and the
    // parts joined.  Blocks of one wave find more room on the CUs, and four
    // waves that share what they load are ahead where there are wide blocks
    // enough or the walks are long; without a window, where they are of every
    // length and parts even them out, sooner.  Whole backward, us, wide and one
    // wave: 64 heads x 512 keys 82 and 70, 8 x 256 47 and 41, 2 x 32 x 768 109
    // and 99, 8 x 1024 80 and 76, 2 key heads of 4 each x 4096 under a window of
    // 512 100 and 91; and 16 x 2000 181 and 195, 8 key heads of 4 each x 1024 114
    // and 120, 4 x 32 x 1024 233 and 242, 8 x 4096 190 and 257; float32 12 x 1000
    // under 256 128 and 111, 8 key heads of 4 each x 1024 281 and 338.
    const bool even = p.s.rule.window < a.queries;
    const int64_t walk = group * std::min(a.queries, p.s.rule.window);
    if (wide_blocks(a.batch, a.kv_heads, a.keys) * group >= 2 * cus || walk >= (even ? 4096 : 1536)) dkv_blocks<T, DT, R, kWide>(p, a, device, on);
    else dkv_blocks<T, DT, 32, 1>(p, a, device, on);
}

template <typename T>
void backward_typed(const AttentionArgs& a, int device) {
    switch ((a.dim + 31) / 32) {
        case 1: return backward_tiles<T, 1>(a, device);
        case 2: return backward_tiles<T, 2>(a, device);
        case 3: return backward_tiles<T, 3>(a, device);
        default: return backward_tiles<T, 4>(a, device);
    }
}

}  // namespace

}  // namespace attention

void launch_attention_backward(int dtype, const AttentionArgs& a, int device) {
    const OnDevice scope(device);
    switch (dtype) {
        case TP_AMD_FLOAT32: attention::backward_typed<float>(a, scope.index()); break;
        case TP_AMD_FLOAT16: attention::backward_typed<f16_t>(a, scope.index()); break;
        case TP_AMD_BFLOAT16: attention::backward_typed<bf16_t>(a, scope.index()); break;
        default: TP_AMD_CHECK(false, "unsupported dtype ", dtype_name(dtype));
    }
}

}  // namespace tp_amd

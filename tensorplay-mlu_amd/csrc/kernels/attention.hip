// Causal attention with a sliding window and first tokens that stay visible,
// forward: prompts and training (a block owns 128 queries of a head), and a
// few queries a sequence over a long cache (the keys split over blocks).
//
// Row p of a head: out = sum_j e^(s_j - l) v_j over the keys it sees,
// s_j = scale q.k_j, l = ln sum_j e^s_j; a row that sees nothing, or that
// stands outside its sequence, gives zeros and l = -inf.  One pass over the
// keys: with m a running bound of the scores (in powers of two) and
// t = sum 2^(s - m), a tile whose scores pass m by more than 2^kSlack scales
// the sums by 2^(m - m') first.  m need not be the maximum, only near enough
// that nothing overflows; most tiles then leave the accumulators alone.
// Scores, statistics and outputs are float32; the probabilities are rounded
// to the operands' type for the matrix instruction, as the values are given
// in it, while t sums them unrounded.

#include <algorithm>

#include "attention_tiles.h"
#include "../allocator.h"
#include "../common.h"
#include "../runtime.h"

namespace tp_amd {

namespace attention {

namespace {

constexpr float kSlack = 8.0f;

struct Forward {
    Shape s;
    TokenRows q, k, v;
    void* out;
    float* lse;
    float scale;  // scale log2 e
    int blocks;   // of 128 queries a head
};

// The running state of a wave's 32 columns (queries).
template <int DT>
struct Columns {
    f32x16 o[DT];
    float m, t;  // t: this lane's share
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = zeros();
        m = -INFINITY;
        t = 0.0f;
    }
    // Scores of NS x 32 keys become probabilities in place.
    template <int NS>
    __device__ __forceinline__ void absorb(f32x16 (&s)[NS], float scale) {
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int e = u == 0 ? 1 : 0; e < 16; ++e) top = fmaxf(top, s[u][e]);
        top = both_halves(top, MaxOf{}) * scale;
        if (__any(top > m + kSlack || (m == -INFINITY && top > m))) {
            const float now = fmaxf(m, top);
            const float turn = now == m ? 1.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            t *= turn;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= turn;
        }
        const float bias = m == -INFINITY ? 0.0f : -m;
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[u][e] = __builtin_amdgcn_exp2f(fmaf(s[u][e], scale, bias));
                t += s[u][e];
            }
    }
};

template <typename T, int DT, int BK>
__global__ __launch_bounds__(4 * kWave, 2) void attention_kernel(Forward p) {
    using S = S_<T>;
    using Keys = Tile<T, DT, BK, 4>;
    constexpr int NS = BK / 32;
    __shared__ __attribute__((aligned(1024))) char k0s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v0s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char k1s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v1s[Keys::kBytes];

    // items: batch, key head, blocks of queries from the last (which sees the
    // most keys) to the first, query head of the group
    const int id = xcd_run(blockIdx.x, gridDim.x);
    const int g = id % p.s.group, rest = id / p.s.group;
    const int qb = p.blocks - 1 - rest % p.blocks, bh = rest / p.blocks;
    const int hk = bh % p.s.kv_heads, b = bh / p.s.kv_heads;
    const int h = hk * p.s.group + g;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, l32 = lane % 32, half = lane / 32;
    const Sequence seq = sequence_of(p.s, b);

    const int mine = qb * 128 + wave * 32 + l32;  // this lane's query
    const bool alive = mine >= seq.first && mine < seq.end;
    const int row = seq.start + mine;
    // the alive rows of the block, and of the wave
    const int b0 = max(qb * 128, seq.first), b1 = min(qb * 128 + 128, seq.end) - 1;
    const int w0 = seq.start + max(qb * 128 + wave * 32, seq.first);
    const int w1 = seq.start + min(qb * 128 + wave * 32 + 32, seq.end) - 1;

    Columns<DT> col;
    col.clear();
    if (b0 <= b1) {
        const int p0 = seq.start + b0, p1 = seq.start + b1;
        const KeyTiles tiles(p.s.rule, p0, p1, BK);
        const S* kh = static_cast<const S*>(p.k.data) + b * p.k.batch + hk * p.k.head;
        const S* vh = static_cast<const S*>(p.v.data) + b * p.v.batch + hk * p.v.head;
        auto keep = [&](int j) { return j <= p1 && (j >= tiles.low_key || j < p.s.rule.sinks); };
        auto issue = [&](int i, char* kt, char* vt) {
            const int r0 = tiles.at(i) * BK;
            Keys::issue(kt, kh, p.k.token, r0, p.s.dim, wave, lane, keep);
            Keys::issue(vt, vh, p.v.token, r0, p.s.dim, wave, lane, keep);
        };
        if (tiles.count > 0) issue(0, k0s, v0s);
        uint4 qf[Keys::kSteps];
        {
            const S* qh = static_cast<const S*>(p.q.data) + b * p.q.batch + h * p.q.head + static_cast<int64_t>(qb * 128) * p.q.token;
            const Rsrc res = buffer_over(qh, static_cast<uint32_t>((127 * p.q.token + p.s.dim) * sizeof(S)));
#pragma unroll
            for (int s = 0; s < Keys::kSteps; ++s) {
                qf[s] = load_fragment<T>(res, alive, static_cast<uint32_t>((wave * 32 + l32) * p.q.token * sizeof(S)), s, half, p.s.dim);
            }
        }
        typename Keys::ByRows rows;
        typename Keys::Transposed cols;
        rows.init(lane);
        cols.init(lane);
        auto step = [&](int i, const char* kt, const char* vt, char* kn, char* vn) {
            meet();  // tile i has landed, and no wave reads the other stage any more
            if (i + 1 < tiles.count) issue(i + 1, kn, vn);
            const int j0 = tiles.at(i) * BK;
            if (!p.s.rule.any_sees(w0, w1, j0, j0 + BK - 1)) return;
            f32x16 s[NS];
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                s[u] = zeros();
#pragma unroll
                for (int f = 0; f < Keys::kSteps; ++f) s[u] = mma<T>(rows.read(kt, u, f), qf[f], s[u]);
            }
            if (!p.s.rule.all_see(w0, w1, j0, j0 + BK - 1)) {
#pragma unroll
                for (int u = 0; u < NS; ++u)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        if (!p.s.rule.sees(row, j0 + 32 * u + row_of(e, half))) s[u][e] = -INFINITY;
                    }
            }
            col.template absorb<NS>(s, p.scale);
#pragma unroll
            for (int u = 0; u < NS; ++u)
#pragma unroll
                for (int f = 0; f < kFragsOf32<T>; ++f) {
                    const uint4 pf = pack_rows<T>(s[u], f);
#pragma unroll
                    for (int d = 0; d < DT; ++d) col.o[d] = mma<T>(cols.read(vt, d, u, f), pf, col.o[d]);
                }
        };
        for (int i = 0; i < tiles.count; i += 2) {
            step(i, k0s, v0s, k1s, v1s);
            if (i + 1 >= tiles.count) break;
            step(i + 1, k1s, v1s, k0s, v0s);
        }
    }
    if (mine >= p.s.queries) return;
    const float total = both_halves(col.t, SumOf{});
    const bool any = alive && total != 0.0f;
    const float inv = any ? 1.0f / total : 0.0f;
    if (half == 0) {
        p.lse[(static_cast<int64_t>(b) * p.s.heads + h) * p.s.queries + mine] = any ? fmaf(col.m, kLn2, logf(total)) : -INFINITY;
    }
    S* out = static_cast<S*>(p.out) + ((static_cast<int64_t>(b) * p.s.queries + mine) * p.s.heads + h) * p.s.dim;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
            const int at = 32 * d + row_of(e, half);
            if (at >= p.s.dim) continue;
            const auto value = [&](int j) { return any ? col.o[d][e + j] * inv : 0.0f; };
            store4<T>(out + at, value(0), value(1), value(2), value(3));
        }
}

template <typename T, int DT>
void forward_tiles(const AttentionArgs& a, int device) {
    constexpr int BK = sizeof(S_<T>) == 2 ? 64 : 32;
    Forward p;
    p.s = shape_of(a);
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.out = a.out;
    p.lse = a.lse;
    p.scale = a.scale * kLog2E;
    p.blocks = (a.queries + 127) / 128;
    const int64_t items = static_cast<int64_t>(a.batch) * a.heads * p.blocks;
    TP_AMD_CHECK(items < (int64_t{1} << 31), "sliding_window_attention: too many rows");
    attention_kernel<T, DT, BK><<<static_cast<unsigned>(items), 4 * kWave, 0, stream(device)>>>(p);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

template <typename T>
void forward_typed(const AttentionArgs& a, int device) {
    switch ((a.dim + 31) / 32) {
        case 1: return forward_tiles<T, 1>(a, device);
        case 2: return forward_tiles<T, 2>(a, device);
        case 3: return forward_tiles<T, 3>(a, device);
        default: return forward_tiles<T, 4>(a, device);
    }
}

}  // namespace

}  // namespace attention

void launch_attention(int dtype, const AttentionArgs& a, int device) {
    const OnDevice scope(device);
    switch (dtype) {
        case TP_AMD_FLOAT32: attention::forward_typed<float>(a, scope.index()); break;
        case TP_AMD_FLOAT16: attention::forward_typed<f16_t>(a, scope.index()); break;
        case TP_AMD_BFLOAT16: attention::forward_typed<bf16_t>(a, scope.index()); break;
        default: TP_AMD_CHECK(false, "unsupported dtype ", dtype_name(dtype));
    }
}

}  // namespace tp_amd

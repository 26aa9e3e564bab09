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

// How far the bound m lies under the scores that set it.  float16 steps by 2^-24
// below 2^-14, and many keys far below the largest can be what a row is made of:
// with its probabilities rounded at 2^7 times their size, 2^15 at most, 2^21 keys
// lose less by those steps than half a step of the result.
template <typename T>
constexpr float kUnder = std::is_same_v<T, f16_t> ? 7.0f : 0.0f;

struct Forward {
    Shape s;
    TokenRows q, k, v;
    void* out;
    float* lse;
    float scale;  // scale log2 e
    int blocks;   // of 128 queries a head
    int pairs;    // batch x key heads
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
    template <typename T, int NS>
    __device__ __forceinline__ void absorb(f32x16 (&s)[NS], float scale) {
        float top = s[0][0];
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
            for (int e = u == 0 ? 1 : 0; e < 16; ++e) top = fmaxf(top, s[u][e]);
        top = both_halves(top, MaxOf{}) * scale - kUnder<T>;
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

// A lane's share of query `mine` of head h: out and l from the sums on bound m.
template <typename T, int DT>
__device__ __forceinline__ void finish_row(const Forward& p, int b, int h, int mine, int half, bool alive, float m, float t,
                                           const Columns<DT>& col) {
    const bool any = alive && t != 0.0f;
    const float inv = any ? 1.0f / t : 0.0f;
    if (half == 0) {
        p.lse[(static_cast<int64_t>(b) * p.s.heads + h) * p.s.queries + mine] = any ? fmaf(m, kLn2, logf(t)) : -INFINITY;
    }
    S_<T>* out = static_cast<S_<T>*>(p.out) + ((static_cast<int64_t>(b) * p.s.queries + mine) * p.s.heads + h) * p.s.dim;
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

// Four elements of query i of head h, and l with the first.
template <typename T>
__device__ __forceinline__ void finish4(const Forward& p, int64_t b, int i, int h, int at, float m, float t, const float (&o)[4]) {
    const bool any = t != 0.0f;
    const float inv = any ? 1.0f / t : 0.0f;
    if (at == 0) p.lse[(b * p.s.heads + h) * p.s.queries + i] = any ? fmaf(m, kLn2, logf(t)) : -INFINITY;
    S_<T>* out = static_cast<S_<T>*>(p.out) + ((b * p.s.queries + i) * p.s.heads + h) * p.s.dim + at;
    const auto value = [&](int j) { return any ? o[j] * inv : 0.0f; };
    store4<T>(out, value(0), value(1), value(2), value(3));
}

// Rows of `out` that hold a NaN and are `bad`, each lane's its own (query i of
// head h at position `row`): see "sums again".
template <typename T>
__device__ __forceinline__ void rows_again(const Forward& p, int b, int hk, int p0, int p1, bool bad, int i, int h, int row) {
    const S_<T>* kh = static_cast<const S_<T>*>(p.k.data) + b * p.k.batch + hk * p.k.head;
    const S_<T>* vh = static_cast<const S_<T>*>(p.v.data) + b * p.v.batch + hk * p.v.head;
    for_each_question(only_beside<T>(p.s, vh, p.v.token, p0, p1, bad, row), [&](int lane) __attribute__((always_inline)) {
        const int iu = __builtin_amdgcn_readlane(i, lane), hu = __builtin_amdgcn_readlane(h, lane);
        const S_<T>* q = static_cast<const S_<T>*>(p.q.data) + b * p.q.batch + iu * p.q.token + hu * p.q.head;
        Two o{0.0f, 0.0f};
        float m = -INFINITY, t = 0.0f;  // t: this lane's share
        for_seen(p.s.rule, __builtin_amdgcn_readlane(row, lane), [&](int j0, uint64_t seen) __attribute__((always_inline)) {
            const int mine = threadIdx.x % kWave;
            const float s = seen >> mine & 1 ? row_product<T>(q, kh + (j0 + mine) * p.k.token, p.s.dim) * p.scale : -INFINITY;
            const float now = fmaxf(m, over_wave(s, MaxOf{}));
            if (now == -INFINITY) return;
            const float turn = __builtin_amdgcn_exp2f(m - now), weight = __builtin_amdgcn_exp2f(s - now);
            m = now;
            t = fmaf(t, turn, weight);
            o.x *= turn;
            o.y *= turn;
            add_rows<T>(o, weight, vh + j0 * p.v.token, p.v.token, seen, p.s.dim);
        });
        const float inv = 1.0f / over_wave(t, SumOf{});
        S_<T>* out = static_cast<S_<T>*>(p.out) + ((static_cast<int64_t>(b) * p.s.queries + iu) * p.s.heads + hu) * p.s.dim;
        store_two<T>(out, p.s.dim, Two{o.x * inv, o.y * inv});
        return i == iu && h == hu;
    });
}

// Of a block of 128 queries, those of a wave.
template <typename T>
__device__ __attribute__((noinline)) void queries_again(const Forward* launched, int b, int hk, int p0, int p1, bool bad, int i, int h, int row) {
    rows_again<T>(as_launched(launched), shared_by_lanes(b), shared_by_lanes(hk), shared_by_lanes(p0), shared_by_lanes(p1), bad, i, h, row);
}

// Whether a row's NaN (if `nan`) is none that its sum has too.
__device__ __forceinline__ bool unexplained(bool nan, float t) { return nan && t > 0.0f && finite(t); }

// A block of four waves owns 128 queries of a head, a wave 32 of them: scores
// are formed transposed, S^T = K Q^T, so that a lane's column is its query, the
// statistics are the lane's own and the probabilities are the next product's
// right operand as they lie in the accumulators.  Queries stay in registers,
// keys and values pass through two stages of LDS, two blocks a CU.
//
// Bound by issue: an exponential, two products, a sum, a maximum and half a
// rounding an element beside the matrix instructions, and with all of them
// running by the card's power, which holds it near 1.9 GHz.  bf16, 32 heads of
// 128 on 8 key heads, 8192 tokens, launched back to back: all earlier keys 523 us,
// 1050 Tflop/s of visible pairs, matrix cores busy 54 % of the cycles, where the
// library's product of 16384 x 16384 makes 1340 to 1370; window 1024 162 to 170 us,
// 770 to 800 Tflop/s, 42 % busy (a block reads 1.18 times the keys its rows see, a
// wave multiplies 1.12 times).  fp16, 4 x 777 queries, 16 heads of 96 on 4 key
// heads, window 1500 of up to 4001 keys: 53 us, 545.
template <typename T, int DT>
__global__ __launch_bounds__(kWide* kWave, sizeof(S_<T>) == 4 && DT == 4 ? 1 : 2) void attention_kernel(Forward p) {
    using S = S_<T>;
    constexpr int BK = sizeof(S) == 2 ? 64 : 32, NS = BK / 32, RB = 32 * kWide;
    using Keys = Tile<T, DT, BK, kWide>;
    __shared__ __attribute__((aligned(1024))) char k0s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v0s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char k1s[Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v1s[Keys::kBytes];

    // Blocks of queries from the last, which sees the most keys, to the first,
    // query heads of the group, then batch and key heads innermost: blocks are
    // dealt over the 8 XCDs in turn, so with a multiple of 8 of those each XCD
    // keeps its own keys and values in its L2, and the short walks come last,
    // where they fill the gaps.
    const int bh = blockIdx.x % p.pairs, rest = blockIdx.x / p.pairs;
    const int g = rest % p.s.group, qb = p.blocks - 1 - rest / p.s.group;
    const int hk = bh % p.s.kv_heads, b = bh / p.s.kv_heads;
    const int h = hk * p.s.group + g;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, l32 = lane % 32, half = lane / 32;
    const Sequence seq = sequence_of(p.s, b);

    const int mine = qb * RB + wave * 32 + l32;  // this lane's query
    const bool alive = mine >= seq.first && mine < seq.end;
    const int row = seq.start + mine;
    // the alive rows of the block, and of the wave
    const int b0 = max(qb * RB, seq.first), b1 = min(qb * RB + RB, seq.end) - 1;
    const int w0 = seq.start + max(qb * RB + wave * 32, seq.first);
    const int w1 = seq.start + min(qb * RB + wave * 32 + 32, seq.end) - 1;

    Columns<DT> col;
    col.clear();
    if (b0 <= b1) {
        const int p0 = seq.start + b0, p1 = seq.start + b1;
        const KeyTiles tiles(p.s.rule, p0, p1, BK);
        const S* kh = static_cast<const S*>(p.k.data) + b * p.k.batch + hk * p.k.head;
        const S* vh = static_cast<const S*>(p.v.data) + b * p.v.batch + hk * p.v.head;
        const KeysSeen keep(p.s.rule, tiles, p1);
        typename Keys::Loads k_loads, v_loads;
        k_loads.init(kh, p.k.token, p.s.dim, wave, lane);
        v_loads.init(vh, p.v.token, p.s.dim, wave, lane);
        auto issue = [&](int i, char* kt, char* vt) {
            const int r0 = tiles.at(i) * BK;
            const bool whole = keep.all(r0, r0 + BK - 1);
            k_loads.issue(kt, r0, wave, whole, keep);
            v_loads.issue(vt, r0, wave, whole, keep);
        };
        if (tiles.count > 0) issue(0, k0s, v0s);
        uint4 qf[Keys::kSteps];
        {
            const S* qh = static_cast<const S*>(p.q.data) + b * p.q.batch + h * p.q.head + static_cast<int64_t>(qb * RB) * p.q.token;
            const Rsrc res = buffer_over(qh, static_cast<uint32_t>(((RB - 1) * p.q.token + p.s.dim) * sizeof(S)));
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
            col.template absorb<T, NS>(s, p.scale);
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
    const float t = both_halves(col.t, SumOf{});
    if (mine < p.s.queries) finish_row<T, DT>(p, b, h, mine, half, alive, col.m, t, col);
    const bool bad = unexplained(alive && holds_nan(col.o), t);
    if (__any(bad)) queries_again<T>(launched_with<Forward>(), b, hk, seq.start + b0, seq.start + b1, bad, mine, h, row);
}

// ---- few queries over many keys -------------------------------------------------

struct Split {
    Forward f;
    int rows, row_tiles;  // packed rows (queries x group) of a key head, tiles of 32 of them
    int tile_rows;        // rows of a tile, but for a key head's last one: fewer
    int splits;
    FastDiv by_splits, by_row_tiles, by_kv_heads, by_group, by_workers;
    // of item i (batch x key head x row tile): m and t, and the sums
    float* stat;  // [items][splits][tile_rows][2]
    float* part;  // [items][splits][tile_rows][dim]
};

// One arrival counter for each item that is split, on a 128-byte line of its
// own (atomics on one line serialize); zero between launches.  A device's
// launches are all on one stream.
constexpr int kCounterStride = 32, kMaxSplitItems = 4096;
__device__ unsigned int split_counters[kMaxSplitItems * kCounterStride];

// Two floats written through to, and read from, the level all XCDs share.
// Relaxed agent-scope stores are acknowledged there before s_waitcnt vmcnt(0)
// returns, so they precede the arrival that is counted after it.
__device__ __forceinline__ void store_shared(float* at, float a, float b) {
    const uint64_t v = static_cast<uint64_t>(__float_as_uint(b)) << 32 | __float_as_uint(a);
    __hip_atomic_store(reinterpret_cast<uint64_t*>(at), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_shared(const float* at) {
    const uint64_t v = __hip_atomic_load(reinterpret_cast<const uint64_t*>(at), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}

// A state (bound m, sum t, four outputs x) added to one on bound `top`.  (A
// bound is a maximum, which passes over NaN: a state that met nothing but NaN
// has m = -inf, as one that met no key, but a sum of NaN.)
__device__ __forceinline__ void add_state(float m, float t, const float4& x, float top, float& total, float (&o)[4]) {
    if (t == 0.0f) return;  // it met no key
    const float turn = __builtin_amdgcn_exp2f(m - top);
    total = fmaf(t, turn, total);
    o[0] = fmaf(x.x, turn, o[0]);
    o[1] = fmaf(x.y, turn, o[1]);
    o[2] = fmaf(x.z, turn, o[2]);
    o[3] = fmaf(x.w, turn, o[3]);
}

// Waves a block: what their private tiles (keys and values, two stages) leave
// room for in LDS.
template <typename T, int DT>
constexpr int kSplitWaves = Tile<T, DT, 32, 1>::kRow == 512 ? 2 : 4;

// What a block of these owns: a split of row tile rt of a key head.
struct SplitItem {
    uint32_t tile, split, rt, b, hk;
    Sequence seq;
    int packed_end, b0, b1;  // its packed rows' end, its first and last alive query
    __device__ __forceinline__ explicit SplitItem(const Split& q) {
        // items: batch, key head, row tile, split
        const uint32_t id = xcd_run(blockIdx.x, gridDim.x);
        tile = fastdiv(id, q.by_splits), split = id - tile * q.splits;
        const uint32_t bh = fastdiv(tile, q.by_row_tiles);
        rt = tile - bh * q.row_tiles;
        b = fastdiv(bh, q.by_kv_heads), hk = bh - b * q.f.s.kv_heads;
    }
    __device__ __forceinline__ void read_sequence(const Split& q) {
        seq = sequence_of(q.f.s, b);
        packed_end = min(static_cast<int>(rt) * 32 + 32, q.rows);
        b0 = max(static_cast<int>(fastdiv(rt * 32, q.by_group)), seq.first);
        b1 = min(static_cast<int>(fastdiv(packed_end - 1, q.by_group)), seq.end - 1);
    }
};

// The rows that a block's threads finished with a NaN: bit k of a thread's `odd`
// for the one of its k-th round, of THREADS quads, QUADS of them a row.
template <typename T, int QUADS, int THREADS>
__device__ __attribute__((noinline)) void tile_again(const Split* launched, unsigned odd) {
    const Split& q = as_launched(launched);
    SplitItem item(q);
    item.read_sequence(q);
    for (int k = 0; __any(odd >> k); ++k) {
        const int packed = item.rt * 32 + (k * THREADS + static_cast<int>(threadIdx.x)) / QUADS, i = fastdiv(packed, q.by_group);
        rows_again<T>(q.f, item.b, item.hk, item.seq.start + item.b0, item.seq.start + item.b1, odd >> k & 1, i,
                      item.hk * q.f.s.group + packed - i * q.f.s.group, item.seq.start + i);
    }
}

// A block owns 32 packed rows of a key head -- all query heads of the group
// and all queries together, so the cache is read once -- and one split of the
// keys they see.  Bound by the cache's bytes: every wave walks a run of 32-key
// tiles of its own, loaded straight into its own part of LDS with the next
// tile's loads always in flight, and meets the others only at the end.  The
// item's last block to arrive adds the splits up, in their order: a second
// launch for it cost 3.9 us where the walk itself takes 7.  bf16, 64 sequences
// of up to 16384 keys, 8 key heads of 128: 546 us, 5.9 TB/s, where a sum
// of 2 GiB reads 6.0; one token over 1024 keys 8.7 us, of which a launch, the
// first loads' way and the arrival are most.
template <typename T, int DT, int AUX>
__global__ __launch_bounds__((kSplitWaves<T, DT> * kWave), 1) void attention_split_kernel(Split q) {
    using S = S_<T>;
    using Keys = Tile<T, DT, 32, 1, AUX>;
    constexpr int W = kSplitWaves<T, DT>;
    __shared__ __attribute__((aligned(1024))) char k0s[W * Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v0s[W * Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char k1s[W * Keys::kBytes];
    __shared__ __attribute__((aligned(1024))) char v1s[W * Keys::kBytes];
    __shared__ float ms[W][32], ts[W][32];
    __shared__ int last;
    const Forward& p = q.f;

    SplitItem item(q);
    const uint32_t tile = item.tile, split = item.split, rt = item.rt, b = item.b, hk = item.hk;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int lane = threadIdx.x % kWave, l32 = lane % 32, half = lane / 32;

    const int packed = rt * 32 + l32;
    const int mine = fastdiv(packed, q.by_group), h = hk * p.s.group + packed - mine * p.s.group;
    // The queries, on their way while the sequence's length is.
    uint4 qf[Keys::kSteps];
    {
        const S* from_row = static_cast<const S*>(p.q.data) + b * p.q.batch + mine * p.q.token + h * p.q.head;
#pragma unroll
        for (int s = 0; s < Keys::kSteps; ++s) {
            const int e = (2 * s + half) * Packet<T>::N;
            qf[s] = packed < q.rows && e < p.s.dim ? *reinterpret_cast<const uint4*>(from_row + e) : make_uint4(0, 0, 0, 0);
        }
    }
    item.read_sequence(q);
    const Sequence& seq = item.seq;
    const bool alive = packed < q.rows && mine >= seq.first && mine < seq.end;
    const int row = seq.start + mine;
    const int packed_end = item.packed_end, b0 = item.b0, b1 = item.b1;

    Columns<DT> col;
    col.clear();
    if (b0 <= b1) {
        const int p0 = seq.start + b0, p1 = seq.start + b1;
        const KeyTiles tiles(p.s.rule, p0, p1, 32);
        const int run = fastdiv(tiles.count + q.splits * W - 1, q.by_workers);
        const int from = min(static_cast<int>(split * W + wave) * run, tiles.count), to = min(from + run, tiles.count);
        if (from < to) {
            const S* kh = static_cast<const S*>(p.k.data) + b * p.k.batch + hk * p.k.head;
            const S* vh = static_cast<const S*>(p.v.data) + b * p.v.batch + hk * p.v.head;
            const KeysSeen keep(p.s.rule, tiles, p1);
            const int at = wave * Keys::kBytes;
            typename Keys::Loads k_loads, v_loads;
            k_loads.init(kh, p.k.token, p.s.dim, 0, lane);
            v_loads.init(vh, p.v.token, p.s.dim, 0, lane);
            auto issue = [&](int i, char* kt, char* vt) __attribute__((always_inline)) {
                const int r0 = tiles.at(i) * 32;
                const bool whole = keep.all(r0, r0 + 31);
                k_loads.issue(kt + at, r0, 0, whole, keep);
                v_loads.issue(vt + at, r0, 0, whole, keep);
            };
            issue(from, k0s, v0s);
#pragma unroll
            for (int s = 0; s < Keys::kSteps; ++s) qf[s] = alive ? qf[s] : make_uint4(0, 0, 0, 0);
            typename Keys::ByRows rows;
            typename Keys::Transposed cols;
            rows.init(lane);
            cols.init(lane);
            auto step = [&](int i, const char* kt, const char* vt, char* kn, char* vn) __attribute__((always_inline)) {
                const bool more = i + 1 < to;
                if (more) {
                    reads_done();
                    issue(i + 1, kn, vn);
                    wait_but<3 * Keys::kIssue>();  // this tile's keys are there
                } else {
                    wait_but<Keys::kIssue>();
                }
                const int j0 = tiles.at(i) * 32;
                f32x16 s[1] = {zeros()};
#pragma unroll
                for (int f = 0; f < Keys::kSteps; ++f) s[0] = mma<T>(rows.read(kt + at, 0, f), qf[f], s[0]);
                if (!p.s.rule.all_see(p0, p1, j0, j0 + 31)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        if (!p.s.rule.sees(row, j0 + row_of(e, half))) s[0][e] = -INFINITY;
                    }
                }
                col.template absorb<T, 1>(s, p.scale);
                if (more) wait_but<2 * Keys::kIssue>();  // and its values
                else wait_but<0>();
#pragma unroll
                for (int f = 0; f < kFragsOf32<T>; ++f) {
                    const uint4 pf = pack_rows<T>(s[0], f);
#pragma unroll
                    for (int d = 0; d < DT; ++d) col.o[d] = mma<T>(cols.read(vt + at, d, 0, f), pf, col.o[d]);
                }
            };
            for (int i = from; i < to; i += 2) {
                step(i, k0s, v0s, k1s, v1s);
                if (i + 1 >= to) break;
                step(i + 1, k1s, v1s, k0s, v0s);
            }
        }
    }
    // The waves' sums in LDS, where their tiles were; then all threads add
    // them up on one bound, a thread four elements of a row, wave 0's first.
    const float t = both_halves(col.t, SumOf{});
    if (half == 0) {
        ms[wave][l32] = alive ? col.m : -INFINITY;
        ts[wave][l32] = alive ? t : 0.0f;
    }
    // Rows of the sums: 32 lanes store at one column of 32 rows, so a row's
    // 16-byte pieces are turned by its number (24 of them: padded instead).
    constexpr int kLine = DT == 3 ? 100 : DT * 32, kSums = 32 * kLine;  // floats a row, a wave
    static_assert(2 * W * Keys::kBytes >= W * kSums * 4, "half of the waves' sums fit where the keys, half where the values were");
    auto piece = [](int r, int quad) { return r * kLine + 4 * (DT == 3 ? quad : quad ^ (r & (DT * 8 - 1))); };
    auto sums_of = [&](int w) { return reinterpret_cast<float*>(w < W / 2 ? k0s : v0s) + w % (W / 2) * kSums; };
    // a wave's tiles may still be read by no one but itself, but its sums lie
    // where others' tiles were
    __syncthreads();
    if (packed < q.rows) {
        float* const at = sums_of(wave);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                store4<float>(at + piece(l32, (32 * d + row_of(e, half)) / 4), col.o[d][e], col.o[d][e + 1], col.o[d][e + 2],
                              col.o[d][e + 3]);
            }
    }
    __syncthreads();
    const int quads = p.s.dim / 4, rows_here = packed_end - rt * 32;
    unsigned odd = 0;  // the rounds of the threads in which this one finished a row with a NaN
    auto finish = [&](int at, int r, int quad, float m, float total, const float (&o)[4]) __attribute__((always_inline)) {
        const int packed_r = rt * 32 + r, i = fastdiv(packed_r, q.by_group);
        finish4<T>(p, b, i, hk * p.s.group + packed_r - i * p.s.group, 4 * quad, m, total, o);
        const float x = (o[0] + o[1]) + (o[2] + o[3]);
        if (unexplained(x != x, total)) odd |= 1u << at / (W * kWave);
    };
    auto again = [&]() __attribute__((always_inline)) {
        if (__any(odd != 0)) tile_again<T, DT * 8, W * kWave>(launched_with<Split>(), odd);
    };
    float* const stat = q.stat + (static_cast<int64_t>(tile) * q.splits + split) * q.tile_rows * 2;
    for (int at = threadIdx.x; at < rows_here * DT * 8; at += W * kWave) {
        const int r = at / (DT * 8), quad = at % (DT * 8);
        if (quad >= quads) continue;
        float m = ms[0][r];
#pragma unroll
        for (int w = 1; w < W; ++w) m = fmaxf(m, ms[w][r]);
        float total = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float4 x = *reinterpret_cast<const float4*>(sums_of(w) + piece(r, quad));
            add_state(ms[w][r], ts[w][r], x, m, total, o);
        }
        if (q.splits == 1) {
            finish(at, r, quad, m, total, o);
            continue;
        }
        if (quad == 0) store_shared(stat + 2 * r, m, total);
        float* part = q.part + ((static_cast<int64_t>(tile) * q.splits + split) * q.tile_rows + r) * p.s.dim + 4 * quad;
        store_shared(part, o[0], o[1]);
        store_shared(part + 2, o[2], o[3]);
    }
    if (q.splits == 1) return again();
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned int* counter = &split_counters[tile * kCounterStride];
        last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == q.splits - 1u;
        if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    // All splits' m and t where the sums were.
    float2* const stats = reinterpret_cast<float2*>(k0s);
    const float* all = q.stat + static_cast<int64_t>(tile) * q.splits * q.tile_rows * 2;
    for (int at = threadIdx.x; at < q.splits * q.tile_rows; at += W * kWave) stats[at] = load_shared(all + 2 * at);
    __syncthreads();
    for (int at = threadIdx.x; at < rows_here * DT * 8; at += W * kWave) {
        const int r = at / (DT * 8), quad = at % (DT * 8);
        if (quad >= quads) continue;
        const int64_t step = static_cast<int64_t>(q.tile_rows) * p.s.dim;
        const float* part = q.part + static_cast<int64_t>(tile) * q.splits * step + r * p.s.dim + 4 * quad;
        float m = -INFINITY;
        for (int s = 0; s < q.splits; ++s) m = fmaxf(m, stats[s * q.tile_rows + r].x);
        float total = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        constexpr int kAhead = 8;  // splits whose loads go out together
        for (int s0 = 0; s0 < q.splits; s0 += kAhead) {
            float2 lo[kAhead], hi[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int s = s0 + k < q.splits ? s0 + k : q.splits - 1;
                lo[k] = load_shared(part + s * step);
                hi[k] = load_shared(part + s * step + 2);
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (s0 + k >= q.splits) break;
                const float2 x = stats[(s0 + k) * q.tile_rows + r];
                add_state(x.x, x.y, make_float4(lo[k].x, lo[k].y, hi[k].x, hi[k].y), m, total, o);
            }
        }
        finish(at, r, quad, m, total, o);
    }
    again();
}

Forward forward_of(const AttentionArgs& a) {
    Forward p;
    p.s = shape_of(a);
    p.q = a.q;
    p.k = a.k;
    p.v = a.v;
    p.out = a.out;
    p.lse = a.lse;
    p.scale = a.scale * kLog2E;
    TP_AMD_CHECK(static_cast<int64_t>(a.batch) * a.kv_heads < (int64_t{1} << 31), "sliding_window_attention: too many heads");
    p.pairs = static_cast<int>(static_cast<int64_t>(a.batch) * a.kv_heads);
    return p;
}

template <typename T, int DT>
void split_tiles(const AttentionArgs& a, int device) {
    Split q;
    q.f = forward_of(a);
    const Rule& rule = q.f.s.rule;
    q.rows = a.queries * q.f.s.group;
    q.row_tiles = (q.rows + 31) / 32;
    q.tile_rows = std::min(q.rows, 32);
    // Tiles of 32 keys that a row tile sees at most (32 packed rows are at most
    // 32 queries), and blocks that fill the device.
    const int64_t near = std::min<int64_t>(a.keys, int64_t{rule.window} + 31) + 31, sinks = std::min(rule.sinks, a.keys) + 31;
    const int64_t tiles = std::min<int64_t>((a.keys + 31) / 32, near / 32 + 1 + sinks / 32);
    const int64_t items = static_cast<int64_t>(a.batch) * a.kv_heads * q.row_tiles;
    constexpr int W = kSplitWaves<T, DT>;
    const int64_t cus = cu_count(device), here = q.tile_rows;
    // Long walks (32 tiles and more a wave) in eight rounds of blocks, which
    // evens out sequences of different lengths: 64 x 16384 keys 546 us against
    // 570 in one; short ones in one, a block costs some 8 us besides its walk:
    // 16 x 2000 keys 17 us against 23 in two.
    const int64_t rounds = tiles * items >= 32 * W * cus ? 8 : 1;
    // The last block reads every split's sums back: no more splits than make
    // that as long as a split's own walk; and their m and t fit in LDS.
    const int64_t walk = tiles * 64 * sizeof(S_<T>), back = here * sizeof(float);
    int64_t splits = std::min({rounds * cus / items, (tiles + W - 1) / W, int64_t(W) * Tile<T, DT, 32, 1>::kBytes / 8 / here});
    while (splits > 1 && splits * splits * back > walk) --splits;
    q.splits = items > kMaxSplitItems ? 1 : static_cast<int>(std::max<int64_t>(1, splits));
    const unsigned grid = grid_of(items * q.splits, W * kWave, "sliding_window_attention");
    q.by_splits = make_fastdiv(static_cast<uint32_t>(q.splits));
    q.by_row_tiles = make_fastdiv(static_cast<uint32_t>(q.row_tiles));
    q.by_kv_heads = make_fastdiv(static_cast<uint32_t>(a.kv_heads));
    q.by_group = make_fastdiv(static_cast<uint32_t>(q.f.s.group));
    q.by_workers = make_fastdiv(static_cast<uint32_t>(q.splits * W));
    Workspace part;
    if (q.splits > 1) {
        const int64_t slots = items * q.splits * here;
        part = Workspace(static_cast<size_t>(slots * (a.dim + 2)) * sizeof(float), device);
        q.part = static_cast<float*>(part.get());
        q.stat = q.part + slots * a.dim;
    }
    // A cache larger than the Infinity Cache is half full of, read once, passes
    // by it: 64 x 16384 keys 558 us against 611; a small one comes from it
    // again (16 x 2000 keys 20.1 us non-temporal, 19.4 so).
    const int64_t bytes = 2 * int64_t{32} * tiles * a.batch * a.kv_heads * a.dim * sizeof(S_<T>);
    auto* kernel = q.row_tiles == 1 && bytes > (int64_t{128} << 20) ? attention_split_kernel<T, DT, kNt> : attention_split_kernel<T, DT, 0>;
    kernel<<<grid, W * kWave, 0, stream(device)>>>(q);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

// The split kernel also takes more packed rows than one tile of 32 where the
// wide blocks are few and a round of its own blocks, one a CU, is enough
// (float32, bound by its products: two rounds).  bf16, 32 heads of 128 on 8 key
// heads over a window of 1024: 64 queries 15.9 us against 27.7 in wide blocks,
// 256 (256 row tiles) 18.0 and 31.0, 512 33.4 and 31.3; float32, 12 heads of 64,
// 1000 queries (384 row tiles) 26.3 and 37.1.  Up to 64 packed rows (two
// tiles) it takes any batch: wide blocks would hold mostly padding.
template <typename T>
bool takes_split(const AttentionArgs& a, int device) {
    const int64_t rows = static_cast<int64_t>(a.queries) * (a.heads / a.kv_heads), cus = cu_count(device);
    const int64_t tiles = static_cast<int64_t>(a.batch) * a.kv_heads * ((rows + 31) / 32);
    return rows <= 64 || tiles <= (sizeof(S_<T>) == 4 ? 2 : 1) * cus;
}

template <typename T, int DT>
void forward_tiles(const AttentionArgs& a, int device) {
    if (takes_split<T>(a, device)) return split_tiles<T, DT>(a, device);
    Forward p = forward_of(a);
    p.blocks = (a.queries + 32 * kWide - 1) / (32 * kWide);
    const int64_t items = static_cast<int64_t>(p.pairs) * p.s.group * p.blocks;
    const unsigned grid = grid_of(items, kWide * kWave, "sliding_window_attention");
    attention_kernel<T, DT><<<grid, kWide * kWave, 0, stream(device)>>>(p);
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

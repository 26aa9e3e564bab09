// Log probabilities of given tokens with the entropy of each row and its
// likeliest tokens, and the gradient of the first two.
//
// For a row x of logits, c the scale: m = max x, S = sum e^(c (x - m)),
// E = sum e^(c (x - m)) c (x - m); the log probability of token t is
// c (x_t - m) - ln S and the entropy ln S - E / S.  The logits are read once:
// each thread keeps its own running m, S and E and rescales them when its
// maximum moves.  Backward, p_j = e^(c (x_j - m)) / S:
//   dx_j = c (da ([j = t] - p_j) - db p_j (ln p_j + H)).
//
// The likeliest tokens come from the same pass.  A block looks at its first
// chunk's largest element of each thread: the `top`-th largest of those in a
// wave is a bound that at least `top` elements reach.  Elements that reach the
// bound go to a list in LDS, in chunks of rising index, so a later element
// that only equals the bound is never wanted.  Where too many reach it (equal
// logits) the list is cut down to its best between packets.
//
// Bound by memory; a row is split over blocks where rows are few, and a second
// kernel joins the splits.

#include <algorithm>

#include "attention.h"
#include "device_common.h"
#include "layers.h"
#include "math_ops.h"
#include "../allocator.h"
#include "../common.h"
#include "../runtime.h"

namespace tp_amd {

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / kWave;
constexpr int kUnits = 4;  // packets a thread and chunk
constexpr float kLowest = -3.402823466e38f;
// What an exponent is held above: 2^-4096 is 0 and times a finite number stays 0.
constexpr float kFloor = -4096.0f;

template <typename T>
using S_ = typename Elem<T>::storage;

struct Plan {
    TokenProbsArgs p;
    int splits;
    int64_t span;  // elements of a split: whole chunks' packets
    float c;       // scale log2 e
    float* part;   // [rows][splits][3]
    uint64_t* part_top;  // [rows][splits][top]
};

// The larger; NaN where either is.
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// Whole numbers in the order of the floats, NaN above all.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t u = __float_as_uint(f);
    if (f != f) return 0xffffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float from_ordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// Larger values first, of equal ones the lower index; an element of -0 counts
// as 0 (`ordered` of v + 0).
__device__ __forceinline__ uint64_t key_of(float v, uint32_t index) {
    return static_cast<uint64_t>(ordered(v + 0.0f)) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xffffffffu - static_cast<uint32_t>(key); }

// Running statistics: the largest logit, S and E (in powers of two) against it.
struct Stats {
    float m, s, e;
};

__device__ __forceinline__ void join(Stats& a, const Stats& b, float c) {
    const float m = larger(a.m, b.m);
    const float da = larger((a.m - m) * c, kFloor), db = larger((b.m - m) * c, kFloor);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    a.e = fmaf(a.s, da, a.e) * fa + fmaf(b.s, db, b.e) * fb;
    a.s = a.s * fa + b.s * fb;
    a.m = m;
}

__device__ __forceinline__ int64_t target_at(const TokenProbsArgs& p, int64_t r) {
    return p.wide_target ? static_cast<const int64_t*>(p.target)[r] : static_cast<const int32_t*>(p.target)[r];
}

// Results of a row from its statistics.  A row without a finite or larger
// logit has the sum 0 and NaN for results.
template <typename T>
__device__ __forceinline__ void write_row(const Plan& w, int64_t r, const Stats& t) {
    const float ls = logf(t.s);
    w.p.stats[2 * r] = t.s == 0.0f ? -__builtin_inff() : t.m;  // every logit -inf
    w.p.stats[2 * r + 1] = ls;
    if (w.p.entropy != nullptr) w.p.entropy[r] = ls - t.e / t.s * kLn2;
    if (w.p.target != nullptr) {
        const int64_t at = target_at(w.p, r);
        float lp = __uint_as_float(0x7fc00000u);
        if (at >= 0 && at < w.p.vocab) {
            lp = fmaf(Elem<T>::load(static_cast<const S_<T>*>(w.p.logits.data)[r * w.p.logits.step + at]) - t.m, w.p.scale, -ls);
        }
        w.p.logprob[r] = lp;
    }
}

__device__ __forceinline__ void write_top(const Plan& w, int64_t r, int i, uint64_t key, const Stats& t) {
    w.p.top_values[r * w.p.top + i] = fmaf(from_ordered(static_cast<uint32_t>(key >> 32)) - t.m, w.p.scale, -logf(t.s));
    w.p.top_index[r * w.p.top + i] = index_of(key);
}

// The skipped row's results.
__device__ __forceinline__ void write_skipped(const Plan& w, int64_t r, int thread, int threads) {
    for (int i = thread; i < w.p.top; i += threads) {
        w.p.top_values[r * w.p.top + i] = 0.0f;
        w.p.top_index[r * w.p.top + i] = -1;
    }
    if (thread != 0) return;
    w.p.logprob[r] = 0.0f;
    w.p.stats[2 * r] = w.p.stats[2 * r + 1] = 0.0f;
    if (w.p.entropy != nullptr) w.p.entropy[r] = 0.0f;
}

// A wave's 64 keys in falling order.
__device__ __forceinline__ uint32_t wave_sorted(uint32_t v) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int size = 2; size <= kWave; size *= 2) {
#pragma unroll
        for (int step = size / 2; step > 0; step /= 2) {
            const uint32_t other = wave_shfl_xor(v, step);
            const bool low = (lane & step) == 0, falling = (lane & size) == 0;
            v = (low == falling) ? (v > other ? v : other) : (v < other ? v : other);
        }
    }
    return v;
}

__device__ __forceinline__ uint64_t wave_largest(uint64_t v) {
#pragma unroll
    for (int m = kWave / 2; m > 0; m /= 2) {
        const uint64_t other = wave_shfl_xor(v, m);
        v = v > other ? v : other;
    }
    return v;
}

// The block's list of candidates: `list` holds `n` keys, `bound` the least
// ordered value worth a look, strictly above it where `strict`.
template <int CAP>
struct Candidates {
    uint64_t list[CAP];
    uint64_t best[kTokenProbsMaxTop];
    uint64_t wave_best[kWaves];
    uint32_t wave_top[kWaves][2];
    uint32_t n;
};

// Cuts the list to its `top` best, in falling order.  All threads; the list
// and n are visible on entry and on return.
template <int CAP>
__device__ void cut(Candidates<CAP>& c, int top) {
    constexpr int PER = (CAP + kBlock - 1) / kBlock;
    const uint32_t n = c.n;
    uint64_t mine[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) mine[i] = threadIdx.x + i * kBlock < n ? c.list[threadIdx.x + i * kBlock] : 0;
    const int want = n < static_cast<uint32_t>(top) ? static_cast<int>(n) : top;
    for (int k = 0; k < want; ++k) {
        uint64_t v = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) v = mine[i] > v ? mine[i] : v;
        v = wave_largest(v);
        if (threadIdx.x % kWave == 0) c.wave_best[threadIdx.x / kWave] = v;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) v = c.wave_best[i] > v ? c.wave_best[i] : v;
        // keys differ (by their index), so one element leaves
#pragma unroll
        for (int i = 0; i < PER; ++i) mine[i] = mine[i] == v ? 0 : mine[i];
        if (threadIdx.x == 0) c.best[k] = v;
        __syncthreads();
    }
    if (threadIdx.x < static_cast<unsigned>(want)) c.list[threadIdx.x] = c.best[threadIdx.x];
    if (threadIdx.x == 0) c.n = want;
    __syncthreads();
}

template <typename T, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(kBlock) void token_log_probs_kernel(Plan w) {
    constexpr int N = Packet<T>::N;
    constexpr int CAP = kBlock * N + kTokenProbsMaxTop;
    __shared__ Stats wave_stats[kWaves];
    __shared__ std::conditional_t<TOP, Candidates<CAP>, int> shared;
    const int64_t r = blockIdx.x / static_cast<unsigned>(w.splits);
    const int split = static_cast<int>(blockIdx.x % static_cast<unsigned>(w.splits));
    if (w.p.target != nullptr && target_at(w.p, r) == w.p.ignore) {
        if (split == 0) write_skipped(w, r, threadIdx.x, kBlock);
        return;
    }
    const int64_t first = split * w.span, end = first + w.span < w.p.vocab ? first + w.span : w.p.vocab;
    const S_<T>* x = static_cast<const S_<T>*>(w.p.logits.data) + r * w.p.logits.step;
    Stats st{kLowest, 0.0f, 0.0f};
    uint32_t bound = 0, have = 0;
    bool strict = false, begun = false;
    if constexpr (TOP) {
        if (threadIdx.x == 0) shared.n = 0;
        __syncthreads();
    }
    for (int64_t base = first; base < end; base += kBlock * N * kUnits) {
        float f[kUnits][N];
        const int64_t at0 = base + threadIdx.x * N;
        uint4 raw[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int64_t at = at0 + u * kBlock * N;
            if (at + N <= end) raw[u] = load_raw_any_nt(x + at);
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int64_t at = at0 + u * kBlock * N;
            if (at + N <= end) {
                unpack<T>(raw[u], f[u]);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) f[u][j] = at + j < end ? Elem<T>::load(x[at + j]) : -__builtin_inff();
            }
        }
        float cm = f[0][0];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
#pragma unroll
            for (int j = 0; j < N; ++j) cm = larger(cm, f[u][j]);
        }
        const float m = larger(st.m, cm);
        {
            const float d = larger((st.m - m) * w.c, kFloor), scale = __builtin_amdgcn_exp2f(d);
            if constexpr (ENTROPY) st.e = fmaf(st.s, d, st.e) * scale;
            st.s *= scale;
            st.m = m;
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float d = larger((f[u][j] - m) * w.c, kFloor), e = __builtin_amdgcn_exp2f(d);
                st.s += e;
                if constexpr (ENTROPY) st.e = fmaf(e, d, st.e);
            }
        }
        if constexpr (TOP) {
            const int top = w.p.top;
            if (!begun) {
                const uint32_t sorted = wave_sorted(ordered(cm + 0.0f));
                const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
                if (lane == top - 1) shared.wave_top[wave][0] = sorted;
                if (lane == (top + kWaves - 1) / kWaves - 1) shared.wave_top[wave][1] = sorted;
                __syncthreads();
                // `top` threads of one wave reach its first number, a quarter as many of every wave the least second one
                uint32_t most = 0, least = 0xffffffffu;
#pragma unroll
                for (int i = 0; i < kWaves; ++i) {
                    most = shared.wave_top[i][0] > most ? shared.wave_top[i][0] : most;
                    least = shared.wave_top[i][1] < least ? shared.wave_top[i][1] : least;
                }
                bound = most > least ? most : least;
                begun = true;
            }
            auto wanted = [&](float v) {
                const uint32_t o = ordered(v + 0.0f);
                return strict ? o > bound : o >= bound;
            };
            uint32_t mine = 0;
            if (wanted(cm)) {
#pragma unroll
                for (int u = 0; u < kUnits; ++u) {
#pragma unroll
                    for (int j = 0; j < N; ++j) mine += at0 + u * kBlock * N + j < end && wanted(f[u][j]) ? 1 : 0;
                }
            }
            uint32_t place = mine ? atomicAdd(&shared.n, mine) : 0;
            __syncthreads();
            const uint32_t total = shared.n;
            __syncthreads();
            if (total <= CAP) {
                if (mine) {
#pragma unroll
                    for (int u = 0; u < kUnits; ++u) {
#pragma unroll
                        for (int j = 0; j < N; ++j) {
                            const int64_t at = at0 + u * kBlock * N + j;
                            if (at < end && wanted(f[u][j])) shared.list[place++] = key_of(f[u][j], static_cast<uint32_t>(at));
                        }
                    }
                }
            } else {
                // packet by packet, the list cut to its best before each
                if (threadIdx.x == 0) shared.n = have;
                __syncthreads();
                for (int u = 0; u < kUnits; ++u) {
                    if (shared.n > static_cast<uint32_t>(top)) {
                        cut(shared, top);
                        bound = static_cast<uint32_t>(shared.list[top - 1] >> 32);
                        strict = true;
                    }
                    __syncthreads();
#pragma unroll
                    for (int j = 0; j < N; ++j) {
                        float v = f[0][j];
#pragma unroll
                        for (int i = 1; i < kUnits; ++i) v = i == u ? f[i][j] : v;
                        const int64_t at = at0 + u * kBlock * N + j;
                        if (at < end && wanted(v)) shared.list[atomicAdd(&shared.n, 1u)] = key_of(v, static_cast<uint32_t>(at));
                    }
                    __syncthreads();
                }
            }
            have = total <= CAP ? total : shared.n;
            // at least `top` elements so far reach the bound, all of lower index than what follows
            strict = true;
        }
    }
    // the threads' statistics as one
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) {
        const Stats other{wave_shfl_xor(st.m, i), wave_shfl_xor(st.s, i), wave_shfl_xor(st.e, i)};
        join(st, other, w.c);
    }
    if (threadIdx.x % kWave == 0) wave_stats[threadIdx.x / kWave] = st;
    __syncthreads();
    st = wave_stats[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) join(st, wave_stats[i], w.c);
    if constexpr (TOP) cut(shared, w.p.top);
    if (w.splits == 1) {
        if (threadIdx.x == 0) write_row<T>(w, r, st);
        if constexpr (TOP) {
            if (threadIdx.x < static_cast<unsigned>(w.p.top)) write_top(w, r, threadIdx.x, shared.list[threadIdx.x], st);
        }
        return;
    }
    const int64_t at = r * w.splits + split;
    if (threadIdx.x == 0) {
        w.part[3 * at] = st.m;
        w.part[3 * at + 1] = st.s;
        w.part[3 * at + 2] = st.e;
    }
    if constexpr (TOP) {
        const unsigned n = shared.n;
        if (threadIdx.x < static_cast<unsigned>(w.p.top)) w.part_top[at * w.p.top + threadIdx.x] = threadIdx.x < n ? shared.list[threadIdx.x] : 0;
    }
}

// A wave joins a row's splits, one a lane; the best of the lanes' lists, each
// in falling order, leave one after another.
template <typename T>
__global__ __launch_bounds__(kWave) void token_log_probs_join_kernel(Plan w) {
    const int64_t r = blockIdx.x;
    const int lane = threadIdx.x;
    if (w.p.target != nullptr && target_at(w.p, r) == w.p.ignore) return;
    Stats st{kLowest, 0.0f, 0.0f};
    const int64_t at = r * w.splits + lane;
    if (lane < w.splits) st = Stats{w.part[3 * at], w.part[3 * at + 1], w.part[3 * at + 2]};
#pragma unroll
    for (int i = 1; i < kWave; i *= 2) {
        const Stats other{wave_shfl_xor(st.m, i), wave_shfl_xor(st.s, i), wave_shfl_xor(st.e, i)};
        join(st, other, w.c);
    }
    if (lane == 0) write_row<T>(w, r, st);
    const int top = w.p.top;
    int next = 0;
    for (int k = 0; k < top; ++k) {
        const uint64_t mine = lane < w.splits && next < top ? w.part_top[at * top + next] : 0;
        const uint64_t v = wave_largest(mine);
        if (mine == v) ++next;
        if (lane == k) write_top(w, r, k, v, st);
    }
}

// dx of kUnits packets a thread; a row's blocks follow one another.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(kBlock) void token_log_probs_backward_kernel(Plan w) {
    constexpr int N = Packet<T>::N;
    const int64_t r = blockIdx.x / static_cast<unsigned>(w.splits);
    const int split = static_cast<int>(blockIdx.x % static_cast<unsigned>(w.splits));
    const int64_t first = split * w.span, end = first + w.span < w.p.vocab ? first + w.span : w.p.vocab;
    const S_<T>* x = static_cast<const S_<T>*>(w.p.logits.data) + r * w.p.logits.step;
    S_<T>* dx = static_cast<S_<T>*>(w.p.dlogits) + r * w.p.vocab;
    int64_t target = -1;
    bool skipped = false;
    float da = 0.0f, db = 0.0f;
    if (w.p.target != nullptr) {
        target = target_at(w.p, r);
        skipped = target == w.p.ignore;
        da = w.p.da != nullptr ? w.p.da[r] : 0.0f;
        if (target < 0 || target >= w.p.vocab) da = __uint_as_float(0x7fc00000u);
    }
    const float m = w.p.stats[2 * r], ls = w.p.stats[2 * r + 1], ls2 = ls * kLog2e;
    float h = 0.0f;
    if constexpr (ENTROPY) db = w.p.db[r], h = w.p.entropy[r];
    auto grad = [&](float v, int64_t at) {
        const float d = v - m;
        const float q = __builtin_amdgcn_exp2f(fmaf(d, w.c, -ls2));
        float g = da;
        if constexpr (ENTROPY) g = fmaf(db, larger(fmaf(d, w.p.scale, -ls), kFloor) + h, g);
        return w.p.scale * ((at == target ? da : 0.0f) - q * g);
    };
    for (int64_t at = first + threadIdx.x * N; at < end; at += kBlock * N) {
        float f[N];
        if (at + N <= end) {
            if (skipped) {
#pragma unroll
                for (int j = 0; j < N; ++j) f[j] = 0.0f;
            } else {
                unpack<T>(load_raw_any_nt(x + at), f);
#pragma unroll
                for (int j = 0; j < N; ++j) f[j] = grad(f[j], at + j);
            }
            store_raw_any_nt(dx + at, pack<T>(f));
        } else {
            for (int64_t i = at; i < end; ++i) dx[i] = Elem<T>::store(skipped ? 0.0f : grad(Elem<T>::load(x[i]), i));
        }
    }
}

Plan plan_of(const TokenProbsArgs& p, int packet, int splits) {
    Plan w{};
    w.p = p;
    w.c = p.scale * kLog2e;
    const int64_t most = std::max<int64_t>(1, (p.vocab + kBlock * packet - 1) / (kBlock * packet));
    const int64_t each = (most + std::min<int64_t>(splits, most) - 1) / std::min<int64_t>(splits, most);
    w.span = each * kBlock * packet;
    w.splits = static_cast<int>((p.vocab + w.span - 1) / w.span);
    return w;
}

void check_extent(const TokenProbsArgs& p) {
    TP_AMD_CHECK(p.vocab > 0 && p.vocab < (int64_t{1} << 31), "token_log_probs: a vocabulary of ", p.vocab);
    TP_AMD_CHECK(p.top >= 0 && p.top <= kTokenProbsMaxTop && p.top <= p.vocab, "token_log_probs: ", p.top, " alternatives of ", p.vocab);
    TP_AMD_CHECK(p.rows < (int64_t{1} << 30), "token_log_probs: ", p.rows, " rows");
}

template <typename T>
void forward_typed(const TokenProbsArgs& p, int device) {
    // About four blocks a CU; a wave joins a row's splits.
    const int64_t want = 4 * cu_count(device);
    Plan w = plan_of(p, Packet<T>::N, static_cast<int>(std::min<int64_t>(kWave, std::max<int64_t>(1, want / p.rows))));
    const int64_t parts = w.splits > 1 ? p.rows * w.splits : 0;
    const Workspace lists(static_cast<size_t>(parts) * p.top * sizeof(uint64_t), device);
    const Workspace part(static_cast<size_t>(parts) * 3 * sizeof(float), device);
    w.part_top = static_cast<uint64_t*>(lists.get());
    w.part = static_cast<float*>(part.get());
    const unsigned blocks = grid_of(p.rows * w.splits, kBlock, "token_log_probs");
    auto* kernel = p.top > 0 ? (p.entropy != nullptr ? token_log_probs_kernel<T, true, true> : token_log_probs_kernel<T, false, true>)
                             : (p.entropy != nullptr ? token_log_probs_kernel<T, true, false> : token_log_probs_kernel<T, false, false>);
    kernel<<<blocks, kBlock, 0, stream(device)>>>(w);
    TP_AMD_HIP_CHECK(hipGetLastError());
    if (w.splits == 1) return;
    token_log_probs_join_kernel<T><<<static_cast<unsigned>(p.rows), kWave, 0, stream(device)>>>(w);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

template <typename T>
void backward_typed(const TokenProbsArgs& p, int device) {
    const Plan w = plan_of(p, Packet<T>::N * kUnits, 1 << 20);
    const unsigned blocks = grid_of(p.rows * w.splits, kBlock, "token_log_probs_backward");
    auto* kernel = p.db != nullptr ? token_log_probs_backward_kernel<T, true> : token_log_probs_backward_kernel<T, false>;
    kernel<<<blocks, kBlock, 0, stream(device)>>>(w);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

}  // namespace

void launch_token_log_probs(int dtype, const TokenProbsArgs& p, int device) {
    if (p.rows <= 0) return;
    check_extent(p);
    const OnDevice scope(device);
    TP_AMD_DISPATCH_TYPED(dtype, forward_typed, p, scope.index());
}

void launch_token_log_probs_backward(int dtype, const TokenProbsArgs& p, int device) {
    if (p.rows <= 0) return;
    check_extent(p);
    const OnDevice scope(device);
    TP_AMD_DISPATCH_TYPED(dtype, backward_typed, p, scope.index());
}

}  // namespace tp_amd

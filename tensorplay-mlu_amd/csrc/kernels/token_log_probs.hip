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
// The likeliest tokens come from the same pass.  A wave holds its 64 best so far
// sorted, one a lane, and the least of the wanted ones as its bound.  Of a chunk
// of logits only those above the bound go on: one by one where few are wanted,
// else through a list in LDS that is sorted and merged into the best whenever it
// holds 64.  Where many lanes have one above (a first chunk, a rising row), the
// `top`-th largest of the lanes' maxima is a bound that `top` elements reach, and
// comes first.
//
// Bound by memory, with the exponentials' issue close behind for 16-bit logits;
// waves share nothing until their ends meet, and have their next chunk's loads
// out.  A row is split over blocks where rows are few, and its last block to
// arrive joins the splits; many short rows go to a wave each.  Kernel times of a
// trace: bf16 4096 x 32000 (262 MB; 42.5 us as an elementwise pass) 48 to 51 us,
// with one alternative 54, backward (524 MB; 85) 87; 1024 x 128000 with five
// alternatives 64 to 68 (50 without), 8 x 32000 with twenty 10.4, 8000 x 1001 with
// one 13 (63 by four waves a row).

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
constexpr int kUnits = 4;  // packets a lane takes at a time: the running maximum moves once for them
constexpr int kMostSplits = 16;
constexpr float kLowest = -3.402823466e38f;
// What an exponent is held above: 2^-4096 is 0 and times a finite number stays 0.
constexpr float kFloor = -4096.0f;

template <typename T>
using S_ = typename Elem<T>::storage;

struct Plan {
    TokenProbsArgs p;
    int64_t first;  // row of the launch
    int splits;
    int64_t span;  // elements of a split: whole chunks' packets
    float c;       // scale log2 e
    uint64_t* part;  // [rows][splits][2 + top]: m and S, E, the best keys
};

// One arrival counter a row that is split, on a 128-byte line of its own (atomics
// on one line serialize); zero between launches.  A device's launches are all on
// one stream.
constexpr int kCounterStride = 32, kMaxSplitRows = 1024;
__device__ unsigned int split_counters[kMaxSplitRows * kCounterStride];

// Words written through to, and read from, the level all XCDs share.  Relaxed
// agent-scope stores are acknowledged there before s_waitcnt vmcnt(0) returns,
// so they precede the arrival that is counted after it.
__device__ __forceinline__ void store_shared(uint64_t* at, uint64_t v) { __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint64_t load_shared(const uint64_t* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

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

// The value of lane ^ STEP (a power of two), or of lane 63 - lane (STEP 63), by
// moves between registers: a few cycles, where an exchange through LDS takes a
// hundred and these networks are chains of them.
template <int STEP>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
    auto dpp = [](uint32_t x, auto control) {
        return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(control)::value, 0xf, 0xf, true));
    };
    using std::integral_constant;
    if constexpr (STEP == 1) {
        return dpp(v, integral_constant<int, 0xb1>{});  // within four lanes: 1 0 3 2
    } else if constexpr (STEP == 2) {
        return dpp(v, integral_constant<int, 0x4e>{});  // 2 3 0 1
    } else if constexpr (STEP == 4) {
        return dpp(dpp(v, integral_constant<int, 0x1b>{}), integral_constant<int, 0x141>{});  // 3 2 1 0, then eight lanes mirrored
    } else if constexpr (STEP == 8) {
        return dpp(v, integral_constant<int, 0x128>{});  // sixteen lanes rotated by 8
    } else if constexpr (STEP == 16) {
        // rows 1 and 3 of the one, 0 and 2 of the other change places
        const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? both[0] : both[1];
    } else if constexpr (STEP == 32) {
        const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? both[0] : both[1];
    } else {
        static_assert(STEP == 63);
        return lane_xor<32>(lane_xor<16>(dpp(v, integral_constant<int, 0x140>{})));  // sixteen lanes mirrored
    }
}
template <int STEP>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
    const uint32_t lo = lane_xor<STEP>(static_cast<uint32_t>(v)), hi = lane_xor<STEP>(static_cast<uint32_t>(v >> 32));
    return static_cast<uint64_t>(hi) << 32 | lo;
}
template <int STEP>
__device__ __forceinline__ float lane_xor(float v) {
    return __uint_as_float(lane_xor<STEP>(__float_as_uint(v)));
}

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

// A wave's lanes as one, in every lane.
template <int STEP = 1>
__device__ __forceinline__ void join_lanes(Stats& st, float c) {
    const Stats other{lane_xor<STEP>(st.m), lane_xor<STEP>(st.s), lane_xor<STEP>(st.e)};
    join(st, other, c);
    if constexpr (STEP < kWave / 2) join_lanes<2 * STEP>(st, c);
}

__device__ __forceinline__ int64_t target_at(const TokenProbsArgs& p, int64_t r) {
    return p.wide_target ? static_cast<const int64_t*>(p.target)[r] : static_cast<const int32_t*>(p.target)[r];
}

// The logit of a row's target, loaded long before it is needed; NaN for a
// target outside the row.
template <typename T>
__device__ __forceinline__ float target_logit(const Plan& w, int64_t r, int64_t target) {
    if (target < 0 || target >= w.p.vocab) return __uint_as_float(0x7fc00000u);
    return Elem<T>::load(static_cast<const S_<T>*>(w.p.logits.data)[r * w.p.logits.step + target]);
}

// Results of a row from its statistics.  A row without a finite or larger
// logit has the sum 0 and NaN for results.
__device__ __forceinline__ void write_row(const Plan& w, int64_t r, const Stats& t, float given) {
    const float ls = logf(t.s);
    w.p.stats[2 * r] = t.s == 0.0f ? -__builtin_inff() : t.m;  // every logit -inf
    w.p.stats[2 * r + 1] = ls;
    if (w.p.entropy != nullptr) w.p.entropy[r] = larger(ls - t.e / t.s * kLn2, 0.0f);  // (rounding may pass 0)
    if (w.p.target != nullptr) w.p.logprob[r] = fmaf(given - t.m, w.p.scale, -ls);
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

// ---- the likeliest tokens ---------------------------------------------------------

template <typename K>
__device__ __forceinline__ K larger_of(K a, K b) { return a > b ? a : b; }
template <typename K>
__device__ __forceinline__ K smaller_of(K a, K b) { return a < b ? a : b; }

// A bitonic network on a wave's 64 keys, one a lane.  Steps STEP, STEP / 2, ..
// 1: runs of 2 STEP lanes sorted, falling or, where lane & SIZE, rising (SIZE
// 64: all falling).
template <int STEP, int SIZE, typename K>
__device__ __forceinline__ K bitonic_steps(K v) {
    const int lane = threadIdx.x % kWave;
    const K other = lane_xor<STEP>(v);
    const K kept = ((lane & STEP) == 0) == ((lane & SIZE) == 0) ? larger_of(v, other) : smaller_of(v, other);
    if constexpr (STEP > 1) return bitonic_steps<STEP / 2, SIZE>(kept);
    else return kept;
}

// In falling order by lane; LANES: the keys past them are 0.
template <int LANES = kWave, int SIZE = 2, typename K>
__device__ __forceinline__ K wave_sorted(K v) {
    v = bitonic_steps<SIZE / 2, SIZE == LANES ? kWave : SIZE>(v);
    if constexpr (SIZE < LANES) return wave_sorted<LANES, 2 * SIZE>(v);
    else return v;
}

// The 64 largest of two falling lists, falling: the larger of each pair from
// opposite ends is a bitonic list of them.
__device__ __forceinline__ uint64_t wave_merged(uint64_t a, uint64_t b) {
    return bitonic_steps<kWave / 2, kWave>(larger_of(a, lane_xor<kWave - 1>(b)));
}

// The block's best in wave 0, from the waves'; all threads.
template <int STRIDE>
__device__ __forceinline__ uint64_t block_merged(uint64_t key, uint64_t (&lists)[kWaves][STRIDE], int lane, int wave) {
    static_assert(kWaves == 4);
    lists[wave][lane] = key;
    __syncthreads();
    if (wave % 2 == 0) {
        key = wave_merged(key, lists[wave + 1][lane]);
        if (wave == 2) lists[2][lane] = key;
    }
    __syncthreads();
    return wave == 0 ? wave_merged(key, lists[2][lane]) : key;
}

// What lanes of one wave wrote to LDS is there for its others.
__device__ __forceinline__ void wave_lds() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ uint64_t lane_key(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane);
    return static_cast<uint64_t>(hi) << 32 | lo;
}

// The value of the lane before (lane 0: 0).
__device__ __forceinline__ uint64_t lane_before(uint64_t v) {
    const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x138, 0xf, 0xf, true);
    const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), 0x138, 0xf, 0xf, true);
    return static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 | static_cast<uint32_t>(lo);
}

// Up to so many wanted, candidates go straight into the best, one after another;
// of more, through the list: bf16 4096 x 32000 by four waves a row (us, one against
// the other) one 69 and 85, five 84 and 96, 16 106 and 115, 20 115 and 115, 32 135
// and 118.  Fewer instructions, but a longer chain of them: few short rows, whose
// waves wait and do not issue, keep to the list (32 x 32000 with five 14.3 and 14.0).
constexpr int kInsertTop = 16;

// A wave's best keys (0: none yet).  DIRECT: up to kInsertTop wanted need no list.
template <bool DIRECT>
struct Best {
    uint64_t key = 0;    // the lane's of the 64 best, falling by lane
    uint64_t bound = 0;  // keys up to it are not wanted: `top` larger ones are known
    float reach = __uint_as_float(0x7fc00000u);  // what is less is below the bound's value (NaN: nothing is)
    uint32_t count = 0;  // keys in the list
    uint64_t* list;      // 128 keys of LDS

    // The list's first 64 into the best.
    __device__ __forceinline__ void flush(int top) {
        const uint32_t lane = threadIdx.x % kWave, kept = count;
        wave_lds();
        const uint64_t mine = lane < count ? list[lane] : 0;
        const uint64_t rest = kWave + lane < count ? list[kWave + lane] : 0;
        wave_lds();
        if (kWave + lane < count) list[lane] = rest;
        count = count > kWave ? count - kWave : 0;
        const bool few = kept <= 16;
        key = wave_merged(key, few ? wave_sorted<16>(mine) : wave_sorted<>(mine));
        raise(lane_key(key, top - 1));
    }

    __device__ __forceinline__ void raise(uint64_t least) {
        if (least <= bound) return;
        bound = least;
        reach = from_ordered(static_cast<uint32_t>(least >> 32));
    }

    // One key of the wave's into the best.
    __device__ __forceinline__ void insert(uint64_t one) {
        const bool greater = key > one;
        const uint32_t place = static_cast<uint32_t>(__popcll(__ballot(greater)));
        const uint64_t before = lane_before(key);
        const uint64_t moved = threadIdx.x % kWave == place ? one : before;
        key = greater ? key : moved;
    }

    // One candidate a lane.
    __device__ __forceinline__ void add(uint64_t candidate, bool wanted, int top) {
        uint64_t lanes = __ballot(wanted);
        if (lanes == 0) return;
        if (DIRECT && top <= kInsertTop && __popcll(lanes) <= 16) {
            for (; lanes != 0; lanes &= lanes - 1) insert(lane_key(candidate, __builtin_ctzll(lanes)));
            raise(lane_key(key, top - 1));
            return;
        }
        const uint32_t before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(lanes >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(lanes), 0u));
        if (wanted) list[count + before] = candidate;
        count += static_cast<uint32_t>(__popcll(lanes));
        if (count >= kWave) flush(top);
    }

    // The elements of a lane's packet, of which those before `end` are there.
    template <int N>
    __device__ __forceinline__ void add_packet(const float (&f)[N], int64_t at, int64_t end, int top) {
        uint32_t left = 0;
#pragma unroll
        for (int j = N - 1; j >= 0; --j) left = left + left + (!(f[j] < reach) ? 1u : 0u);
        if (at + N > end) left = at < end ? left & ((1u << static_cast<uint32_t>(end - at)) - 1) : 0u;
        // one element a lane and round: hardly ever more than one or two
        while (__ballot(left != 0) != 0) {
            const uint32_t j = __builtin_ctz(left | 1u << 31);
            float v = f[0];
#pragma unroll
            for (int i = 1; i < N; ++i) v = j == static_cast<uint32_t>(i) ? f[i] : v;
            const uint64_t candidate = key_of(v, static_cast<uint32_t>(at) + j);
            add(candidate, left != 0 && candidate > bound, top);
            left &= left - 1;
        }
    }
};

// WAVES waves a row's split: four of a block's, or one.
template <typename T, int U, int WAVES, bool ENTROPY, bool TOP>
__global__ __launch_bounds__(kBlock) void token_log_probs_kernel(Plan w) {
    constexpr int N = Packet<T>::N, kTeam = WAVES * kWave;
    constexpr int64_t kChunk = kTeam * N * U;
    __shared__ Stats wave_stats[kWaves];
    __shared__ uint64_t lists[kWaves][TOP ? 2 * kWave : 1];
    __shared__ bool last;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int64_t r = w.first + (WAVES == 1 ? static_cast<int64_t>(blockIdx.x) * kWaves + wave : blockIdx.x / static_cast<unsigned>(w.splits));
    const int split = WAVES == 1 ? 0 : static_cast<int>(blockIdx.x % static_cast<unsigned>(w.splits));
    if (WAVES == 1 && r >= w.p.rows) return;
    const int mine = WAVES == 1 ? lane : static_cast<int>(threadIdx.x);  // of the team
    float given = 0.0f;
    if (w.p.target != nullptr) {
        const int64_t target = target_at(w.p, r);
        if (target == w.p.ignore) {
            if (split == 0) write_skipped(w, r, mine, kTeam);
            return;
        }
        given = target_logit<T>(w, r, target);
    }
    const int64_t first = split * w.span, end = first + w.span < w.p.vocab ? first + w.span : w.p.vocab;
    const S_<T>* x = static_cast<const S_<T>*>(w.p.logits.data) + r * w.p.logits.step;
    const int top = w.p.top;
    Stats st{kLowest, 0.0f, 0.0f};
    Best<(U > 1)> best;
    if constexpr (TOP) best.list = lists[wave];
    // unit u of a chunk lies at base + (u kTeam + mine) N: every wave has its share of a last short one
    uint4 next[U];
    auto fetch = [&](int64_t base) {
        if (base + kChunk <= end) {
#pragma unroll
            for (int u = 0; u < U; ++u) next[u] = load_raw_any_nt(x + base + (u * kTeam + mine) * N);
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = base + (u * kTeam + mine) * N;
                if (at + N <= end) next[u] = load_raw_any_nt(x + at);
            }
        }
    };
    if (first < end) fetch(first);
    for (int64_t base = first; base < end; base += kChunk) {
        float f[U][N], um[U];
        const bool whole = base + kChunk <= end;
        // units of which this wave has any element
        const int64_t left = end - base - (WAVES == 1 ? 0 : wave * (kWave * N));
        const int units = whole ? U : left <= 0 ? 0 : static_cast<int>(min<int64_t>(U, (left + kTeam * N - 1) / (kTeam * N)));
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= units) break;
            const int64_t at = base + (u * kTeam + mine) * N;
            if (whole || at + N <= end) {
                unpack<T>(next[u], f[u]);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) f[u][j] = at + j < end ? Elem<T>::load(x[at + j]) : -__builtin_inff();
            }
        }
        if (base + kChunk < end) fetch(base + kChunk);
        float cm = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= units) break;
            um[u] = f[u][0];
#pragma unroll
            for (int j = 1; j < N; ++j) um[u] = larger(um[u], f[u][j]);
            cm = larger(cm, um[u]);
        }
        const float m = larger(st.m, cm);
        {
            const float d = larger((st.m - m) * w.c, kFloor), scale = __builtin_amdgcn_exp2f(d);
            if constexpr (ENTROPY) st.e = fmaf(st.s, d, st.e) * scale;
            st.s *= scale;
            st.m = m;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (u >= units) break;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if constexpr (ENTROPY) {
                    const float d = larger((f[u][j] - m) * w.c, kFloor), e = __builtin_amdgcn_exp2f(d);
                    st.s += e;
                    st.e = fmaf(e, d, st.e);
                } else {
                    st.s += __builtin_amdgcn_exp2f((f[u][j] - m) * w.c);
                }
            }
        }
        if constexpr (TOP) {
            const uint64_t above = __ballot(!(cm < best.reach));
            if (__popcll(above) >= (U > 1 && top <= kInsertTop ? top + 6 : top)) {
                const uint32_t reached = __builtin_amdgcn_readlane(wave_sorted(ordered(cm + 0.0f)), top - 1);
                best.raise((static_cast<uint64_t>(reached) << 32) - 1);
            }
            if (above != 0) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (u >= units) break;
                    if (__ballot(!(um[u] < best.reach)) != 0) best.add_packet(f[u], base + (u * kTeam + mine) * N, end, top);
                }
                // a closer bound for the chunks to come
                if (best.count >= static_cast<uint32_t>(top) && base + kChunk < end) best.flush(top);
            }
        }
    }
    join_lanes(st, w.c);
    if constexpr (TOP) {
        if (best.count > 0) best.flush(top);
    }
    if constexpr (WAVES > 1) {
        static_assert(WAVES == kWaves);
        if (lane == 0) wave_stats[wave] = st;
        if constexpr (TOP) best.key = block_merged(best.key, lists, lane, wave);
        else __syncthreads();
        st = wave_stats[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) join(st, wave_stats[i], w.c);
        if (w.splits > 1) {
            const int words = 2 + top;
            uint64_t* const parts = w.part + r * w.splits * words;
            if (wave == 0) {
                uint64_t* part = parts + split * words;
                if (lane == 0) {
                    store_shared(part, static_cast<uint64_t>(__float_as_uint(st.s)) << 32 | __float_as_uint(st.m));
                    store_shared(part + 1, __float_as_uint(st.e));
                }
                if (TOP && lane < top) store_shared(part + 2 + lane, best.key);
                __builtin_amdgcn_s_waitcnt(0);
            }
            __syncthreads();
            if (threadIdx.x == 0) {
                unsigned int* counter = &split_counters[r * kCounterStride];
                last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == w.splits - 1u;
                if (last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (!last) return;
            // the splits' statistics one a lane, their lists one after another by every wave
            st = Stats{kLowest, 0.0f, 0.0f};
            if (lane < w.splits) {
                const uint64_t ms = load_shared(parts + lane * words), e = load_shared(parts + lane * words + 1);
                st = Stats{__uint_as_float(static_cast<uint32_t>(ms)), __uint_as_float(static_cast<uint32_t>(ms >> 32)),
                           __uint_as_float(static_cast<uint32_t>(e))};
            }
            if constexpr (TOP) {
                uint64_t keys[kMostSplits / kWaves];
#pragma unroll
                for (int i = 0; i < kMostSplits / kWaves; ++i) {
                    const int from = wave + i * kWaves;
                    keys[i] = from < w.splits && lane < top ? load_shared(parts + from * words + 2 + lane) : 0;
                }
                best.key = keys[0];
#pragma unroll
                for (int i = 1; i < kMostSplits / kWaves; ++i) {
                    if (wave + i * kWaves < w.splits) best.key = wave_merged(best.key, keys[i]);
                }
                best.key = block_merged(best.key, lists, lane, wave);
            }
            join_lanes(st, w.c);
        }
        if (wave != 0) return;
    }
    if (lane == 0) write_row(w, r, st, given);
    if (TOP && lane < top) write_top(w, r, lane, best.key, st);
}

// dx of a span a block; a row's blocks follow one another.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(kBlock) void token_log_probs_backward_kernel(Plan w) {
    constexpr int N = Packet<T>::N;
    const int64_t r = w.first + blockIdx.x / static_cast<unsigned>(w.splits);
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

// Rows in at most `splits` spans of whole steps of `step` elements.
Plan plan_of(const TokenProbsArgs& p, int64_t step, int64_t splits) {
    Plan w{};
    w.p = p;
    w.c = p.scale * kLog2e;
    const int64_t steps = (p.vocab + step - 1) / step, most = std::min(std::max<int64_t>(splits, 1), steps);
    w.span = (steps + most - 1) / most * step;
    w.splits = static_cast<int>((p.vocab + w.span - 1) / w.span);
    return w;
}

void check_extent(const TokenProbsArgs& p) {
    TP_AMD_CHECK(p.vocab > 0 && p.vocab < (int64_t{1} << 31), "token_log_probs: a vocabulary of ", p.vocab);
    TP_AMD_CHECK(p.top >= 0 && p.top <= kTokenProbsMaxTop && p.top <= p.vocab, "token_log_probs: ", p.top, " alternatives of ", p.vocab);
    TP_AMD_CHECK(p.rows < kMaxRows, "token_log_probs: ", p.rows, " rows");
}

// The kernel over all rows, `per_block` of them a block or `splits` blocks each:
// more of them than one launch takes go in several.
template <typename Kernel>
void launch_rows(Kernel* kernel, Plan w, int64_t per_block, int device) {
    const int64_t at_once = most_blocks(kBlock) / w.splits * per_block;
    for (w.first = 0; w.first < w.p.rows; w.first += at_once) {
        const int64_t rows = std::min(at_once, w.p.rows - w.first);
        kernel<<<static_cast<unsigned>((rows + per_block - 1) / per_block * w.splits), kBlock, 0, stream(device)>>>(w);
        TP_AMD_HIP_CHECK(hipGetLastError());
    }
}

template <typename T, int U, int WAVES>
void forward_units(const TokenProbsArgs& p, int64_t splits, int device) {
    Plan w = plan_of(p, static_cast<int64_t>(WAVES) * kWave * Packet<T>::N * U, p.rows > kMaxSplitRows ? 1 : std::min<int64_t>(splits, kMostSplits));
    const Workspace part(w.splits > 1 ? static_cast<size_t>(p.rows * w.splits) * (2 + p.top) * sizeof(uint64_t) : 0, device);
    w.part = static_cast<uint64_t*>(part.get());
    auto* kernel = p.top > 0 ? (p.entropy != nullptr ? token_log_probs_kernel<T, U, WAVES, true, true> : token_log_probs_kernel<T, U, WAVES, false, true>)
                             : (p.entropy != nullptr ? token_log_probs_kernel<T, U, WAVES, true, false> : token_log_probs_kernel<T, U, WAVES, false, false>);
    launch_rows(kernel, w, WAVES == 1 ? kWaves : 1, device);
}

template <typename T>
void forward_typed(const TokenProbsArgs& p, int device) {
    constexpr int64_t kPass = static_cast<int64_t>(kBlock) * Packet<T>::N;  // of a block, a packet a lane
    const int64_t cus = cu_count(device);
    // A wave a row where rows of few chunks fill the device by themselves: 8000 x
    // 1001 15 us (63 by four), but 8192 x 32000 105 (96).  Alternatives cost every
    // wave its own bound, list and merges: a wave a row also of longer rows, the
    // longer the more of them there are: with five 4096 x 32000 76 (86), 8212 x
    // 65000 242 (258), 4120 x 50257 130 (122).  Else a block a split, four packets a
    // lane.  Rows too few to fill the device so, and short enough that sixteen splits
    // of one packet a lane cover them, take those: 8 x 32000 10.4 us (four splits of
    // four packets 11.0).  Two packets a lane instead of four: 1024 x 128000 64 us
    // against 54.
    const int64_t by_wave = p.top > 0 ? std::max<int64_t>(8, p.rows / cus) : 8;
    if (p.rows >= 16 * cus && p.vocab <= by_wave * kPass) forward_units<T, kUnits, 1>(p, 1, device);
    else if (p.vocab > kMostSplits * kPass || p.rows >= 2 * cus) forward_units<T, kUnits, kWaves>(p, 4 * cus / p.rows, device);
    else forward_units<T, 1, kWaves>(p, 2 * cus / p.rows, device);
}

template <typename T>
void backward_typed(const TokenProbsArgs& p, int device) {
    const Plan w = plan_of(p, kBlock * Packet<T>::N * 4, p.vocab);
    launch_rows(p.db != nullptr ? token_log_probs_backward_kernel<T, true> : token_log_probs_backward_kernel<T, false>, w, 1, device);
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

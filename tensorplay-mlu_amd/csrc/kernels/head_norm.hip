// Norm of every head's query and key with the position rotation in the same
// pass, forward and backward.
//
// For a head's row x of D elements: r = (mean x^2 + eps)^-1/2, n = r x w, and
// the first R elements of n turn in R / 2 pairs (a, b) -> (a c - b s,
// b c + a s) with c, s from the position's row of a table.  Pair j is
// elements (j, j + R / 2), or (2 j, 2 j + 1) when interleaved; elements past
// R keep n, whatever lies beside them in a lane.  Backward, with g the gradient turned back, u = g w and
// m = x r: dx = r (u - m mean(u m)), dw = sum over rows of g m.
//
// Bound by memory: a row is read once (backward: x and dy) and written once.
// A group of G lanes owns a row, each lane `UPL` units of two V-element
// packets laid out so that both elements of a pair sit in one lane: packets u
// and u + R / 2 / V, or two neighbouring packets.  The rotation then needs no
// exchange, and the row's one sum is log2 G lane exchanges.  V is a 16-byte
// packet where R / 2 and D - R are whole packets (rows may start at any
// element, unaligned 16-byte loads cost nothing here), else single elements.
// A group takes ROWS heads of one token in a row: their loads go out together
// and the table's row, as many bytes as a 16-bit head, is read once for all.
//
// bf16, 40 heads of 128: 8192 tokens forward 32 us, 5.4 TB/s; 4 x 2048 backward
// 46 us, 5.5 TB/s, and 4 us for the weights' sums over blocks (2 GiB read and
// written by a plain elementwise pass: 6.35 TB/s).  8 tokens 3.5 us, a launch's
// own time.  float32, 3001 tokens, 24 heads of 80 of which 40 turn as neighbours:
// 12 us forward, 3.9 TB/s, 15 and 4 us backward (6 of a group's 16 lanes hold
// nothing there).

#include <algorithm>
#include <type_traits>

#include "attention.h"
#include "device_common.h"
#include "../allocator.h"
#include "../common.h"
#include "../runtime.h"

namespace tp_amd {

namespace {

constexpr int kBlock = 256;

template <typename T>
using S_ = typename Elem<T>::storage;

// What the kernels derive from the arguments once, on the host.
struct HeadNormPlan {
    HeadNormArgs p;
    FastDiv by_inner, by_slots;
    uint32_t slots;  // groups of ROWS heads a token takes, queries' first
    uint32_t q_slots;
    uint32_t tokens;
    int lanes;  // G
    int turns;  // units that rotate
    int units;
    float inv_dim;
};

__device__ __forceinline__ int64_t position_of(const HeadNormArgs& p, int64_t o, int64_t i) {
    const int64_t at = o * p.pos_outer + i * p.pos_inner;
    return p.wide_positions ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
}

// The element a lane's unit starts at, and its second packet's distance; the
// last unit past R may lack the second packet.
template <int V, bool INTER>
struct Unit {
    int first, second;
    bool in, both, turns;
    __device__ __forceinline__ Unit(const HeadNormPlan& w, int u) {
        in = u < w.units;
        turns = u < w.turns;
        first = turns ? (INTER ? 2 * u * V : u * V) : w.p.rotary + (u - w.turns) * 2 * V;
        second = turns && !INTER ? first + w.p.rotary / 2 : first + V;
        both = in && second < w.p.dim;
    }
};

// Elements as float32 pairs: a[j] and b[j] turn together.
template <typename T, int V, bool INTER>
__device__ __forceinline__ void load_unit(const S_<T>* row, const Unit<V, INTER>& u, float (&a)[V], float (&b)[V]) {
    float f[2 * V];
#pragma unroll
    for (int j = 0; j < 2 * V; ++j) f[j] = 0.0f;
    if constexpr (V == Packet<T>::N) {
        float lo[V], hi[V];
        if (u.in) {
            unpack<T>(load_raw_any(row + u.first), lo);
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = lo[j];
        }
        if (u.both) {
            unpack<T>(load_raw_any(row + u.second), hi);
#pragma unroll
            for (int j = 0; j < V; ++j) f[V + j] = hi[j];
        }
    } else {
        if (u.in) f[0] = Elem<T>::load(row[u.first]);
        if (u.both) f[1] = Elem<T>::load(row[u.second]);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
        a[j] = INTER ? f[2 * j] : f[j];
        b[j] = INTER ? f[2 * j + 1] : f[V + j];
    }
}

template <typename T, int V, bool INTER>
__device__ __forceinline__ void store_unit(S_<T>* row, const Unit<V, INTER>& u, const float (&a)[V], const float (&b)[V]) {
    float lo[V], hi[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        if constexpr (INTER) {
            (2 * j < V ? lo[2 * j] : hi[2 * j - V]) = a[j];
            (2 * j + 1 < V ? lo[2 * j + 1] : hi[2 * j + 1 - V]) = b[j];
        } else {
            lo[j] = a[j];
            hi[j] = b[j];
        }
    }
    if constexpr (V == Packet<T>::N) {
        if (u.in) store_raw_any_nt(row + u.first, pack<T>(lo));
        if (u.both) store_raw_any_nt(row + u.second, pack<T>(hi));
    } else {
        if (u.in) row[u.first] = Elem<T>::store(lo[0]);
        if (u.both) row[u.second] = Elem<T>::store(hi[0]);
    }
}

// cos and sin of a lane's V pairs; 1 and 0 past R.  A position outside the
// table reads nothing and turns its rows to NaN.
template <int V>
__device__ __forceinline__ void load_turn(const HeadNormPlan& w, int64_t pos, int u, float (&c)[V], float (&s)[V]) {
    const bool known = pos >= 0 && pos < w.p.table_rows;
    const float other = known ? 1.0f : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        c[j] = other;
        s[j] = 0.0f;
    }
    if (!known || u >= w.turns) return;
    const float* row = w.p.table + pos * w.p.rotary + u * V;
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int j = 0; j < V; j += 4) {
            const uint4 x = load_raw_any(row + j), y = load_raw_any(row + w.p.rotary / 2 + j);
            const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                c[j + e] = __uint_as_float(xs[e]);
                s[j + e] = __uint_as_float(ys[e]);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            c[j] = row[j];
            s[j] = row[w.p.rotary / 2 + j];
        }
    }
}

template <typename T, int V, bool INTER>
__device__ __forceinline__ void load_weight(const void* weight, const Unit<V, INTER>& u, float (&a)[V], float (&b)[V]) {
    if (weight != nullptr) {
        load_unit<T, V, INTER>(static_cast<const S_<T>*>(weight), u, a, b);
        return;
    }
#pragma unroll
    for (int j = 0; j < V; ++j) a[j] = b[j] = 1.0f;
}

// Sum over the G lanes of a group (a power of two).
__device__ __forceinline__ float group_sum(float v, int lanes) {
    for (int m = 1; m < lanes; m *= 2) v += wave_shfl_xor(v, m);
    return v;
}

template <typename T, int V, int UPL, bool INTER, int ROWS>
__global__ __launch_bounds__(kBlock) void head_norm_kernel(HeadNormPlan w) {
    using U = Unit<V, INTER>;
    const int lane = threadIdx.x & (w.lanes - 1);
    const uint32_t group = blockIdx.x * (kBlock / w.lanes) + threadIdx.x / w.lanes;
    const uint32_t token = fastdiv(group, w.by_slots);
    if (token >= w.tokens) return;
    const uint32_t slot = group - token * w.slots;
    const bool key = slot >= w.q_slots;
    const HeadNormSide& side = w.p.side[key];
    const int h0 = static_cast<int>(key ? slot - w.q_slots : slot) * ROWS;
    const uint32_t o = fastdiv(token, w.by_inner), i = token - o * static_cast<uint32_t>(w.p.inner);
    const S_<T>* x = static_cast<const S_<T>*>(side.x.data) + o * side.x.outer + i * side.x.inner + h0 * side.x.head;

    float a[ROWS][UPL][V], b[ROWS][UPL][V];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        // a head past the last is the last one over again: not stored
        const int64_t at = (h0 + r < side.heads ? r : side.heads - 1 - h0) * side.x.head;
#pragma unroll
        for (int k = 0; k < UPL; ++k) load_unit<T, V, INTER>(x + at, U(w, lane + k * w.lanes), a[r][k], b[r][k]);
    }
    const int64_t pos = position_of(w.p, o, i);
    float scale[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < UPL; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) sum = fmaf(a[r][k][j], a[r][k][j], fmaf(b[r][k][j], b[r][k][j], sum));
        sum = group_sum(sum, w.lanes);
        scale[r] = 1.0f / sqrtf(fmaf(sum, w.inv_dim, w.p.eps));
    }
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const int u = lane + k * w.lanes;
        const U unit(w, u);
        float c[V], s[V], wa[V], wb[V];
        load_turn<V>(w, pos, u, c, s);
        load_weight<T, V, INTER>(side.weight, unit, wa, wb);
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            if (h0 + r >= side.heads) break;
            float ya[V], yb[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float na = a[r][k][j] * scale[r] * wa[j], nb = b[r][k][j] * scale[r] * wb[j];
                ya[j] = na * c[j], yb[j] = nb * c[j];
                if (unit.turns) {
                    ya[j] -= nb * s[j];
                    yb[j] += na * s[j];
                }
            }
            const int64_t row = static_cast<int64_t>(token) * side.heads + h0 + r;
            store_unit<T, V, INTER>(static_cast<S_<T>*>(side.out) + row * w.p.dim, unit, ya, yb);
            if (k == 0 && lane == 0) side.rstd[row] = scale[r];
        }
    }
}

// Groups walk a side's rows (blockIdx.y), every group the same number apart,
// and keep their columns' running dw; a block adds its groups' in LDS and
// writes one float32 row of `part`, which head_norm_fold_kernel adds up in
// block order: the same bits every time.
template <typename T, int V, int UPL, bool INTER>
__global__ __launch_bounds__(kBlock) void head_norm_backward_kernel(HeadNormPlan w, float* part) {
    using U = Unit<V, INTER>;
    extern __shared__ float fold[];  // [groups][dim]
    const HeadNormSide& side = w.p.side[blockIdx.y];
    const int lane = threadIdx.x & (w.lanes - 1), groups = kBlock / w.lanes, mine = threadIdx.x / w.lanes;
    const uint32_t rows = w.tokens * static_cast<uint32_t>(side.heads);
    const uint32_t step = gridDim.x * groups;
    const bool sums = side.dweight != nullptr;
    float wa[UPL][V], wb[UPL][V], da[UPL][V], db[UPL][V];
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        load_weight<T, V, INTER>(side.weight, U(w, lane + k * w.lanes), wa[k], wb[k]);
#pragma unroll
        for (int j = 0; j < V; ++j) da[k][j] = db[k][j] = 0.0f;
    }
    for (uint32_t row = blockIdx.x * groups + mine; row < rows; row += step) {
        const uint32_t token = row / static_cast<uint32_t>(side.heads), h = row - token * side.heads;
        const uint32_t o = fastdiv(token, w.by_inner), i = token - o * static_cast<uint32_t>(w.p.inner);
        const S_<T>* x = static_cast<const S_<T>*>(side.x.data) + o * side.x.outer + i * side.x.inner + h * side.x.head;
        const S_<T>* dy = static_cast<const S_<T>*>(side.dy.data) + o * side.dy.outer + i * side.dy.inner + h * side.dy.head;
        const float r = side.rstd[row];
        const int64_t pos = position_of(w.p, o, i);
        float ma[UPL][V], mb[UPL][V], ua[UPL][V], ub[UPL][V];
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
            const int u = lane + k * w.lanes;
            const U unit(w, u);
            float c[V], s[V], ga[V], gb[V];
            load_unit<T, V, INTER>(x, unit, ma[k], mb[k]);
            load_unit<T, V, INTER>(dy, unit, ga, gb);
            load_turn<V>(w, pos, u, c, s);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                float ta = ga[j] * c[j], tb = gb[j] * c[j];
                if (unit.turns) {
                    ta += gb[j] * s[j];
                    tb -= ga[j] * s[j];
                }
                ma[k][j] *= r;
                mb[k][j] *= r;
                da[k][j] = fmaf(ta, ma[k][j], da[k][j]);
                db[k][j] = fmaf(tb, mb[k][j], db[k][j]);
                ua[k][j] = ta * wa[k][j];
                ub[k][j] = tb * wb[k][j];
                sum = fmaf(ua[k][j], ma[k][j], fmaf(ub[k][j], mb[k][j], sum));
            }
        }
        if (side.out == nullptr) continue;
        const float mean = group_sum(sum, w.lanes) * w.inv_dim;
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
            float xa[V], xb[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                xa[j] = r * fmaf(-ma[k][j], mean, ua[k][j]);
                xb[j] = r * fmaf(-mb[k][j], mean, ub[k][j]);
            }
            store_unit<T, V, INTER>(static_cast<S_<T>*>(side.out) + static_cast<int64_t>(row) * w.p.dim,
                                    U(w, lane + k * w.lanes), xa, xb);
        }
    }
    if (!sums) return;  // the same for the whole block
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const U unit(w, lane + k * w.lanes);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int ea = INTER ? unit.first + 2 * j : unit.first + j;
            const int eb = INTER ? unit.first + 2 * j + 1 : unit.second + j;
            // past R the two packets are neighbours whatever the pairing, so
            // an interleaved unit's elements run on in either case
            if (unit.in && ea < w.p.dim) fold[mine * w.p.dim + ea] = da[k][j];
            if (unit.in && eb < w.p.dim) fold[mine * w.p.dim + eb] = db[k][j];
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < w.p.dim; d += kBlock) {
        float t = 0.0f;
        for (int g = 0; g < groups; ++g) t += fold[g * w.p.dim + d];
        part[(static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * w.p.dim + d] = t;
    }
}

// dw of column d = the blocks' partials in order: 16 runs of blocks, one a
// wave, then the runs in order.  64 columns a block.
constexpr int kFoldWaves = 16;

template <typename T>
__global__ __launch_bounds__(kFoldWaves* kWave) void head_norm_fold_kernel(const float* part, int blocks, int dim,
                                                                           S_<T>* dq, S_<T>* dk) {
    __shared__ float run[kFoldWaves][kWave];
    S_<T>* out = blockIdx.y ? dk : dq;
    if (out == nullptr) return;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, d = blockIdx.x * kWave + lane;
    const int per = (blocks + kFoldWaves - 1) / kFoldWaves;
    float t = 0.0f;
    if (d < dim) {
        const float* at = part + static_cast<int64_t>(blockIdx.y) * blocks * dim + d;
        const int end = (wave + 1) * per < blocks ? (wave + 1) * per : blocks;
#pragma unroll 8
        for (int b = wave * per; b < end; ++b) t += at[static_cast<int64_t>(b) * dim];
    }
    run[wave][lane] = t;
    __syncthreads();
    if (wave != 0 || d >= dim) return;
    for (int k = 1; k < kFoldWaves; ++k) t += run[k][lane];
    out[d] = Elem<T>::store(t);
}

// Packets where every packet of a row is whole and a row takes at most a wave.
template <typename T>
bool whole_packets(const HeadNormArgs& p) {
    constexpr int V = Packet<T>::N;
    return p.rotary % (2 * V) == 0 && (p.dim - p.rotary) % V == 0 && p.dim <= 2 * V * kWave;
}

HeadNormPlan plan_of(const HeadNormArgs& p, int v, int rows) {
    HeadNormPlan w;
    w.p = p;
    w.tokens = static_cast<uint32_t>(p.outer * p.inner);
    w.by_inner = make_fastdiv(static_cast<uint32_t>(std::max<int64_t>(p.inner, 1)));
    w.q_slots = static_cast<uint32_t>((p.side[0].heads + rows - 1) / rows);
    w.slots = w.q_slots + static_cast<uint32_t>((p.side[1].heads + rows - 1) / rows);
    w.by_slots = make_fastdiv(std::max(w.slots, 1u));
    w.turns = p.rotary / 2 / v;
    w.units = w.turns + (p.dim - p.rotary + 2 * v - 1) / (2 * v);
    w.lanes = 1;
    while (w.lanes < w.units && w.lanes < kWave) w.lanes *= 2;
    w.inv_dim = 1.0f / static_cast<float>(p.dim);
    return w;
}

template <typename T, int V, int UPL, int ROWS>
void forward_rows(const HeadNormArgs& p, int device) {
    const HeadNormPlan w = plan_of(p, V, ROWS);
    const uint64_t groups = static_cast<uint64_t>(w.tokens) * w.slots;
    const unsigned blocks = grid_of(static_cast<int64_t>((groups * w.lanes + kBlock - 1) / kBlock), kBlock, "qk_norm_rope");
    auto* kernel = p.interleaved ? head_norm_kernel<T, V, UPL, true, ROWS> : head_norm_kernel<T, V, UPL, false, ROWS>;
    kernel<<<blocks, kBlock, 0, stream(device)>>>(w);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

// Four heads a group where that still leaves sixteen waves a CU: bf16 8192
// tokens x 40 heads of 128 31.5 us (two heads 33.8, one 34.5); 8 tokens 5.9
// against 3.7 with one.
template <typename T, int V, int UPL>
void forward_units(const HeadNormArgs& p, int device) {
    const HeadNormPlan w = plan_of(p, V, 4);
    const uint64_t waves = static_cast<uint64_t>(w.tokens) * w.slots * w.lanes / kWave;
    if (UPL == 1 && waves >= 16 * static_cast<uint64_t>(cu_count(device))) forward_rows<T, V, UPL, UPL == 1 ? 4 : 1>(p, device);
    else forward_rows<T, V, UPL, 1>(p, device);
}

template <typename T, int V, int UPL>
void backward_units(const HeadNormArgs& p, int device) {
    const HeadNormPlan w = plan_of(p, V, 1);
    const int groups = kBlock / w.lanes;
    const int64_t most = static_cast<int64_t>(w.tokens) * std::max(p.side[0].heads, p.side[1].heads);
    const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((most + groups - 1) / groups, 4 * cu_count(device)));
    const bool sums = p.side[0].dweight != nullptr || p.side[1].dweight != nullptr;
    const Workspace part(sums ? static_cast<size_t>(2 * blocks * p.dim) * sizeof(float) : 0, device);
    const size_t lds = sums ? static_cast<size_t>(groups * p.dim) * sizeof(float) : 0;
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    auto* kernel = p.interleaved ? head_norm_backward_kernel<T, V, UPL, true> : head_norm_backward_kernel<T, V, UPL, false>;
    kernel<<<grid, kBlock, lds, stream(device)>>>(w, static_cast<float*>(part.get()));
    TP_AMD_HIP_CHECK(hipGetLastError());
    if (!sums) return;
    head_norm_fold_kernel<T><<<dim3(static_cast<unsigned>((p.dim + kWave - 1) / kWave), 2), kFoldWaves * kWave, 0, stream(device)>>>(
        static_cast<const float*>(part.get()), static_cast<int>(blocks), p.dim, static_cast<S_<T>*>(p.side[0].dweight),
        static_cast<S_<T>*>(p.side[1].dweight));
    TP_AMD_HIP_CHECK(hipGetLastError());
}

// Rows and groups of lanes are counted in 32 bits, those past the last row's
// in its block among them.
void check_extent(const HeadNormArgs& p) {
    const int64_t rows = p.outer * p.inner * (static_cast<int64_t>(p.side[0].heads) + p.side[1].heads);
    TP_AMD_CHECK(p.dim > 0 && p.dim <= kHeadNormMaxDim && p.rotary >= 0 && p.rotary <= p.dim && p.rotary % 2 == 0,
                 "qk_norm_rope: heads of ", p.dim, " with ", p.rotary, " rotated elements");
    TP_AMD_CHECK(rows < (int64_t{1} << 30), "qk_norm_rope: ", rows, " rows of heads");
}

template <typename T>
void forward_typed(const HeadNormArgs& p, int device) {
    if (whole_packets<T>(p)) forward_units<T, Packet<T>::N, 1>(p, device);
    else if (p.dim <= 2 * kWave) forward_units<T, 1, 1>(p, device);
    else forward_units<T, 1, 8>(p, device);
}

template <typename T>
void backward_typed(const HeadNormArgs& p, int device) {
    if (whole_packets<T>(p)) backward_units<T, Packet<T>::N, 1>(p, device);
    else if (p.dim <= 2 * kWave) backward_units<T, 1, 1>(p, device);
    else backward_units<T, 1, 8>(p, device);
}

}  // namespace

#define TP_AMD_DISPATCH_FLOAT(dtype, FN, ...)                       \
    switch (dtype) {                                                \
        case TP_AMD_FLOAT32: FN<float>(__VA_ARGS__); break;         \
        case TP_AMD_FLOAT16: FN<f16_t>(__VA_ARGS__); break;         \
        case TP_AMD_BFLOAT16: FN<bf16_t>(__VA_ARGS__); break;       \
        default: TP_AMD_CHECK(false, "unsupported dtype ", dtype_name(dtype)); \
    }

void launch_head_norm(int dtype, const HeadNormArgs& p, int device) {
    check_extent(p);
    const OnDevice scope(device);
    TP_AMD_DISPATCH_FLOAT(dtype, forward_typed, p, scope.index());
}

void launch_head_norm_backward(int dtype, const HeadNormArgs& p, int device) {
    check_extent(p);
    const OnDevice scope(device);
    TP_AMD_DISPATCH_FLOAT(dtype, backward_typed, p, scope.index());
}

}  // namespace tp_amd

// The join of a block to its residual stream, with the norms on both sides of
// it, forward and backward.
//
// For a row x of the residual and y of the branch: n = y r1 w1 with r1 =
// (mean y^2 + e1)^-1/2 (or n = y), u = drop(n), z = a x + b g u, and h =
// z r2 w2 with r2 = (mean z^2 + e2)^-1/2.  Backward, with m1 = y r1, m2 = z r2
// and v = dh w2: c = mean(v m2), G = dz + r2 (v - m2 c), dx = a G,
// q = drop(b g G), dg = sum b u G, dw1 = sum q m1, dw2 = sum dh m2,
// dy = r1 (q w1 - m1 mean(q w1 m1)).  z is formed again from x and y in
// float32, the same bytes as reading it back rounded.  G is linear in c, so
// the row's sums that need G are two sums each that do not, and all go through
// one exchange: sum(k G) = sum(k (dz + r2 v)) - c sum(k r2 m2).
//
// Bound by memory: forward reads x and y and writes z and h, backward reads x,
// y, dz and dh and writes dx and dy.  A team of threads owns a row in
// registers, at most 16 elements a thread: lanes of one wave for rows of up to
// 64 packets (no barrier), a whole block for wider ones.

#include <algorithm>

#include "attention.h"
#include "device_common.h"
#include "layers.h"
#include "../allocator.h"
#include "../common.h"
#include "../runtime.h"

namespace tp_amd {

namespace {

constexpr int kBlock = 256;
constexpr int kMaxWaves = 16;

template <typename T>
using S_ = typename Elem<T>::storage;

// What the kernels derive from the arguments once, on the host.
struct Plan {
    ResidualNormArgs p;
    FastDiv by_gate;   // rows to gate rows
    int lanes;         // of a team within a wave (a power of two)
    float inv_dim;
    // backward: blocks walk `groups` groups of `group_rows` rows, `per_group` blocks a group
    int64_t groups, group_rows;
    int per_group;
    bool gate_sums;  // the gate's gradient is summed over a group's rows
    float *part1, *part2, *part_gate;  // [blocks][dim]; the gate's [blocks][dim or 1]
};

// Elements at .. at + N of a row of `dim`, as they lie; zeros past its end.
template <typename T>
__device__ __forceinline__ uint4 load_units(const S_<T>* row, int at, int dim) {
    constexpr int N = Packet<T>::N;
    if (at + N <= dim) return load_raw_any(row + at);
    S_<T> v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = at + j < dim ? row[at + j] : S_<T>{};
    uint4 raw;
    __builtin_memcpy(&raw, v, 16);
    return raw;
}

template <typename T>
__device__ __forceinline__ void store_units(S_<T>* row, int at, int dim, const float (&f)[Packet<T>::N]) {
    constexpr int N = Packet<T>::N;
    if (at + N <= dim) {
        store_raw_any_nt(row + at, pack<T>(f));
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (at + j < dim) row[at + j] = Elem<T>::store(f[j]);
    }
}

// A row of weights (null: ones).
template <typename T>
__device__ __forceinline__ void load_weights(const void* w, int at, int dim, float (&f)[Packet<T>::N]) {
    constexpr int N = Packet<T>::N;
    if (w != nullptr) {
        unpack<T>(load_units<T>(static_cast<const S_<T>*>(w), at, dim), f);
        return;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) f[j] = 1.0f;
}

// The gate's row of row r: its elements, or the one for all.
template <typename T>
__device__ __forceinline__ void load_gate(const Plan& w, int64_t r, int at, float (&f)[Packet<T>::N]) {
    constexpr int N = Packet<T>::N;
    if (w.p.gate.data == nullptr) {
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = 1.0f;
        return;
    }
    const S_<T>* row = static_cast<const S_<T>*>(w.p.gate.data) + fastdiv(static_cast<uint32_t>(r), w.by_gate) * w.p.gate.step;
    if (w.p.gate_one) {
        const float g = Elem<T>::load(*row);
#pragma unroll
        for (int j = 0; j < N; ++j) f[j] = g;
        return;
    }
    unpack<T>(load_units<T>(row, at, w.p.dim), f);
}

// Bit j: is element at + j of row r kept.
template <int N>
__device__ __forceinline__ uint32_t drawn(const Plan& w, const DropKey& key, int64_t r, int at) {
    if (!w.p.drops) return (1u << N) - 1;
    return keep_bits<N>(key, static_cast<uint64_t>(r) * static_cast<uint64_t>(w.p.dim) + static_cast<uint64_t>(at));
}

// Sums of K values over a team, each in a fixed order.  Blocks: the waves'
// sums meet in LDS, two buffers in turn, so one barrier a call: a wave that
// writes a buffer again has passed the barrier of the call between, which the
// others reach only after their reads.
template <bool BLOCK, int K>
__device__ __forceinline__ void team_sums(float (&v)[K], int lanes, float (&red)[2][K][kMaxWaves], int& turn) {
    if constexpr (!BLOCK) {
        for (int m = 1; m < lanes; m *= 2) {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += wave_shfl_xor(v[k], m);
        }
    } else {
        const int wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = wave_allreduce(v[k], [](float a, float b) { return a + b; });
        if (threadIdx.x % kWave == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) red[turn][k][wave] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = 0.0f;
            for (int i = 0; i < waves; ++i) t += red[turn][k][i];
            v[k] = t;
        }
        turn ^= 1;
    }
}

template <typename T, int UPL, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? kMaxWaves* kWave : kBlock) void residual_norm_kernel(Plan w) {
    constexpr int N = Packet<T>::N;
    __shared__ float red[2][1][kMaxWaves];
    const int lanes = BLOCK ? blockDim.x : w.lanes;
    const int lane = BLOCK ? threadIdx.x : threadIdx.x & (w.lanes - 1);
    const int64_t r = BLOCK ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * (kBlock / w.lanes) + threadIdx.x / w.lanes;
    if (r >= w.p.rows) return;  // whole teams: a team never spans waves that differ here
    const int dim = w.p.dim;
    const S_<T>* x = static_cast<const S_<T>*>(w.p.x.data) + r * w.p.x.step;
    int turn = 0;
    uint4 rx[UPL], ry[UPL];
#pragma unroll
    for (int k = 0; k < UPL; ++k) rx[k] = load_units<T>(x, (lane + k * lanes) * N, dim);
    float z[UPL][N];
    if (w.p.y.data == nullptr) {
#pragma unroll
        for (int k = 0; k < UPL; ++k) unpack<T>(rx[k], z[k]);
    } else {
        const S_<T>* y = static_cast<const S_<T>*>(w.p.y.data) + r * w.p.y.step;
#pragma unroll
        for (int k = 0; k < UPL; ++k) ry[k] = load_units<T>(y, (lane + k * lanes) * N, dim);
        float r1 = 1.0f;
        if (w.p.norm1) {
            float s[1] = {0.0f};
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
                float f[N];
                unpack<T>(ry[k], f);
#pragma unroll
                for (int j = 0; j < N; ++j) s[0] = fmaf(f[j], f[j], s[0]);
            }
            team_sums<BLOCK, 1>(s, lanes, red, turn);
            r1 = 1.0f / sqrtf(fmaf(s[0], w.inv_dim, w.p.eps1));
            if (lane == 0) w.p.r1[r] = r1;
        }
        const DropKey key(w.p.drop);
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
            const int at = (lane + k * lanes) * N;
            float fx[N], fy[N], w1[N], g[N];
            unpack<T>(rx[k], fx);
            unpack<T>(ry[k], fy);
            load_gate<T>(w, r, at, g);
            load_weights<T>(w.p.norm1 ? w.p.w1 : nullptr, at, dim, w1);
            const uint32_t keep = drawn<N>(w, key, r, at);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                float u = fy[j] * r1 * w1[j];
                if (w.p.drops) u = keep >> j & 1 ? u * w.p.drop.scale : 0.0f;
                z[k][j] = fmaf(w.p.a, fx[j], w.p.b * (g[j] * u));
            }
            store_units<T>(static_cast<S_<T>*>(w.p.z) + r * dim, at, dim, z[k]);
        }
    }
    if (!w.p.norm2) return;
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const int at = (lane + k * lanes) * N;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            // an element past the row's end is no part of it, whatever the factors make of it
            const float t = at + j < dim ? z[k][j] : 0.0f;
            s[0] = fmaf(t, t, s[0]);
        }
    }
    team_sums<BLOCK, 1>(s, lanes, red, turn);
    const float r2 = 1.0f / sqrtf(fmaf(s[0], w.inv_dim, w.p.eps2));
    if (lane == 0) w.p.r2[r] = r2;
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const int at = (lane + k * lanes) * N;
        float w2[N];
        load_weights<T>(w.p.w2, at, dim, w2);
#pragma unroll
        for (int j = 0; j < N; ++j) w2[j] *= z[k][j] * r2;
        store_units<T>(static_cast<S_<T>*>(w.p.h) + r * dim, at, dim, w2);
    }
}

// Adds the teams' column sums of a block (one team: they stand) and writes
// them to `out` as float32, or as the result where there is nothing to add.
template <typename T, int UPL, bool BLOCK>
__device__ __forceinline__ void fold_teams(const float (&sum)[UPL][Packet<T>::N], int lanes, int lane, int dim, float* fold, float* out,
                                           S_<T>* result) {
    constexpr int N = Packet<T>::N;
    if constexpr (BLOCK) {
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
            const int at = (lane + k * lanes) * N;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (at + j >= dim) continue;
                if (result != nullptr) result[at + j] = Elem<T>::store(sum[k][j]);
                else out[at + j] = sum[k][j];
            }
        }
    } else {
        const int teams = kBlock / lanes, mine = threadIdx.x / lanes;
        __syncthreads();  // the previous use of fold is done
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int at = (lane + k * lanes) * N + j;
                if (at < dim) fold[mine * dim + at] = sum[k][j];
            }
        }
        __syncthreads();
        for (int d = threadIdx.x; d < dim; d += kBlock) {
            float t = 0.0f;
            for (int g = 0; g < teams; ++g) t += fold[g * dim + d];
            if (result != nullptr) result[d] = Elem<T>::store(t);
            else out[d] = t;
        }
    }
}

template <typename T, int UPL, bool BLOCK>
__global__ __launch_bounds__(BLOCK ? kMaxWaves* kWave : kBlock) void residual_norm_backward_kernel(Plan w) {
    constexpr int N = Packet<T>::N, K = 5;
    extern __shared__ float fold[];  // [teams][dim] where teams share a block
    __shared__ float red[2][K][kMaxWaves];
    const int lanes = BLOCK ? blockDim.x : w.lanes;
    const int lane = BLOCK ? threadIdx.x : threadIdx.x & (w.lanes - 1);
    const int teams = BLOCK ? 1 : kBlock / w.lanes, mine = BLOCK ? 0 : threadIdx.x / w.lanes;
    const int dim = w.p.dim;
    const bool branch = w.p.y.data != nullptr, gate_row = w.p.dgate != nullptr && !w.gate_sums;
    int turn = 0;
    const DropKey key(w.p.drop);
    const float scale = w.p.drops ? w.p.drop.scale : 1.0f;
    float s1[UPL][N], s2[UPL][N];
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
#pragma unroll
        for (int j = 0; j < N; ++j) s1[k][j] = s2[k][j] = 0.0f;
    }
    for (int64_t group = blockIdx.x / w.per_group; group < w.groups; group += gridDim.x / w.per_group) {
        float sg[UPL][N];
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
#pragma unroll
            for (int j = 0; j < N; ++j) sg[k][j] = 0.0f;
        }
        const int64_t end = (group + 1) * w.group_rows;
        for (int64_t r = group * w.group_rows + static_cast<int64_t>(blockIdx.x % w.per_group) * teams + mine; r < end;
             r += static_cast<int64_t>(w.per_group) * teams) {
            const float r1 = w.p.norm1 ? w.p.r1[r] : 1.0f, r2 = w.p.norm2 ? w.p.r2[r] : 0.0f;
            float x[UPL][N], y[UPL][N], d[UPL][N], v[UPL][N];
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
                const int at = (lane + k * lanes) * N;
                unpack<T>(load_units<T>(static_cast<const S_<T>*>(w.p.x.data) + r * w.p.x.step, at, dim), x[k]);
                if (branch) unpack<T>(load_units<T>(static_cast<const S_<T>*>(w.p.y.data) + r * w.p.y.step, at, dim), y[k]);
                if (w.p.dz.data != nullptr) unpack<T>(load_units<T>(static_cast<const S_<T>*>(w.p.dz.data) + r * w.p.dz.step, at, dim), d[k]);
                if (w.p.norm2) unpack<T>(load_units<T>(static_cast<const S_<T>*>(w.p.dh.data) + r * w.p.dh.step, at, dim), v[k]);
            }
            // x becomes m2 = z r2, y becomes m1, d becomes dz + r2 v
            float f[UPL][N], u[UPL][N];  // f: b g / (1 - p), u: b drop(n), the other factor of dg
            uint32_t keep[UPL];
            float sums[K] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
                const int at = (lane + k * lanes) * N;
                float w1[N], w2[N], g[N];
                load_weights<T>(w.p.norm1 ? w.p.w1 : nullptr, at, dim, w1);
                load_weights<T>(w.p.w2, at, dim, w2);
                load_gate<T>(w, r, at, g);
                keep[k] = branch ? drawn<N>(w, key, r, at) : 0;
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const bool in = at + j < dim, kept = keep[k] >> j & 1;
                    if (w.p.dz.data == nullptr) d[k][j] = 0.0f;
                    float z = w.p.a * x[k][j];
                    f[k][j] = u[k][j] = 0.0f;
                    if (branch) {
                        y[k][j] *= r1;
                        u[k][j] = kept && in ? w.p.b * (y[k][j] * w1[j] * scale) : 0.0f;
                        f[k][j] = w.p.b * (g[j] * scale);
                        z = fmaf(g[j], u[k][j], z);
                    }
                    x[k][j] = 0.0f;
                    if (w.p.norm2 && in) {
                        x[k][j] = z * r2;
                        s2[k][j] = fmaf(v[k][j], x[k][j], s2[k][j]);
                        v[k][j] *= w2[j];
                        sums[0] = fmaf(v[k][j], x[k][j], sums[0]);
                        d[k][j] = fmaf(r2, v[k][j], d[k][j]);
                    }
                    if (w.p.norm1 && kept && in) {
                        const float t = f[k][j] * w1[j] * y[k][j];
                        sums[1] = fmaf(t, d[k][j], sums[1]);
                        sums[2] = fmaf(t * r2, x[k][j], sums[2]);
                    }
                    if (gate_row && w.p.gate_one && in) {
                        sums[3] = fmaf(u[k][j], d[k][j], sums[3]);
                        sums[4] = fmaf(u[k][j] * r2, x[k][j], sums[4]);
                    }
                }
            }
            team_sums<BLOCK, K>(sums, lanes, red, turn);
            const float c = sums[0] * w.inv_dim;
            const float c1 = fmaf(-c, sums[2], sums[1]) * w.inv_dim;
            if (gate_row && w.p.gate_one && lane == 0) static_cast<S_<T>*>(w.p.dgate)[r] = Elem<T>::store(fmaf(-c, sums[4], sums[3]));
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
                const int at = (lane + k * lanes) * N;
                float w1[N], dx[N], dy[N], dg[N];
                load_weights<T>(w.p.norm1 ? w.p.w1 : nullptr, at, dim, w1);
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const float G = fmaf(-c * r2, x[k][j], d[k][j]);
                    dx[j] = w.p.a * G;
                    const float q = keep[k] >> j & 1 ? f[k][j] * G : 0.0f;
                    dg[j] = u[k][j] * G;
                    sg[k][j] += dg[j];
                    dy[j] = q;
                    if (w.p.norm1) {
                        s1[k][j] = fmaf(q, y[k][j], s1[k][j]);
                        dy[j] = r1 * fmaf(-c1, y[k][j], q * w1[j]);
                    }
                }
                if (w.p.dx != nullptr) store_units<T>(static_cast<S_<T>*>(w.p.dx) + r * dim, at, dim, dx);
                if (w.p.dy != nullptr) store_units<T>(static_cast<S_<T>*>(w.p.dy) + r * dim, at, dim, dy);
                if (gate_row && !w.p.gate_one) store_units<T>(static_cast<S_<T>*>(w.p.dgate) + r * dim, at, dim, dg);
            }
        }
        if (!w.gate_sums) continue;
        if (w.p.gate_one) {
            // one number a group: over the columns, and over the teams of a block
            float t = 0.0f;
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
#pragma unroll
                for (int j = 0; j < N; ++j) t += (lane + k * lanes) * N + j < dim ? sg[k][j] : 0.0f;
            }
            t = wave_allreduce(t, [](float a, float b) { return a + b; });
            __syncthreads();
            if (threadIdx.x % kWave == 0) red[0][0][threadIdx.x / kWave] = t;
            __syncthreads();
            if (threadIdx.x == 0) {
                t = 0.0f;
                for (unsigned i = 0; i < blockDim.x / kWave; ++i) t += red[0][0][i];
                if (w.per_group == 1) static_cast<S_<T>*>(w.p.dgate)[group] = Elem<T>::store(t);
                else w.part_gate[blockIdx.x] = t;
            }
            __syncthreads();
        } else {
            fold_teams<T, UPL, BLOCK>(sg, lanes, lane, dim, fold, w.part_gate + static_cast<int64_t>(blockIdx.x) * dim,
                                      w.per_group == 1 ? static_cast<S_<T>*>(w.p.dgate) + group * dim : nullptr);
        }
    }
    const int64_t at = static_cast<int64_t>(blockIdx.x) * dim;
    if (w.p.dw1 != nullptr) fold_teams<T, UPL, BLOCK>(s1, lanes, lane, dim, fold, w.part1 + at, nullptr);
    if (w.p.dw2 != nullptr) fold_teams<T, UPL, BLOCK>(s2, lanes, lane, dim, fold, w.part2 + at, nullptr);
}

// Column sums of the blocks' partials in a fixed order: blockIdx.y names the
// result, 64 columns a block, 16 runs of partial rows, one a wave, then the
// runs in order.
struct Fold {
    const float* part;
    void* out;
    int64_t rows;    // partial rows of one result row
    int64_t width;   // columns
};
struct Folds {
    Fold f[3];
};

constexpr int kFoldWaves = 16;

template <typename T>
__global__ __launch_bounds__(kFoldWaves* kWave) void residual_norm_fold_kernel(Folds folds) {
    __shared__ float run[kFoldWaves][kWave];
    // blockIdx.y: 0 and 1 the weights, 2 + g the gate's row g
    const int which = blockIdx.y < 2 ? blockIdx.y : 2;
    const Fold& f = folds.f[which];
    if (f.out == nullptr) return;
    const int64_t row = which == 2 ? static_cast<int64_t>(blockIdx.y) - 2 : 0;
    const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
    const int64_t d = static_cast<int64_t>(blockIdx.x) * kWave + lane;
    const int64_t per = (f.rows + kFoldWaves - 1) / kFoldWaves;
    float t = 0.0f;
    if (d < f.width) {
        const float* at = f.part + row * f.rows * f.width + d;
        const int64_t end = (wave + 1) * per < f.rows ? (wave + 1) * per : f.rows;
#pragma unroll 8
        for (int64_t b = wave * per; b < end; ++b) t += at[b * f.width];
    }
    run[wave][lane] = t;
    __syncthreads();
    if (wave != 0 || d >= f.width) return;
    for (int k = 1; k < kFoldWaves; ++k) t += run[k][lane];
    static_cast<S_<T>*>(f.out)[row * f.width + d] = Elem<T>::store(t);
}

// How a row's team lies.
struct Shape {
    int upl;
    bool block;
    int threads, lanes, teams;
};

template <typename T>
Shape shape_of(int dim) {
    const int packets = (dim + Packet<T>::N - 1) / Packet<T>::N;
    Shape s{1, packets > kWave, kBlock, 1, 1};
    if (!s.block) {
        while (s.lanes < packets) s.lanes *= 2;
        s.teams = kBlock / s.lanes;
        return s;
    }
    while ((packets + s.upl - 1) / s.upl > kMaxWaves * kWave) s.upl *= 2;
    s.threads = ((packets + s.upl - 1) / s.upl + kWave - 1) / kWave * kWave;
    s.lanes = s.threads;
    return s;
}

Plan plan_of(const ResidualNormArgs& p, const Shape& s) {
    Plan w{};
    w.p = p;
    w.by_gate = make_fastdiv(static_cast<uint32_t>(std::max<int64_t>(p.rows_per_gate, 1)));
    w.lanes = s.lanes;
    w.inv_dim = 1.0f / static_cast<float>(p.dim);
    return w;
}

void check_extent(const ResidualNormArgs& p) {
    TP_AMD_CHECK(p.dim > 0 && p.dim <= kResidualNormMaxDim, "residual_norm: rows of ", p.dim);
    TP_AMD_CHECK(p.rows < (int64_t{1} << 30), "residual_norm: ", p.rows, " rows");
}

template <typename T>
void forward_typed(const ResidualNormArgs& p, int device) {
    const Shape s = shape_of<T>(p.dim);
    const Plan w = plan_of(p, s);
    const unsigned blocks = grid_of((p.rows + s.teams - 1) / s.teams, s.threads, "residual_norm");
    auto* kernel = !s.block ? residual_norm_kernel<T, 1, false> : s.upl == 1 ? residual_norm_kernel<T, 1, true>
                   : s.upl == 2 ? residual_norm_kernel<T, 2, true> : residual_norm_kernel<T, 16 / Packet<T>::N, true>;
    kernel<<<blocks, s.threads, 0, stream(device)>>>(w);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

template <typename T>
void backward_typed(const ResidualNormArgs& p, int device) {
    const Shape s = shape_of<T>(p.dim);
    Plan w = plan_of(p, s);
    // About two blocks a CU walk the rows, each group of rows that shares a
    // gate's row by blocks of its own.
    const int64_t most = 2 * cu_count(device);
    w.gate_sums = p.dgate != nullptr && p.rows_per_gate > 1;
    w.groups = w.gate_sums ? p.rows / p.rows_per_gate : 1;
    w.group_rows = w.gate_sums ? p.rows_per_gate : p.rows;
    w.per_group = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((w.group_rows + s.teams - 1) / s.teams, most / std::max<int64_t>(w.groups, 1))));
    const int64_t blocks = std::min<int64_t>(std::max<int64_t>(w.groups, 1), most) * w.per_group;
    const int64_t gate_width = p.gate_one ? 1 : p.dim;
    const bool gate_part = w.gate_sums && w.per_group > 1;
    const Workspace part(static_cast<size_t>(blocks * ((p.dw1 != nullptr) + (p.dw2 != nullptr)) * p.dim + (gate_part ? blocks * gate_width : 0)) *
                             sizeof(float), device);
    float* next = static_cast<float*>(part.get());
    if (p.dw1 != nullptr) w.part1 = next, next += blocks * p.dim;
    if (p.dw2 != nullptr) w.part2 = next, next += blocks * p.dim;
    if (gate_part) w.part_gate = next;
    const bool sums = p.dw1 != nullptr || p.dw2 != nullptr || w.gate_sums;
    const size_t lds = sums && !s.block ? static_cast<size_t>(s.teams) * p.dim * sizeof(float) : 0;
    auto* kernel = !s.block ? residual_norm_backward_kernel<T, 1, false> : s.upl == 1 ? residual_norm_backward_kernel<T, 1, true>
                   : s.upl == 2 ? residual_norm_backward_kernel<T, 2, true> : residual_norm_backward_kernel<T, 16 / Packet<T>::N, true>;
    kernel<<<static_cast<unsigned>(blocks), s.threads, lds, stream(device)>>>(w);
    TP_AMD_HIP_CHECK(hipGetLastError());
    if (p.dw1 == nullptr && p.dw2 == nullptr && !gate_part) return;
    Folds folds{};
    folds.f[0] = Fold{w.part1, p.dw1, blocks, p.dim};
    folds.f[1] = Fold{w.part2, p.dw2, blocks, p.dim};
    folds.f[2] = Fold{w.part_gate, gate_part ? p.dgate : nullptr, w.per_group, gate_width};
    const dim3 grid(static_cast<unsigned>((p.dim + kWave - 1) / kWave), static_cast<unsigned>(gate_part ? 2 + w.groups : 2));
    residual_norm_fold_kernel<T><<<grid, kFoldWaves * kWave, 0, stream(device)>>>(folds);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

}  // namespace

void launch_residual_norm(int dtype, const ResidualNormArgs& p, int device) {
    check_extent(p);
    if (p.rows <= 0) return;
    const OnDevice scope(device);
    TP_AMD_DISPATCH_TYPED(dtype, forward_typed, p, scope.index());
}

void launch_residual_norm_backward(int dtype, const ResidualNormArgs& p, int device) {
    check_extent(p);
    if (p.rows <= 0) return;
    const OnDevice scope(device);
    TP_AMD_DISPATCH_TYPED(dtype, backward_typed, p, scope.index());
}

}  // namespace tp_amd

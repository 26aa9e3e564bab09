// The join of a block to its residual stream, backward.
//
// With m1 = y r1, u = b drop(m1 w1), z = a x + g u, m2 = z r2 and v = dh w2:
// c = mean(v m2), G = dz + r2 (v - m2 c), dx = a G, q = b g G / (1 - p) where
// kept, dg = sum u G, dw1 = sum q m1, dw2 = sum dh m2, dy = r1 (q w1 -
// m1 mean(q w1 m1)).  z is formed again from x and y in float32, the same bytes
// as reading it back rounded.  With d = dz + r2 v, G = d - c r2 m2 is linear in
// c, and q w1 m1 = g u G: the row's sums need no G, sum(g u G) = sum(g u d) -
// c r2 sum(g u m2), and all go through one exchange (one barrier a row).
//
// Teams walk rows and keep their columns' running sums: of dh m2, and of E m1
// with E = b G / (1 - p) where kept, which is both dw1 = sum g E m1 and dg =
// sum w1 E m1 where the rows of a walk share their gate (the rows of one gate are
// walked together for that).  A block adds its teams' in LDS and writes one
// float32 row of partials, which a second kernel adds up in block order: the
// same bits every time.
//
// Bound by memory: x, y, dz and dh are read once, dx and dy written once; a row
// of more than 1024 packets is read a second time, from L2, as its sums and it
// do not fit the registers.  What was worked on at a time decides: a part of
// four elements after the other, and the sums made where their terms are
// (left alone, the compiler moves the additions past the exchange, keeps every
// term for them and spills).  bf16 8192 x 4096 (403 MB; an elementwise pass of
// it 65 us): 70 us with one norm, 79 with both and a gate, 90 with dropout too,
// and 5 us for the fold; 1700 x 16384 100 (54), float32 3003 x 1000 19 (12).  Masking
// every product of a dropped element is 1 of the 90, and of 28 for float16 rows of
// 768.

#include "attention.h"
#include "residual_norm_rows.h"
#include "../allocator.h"
#include "../runtime.h"

namespace tp_amd {

namespace {

using namespace residual;

// One unit of a row, as loaded.
template <typename T, int V, Gate GATE>
struct Loaded {
    Raw<T, V> x, y, dz, dh, g;

    // ONCE: nothing of it is read again.
    template <bool ONCE>
    __device__ __forceinline__ void load(const Plan& w, int64_t r, int at) {
        auto take = [&](const Rows& t) {
            const S_<T>* p = element<T>(static_cast<const S_<T>*>(t.data) + r * t.step, at);
            return load_unit<T, V, ONCE>(p);
        };
        x = take(w.p.x);
        y = take(w.p.y);
        dz = take(w.p.dz);
        dh = take(w.p.dh);
        g = load_gate<T, V, GATE>(w, r, at);
    }
};

struct RowScalars {
    float r1, r2;
};

// g b drop(m1 w1) of one element, kept by bit j: whatever m1, w1 and g hold, 0
// where it is dropped.  (A gate that is not finite makes the forward's sum of a
// dropped element NaN and r2 with it: so are m2 and the norm's gradient here.)
template <bool NORM, bool DROP, bool GATED>
__device__ __forceinline__ float branch_of(float m1, float w1, float g, float bs, uint32_t keep, int j) {
    float u = m1 * bs;
    if constexpr (NORM) u *= w1;
    if constexpr (GATED) u *= g;
    if constexpr (DROP) u = kept(u, keep, j);
    return u;
}

// A column's or row's sum times the gate or weight it has in common: elements
// that were all dropped make it 0, whatever that factor holds.
template <bool DROP>
__device__ __forceinline__ float shared_factor(float sum, float factor) {
    return DROP && sum == 0.0f ? 0.0f : sum * factor;
}

// What a part of a unit gives from its loads and weights: m1, m2 and d = dz +
// r2 v, which both phases take, v = dh w2 and t = g u (a row's one gate left
// out).
template <int P>
struct Terms {
    float m1[P], m2[P], d[P];
};

template <typename T, int V, bool NORM, bool DROP, Gate GATE>
__device__ __forceinline__ void terms_of(const Plan& w, const Loaded<T, V, GATE>& in, const Raw<T, V>& rw1, const Raw<T, V>& rw2,
                                         const RowScalars& row, float bs, uint32_t keep, int bit, int part, Terms<kPart<V>>& out,
                                         float (&dh)[kPart<V>], float (&v)[kPart<V>], float (&t)[kPart<V>]) {
    constexpr int P = kPart<V>;
    float w1[P], w2[P], g[P], x[P];
    expand_part<T, V>(in.x, part, x);
    expand_part<T, V>(in.y, part, out.m1);
    expand_part<T, V>(in.dz, part, out.d);
    expand_part<T, V>(in.dh, part, dh);
    expand_part<T, V>(rw2, part, w2);
    if constexpr (NORM) expand_part<T, V>(rw1, part, w1);
    if constexpr (GATE != kNoGate) expand_part<T, V>(in.g, part, g);
#pragma unroll
    for (int j = 0; j < P; ++j) {
        if constexpr (NORM) out.m1[j] *= row.r1;
        t[j] = branch_of<NORM, DROP, GATE == kGateRow>(out.m1[j], NORM ? w1[j] : 1.0f, GATE == kGateRow ? g[j] : 1.0f, bs, keep, bit + j);
        out.m2[j] = fmaf(w.p.a, x[j], GATE == kGateOne ? g[j] * t[j] : t[j]) * row.r2;
        if (!w.p.norm2) out.m2[j] = 0.0f;  // (z may be infinite)
        v[j] = dh[j] * w2[j];
        out.d[j] = fmaf(row.r2, v[j], out.d[j]);
    }
}

// Adds the teams' column sums of a block and hands each column's to `take`.
template <int V, int UPL, typename Take>
__device__ __forceinline__ void fold_teams(const Plan& w, const float (&sum)[UPL][V], int lane, int team, float* fold, Take&& take) {
    const int dim = w.p.dim;
    __syncthreads();  // the previous use of fold is done
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const Place<V> at(lane + k * w.lanes, dim);
        if (!at.own) continue;
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if (j >= at.skip) fold[team * dim + at.at + j] = sum[k][j];
        }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < dim; d += blockDim.x) {
        float t = 0.0f;
        for (int g = 0; g < w.teams; ++g) t += fold[g * dim + d];
        take(d, t);
    }
}

template <typename T, int V, int UPL, bool WAVES, bool NORM, bool DROP, Gate GATE>
__global__ __launch_bounds__(WAVES ? kMaxWaves* kWave : 256, 4) void residual_norm_backward_kernel(Plan w) {
    constexpr int K = 3, P = kPart<V>;
    constexpr bool HELD = UPL == 1;  // a row stays in registers between the phases; else it is read again (from L2)
    extern __shared__ float fold[];  // [teams][dim]
    __shared__ float red[2][K][kMaxWaves];
    const int lane = threadIdx.x % w.lanes, dim = w.p.dim;
    // (whole waves: a scalar, and with it the rows' addresses)
    const int team = WAVES ? __builtin_amdgcn_readfirstlane(threadIdx.x / w.lanes) : threadIdx.x / w.lanes;
    int turn = 0;
    const DropKey key(w.p.drop);
    const float bs = DROP ? w.p.b * w.p.drop.scale : w.p.b;
    const bool each = w.p.rows_per_gate == 1;  // a gate of its own for every row
    float s2[UPL][V];
    Raw<T, V> rw1, rw2;
    // (a row read again has its weights in memory, ones where there are none)
    auto weights = [&](int at) {
        if constexpr (NORM) rw1 = !HELD || w.p.w1 != nullptr ? load_unit<T, V, false>(element<T>(w.p.w1, at)) : ones<T, V>();
        rw2 = !HELD || w.p.w2 != nullptr ? load_unit<T, V, false>(element<T>(w.p.w2, at)) : ones<T, V>();
    };
    if (HELD) weights(Place<V>(lane, dim).at);
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
#pragma unroll
        for (int j = 0; j < V; ++j) s2[k][j] = 0.0f;
    }
    auto scalars = [&](int64_t r) { return RowScalars{NORM ? w.p.r1[r] : 1.0f, w.p.norm2 ? w.p.r2[r] : 0.0f}; };
    for (int64_t group = blockIdx.x / w.per_group; group < w.groups; group += gridDim.x / w.per_group) {
        float se[UPL][V];  // sum of E m1, or of g E m1 where every row has a gate of its own
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
#pragma unroll
            for (int j = 0; j < V; ++j) se[k][j] = 0.0f;
        }
        // rows of the block's teams, every block of the group in turn
        const int64_t end = (group + 1) * w.group_rows, step = static_cast<int64_t>(w.per_group) * w.teams;
        int64_t base = group * w.group_rows + static_cast<int64_t>(blockIdx.x % w.per_group) * w.teams;
        for (; base < end; base += step) {
            const int64_t r = base + team;
            const bool there = r < end;
            const int here = stays(lane);
            if (HELD) stay(rw1), stay(rw2);
            Loaded<T, V, GATE> in;
            RowScalars row{1.0f, 0.0f};
            if (there) row = scalars(r);
            Terms<P> terms[HELD ? V / P : 1];
            uint32_t keep = 0;  // V bits a unit
            float sums[K] = {0.0f, 0.0f, 0.0f};
            if (there) {
#pragma unroll
                for (int k = 0; k < UPL; ++k) {
                    const Place<V> at((HELD ? here : stays(lane)) + k * w.lanes, dim);
                    in.template load<HELD>(w, r, at.at);
                    if (!HELD) weights(at.at);
                    if constexpr (DROP) {
                        keep |= (drawn<V>(w, key, r, at.at) & ((1u << V) - 1)) << (k * V);
                        now(keep);
                    }
#pragma unroll
                    for (int i = 0; i < V / P; ++i) {
                        Terms<P>& o = terms[HELD ? i : 0];
                        float dh[P], v[P], t[P];
                        terms_of<T, V, NORM, DROP, GATE>(w, in, rw1, rw2, row, bs, keep, k * V + i * P, i, o, dh, v, t);
#pragma unroll
                        for (int j = 0; j < P; ++j) {
                            s2[k][i * P + j] = fmaf(dh[j], o.m2[j], s2[k][i * P + j]);
                            now(s2[k][i * P + j]);
                        }
                        if (w.ragged) {
#pragma unroll
                            for (int j = 0; j < P; ++j) {
                                v[j] = i * P + j < at.skip ? 0.0f : v[j];
                                t[j] = i * P + j < at.skip ? 0.0f : t[j];
                            }
                        }
#pragma unroll
                        for (int j = 0; j < P; ++j) {
                            sums[0] = fmaf(v[j], o.m2[j], sums[0]);
                            if constexpr (NORM || GATE == kGateOne) {
                                // (a dropped element has no part in a sum, whatever its gradient)
                                sums[1] = fmaf(t[j], DROP ? kept(o.d[j], keep, k * V + i * P + j) : o.d[j], sums[1]);
                                sums[2] = fmaf(t[j], o.m2[j], sums[2]);
                            }
                        }
                        now(sums[0]), now(sums[1]), now(sums[2]);
                        __builtin_amdgcn_sched_barrier(0);  // one part after the other: fewer registers
                    }
                }
            }
            team_sums<WAVES, K>(sums, w.lanes, red, turn);
            if (!there) continue;
            const float cr = sums[0] * w.inv_dim * row.r2;  // c r2
            const float tg = fmaf(-cr, sums[2], sums[1]);   // sum of t G
            float one = 1.0f;
            if constexpr (GATE == kGateOne) {
                float g[P];
                expand_part<T, V>(in.g, 0, g);
                one = g[0];
                if (each && w.p.dgate != nullptr && lane == 0) static_cast<S_<T>*>(w.p.dgate)[r] = Elem<T>::store(tg);
            }
            const float c1 = shared_factor<DROP>(tg, one) * w.inv_dim;
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
                const Place<V> at((HELD ? here : stays(lane)) + k * w.lanes, dim);
                if (!HELD) {
                    in.template load<true>(w, r, at.at);
                    weights(at.at);
                }
                float dx[V], dy[V], dg[V];
#pragma unroll
                for (int i = 0; i < V / P; ++i) {
                    Terms<P>& o = terms[HELD ? i : 0];
                    if constexpr (!HELD) {
                        float dh[P], v[P], t[P];
                        terms_of<T, V, NORM, DROP, GATE>(w, in, rw1, rw2, row, bs, keep, k * V + i * P, i, o, dh, v, t);
                    }
                    float w1[P], g[P];
                    if constexpr (NORM) expand_part<T, V>(rw1, i, w1);
                    if constexpr (GATE != kNoGate) expand_part<T, V>(in.g, i, g);
#pragma unroll
                    for (int j = 0; j < P; ++j) {
                        const int e = i * P + j;
                        const float G = fmaf(-cr, o.m2[j], o.d[j]);
                        dx[e] = w.p.a * G;
                        // Of a dropped element every product is masked, not G alone: m1, w1
                        // and the gate need not be finite.
                        const auto drop = [&](float v) { return DROP ? kept(v, keep, k * V + e) : v; };
                        const float E = bs * G, q = GATE != kNoGate ? E * g[j] : E;
                        if constexpr (NORM || GATE != kNoGate) {
                            se[k][e] = fmaf(drop(GATE != kNoGate && each ? q : E), drop(o.m1[j]), se[k][e]);
                            now(se[k][e]);
                        }
                        if constexpr (GATE == kGateRow) dg[e] = drop(NORM ? E * o.m1[j] * w1[j] : E * o.m1[j]);
                        dy[e] = NORM ? row.r1 * fmaf(-c1, o.m1[j], drop(q * w1[j])) : drop(q);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (!at.own) continue;
                if (w.p.dx != nullptr) store_unit<T, V>(element<T>(static_cast<S_<T>*>(w.p.dx) + r * dim, at.at), dx);
                if (w.p.dy != nullptr) store_unit<T, V>(element<T>(static_cast<S_<T>*>(w.p.dy) + r * dim, at.at), dy);
                if constexpr (GATE == kGateRow) {
                    if (each && w.p.dgate != nullptr) store_unit<T, V>(element<T>(static_cast<S_<T>*>(w.p.dgate) + r * dim, at.at), dg);
                }
            }
        }
        // the group's part of dw1, and its dg
        const S_<T>* gate = static_cast<const S_<T>*>(w.p.gate.data) + (each ? 0 : group * w.p.gate.step);
        const bool first = group == blockIdx.x / w.per_group;
        float* part1 = w.p.dw1 != nullptr ? w.part1 + static_cast<int64_t>(blockIdx.x) * dim : nullptr;
        float one = 0.0f;
        if ((NORM && part1 != nullptr) || w.gate_sums) {
            fold_teams<V, UPL>(w, se, stays(lane), team, fold, [&](int d, float t) {
                if (NORM && part1 != nullptr) {
                    const float f = GATE == kNoGate || each ? t : shared_factor<DROP>(t, Elem<T>::load(GATE == kGateOne ? *gate : gate[d]));
                    part1[d] = first ? f : part1[d] + f;
                }
                if (GATE == kNoGate || !w.gate_sums) return;
                if (NORM && w.p.w1 != nullptr) t = shared_factor<DROP>(t, Elem<T>::load(static_cast<const S_<T>*>(w.p.w1)[d]));
                if (GATE == kGateOne) one += t;
                else if (w.per_group == 1) static_cast<S_<T>*>(w.p.dgate)[group * dim + d] = Elem<T>::store(t);
                else w.part_gate[static_cast<int64_t>(blockIdx.x) * dim + d] = t;
            });
        }
        if (GATE == kGateOne && w.gate_sums) {
            // one number a group: over the columns
            one = wave_allreduce(one, [](float a, float b) { return a + b; });
            __syncthreads();
            if (threadIdx.x % kWave == 0) red[0][0][threadIdx.x / kWave] = one;
            __syncthreads();
            if (threadIdx.x == 0) {
                one = 0.0f;
                for (unsigned i = 0; i < blockDim.x / kWave; ++i) one += red[0][0][i];
                if (w.per_group == 1) static_cast<S_<T>*>(w.p.dgate)[group] = Elem<T>::store(one);
                else w.part_gate[blockIdx.x] = one;
            }
            __syncthreads();
        }
    }
    if (w.p.dw2 != nullptr) {
        float* part2 = w.part2 + static_cast<int64_t>(blockIdx.x) * dim;
        fold_teams<V, UPL>(w, s2, stays(lane), team, fold, [&](int d, float t) { part2[d] = t; });
    }
}

// Column sums of the blocks' partials in a fixed order: blockIdx.y names the
// result, 64 columns a block, 16 runs of partial rows, one a wave, then the
// runs in order.
struct Fold {
    const float* part;
    void* out;
    int64_t rows;   // partial rows of one result row
    int64_t width;  // columns
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

// A row of zeros and one of ones for operands that are not there.
template <typename T>
__global__ void residual_norm_rows_kernel(S_<T>* zeros, S_<T>* one, int dim) {
    const int d = blockIdx.x * blockDim.x + threadIdx.x;
    if (d >= dim) return;
    zeros[d] = Elem<T>::store(0.0f);
    one[d] = Elem<T>::store(1.0f);
}

template <typename T>
void backward_typed(const ResidualNormArgs& given, int device) {
    const Shape s = shape_of<T>(given.dim, 512, kMaxWaves * kWave);
    // The kernel reads every operand without asking whether it is there: branches
    // around its loads cost registers and the order of the loads.
    ResidualNormArgs p = given;
    if (!p.norm2) p.x.data = nullptr, p.w2 = nullptr;  // (only the norm's gradient needs them)
    Workspace rows;
    const bool reread = s.upl > 1;
    if (p.x.data == nullptr || p.y.data == nullptr || p.dz.data == nullptr || p.dh.data == nullptr || (reread && ((p.norm1 && p.w1 == nullptr) || p.w2 == nullptr))) {
        rows = Workspace(2 * sizeof(S_<T>) * p.dim, device);
        S_<T>*zeros = static_cast<S_<T>*>(rows.get()), *one = zeros + p.dim;
        residual_norm_rows_kernel<T><<<(p.dim + 255) / 256, 256, 0, stream(device)>>>(zeros, one, p.dim);
        TP_AMD_HIP_CHECK(hipGetLastError());
        for (Rows* t : {&p.x, &p.y, &p.dz, &p.dh}) {
            if (t->data == nullptr) *t = Rows{zeros, 0};
        }
        if (reread && p.w1 == nullptr) p.w1 = one;
        if (reread && p.w2 == nullptr) p.w2 = one;
    }
    Plan w = plan_of(p, s);
    // Blocks of 16 waves a CU walk the rows, each group of rows that shares a
    // gate's row by blocks of its own.
    const int64_t most = std::max<int64_t>(1, 1024 / s.threads()) * cu_count(device);
    w.gate_sums = p.dgate != nullptr && p.rows_per_gate > 1;
    // (also where the gate's gradient is not wanted: the other sums keep their order)
    const bool grouped = p.gate.data != nullptr && p.rows_per_gate > 1;
    w.groups = grouped ? p.rows / p.rows_per_gate : 1;
    w.group_rows = grouped ? p.rows_per_gate : p.rows;
    w.per_group = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((w.group_rows + s.teams - 1) / s.teams, most / w.groups)));
    const int64_t blocks = std::min<int64_t>(w.groups, most) * w.per_group;
    const int64_t gate_width = p.gate_one ? 1 : p.dim;
    const bool gate_part = w.gate_sums && w.per_group > 1;
    const Workspace part(static_cast<size_t>(blocks * ((p.dw1 != nullptr) + (p.dw2 != nullptr)) * p.dim + (gate_part ? blocks * gate_width : 0)) *
                             sizeof(float), device);
    float* next = static_cast<float*>(part.get());
    if (p.dw1 != nullptr) w.part1 = next, next += blocks * p.dim;
    if (p.dw2 != nullptr) w.part2 = next, next += blocks * p.dim;
    if (gate_part) w.part_gate = next;
    const size_t lds = static_cast<size_t>(s.teams) * p.dim * sizeof(float);
    auto* kernel = TP_AMD_RESIDUAL_KERNEL(residual_norm_backward_kernel, T, s, p);
    kernel<<<static_cast<unsigned>(blocks), s.threads(), lds, stream(device)>>>(w);
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

void launch_residual_norm_backward(int dtype, const ResidualNormArgs& p, int device) {
    check_extent(p);
    if (p.rows <= 0) return;
    const OnDevice scope(device);
    TP_AMD_DISPATCH_TYPED(dtype, backward_typed, p, scope.index());
}

}  // namespace tp_amd

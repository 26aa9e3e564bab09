// The join of a block to its residual stream, with the norms on both sides of
// it, forward.
//
// For a row x of the residual and y of the branch: n = y r1 w1 with r1 =
// (mean y^2 + e1)^-1/2 (or n = y), u = drop(n), z = a x + b g u, and h =
// z r2 w2 with r2 = (mean z^2 + e2)^-1/2, of z before its rounding.
//
// Bound by memory: x and y are read once, z and h written once.  A row's loads,
// its gate's and weights' among them, go out together, the keep bits are drawn
// while they are on their way.  bf16, 8192 x 4096 (268 MB; an elementwise pass of
// it 43.5 us): 46 us with one norm, 51 with both and a gate, 53 with dropout too
// (the generator's 20 products of 32 bits an element's block of 4 are the rest).
// 8 x 4096 3.2 us, a launch's own time.

#include "attention.h"
#include "residual_norm_rows.h"
#include "../runtime.h"

namespace tp_amd {

namespace {

using namespace residual;

template <typename T, int V, int UPL, bool WAVES, bool NORM, bool DROP, Gate GATE>
__global__ __launch_bounds__(kMaxWaves* kWave) void residual_norm_kernel(Plan w) {
    __shared__ float red[2][1][kMaxWaves];
    const int lane = threadIdx.x % w.lanes;
    // (whole waves: a scalar, and with it the rows' addresses)
    const int team = WAVES ? __builtin_amdgcn_readfirstlane(threadIdx.x / w.lanes) : threadIdx.x / w.lanes;
    const int64_t r0 = w.first + static_cast<int64_t>(blockIdx.x) * w.teams + team;
    // a team past the last row goes through the last one again and stores nothing
    const bool there = r0 < w.p.rows;
    const int64_t r = there ? r0 : w.p.rows - 1;
    const int dim = w.p.dim;
    const S_<T>* x = static_cast<const S_<T>*>(w.p.x.data) + r * w.p.x.step;
    const S_<T>* y = static_cast<const S_<T>*>(w.p.y.data) + r * w.p.y.step;
    const bool branch = w.p.y.data != nullptr;
    int turn = 0;
    Raw<T, V> rx[UPL], ry[UPL], rg[UPL], rw1[UPL], rw2[UPL];
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const Place<V> at(lane + k * w.lanes, dim);
        rx[k] = load_unit<T, V, true>(element<T>(x, at.at));
        if (branch) ry[k] = load_unit<T, V, true>(element<T>(y, at.at));
    }
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const Place<V> at(lane + k * w.lanes, dim);
        rg[k] = load_gate<T, V, GATE>(w, r, at.at);
        if constexpr (NORM) rw1[k] = w.p.w1 != nullptr ? load_unit<T, V, false>(element<T>(w.p.w1, at.at)) : ones<T, V>();
        if (w.p.norm2) rw2[k] = w.p.w2 != nullptr ? load_unit<T, V, false>(element<T>(w.p.w2, at.at)) : ones<T, V>();
    }
    // (drawn while the loads are on their way)
    uint32_t keep[UPL];
    if constexpr (DROP) {
        const DropKey key(w.p.drop);
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
            keep[k] = drawn<V>(w, key, r, Place<V>(lane + k * w.lanes, dim).at);
            now(keep[k]);
        }
    }
    float z[UPL][V];
    if (!branch) {
#pragma unroll
        for (int k = 0; k < UPL; ++k) expand<T, V>(rx[k], z[k]);
    } else {
        float r1 = 1.0f;
        if constexpr (NORM) {
            float s[1] = {0.0f};
#pragma unroll
            for (int k = 0; k < UPL; ++k) {
                const Place<V> at(lane + k * w.lanes, dim);
                float f[V];
                expand<T, V>(ry[k], f);
                if (w.ragged) {
#pragma unroll
                    for (int j = 0; j < V; ++j) f[j] = j < at.skip ? 0.0f : f[j];
                }
#pragma unroll
                for (int j = 0; j < V; ++j) s[0] = fmaf(f[j], f[j], s[0]);
            }
            team_sums<WAVES, 1>(s, w.lanes, red, turn);
            r1 = 1.0f / sqrtf(fmaf(s[0], w.inv_dim, w.p.eps1));
            if (lane == 0 && there) w.p.r1[r] = r1;
        }
#pragma unroll
        for (int k = 0; k < UPL; ++k) {
            const Place<V> at(lane + k * w.lanes, dim);
            float x_[V], u[V], w1[V], g[V];
            expand<T, V>(rx[k], x_);
            expand<T, V>(ry[k], u);
            if constexpr (NORM) expand<T, V>(rw1[k], w1);
            if constexpr (GATE != kNoGate) expand<T, V>(rg[k], g);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if constexpr (NORM) u[j] *= r1 * w1[j];
                if constexpr (DROP) u[j] = kept(u[j] * w.p.drop.scale, keep[k], j);
                if constexpr (GATE != kNoGate) u[j] *= g[j];
                z[k][j] = fmaf(w.p.a, x_[j], w.p.b * u[j]);
            }
            if (at.own && there) store_unit<T, V>(element<T>(static_cast<S_<T>*>(w.p.z) + r * dim, at.at), z[k]);
        }
    }
    if (!w.p.norm2) return;
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const Place<V> at(lane + k * w.lanes, dim);
        float f[V];
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = z[k][j];
        if (w.ragged) {
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = j < at.skip ? 0.0f : f[j];
        }
#pragma unroll
        for (int j = 0; j < V; ++j) s[0] = fmaf(f[j], f[j], s[0]);
    }
    team_sums<WAVES, 1>(s, w.lanes, red, turn);
    const float r2 = 1.0f / sqrtf(fmaf(s[0], w.inv_dim, w.p.eps2));
    if (lane == 0 && there) w.p.r2[r] = r2;
#pragma unroll
    for (int k = 0; k < UPL; ++k) {
        const Place<V> at(lane + k * w.lanes, dim);
        float h[V];
        expand<T, V>(rw2[k], h);
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] *= z[k][j] * r2;
        if (at.own && there) store_unit<T, V>(element<T>(static_cast<S_<T>*>(w.p.h) + r * dim, at.at), h);
    }
}

// 16-bit rows of a full device whose units lie between a half and three quarters
// of a power of two of lanes: a quarter of the lanes, three units each.  Lanes
// that hold nothing draw and wait like the others, and a row's sums take fewer
// moves.  bf16 with dropout 7812 x 768 16.8 -> 11.8 us, 9983 x 601 21.0 -> 17.8,
// 5454 x 1100 18.2 -> 16.5; without 11.6 -> 10.1, 13.6 -> 13.4 and 11.9 -> 12.7, so
// rows without dropout that fill less than three quarters of the units stay as they
// are.  Not kept: float32 (5.9 M elements: 22.4 -> 21.3 us in rows of 384, 19.8 ->
// 21.4 of 768), four lanes for rows of 72 (21.4 -> 24.1), and two or four units for
// powers of two (5859 x 1024 13.7 -> 13.2, 2929 x 2048 14 -> 20).
inline bool three_units(int units, bool drops, int& lanes) {
    int few = 16;
    while (few < kWave && 3 * few < units) few *= 2;
    if (units <= 2 * few || units > 3 * few || (!drops && 4 * units < 9 * few)) return false;
    lanes = few;
    return true;
}

template <typename T>
void forward_typed(const ResidualNormArgs& p, int device) {
    // Of rows that fill the device wide ones go to fewer threads, which wait for
    // each other less: bf16 8192 x 4096 with dropout 57 -> 53 us, 3400 x 8192 49 ->
    // 44; eight rows of 4096 3.2 us by 512 threads, 3.6 by 256.  Just past the border
    // lanes lie idle either way: with one norm and both, 13618 x 2056 43 and 46 us (41
    // and 51 by one packet a thread), 5600 x 5000 43 and 45 (42 and 54),
    // float32 13618 x 1028 44 and 45 (42 and 47), 10937 x 1280 39 and 41 (38 and 41).
    const bool many = p.rows >= 2 * cu_count(device);
    Shape s = shape_of<T>(p.dim, 256, many ? 256 : kMaxWaves * kWave);
    bool three = false;
    if constexpr (sizeof(S_<T>) == 2) {
        three = many && s.unit > 1 && three_units((p.dim + s.unit - 1) / s.unit, p.drops, s.lanes);
        if (three) s.upl = 3, s.waves = false, s.teams = 256 / s.lanes;
    }
    Plan w = plan_of(p, s);
    auto* kernel = TP_AMD_RESIDUAL_KERNEL(residual_norm_kernel, T, s, p);
    if constexpr (sizeof(S_<T>) == 2) {
        if (three) kernel = TP_AMD_RESIDUAL_FORM(residual_norm_kernel, T, Packet<T>::N, 3, false, p);
    }
    // (more rows than one launch takes go in several)
    const int64_t at_once = most_blocks(s.threads()) * s.teams;
    for (; w.first < p.rows; w.first += at_once) {
        const int64_t rows = std::min(at_once, p.rows - w.first);
        kernel<<<static_cast<unsigned>((rows + s.teams - 1) / s.teams), s.threads(), 0, stream(device)>>>(w);
        TP_AMD_HIP_CHECK(hipGetLastError());
    }
}

}  // namespace

void launch_residual_norm(int dtype, const ResidualNormArgs& p, int device) {
    check_extent(p);
    if (p.rows <= 0) return;
    const OnDevice scope(device);
    TP_AMD_DISPATCH_TYPED(dtype, forward_typed, p, scope.index());
}

}  // namespace tp_amd

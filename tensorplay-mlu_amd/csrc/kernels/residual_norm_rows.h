// What the forward and the backward of the residual join share
// (residual_norm.hip, residual_norm_backward.hip): how a row lies over
// threads, and the loads, sums and draws of a row.
//
// A team of threads owns a row, UPL units of V elements a thread: lanes of one
// wave for rows of up to 64 units (no barrier; of up to 192 in the forward's
// form of three units a lane), whole waves for wider ones,
// several teams a block where they fit.  V is a 16-byte packet, or one element
// for rows shorter than that.  The unit that ends a row starts
// early enough to be whole: the elements that it shares with the unit before
// it are computed twice, to the same bits, and left out of sums.
#pragma once

#include <algorithm>
#include <type_traits>

#include "device_common.h"
#include "layers.h"
#include "../common.h"

namespace tp_amd {
namespace residual {

constexpr int kMaxWaves = 16;

template <typename T>
using S_ = typename Elem<T>::storage;

enum Gate { kNoGate, kGateRow, kGateOne };

// What the kernels derive from the arguments once, on the host.
struct Plan {
    ResidualNormArgs p;
    FastDiv by_gate;  // rows to gate rows
    int lanes;        // threads of a team
    int teams;        // of a block
    bool ragged;      // a thread's units hold elements of no row or of two units
    bool low;         // every generator's block has a number below 2^32
    float inv_dim;
    int64_t first;  // forward: row of the launch
    // backward: blocks walk `groups` groups of `group_rows` rows, `per_group` blocks a group
    int64_t groups, group_rows;
    int per_group;
    bool gate_sums;                    // the gate's gradient is summed over a group's rows
    float *part1, *part2, *part_gate;  // [blocks][dim]; the gate's [blocks][dim or 1]
};

// A unit as it lies: a packet, or one element.
template <typename T, int V>
using Raw = std::conditional_t<V == 1, S_<T>, uint4>;

// At any element address; ONCE: nothing of it is read again.
template <typename T, int V, bool ONCE>
__device__ __forceinline__ Raw<T, V> load_unit(const S_<T>* p) {
    if constexpr (V == 1) return *p;
    else return ONCE ? load_raw_any_nt(p) : load_raw_any(p);
}

template <typename T, int V>
__device__ __forceinline__ void expand(const Raw<T, V>& raw, float (&f)[V]) {
    if constexpr (V == 1) f[0] = Elem<T>::load(raw);
    else unpack<T>(raw, f);
}

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> ones() {
    float f[V];
#pragma unroll
    for (int j = 0; j < V; ++j) f[j] = 1.0f;
    if constexpr (V == 1) return Elem<T>::store(f[0]);
    else return pack<T>(f);
}

// Keeps what is made of a unit, or of a lane, inside the loop that uses it: made
// once before a loop over rows, conversions would hold twice the registers, and
// the masks of a row's end a pair of scalars an element.
template <typename R>
__device__ __forceinline__ void stay(R& raw) {
    if constexpr (sizeof(R) == 16) asm volatile("" : "+v"(raw.x), "+v"(raw.y), "+v"(raw.z), "+v"(raw.w));
}
__device__ __forceinline__ int stays(int lane) {
    asm volatile("" : "+v"(lane));
    return lane;
}
// A value that is needed later (a sum a row later, keep bits a phase later),
// made here and not where its operands would have to wait for it.
template <typename F>
__device__ __forceinline__ void now(F& v) {
    asm volatile("" : "+v"(v));
}

// Elements of a unit that are worked on at a time, so that what they need fits
// the registers beside what stays: four, half a 16-bit packet.
template <int V>
constexpr int kPart = V < 4 ? V : 4;

// Part i of a unit as float32.
template <typename T, int V>
__device__ __forceinline__ void expand_part(const Raw<T, V>& raw, int i, float (&f)[kPart<V>]) {
    if constexpr (kPart<V> == V) {
        expand<T, V>(raw, f);
    } else {
        const uint32_t a = i ? raw.z : raw.x, b = i ? raw.w : raw.y;
        if constexpr (std::is_same_v<T, bf16_t>) {
            f[0] = __uint_as_float(a << 16), f[1] = __uint_as_float(a & 0xffff0000u);
            f[2] = __uint_as_float(b << 16), f[3] = __uint_as_float(b & 0xffff0000u);
        } else {
            f[0] = f16_to_float(static_cast<uint16_t>(a & 0xffffu)), f[1] = f16_to_float(static_cast<uint16_t>(a >> 16));
            f[2] = f16_to_float(static_cast<uint16_t>(b & 0xffffu)), f[3] = f16_to_float(static_cast<uint16_t>(b >> 16));
        }
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_unit(S_<T>* p, const float (&f)[V]) {
    if constexpr (V == 1) *p = Elem<T>::store(f[0]);
    else store_raw_any_nt(p, pack<T>(f));
}

// A unit's first element and how many of its first ones are not its own.
template <int V>
struct Place {
    int at, skip;
    bool own;  // any is
    __device__ __forceinline__ Place(int unit, int dim) {
        const int first = unit * V, last = dim - V;
        at = first < last ? first : last;
        skip = first - at;
        own = first < dim;
    }
};

// Element `at` of a row: the offset in 32 bits, so that a row all lanes share
// is addressed by a scalar and one register.
template <typename T>
__device__ __forceinline__ const S_<T>* element(const void* row, int at) {
    return reinterpret_cast<const S_<T>*>(static_cast<const char*>(row) + static_cast<uint32_t>(at) * static_cast<uint32_t>(sizeof(S_<T>)));
}
template <typename T>
__device__ __forceinline__ S_<T>* element(void* row, int at) {
    return reinterpret_cast<S_<T>*>(static_cast<char*>(row) + static_cast<uint32_t>(at) * static_cast<uint32_t>(sizeof(S_<T>)));
}

// The gate's unit of row r: of its row, or its one element (in every place).
template <typename T, int V, Gate GATE>
__device__ __forceinline__ Raw<T, V> load_gate(const Plan& w, int64_t r, int at) {
    if constexpr (GATE == kNoGate) return Raw<T, V>{};
    const S_<T>* row = static_cast<const S_<T>*>(w.p.gate.data) + fastdiv(static_cast<uint32_t>(r), w.by_gate) * w.p.gate.step;
    if constexpr (GATE == kGateRow || V == 1) {
        return load_unit<T, V, false>(GATE == kGateRow ? element<T>(row, at) : row);
    } else {
        const uint32_t one = sizeof(S_<T>) == 4 ? __builtin_bit_cast(uint32_t, static_cast<float>(Elem<T>::load(*row)))
                                                : static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(row)) * 0x10001u;
        return make_uint4(one, one, one, one);
    }
}

// Bit j: is element at + j of row r kept.
template <int V>
__device__ __forceinline__ uint32_t drawn(const Plan& w, const DropKey& key, int64_t r, int at) {
    const uint64_t e = static_cast<uint64_t>(r) * static_cast<uint64_t>(w.p.dim) + static_cast<uint64_t>(at);
    return w.low ? keep_bits_at<V, true>(key, e) : keep_bits_at<V, false>(key, e);
}

// Sums of K values over a team, each in a fixed order.  Waves: their sums meet
// in LDS, two buffers in turn, so one barrier a call: a wave that writes a
// buffer again has passed the barrier of the call between, which the others
// reach only after their reads.
template <bool WAVES, int K>
__device__ __forceinline__ void team_sums(float (&v)[K], int lanes, float (&red)[2][K][kMaxWaves], int& turn) {
    if constexpr (!WAVES) {
        for (int m = 1; m < lanes; m *= 2) {
#pragma unroll
            for (int k = 0; k < K; ++k) v[k] += wave_shfl_xor(v[k], m);
        }
    } else {
        const int wave = threadIdx.x / kWave, waves = lanes / kWave, first = wave / waves * waves;
        const auto plus = [](float a, float b) { return a + b; };
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = wave_allreduce(v[k], plus);
        if (threadIdx.x % kWave == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) red[turn][k][wave] = v[k];
        }
        __syncthreads();
        // every row of 16 lanes reads the team's sums and adds them up: one trip to LDS
        const int one = threadIdx.x % kMaxWaves;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = red[turn][k][first + (one < waves ? one : 0)];
            t = one < waves ? t : 0.0f;
            t += row_ror<8>(t);
            t += row_ror<4>(t);
            t += row_ror<2>(t);
            v[k] = t + row_ror<1>(t);
        }
        turn ^= 1;
    }
}

// How a row's team lies.
struct Shape {
    int upl;      // units a thread
    int unit;     // V
    bool waves;   // a team is whole waves
    int lanes, teams;
    int threads() const { return lanes * teams; }
};

// Teams of `most` threads a block at most, or one team; rows of more than
// `single` packets go 16 elements a thread.
template <typename T>
Shape shape_of(int dim, int most, int single) {
    constexpr int N = Packet<T>::N;
    Shape s{1, dim < N ? 1 : N, false, 1, 1};
    const int units = (dim + s.unit - 1) / s.unit;
    s.waves = units > kWave;
    if (!s.waves) {
        while (s.lanes < units) s.lanes *= 2;
        s.teams = 256 / s.lanes;
        return s;
    }
    if (units > single) s.upl = 16 / N;
    s.lanes = ((dim + s.unit * s.upl - 1) / (s.unit * s.upl) + kWave - 1) / kWave * kWave;
    s.teams = std::max(1, most / s.lanes);
    return s;
}

inline Plan plan_of(const ResidualNormArgs& p, const Shape& s) {
    Plan w{};
    w.p = p;
    w.by_gate = make_fastdiv(static_cast<uint32_t>(std::max<int64_t>(p.rows_per_gate, 1)));
    w.lanes = s.lanes;
    w.teams = s.teams;
    w.low = p.rows * p.dim / 4 + 4 < (int64_t{1} << 32);
    w.ragged = s.lanes * s.upl * s.unit != p.dim;
    w.inv_dim = 1.0f / static_cast<float>(p.dim);
    return w;
}

inline void check_extent(const ResidualNormArgs& p) {
    TP_AMD_CHECK(p.dim > 0 && p.dim <= kResidualNormMaxDim, "residual_norm: rows of ", p.dim);
    TP_AMD_CHECK(p.rows < kMaxRows, "residual_norm: ", p.rows, " rows");
}

// The kernel of a form: KERNEL<T, V, UPL, WAVES, NORM, DROP, GATE> by shape,
// branch's norm, dropout and gate.
#define TP_AMD_RESIDUAL_GATE(KERNEL, T, V, UPL, WAVES, NORM, DROP, p)                                            \
    ((p).gate.data == nullptr ? KERNEL<T, V, UPL, WAVES, NORM, DROP, kNoGate>                                    \
     : (p).gate_one           ? KERNEL<T, V, UPL, WAVES, NORM, DROP, kGateOne>                                   \
                              : KERNEL<T, V, UPL, WAVES, NORM, DROP, kGateRow>)
#define TP_AMD_RESIDUAL_FORM(KERNEL, T, V, UPL, WAVES, p)                                                        \
    ((p).norm1 ? ((p).drops ? TP_AMD_RESIDUAL_GATE(KERNEL, T, V, UPL, WAVES, true, true, p)                      \
                            : TP_AMD_RESIDUAL_GATE(KERNEL, T, V, UPL, WAVES, true, false, p))                    \
               : ((p).drops ? TP_AMD_RESIDUAL_GATE(KERNEL, T, V, UPL, WAVES, false, true, p)                     \
                            : TP_AMD_RESIDUAL_GATE(KERNEL, T, V, UPL, WAVES, false, false, p)))
#define TP_AMD_RESIDUAL_KERNEL(KERNEL, T, s, p)                                                                  \
    (!(s).waves      ? ((s).unit == 1 ? TP_AMD_RESIDUAL_FORM(KERNEL, T, 1, 1, false, p)                          \
                                      : TP_AMD_RESIDUAL_FORM(KERNEL, T, Packet<T>::N, 1, false, p))              \
     : (s).upl == 1  ? TP_AMD_RESIDUAL_FORM(KERNEL, T, Packet<T>::N, 1, true, p)                                 \
                     : TP_AMD_RESIDUAL_FORM(KERNEL, T, Packet<T>::N, 16 / Packet<T>::N, true, p))

}  // namespace residual
}  // namespace tp_amd

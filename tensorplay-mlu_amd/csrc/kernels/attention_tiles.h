// Device-side pieces the attention kernels share: which keys a row sees, the
// matrix instruction on 16-byte fragments, and LDS tiles of keys, values or
// queries that are read both by rows and transposed.
//
// All kernels form scores with the keys (or queries) of an LDS tile as rows
// and a wave's own 32 queries (or keys) as columns.  A 32 x 32 accumulator
// gives a lane column lane % 32 and rows 8 g + 4 (lane / 32) + r in element
// 4 g + r: exactly the rows a fragment of the next product's right operand
// needs in that lane, if the left operand takes its rows in the same order.
// So probabilities go from one product to the next in the registers they were
// formed in, and a column's maximum and sum are a lane's own, but for one
// exchange between the two halves of the wave.
#pragma once

#include <type_traits>
#include <utility>

#include "attention.h"
#include "device_common.h"

namespace tp_amd {
namespace attention {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void* LdsPtr;

// f(0), f(1), ... with compile-time arguments.
template <typename F, int... N>
__device__ __forceinline__ void unrolled(const F& f, std::integer_sequence<int, N...>) {
    (f(std::integral_constant<int, N>{}), ...);
}

template <typename T>
using S_ = typename Elem<T>::storage;

// Positions lie under it in magnitude, so differences of them fit an int.
constexpr int kNoWindow = 1 << 30;

// What a row sees: keys j <= p of which j > p - window or j < sinks.
struct Rule {
    int window;  // kNoWindow: every earlier key
    int sinks;
    __device__ __forceinline__ bool sees(int p, int j) const { return j <= p && (j > p - window || j < sinks); }
    // Keys that row p sees, no fewer than any row before it.
    __device__ __forceinline__ int count_seen(int p) const { return p - window < sinks ? p + 1 : window + sinks; }
    // Every row of p0 .. p1 sees all of the keys k0 .. k1.
    __device__ __forceinline__ bool all_see(int p0, int p1, int k0, int k1) const {
        return k1 <= p0 && (k0 > p1 - window || k1 < sinks);
    }
    // Some row of p0 .. p1 sees some key of k0 .. k1.
    __device__ __forceinline__ bool any_sees(int p0, int p1, int k0, int k1) const {
        return p0 <= p1 && k0 <= p1 && (k1 > p0 - window || k0 < sinks);
    }
};

// A sequence of the batch: query i stands at position start + i and is alive
// when that lies in [0, length).
struct Sequence {
    int length, start;
    int first, end;  // its alive queries
};

struct Shape {
    int queries, keys, heads, kv_heads, group, dim;
    Rule rule;
    const void *lengths, *starts;
    bool wide_lengths, wide_starts;
    int64_t lengths_step, starts_step;
};

__device__ __forceinline__ int64_t read_index(const void* p, bool wide, int64_t at) {
    return wide ? static_cast<const int64_t*>(p)[at] : static_cast<const int32_t*>(p)[at];
}

// Lengths past the keys count as all keys, negative ones as none; a start
// that leaves no query alive is held to one that fits 32 bits and does too.
__device__ __forceinline__ Sequence sequence_of(const Shape& s, int b) {
    Sequence q;
    int64_t length = s.keys;
    if (s.lengths != nullptr) {
        length = read_index(s.lengths, s.wide_lengths, b * s.lengths_step);
        length = length < 0 ? 0 : length > s.keys ? s.keys : length;
    }
    int64_t start = length - s.queries;
    if (s.starts != nullptr) {
        start = read_index(s.starts, s.wide_starts, b * s.starts_step);
        start = start < -s.queries ? -s.queries : start > s.keys ? s.keys : start;
    }
    q.length = __builtin_amdgcn_readfirstlane(static_cast<int>(length));
    q.start = __builtin_amdgcn_readfirstlane(static_cast<int>(start));
    q.first = q.start < 0 ? -q.start : 0;
    q.end = q.length - q.start < s.queries ? q.length - q.start : s.queries;
    return q;
}

// The key tiles of BK that rows p0 .. p1 (alive, p0 <= p1) see: `sinks` tiles
// from key 0 on, then `count - sinks` from tile `low` on.
struct KeyTiles {
    int sinks, low, count;
    int low_key;  // the window's first key
    __device__ __forceinline__ KeyTiles(const Rule& r, int p0, int p1, int bk) {
        low_key = p0 - r.window + 1 > 0 ? p0 - r.window + 1 : 0;
        low = low_key / bk;
        const int s = r.sinks < p1 + 1 ? r.sinks : p1 + 1;
        sinks = (s + bk - 1) / bk;
        if (sinks > low) sinks = low;
        const int near = p1 / bk - low + 1;
        count = sinks + (near > 0 ? near : 0);
    }
    __device__ __forceinline__ int at(int i) const { return i < sinks ? i : low + i - sinks; }
};

// Keys that some row of a block sees, which are the ones it reads: up to the
// last row's position, from the first row's window on or among the first.
struct KeysSeen {
    int last, low_key, sinks;
    __device__ __forceinline__ KeysSeen(const Rule& r, const KeyTiles& t, int p1) : last(p1), low_key(t.low_key), sinks(r.sinks) {}
    __device__ __forceinline__ bool operator()(int j) const { return j <= last && (j >= low_key || j < sinks); }
    __device__ __forceinline__ bool all(int k0, int k1) const { return k1 <= last && (k0 >= low_key || k1 < sinks); }
};

// ---- matrix instruction ---------------------------------------------------------

// C += A B on fragments of 16 bytes a lane: 16 steps of the inner axis for
// 16-bit types, 8 for float32 (lane half h holds 4 h .. 4 h + 3 of them).
template <typename T>
__device__ __forceinline__ f32x16 mma(const uint4& a, const uint4& b, f32x16 c) {
    if constexpr (std::is_same_v<T, float>) {
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.x), __uint_as_float(b.x), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.y), __uint_as_float(b.y), c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.z), __uint_as_float(b.z), c, 0, 0, 0);
        return __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(a.w), __uint_as_float(b.w), c, 0, 0, 0);
    } else if constexpr (std::is_same_v<T, bf16_t>) {
        typedef __bf16 V __attribute__((ext_vector_type(8)));
        V x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
    } else {
        typedef _Float16 V __attribute__((ext_vector_type(8)));
        V x, y;
        __builtin_memcpy(&x, &a, 16);
        __builtin_memcpy(&y, &b, 16);
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
    }
}

// Row that element e of a 32 x 32 accumulator holds.
__device__ __forceinline__ int row_of(int e, int half) { return 8 * (e / 4) + 4 * half + e % 4; }

__device__ __forceinline__ f32x16 zeros() {
    f32x16 z;
#pragma unroll
    for (int e = 0; e < 16; ++e) z[e] = 0.0f;
    return z;
}

// Fragments in which one 32 x 32 accumulator's rows feed the next product.
template <typename T>
constexpr int kFragsOf32 = sizeof(S_<T>) == 4 ? 4 : 2;

// Fragment f of them, rounded to T (float32: as it is).
template <typename T>
__device__ __forceinline__ uint4 pack_rows(const f32x16& s, int f) {
    constexpr int N = Packet<T>::N;
    float v[N];
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = s[N * f + j];
    return pack<T>(v);
}

// op over the two lanes of a column (the halves of the wave), in both.
template <typename Op>
__device__ __forceinline__ float both_halves(float v, Op op) {
    const uint32_t u = __float_as_uint(v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // {low, low}, {high, high}
    return op(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

struct MaxOf {
    __device__ __forceinline__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct SumOf {
    __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};

// ---- LDS tiles ---------------------------------------------------------------------

// R token rows of DT x 32 elements, filled by W waves with loads straight
// into LDS (16 bytes a lane, cache policy AUX).  Rows are padded to a power of two bytes, and the
// 16-byte chunk c of row r lies at slot c ^ swizzle(r): 16 rows at one chunk
// (a fragment read by rows) take 16 different sixteenths of LDS's 256 bytes a
// clock, and 4 consecutive rows at 64 bytes (half a transposed read) its four
// quarters.
template <typename T, int DT, int R, int W, int AUX = 0>
struct Tile {
    using S = S_<T>;
    static constexpr int E = sizeof(S);
    static constexpr int kUsed = DT * 32 * E;
    static constexpr int kRow = kUsed <= 64 ? 64 : kUsed <= 128 ? 128 : kUsed <= 256 ? 256 : 512;
    static constexpr int kChunks = kRow / 16;
    static constexpr int kBytes = R * kRow;
    static constexpr int kPerLoad = 1024 / kRow;  // rows a load instruction fills
    static constexpr int kIssue = kBytes / 1024 / W;
    static constexpr int kSteps = kUsed / 32;  // fragments along a row
    static_assert(kIssue * 1024 * W == kBytes, "the waves share a tile's loads evenly");

    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (kRow == 64) return (r >> 2) & 3;
        else if constexpr (kRow == 128) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        else return ((r & 3) << 2) | ((r >> 2) & 3);
    }

    // A wave's loads of tiles of one tensor, whose token rows lie `step`
    // elements apart from `head` on.
    struct Loads {
        // the swizzle repeats every 16 rows
        static constexpr int kPeriod = kPerLoad * W >= 16 ? 1 : 16 / (kPerLoad * W);
        const S* head;
        int64_t step;
        uint32_t records;       // bytes from a load's first row to its last one's end
        uint32_t off[kPeriod];  // a lane's place in the rows of load i % kPeriod
        int row;                // and its row in load 0

        __device__ __forceinline__ void init(const S* first, int64_t step_, int dim, int wave, int lane) {
            step = step_;
            head = first + wave * kPerLoad * step;
            records = static_cast<uint32_t>(((kPerLoad - 1) * step + dim) * E);
            row = wave * kPerLoad + lane / kChunks;
            unrolled([&](auto i) __attribute__((always_inline)) {
                const int chunk = (lane % kChunks) ^ swizzle(i * W * kPerLoad + row);
                off[i] = chunk * 16 < dim * E ? static_cast<uint32_t>(lane / kChunks * step * E) + chunk * 16 : kOutOfRange;
            }, std::make_integer_sequence<int, kPeriod>{});
        }

        // Rows r0 .. r0 + R - 1 into `tile`: all of them if `whole`, else row r
        // if keep(r), the others as zeros.
        template <typename Keep>
        __device__ __forceinline__ void issue(char* tile, int r0, int wave, bool whole, const Keep& keep) const {
            const S* from = head + r0 * step;
            if (whole) {
                unrolled([&](auto i) __attribute__((always_inline)) { load(i, tile, from, wave, off[i % kPeriod]); }, std::make_integer_sequence<int, kIssue>{});
            } else {
                unrolled([&](auto i) __attribute__((always_inline)) { load(i, tile, from, wave, keep(r0 + row + i * W * kPerLoad) ? off[i % kPeriod] : kOutOfRange); },
                         std::make_integer_sequence<int, kIssue>{});
            }
        }

    private:
        __device__ __forceinline__ void load(int i, char* tile, const S* from, int wave, uint32_t at) const {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(buffer_over(from + i * W * kPerLoad * step, records),
                                                     (LdsPtr)(tile + (i * W + wave) * 1024), 16, at, 0, 0, AUX);
        }
    };

    // A lane's offsets for reading 32 rows (lane % 32) at fragment s of them.
    struct ByRows {
        int off[kSteps];
        __device__ __forceinline__ void init(int lane) {
            const int l32 = lane % 32, half = lane / 32;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) off[s] = l32 * kRow + (((2 * s + half) ^ swizzle(l32)) << 4);
        }
        // rows 32 u ..
        __device__ __forceinline__ uint4 read(const char* tile, int u, int s) const {
            return *reinterpret_cast<const uint4*>(tile + 32 * u * kRow + off[s]);
        }
    };

    // Transposed: 32 columns (32 t + lane % 32) by fragment f of rows 32 u ..
    // in the order pack_rows has them.
    struct Transposed {
        int lo[DT];
        __device__ __forceinline__ void init(int lane) {
            const int l32 = lane % 32, half = lane / 32;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                if constexpr (E == 2) {
                    // lane p of a 16-lane group addresses row p / 4 of four
                    // and 8 bytes of it; it gets column p of the four rows
                    const int p = lane % 16, row = 4 * half + p / 4, col = 32 * t + (lane & 16) + 4 * (p % 4);
                    lo[t] = row * kRow + (((col / 8) ^ swizzle(row)) << 4) + (col % 8) * 2;
                } else {
                    const int row = 4 * half, col = 32 * t + l32;
                    lo[t] = row * kRow + (((col / 4) ^ swizzle(row)) << 4) + (col % 4) * 4;
                }
            }
        }
        __device__ __forceinline__ uint4 read(const char* tile, int t, int u, int f) const {
            uint4 v;
            if constexpr (E == 2) {
                typedef short short4_t __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) short4_t* Ptr;
                const char* q = tile + (32 * u + 16 * f) * kRow;
                // eight rows on, bit 1 of the swizzle turns
                const short4_t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(q + lo[t]));
                const short4_t b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(q + 8 * kRow + (lo[t] ^ 32)));
                __builtin_memcpy(&v, &a, 8);
                __builtin_memcpy(reinterpret_cast<char*>(&v) + 8, &b, 8);
            } else {
                // row 8 f + 4 half + j: bits 0 and 1 turn chunk bits 2 and 3
                // (wide rows) or bit 1 turns chunk bit 2, bit 3 chunk bit 1
                const char* q = tile + (32 * u + 8 * f) * kRow;
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int turn = (swizzle(8 * f + j) ^ swizzle(0)) << 4;
                    w[j] = *reinterpret_cast<const uint32_t*>(q + j * kRow + (lo[t] ^ turn));
                }
                v = make_uint4(w[0], w[1], w[2], w[3]);
            }
            return v;
        }
    };
};

// 16 bytes a lane of a wave's own 32 rows, straight from memory: fragment s of
// row `row` (zeros when not `in`).
template <typename T>
__device__ __forceinline__ uint4 load_fragment(Rsrc res, bool in, uint32_t row_bytes, int s, int half, int dim) {
    constexpr int E = sizeof(S_<T>);
    const uint32_t at = (2 * s + half) * 16;
    return buffer_load16_cached(res, in && at < static_cast<uint32_t>(dim * E) ? row_bytes + at : kOutOfRange);
}

// Four consecutive elements of a dense row.
template <typename T>
__device__ __forceinline__ void store4(S_<T>* at, float a, float b, float c, float d) {
    const S_<T> v[4] = {Elem<T>::store(a), Elem<T>::store(b), Elem<T>::store(c), Elem<T>::store(d)};
    if constexpr (sizeof(v) == 8) *reinterpret_cast<uint2*>(at) = __builtin_bit_cast(uint2, v);
    else *reinterpret_cast<uint4*>(at) = __builtin_bit_cast(uint4, v);
}

// ---- sums again ----------------------------------------------------------------------
//
// A matrix instruction sums over all rows of a tile, and what a column does not
// see has a factor of 0 there: beside a value that is not finite that is NaN, in
// columns that never saw it.  So a wave that finds a NaN in its sums at the end of
// its walk looks for such values among the rows its block has read.  A column
// whose elements that hold one are those of rows it sees keeps what it has; one
// that has an element's from a row that only shared a tile with it is summed again
// over what it sees, all lanes on one column.  The test is one sum of the
// accumulators.  What follows it stands in functions of its own, where it costs
// the walks no registers; the search reads the rows once more, and the columns
// beside a value, fewer than a block has, take some 0.2 us a row each: 8192
// tokens, 32 heads of 128 on 8, forward and backward 3.4 ms, with one infinity in
// the value of token 4000 22, in the gradient of its result 91.

// Whether the sums hold a NaN (or infinities of both signs).
template <int DT>
__device__ __forceinline__ bool holds_nan(const f32x16 (&sums)[DT]) {
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e % 4] += sums[d][e];
    const float all = (x[0] + x[1]) + (x[2] + x[3]);
    return all != all;
}

__device__ __forceinline__ bool finite(float x) { return x - x == 0.0f; }

// The kernel's argument, for a function that it calls: as it was launched, so
// that the kernel's own stays in registers.  The function takes its fields by
// scalar loads, and what all lanes share of its other arguments into scalars.
template <typename Args>
__device__ __forceinline__ const Args* launched_with() {
    return (const Args*)__builtin_amdgcn_kernarg_segment_ptr();
}
template <typename Args>
__device__ __forceinline__ const Args& as_launched(const Args* at) {
    const uint64_t a = reinterpret_cast<uint64_t>(at);
    const uint64_t shared = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32)))) << 32 |
                            static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a)));
    return *(const Args*)(__attribute__((address_space(4))) const Args*)shared;
}
__device__ __forceinline__ int shared_by_lanes(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Whether all elements of a token row are finite.
template <typename T>
__device__ __forceinline__ bool row_is_finite(const S_<T>* row, int dim) {
    constexpr int N = Packet<T>::N;
    float none = 0.0f;
#pragma unroll 1
    for (int d = 0; d < dim; d += N) {
        float x[N];
        unpack<T>(*reinterpret_cast<const uint4*>(row + d), x);
#pragma unroll
        for (int j = 0; j < N; ++j) none = fmaf(x[j], 0.0f, none);
    }
    return none == none;
}

// A lane's two elements of a token row that all lanes share (the last two again
// in lanes past its end).
struct Two {
    float x, y;
};
template <typename T>
__device__ __forceinline__ Two two_of(const S_<T>* row, int dim) {
    const int at = min(2 * static_cast<int>(threadIdx.x % kWave), dim - 2);
    struct alignas(2 * sizeof(S_<T>)) Pair {
        S_<T> x, y;
    };
    const Pair v = *reinterpret_cast<const Pair*>(row + at);
    return Two{Elem<T>::load(v.x), Elem<T>::load(v.y)};
}
template <typename T>
__device__ __forceinline__ void store_two(S_<T>* row, int dim, const Two& v) {
    const int at = 2 * (threadIdx.x % kWave);
    if (at >= dim) return;
    row[at] = Elem<T>::store(v.x);
    row[at + 1] = Elem<T>::store(v.y);
}
__device__ __forceinline__ void add_two(Two& sum, float f, const Two& v) {
    sum.x = fmaf(f, v.x, sum.x);
    sum.y = fmaf(f, v.y, sum.y);
}

// Product of a lane's row with another.
template <typename T>
__device__ __forceinline__ float row_product(const S_<T>* a, const S_<T>* b, int dim) {
    float sum = 0.0f;
#pragma unroll 2
    for (int d = 0; d < dim; d += Packet<T>::N) {
        float x[Packet<T>::N], y[Packet<T>::N];
        unpack<T>(*reinterpret_cast<const uint4*>(a + d), x);
        unpack<T>(*reinterpret_cast<const uint4*>(b + d), y);
#pragma unroll
        for (int j = 0; j < Packet<T>::N; ++j) sum = fmaf(x[j], y[j], sum);
    }
    return sum;
}

__device__ __forceinline__ float from_lane(float v, int lane) {
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// Elements of a row, as bits: those at 2 l and at 2 l + 1.
struct Elements {
    uint64_t x, y;
    __device__ __forceinline__ void add(const Elements& e, bool if_) {
        x |= if_ ? e.x : 0;
        y |= if_ ? e.y : 0;
    }
    __device__ __forceinline__ bool all_in(const Elements& e) const { return ((x & ~e.x) | (y & ~e.y)) == 0; }
};

__device__ __forceinline__ Elements all_elements(int dim) {
    const uint64_t half = dim == 2 * kWave ? ~uint64_t{0} : (uint64_t{1} << dim / 2) - 1;
    return Elements{half, half};
}

// Those of a row that all lanes share which are not finite.
template <typename T>
__device__ __forceinline__ Elements odd_elements(const S_<T>* row, int dim) {
    const Two v = two_of<T>(row, dim);
    const bool in = 2 * static_cast<int>(threadIdx.x % kWave) < dim;
    return Elements{__ballot(in && !finite(v.x)), __ballot(in && !finite(v.y))};
}

// sum += the lanes' f times their rows (lane l's `step` l elements from `rows`
// on), of the lanes in `seen`, which is not 0.
template <typename T>
__device__ __forceinline__ void add_rows(Two& sum, float f, const S_<T>* rows, int64_t step, uint64_t seen, int dim) {
    const int first = __ffsll(static_cast<unsigned long long>(seen)) - 1;
#pragma unroll 16
    for (int l = 0; l < kWave; ++l) {
        // (bits, not a branch: the loads go out together)
        const uint32_t in = -static_cast<uint32_t>(seen >> l & 1);
        const Two v = two_of<T>(rows + (in ? l : first) * step, dim);
        auto part = [&](float x) { return __uint_as_float(__float_as_uint(x) & in); };
        add_two(sum, part(from_lane(f, l)), Two{part(v.x), part(v.y)});
    }
}

// The wave's lanes together.
template <typename Op>
__device__ __forceinline__ float over_wave(float v, Op op) {
    for (int m = 1; m < kWave; m *= 2) v = op(v, wave_shfl_xor(v, m));
    return v;
}

// f(j0, seen) for the keys that row p sees: 64 of them from j0 on, one a lane,
// those in `seen`.
template <typename F>
__device__ __forceinline__ void for_seen(const Rule& r, int p, const F& f) {
    const KeyTiles tiles(r, p, p, kWave);
    for (int i = 0; i < tiles.count; ++i) {
        const int j0 = tiles.at(i) * kWave;
        const uint64_t seen = __ballot(r.sees(p, j0 + static_cast<int>(threadIdx.x % kWave)));
        if (seen != 0) f(j0, seen);
    }
}

// Of the lanes that ask (`bad`, on row `row`): those with an element that is not
// finite in a key which rows p0 .. p1 read and theirs does not see, and in none
// that theirs sees.  `rows` is the first key's row of the tensor.
template <typename T>
__device__ __forceinline__ bool only_beside(const Shape& s, const S_<T>* rows, int64_t step, int p0, int p1, bool bad, int row) {
    const KeyTiles tiles(s.rule, p0, p1, kWave);
    const KeysSeen keep(s.rule, tiles, p1);
    const Elements all = all_elements(s.dim);
    Elements own{0, 0}, beside{0, 0};
    for (int i = 0; i < tiles.count && __any(bad && !all.all_in(own)); ++i) {
        const int j0 = tiles.at(i) * kWave, mine = j0 + static_cast<int>(threadIdx.x % kWave);
        uint64_t found = __ballot(keep(mine) && !row_is_finite<T>(rows + mine * step, s.dim));
        for (; found != 0; found &= found - 1) {
            const int j = j0 + __ffsll(static_cast<unsigned long long>(found)) - 1;
            const Elements odd = odd_elements<T>(rows + j * step, s.dim);
            const bool sees = s.rule.sees(row, j);
            own.add(odd, sees);
            beside.add(odd, !sees);
        }
    }
    return bad && !beside.all_in(own);
}

// f(lane) for the first lane that asks, and again until no lane does that f has
// not answered: f returns whether a lane's question is the same.
template <typename F>
__device__ __forceinline__ void for_each_question(bool asks, const F& f) {
    for (uint64_t left = __ballot(asks); left != 0;) left &= ~__ballot(f(__ffsll(static_cast<unsigned long long>(left)) - 1));
}

// Waits until this wave's loads have landed and its LDS reads are done, then
// meets the block's other waves.  (Not __syncthreads(): the compiler would
// place the wait where it likes among the loads into LDS.)
__device__ __forceinline__ void meet() {
    __builtin_amdgcn_s_waitcnt(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// This wave's LDS reads are done: what they read may be filled again.
__device__ __forceinline__ void reads_done() {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// The same as meet() for one wave's own tile, its N latest loads left in flight.
template <int N>
__device__ __forceinline__ void wait_but() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | ((N >> 4) << 14));  // vmcnt(N) lgkmcnt(0)
    asm volatile("" ::: "memory");
}

// Work item `id` of `total` for block `bid`: each XCD (blocks are dealt over
// the 8 in turn) takes a run of neighbouring items, which share keys and
// values in its L2.
__device__ __forceinline__ int xcd_run(int bid, int total) {
    const int xcd = bid % 8, q = total / 8, rest = total % 8;
    return xcd * q + (xcd < rest ? xcd : rest) + bid / 8;
}

constexpr float kLog2E = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// Blocks own 32 rows a wave: of kWide waves where those are enough to give the
// CUs work, else of one.
constexpr int kWide = 4;

inline int64_t wide_blocks(int64_t batch, int64_t heads, int64_t rows) {
    return batch * heads * ((rows + 32 * kWide - 1) / (32 * kWide));
}

inline Shape shape_of(const AttentionArgs& a) {
    Shape s;
    s.queries = a.queries;
    s.keys = a.keys;
    s.heads = a.heads;
    s.kv_heads = a.kv_heads;
    s.group = a.heads / a.kv_heads;
    s.dim = a.dim;
    // a window that reaches every key is none
    s.rule.window = a.window < 0 || a.window >= static_cast<int64_t>(a.keys) + a.queries ? kNoWindow : static_cast<int>(a.window);
    s.rule.sinks = s.rule.window == kNoWindow ? 0 : static_cast<int>(a.sinks < a.keys ? a.sinks : a.keys);
    s.lengths = a.lengths;
    s.starts = a.starts;
    s.wide_lengths = a.wide_lengths;
    s.wide_starts = a.wide_starts;
    s.lengths_step = a.lengths_step;
    s.starts_step = a.starts_step;
    return s;
}

}  // namespace attention
}  // namespace tp_amd

// Dropout whose mask is never stored: out = keep ? x / (1 - p) : 0, the keep
// bits drawn again from the element's place and the seed wherever they are
// needed, so the backward is the same kernel on the gradient.
//
// Bound by memory, the generator (20 products of 32 bits a block of four
// elements) close behind: bf16 8192 x 4096, 134 MB, 24 us, 5.6 TB/s (an
// elementwise pass 6.2), 26 before its rounds took three-way xors and a
// scalar high word.

#include <algorithm>

#include "device_common.h"
#include "layers.h"
#include "../common.h"
#include "../runtime.h"

namespace tp_amd {

namespace {

constexpr int kBlock = 256;

template <typename T>
using S_ = typename Elem<T>::storage;

// The float32 product as computed: the compiler would fold it into the 16-bit
// conversion as fma(a, b, +0), which turns a -0 product into +0.
__device__ __forceinline__ float opaque(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

// One 16-byte packet a thread and step; the last one may be short.
template <typename T>
__global__ __launch_bounds__(kBlock) void seeded_dropout_kernel(const S_<T>* x, S_<T>* out, int64_t n, DropArgs args) {
    constexpr int N = Packet<T>::N;
    const DropKey key(args);
    const int64_t step = static_cast<int64_t>(gridDim.x) * kBlock * N;
    for (int64_t e = (static_cast<int64_t>(blockIdx.x) * kBlock + threadIdx.x) * N; e < n; e += step) {
        // a wave's packets start at a multiple of their length: one high word for all of them
        const uint64_t block = static_cast<uint64_t>(e) >> 2;
        const uint32_t keep = keep_blocks<N / 4>(key, static_cast<uint32_t>(block),
                                                 __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(block >> 32)));
        if (e + N <= n) {
            float f[N];
            unpack<T>(load_raw_any_nt(x + e), f);
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = kept(opaque(f[j] * args.scale), keep, j);
            store_raw_any_nt(out + e, pack<T>(f));
        } else {
            for (int j = 0; e + j < n; ++j) out[e + j] = Elem<T>::store(kept(opaque(Elem<T>::load(x[e + j]) * args.scale), keep, j));
        }
    }
}

template <typename T>
void dropout_typed(int64_t n, const void* x, const DropArgs& drop, void* out, int device) {
    constexpr int64_t per_block = static_cast<int64_t>(kBlock) * Packet<T>::N;
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((n + per_block - 1) / per_block, 1 << 20));
    seeded_dropout_kernel<T><<<blocks, kBlock, 0, stream(device)>>>(static_cast<const S_<T>*>(x), static_cast<S_<T>*>(out), n, drop);
    TP_AMD_HIP_CHECK(hipGetLastError());
}

}  // namespace

void launch_seeded_dropout(int dtype, int64_t n, const void* x, const DropArgs& drop, void* out, int device) {
    if (n <= 0) return;
    const OnDevice scope(device);
    TP_AMD_DISPATCH_TYPED(dtype, dropout_typed, n, x, drop, out, scope.index());
}

}  // namespace tp_amd

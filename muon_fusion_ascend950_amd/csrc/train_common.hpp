// train_common.hpp — what the operators of include/muon_train.h share: row access in
// 16-byte pieces at any alignment, reductions over a wave and a workgroup in a fixed
// order, and the error report of their C entries.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <cstdio>

#include "muon_train.h"
#include "polar_kernels.h"
#include "polar_tile.hpp"

namespace muon_train {

using muon_polar::bf16_bits_to_f32;
using muon_polar::f32_to_bf16_bits;
using muon_polar::u32x4;

inline int invalid(const char *msg) {
    return muon_polar::report(MUON_POLAR_ERR_INVALID_ARGUMENT, msg);
}
// A launch has at most 2^32 - 1 threads; one with more came back as done, only the rest past a
// multiple of 2^32 having run.
constexpr int64_t kMaxThreads = UINT32_MAX;

// The launches of one call.  Each gives its own status: hipGetLastError would also give an
// error that some earlier HIP call of the thread left behind.
struct Launches {
    hipStream_t stream;
    hipError_t status = hipSuccess;
    template <class... P, class... A>
    void operator()(void (*kernel)(P...), dim3 grid, int threads, const A &...a) {
        if (status == hipSuccess && int64_t(grid.x) * threads > kMaxThreads) status = hipErrorInvalidConfiguration;
        if (status != hipSuccess) return;
        auto launch = [&](P... p) {
            void *args[] = {const_cast<void *>(static_cast<const void *>(&p))...};
            status = hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, dim3(threads), args, 0, stream);
        };
        launch(a...);
    }
    int result(const char *what) const {
        if (status == hipSuccess) return MUON_POLAR_OK;
        char msg[256];
        snprintf(msg, sizeof msg, "%s: %s", what, hipGetErrorString(status));
        return muon_polar::report(MUON_POLAR_ERR_HIP, msg);
    }
};

// Whether two buffers meet (a null one meets none).
inline bool meet(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
    const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return a && b && x < y + static_cast<uintptr_t>(b_bytes) && y < x + static_cast<uintptr_t>(a_bytes);
}

// Compute units of the current device (asked once per device), or 0 with an error.
int compute_units() noexcept;

// ------------------------------------------------------------------ element types
struct F32 {
    using Raw = float;
};
struct Bf16 {
    using Raw = uint16_t;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_bits_to_f32(v); }

// Element i of a vector of either type (uniform branch).
__device__ __forceinline__ float load_any(const void *p, int64_t i, int dtype) {
    return dtype == MUON_TRAIN_BF16 ? bf16_bits_to_f32(static_cast<const uint16_t *>(p)[i])
                                    : static_cast<const float *>(p)[i];
}
__device__ __forceinline__ void store_any(void *p, int64_t i, int dtype, float v) {
    if (dtype == MUON_TRAIN_BF16)
        static_cast<uint16_t *>(p)[i] = f32_to_bf16_bits(v);
    else
        static_cast<float *>(p)[i] = v;
}

// Eight consecutive elements as they lie in memory.  Loads and stores of whole pieces are
// 16-byte accesses at any address (global memory takes them unaligned); a piece that a
// row's end cuts goes element by element.
template <class T>
struct Piece;
template <>
struct Piece<Bf16> {
    u32x4 v;
    __device__ __forceinline__ void load(const uint16_t *p, int valid) {
        if (valid >= 8) {
            __builtin_memcpy(&v, p, 16);
        } else {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = i < valid ? p[i] : 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = h[2 * i] | (h[2 * i + 1] << 16);
        }
    }
    __device__ __forceinline__ void zero() { v = u32x4{0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(v[i] << 16);
            f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = f32_to_bf16_bits(f[2 * i]) | uint32_t(f32_to_bf16_bits(f[2 * i + 1])) << 16;
    }
    __device__ __forceinline__ void store(uint16_t *p, int valid) const {
        if (valid >= 8) {
            __builtin_memcpy(p, &v, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < valid) p[i] = static_cast<uint16_t>(v[i / 2] >> (16 * (i & 1)));
        }
    }
};
template <>
struct Piece<F32> {
    u32x4 v[2];
    __device__ __forceinline__ void load(const float *p, int valid) {
        if (valid >= 8) {
            __builtin_memcpy(v, p, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = i < valid ? __float_as_uint(p[i]) : 0u;
        }
    }
    __device__ __forceinline__ void zero() { v[0] = v[1] = u32x4{0u, 0u, 0u, 0u}; }
    __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(v[i / 4][i % 4]);
    }
    __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i / 4][i % 4] = __float_as_uint(f[i]);
    }
    __device__ __forceinline__ void store(float *p, int valid) const {
        if (valid >= 8) {
            __builtin_memcpy(p, v, 32);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < valid) p[i] = __uint_as_float(v[i / 4][i % 4]);
        }
    }
};

// Eight elements of a vector of either type as fp32 (missing ones 0).
__device__ __forceinline__ void load8_any(const void *p, int64_t at, int valid, int dtype,
                                          float (&f)[8]) {
    if (dtype == MUON_TRAIN_BF16) {
        Piece<Bf16> t;
        t.load(static_cast<const uint16_t *>(p) + at, valid);
        t.get(f);
    } else {
        Piece<F32> t;
        t.load(static_cast<const float *>(p) + at, valid);
        t.get(f);
    }
}
__device__ __forceinline__ void store8_any(void *p, int64_t at, int valid, int dtype,
                                           const float (&f)[8]) {
    if (dtype == MUON_TRAIN_BF16) {
        Piece<Bf16> t;
        t.set(f);
        t.store(static_cast<uint16_t *>(p) + at, valid);
    } else {
        Piece<F32> t;
        t.set(f);
        t.store(static_cast<float *>(p) + at, valid);
    }
}

// --------------------------------------------------------------------- reductions
// Over a wave by DPP (adds within rows of 16 lanes, then from row to row): the total is in
// lane 63 and read from there into a scalar, so every lane holds the same bits.
template <int kCtrl, int kRowMask>
__device__ __forceinline__ float dpp(float old, float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(old), __float_as_uint(v),
                                                       kCtrl, kRowMask, 0xf, false));
}
constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kRowHalfMirror = 0x141, kRowMirror = 0x140,
              kRowBcast15 = 0x142, kRowBcast31 = 0x143;

__device__ __forceinline__ float wave_total(float v) {
    v += dpp<kQuadXor1, 0xf>(0.0f, v);
    v += dpp<kQuadXor2, 0xf>(0.0f, v);
    v += dpp<kRowHalfMirror, 0xf>(0.0f, v);
    v += dpp<kRowMirror, 0xf>(0.0f, v);
    v += dpp<kRowBcast15, 0xa>(0.0f, v);
    v += dpp<kRowBcast31, 0xc>(0.0f, v);
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
    v = fmaxf(v, dpp<kQuadXor1, 0xf>(v, v));
    v = fmaxf(v, dpp<kQuadXor2, 0xf>(v, v));
    v = fmaxf(v, dpp<kRowHalfMirror, 0xf>(v, v));
    v = fmaxf(v, dpp<kRowMirror, 0xf>(v, v));
    v = fmaxf(v, dpp<kRowBcast15, 0xa>(v, v));
    v = fmaxf(v, dpp<kRowBcast31, 0xc>(v, v));
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// Over a workgroup of NW waves, N values at once: wave totals meet in LDS and every thread
// adds them in wave order.  Successive calls alternate between two sets of LDS words, so
// one barrier each is enough: a wave writes a set again only past the barrier of the call
// between, which every wave reaches after its last read of that set.
template <int NW, int N>
struct BlockSum {
    float (*red)[NW * N];  // [2][NW * N] in LDS
    int turn = 0;
    __device__ __forceinline__ explicit BlockSum(float (*lds)[NW * N]) : red(lds) {}
    template <int K>
    __device__ __forceinline__ void sum(float (&v)[K]) {
        static_assert(K <= N, "room for K values a wave");
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = wave_total(v[k]);
        if constexpr (NW == 1) return;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) red[turn][wave * N + k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = red[turn][k];
#pragma unroll
            for (int w = 1; w < NW; ++w) t += red[turn][w * N + k];
            v[k] = t;
        }
        turn ^= 1;
    }
    __device__ __forceinline__ float sum(float a) {
        float v[1] = {a};
        sum(v);
        return v[0];
    }
    template <int K>
    __device__ __forceinline__ void max(float (&v)[K]) {
        static_assert(K <= N, "room for K values a wave");
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = wave_max(v[k]);
        if constexpr (NW == 1) return;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) red[turn][wave * N + k] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float t = red[turn][k];
#pragma unroll
            for (int w = 1; w < NW; ++w) t = fmaxf(t, red[turn][w * N + k]);
            v[k] = t;
        }
        turn ^= 1;
    }
};

}  // namespace muon_train

// train_fp8.hip — e4m3 values with a scale for each block of 128, and products of matrices
// held so (include/muon_train.h; the formulas are there).
#include "train_common.hpp"

#include <type_traits>
#include <utility>

namespace muon_train {

namespace {

using muon_polar::f32x4;
using muon_polar::u32x2;
using i32x8 = int32_t __attribute__((ext_vector_type(8)));
using muon_polar::i32x4;

constexpr int kBlock = 128;
using u32x4_any = uint32_t __attribute__((ext_vector_type(4), aligned(2)));  // at any element's address

// f(0), f(1), ..., f(N - 1) with the index a compile-time constant.
template <class F, int... I>
__device__ __forceinline__ void static_for_seq(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F &&f) {
    static_for_seq(f, std::make_integer_sequence<int, N>{});
}

// ------------------------------------------------------------------------- quantising
// One workgroup takes a tile of 128 x 128 elements: thread t the rows 8·(t / 16) .. + 7 and
// the columns 8·(t % 16) .. + 7.  Magnitudes are compared as integers, which orders NaN
// above the infinities and those above all numbers, so that either reaches the scale.
constexpr int kQuantThreads = 256;
constexpr int kTilePitch = kBlock + 16;  // bytes from column to column of the turned tile

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
    return __builtin_amdgcn_update_dpp(v, v, kCtrl, 0xf, 0xf, false);
}
// Over the 16 lanes of a row of the wave.
__device__ __forceinline__ uint32_t row_umax(uint32_t v) {
    v = umax(v, dpp_u32<kQuadXor1>(v));
    v = umax(v, dpp_u32<kQuadXor2>(v));
    v = umax(v, dpp_u32<kRowHalfMirror>(v));
    return umax(v, dpp_u32<kRowMirror>(v));
}
__device__ __forceinline__ float scale_of(uint32_t amax) {
    const float s = __uint_as_float(amax) * (1.0f / 448.0f);
    return s >= 0x1p-126f || s != s ? s : 0x1p-126f;
}
// Eight values as e4m3, in order.
__device__ __forceinline__ u32x2 to_fp8(const float (&f)[8], const float (&inv)[8]) {
    int lo = 0, hi = 0;
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0] * inv[0], f[1] * inv[1], lo, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2] * inv[2], f[3] * inv[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4] * inv[4], f[5] * inv[5], hi, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6] * inv[6], f[7] * inv[7], hi, true);
    return u32x2{uint32_t(lo), uint32_t(hi)};
}

using QuantArgs = muon_train_fp8_quantize_args;

template <class T, int kRows>
__global__ __launch_bounds__(kQuantThreads) void quantize_kernel(QuantArgs a, int col_tiles) {
    using Raw = typename T::Raw;
    __shared__ uint32_t col_max[4][kBlock];
    __shared__ uint8_t turned[kBlock * kTilePitch];
    const int tid = threadIdx.x, wave = tid >> 6;
    const int64_t tile_r = blockIdx.x / col_tiles, tile_c = blockIdx.x % col_tiles;
    const int64_t row0 = tile_r * kBlock + 8 * (tid >> 4), col0 = tile_c * kBlock + 8 * (tid & 15);
    const int64_t padded_cols = int64_t(col_tiles) * kBlock;
    const int64_t padded_rows = (a.rows + kBlock - 1) / kBlock * kBlock;
    const int64_t left = a.cols - col0;
    const int valid = left < 0 ? 0 : left > 8 ? 8 : int(left);

    float x[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        Piece<T> p;
        if (row0 + i < a.rows)
            p.load(static_cast<const Raw *>(a.x) + (row0 + i) * a.ld_x + col0, valid);
        else
            p.zero();
        p.get(x[i]);
    }
    float inv[8];
    if constexpr (kRows == 1) {
        if (a.values) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t m = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) m = umax(m, magnitude(x[i][e]));
                const float s = scale_of(row_umax(m)), r = 1.0f / s;
#pragma unroll
                for (int e = 0; e < 8; ++e) inv[e] = r;
                if (row0 + i < a.rows) {
                    const u32x2 q = to_fp8(x[i], inv);
                    __builtin_memcpy(static_cast<uint8_t *>(a.values) + (row0 + i) * padded_cols + col0, &q, 8);
                    if ((tid & 15) == 0) a.scales[tile_c * a.rows + row0 + i] = s;
                }
            }
        }
        if (!a.values_t) return;
    }
    // magnitudes of the columns (of the whole tile: blocks of 128 rows)
    uint32_t cm[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = umax(m, magnitude(x[i][e]));
        m = umax(m, __shfl_xor(m, 16));
        cm[e] = umax(m, __shfl_xor(m, 32));
    }
    if constexpr (kRows == kBlock) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = umax(m, cm[e]);
        m = row_umax(m);
        if ((tid & 63) == 0) col_max[wave][0] = m;
        __syncthreads();
        m = umax(umax(col_max[0][0], col_max[1][0]), umax(col_max[2][0], col_max[3][0]));
        const float s = scale_of(m), r = 1.0f / s;
#pragma unroll
        for (int e = 0; e < 8; ++e) inv[e] = r;
        if (tid == 0) a.scales[tile_r * col_tiles + tile_c] = s;
        if (a.values) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (row0 + i < a.rows) {
                    const u32x2 q = to_fp8(x[i], inv);
                    __builtin_memcpy(static_cast<uint8_t *>(a.values) + (row0 + i) * padded_cols + col0, &q, 8);
                }
        }
        if (!a.values_t) return;
    } else {
        if ((tid & 63) < 16) {
#pragma unroll
            for (int e = 0; e < 8; ++e) col_max[wave][8 * (tid & 15) + e] = cm[e];
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = 8 * (tid & 15) + e;
            const uint32_t m = umax(umax(col_max[0][c], col_max[1][c]), umax(col_max[2][c], col_max[3][c]));
            const float s = scale_of(m);
            inv[e] = 1.0f / s;
            if ((tid >> 4) == 0 && col0 + e < a.cols) a.scales_t[tile_r * a.cols + col0 + e] = s;
        }
    }
    // the tile turned: eight rows of a column are eight bytes in a line
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float f[8], r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = x[i][e], r[i] = inv[e];
        const u32x2 q = to_fp8(f, r);
        *reinterpret_cast<u32x2 *>(turned + (8 * (tid & 15) + e) * kTilePitch + 8 * (tid >> 4)) = q;
    }
    __syncthreads();
#pragma unroll
    for (int pass = 0; pass < 4; ++pass) {
        const int c = 32 * pass + (tid >> 3), b = 16 * (tid & 7);
        const int64_t col = tile_c * kBlock + c;
        if (col < a.cols)
            *reinterpret_cast<u32x4 *>(static_cast<uint8_t *>(a.values_t) + col * padded_rows +
                                       tile_r * kBlock + b) =
                *reinterpret_cast<const u32x4 *>(turned + c * kTilePitch + b);
    }
    // tests/isa_hazards.py reads the code in address order, past the program's
    // end: two wait states keep it from pairing the last store with the block laid out there.
    asm volatile("s_nop 1");
}

// Rows alone, for matrices of too few tiles to fill the card: a workgroup takes 16 rows of a
// block column, a thread eight elements, so that a small call waits for one load.
template <class T>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(QuantArgs a, int col_tiles) {
    const int64_t row = int64_t(blockIdx.x / col_tiles) * 16 + (threadIdx.x >> 4);
    const int64_t tile_c = blockIdx.x % col_tiles, col0 = tile_c * kBlock + 8 * (threadIdx.x & 15);
    if (row >= a.rows) return;  // whole rows of 16 lanes
    const int64_t left = a.cols - col0;
    Piece<T> p;
    p.load(static_cast<const typename T::Raw *>(a.x) + row * a.ld_x + col0, left < 0 ? 0 : left > 8 ? 8 : int(left));
    float x[8], inv[8];
    p.get(x);
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = umax(m, magnitude(x[e]));
    const float s = scale_of(row_umax(m)), r = 1.0f / s;
#pragma unroll
    for (int e = 0; e < 8; ++e) inv[e] = r;
    const u32x2 q = to_fp8(x, inv);
    __builtin_memcpy(static_cast<uint8_t *>(a.values) + row * (int64_t(col_tiles) * kBlock) + col0, &q, 8);
    if ((threadIdx.x & 15) == 0) a.scales[tile_c * a.rows + row] = s;
}

// -------------------------------------------------------------------------- products
// v_mfma_f32_16x16x128_f8f6f4 on e4m3 values: lane l supplies 32 consecutive values (k-part
// l / 16 of the 128) of row l % 16 of A and of column l % 16 of B, and receives
// D[4·(l / 16) + j][l % 16], j = 0 .. 3.  Each row's values count times 2^(e − 127) of its lane's
// exponent e, 0 to 254, which is byte kB of eb for b.
template <int kB = 0>
__device__ __forceinline__ f32x4 mfma_fp8(i32x8 a, uint32_t ea, i32x8 b, uint32_t eb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0,
                                                            static_cast<int>(ea), kB, static_cast<int>(eb));
}

// The product of two scales may leave fp32's range where the result does not: large ones at
// blocks whose values meet zeros would be infinity times 0, small ones would lose the sums they
// multiply.  Such scales are taken apart, s = mantissa·2^(exponent − 127): the exponents go into
// the MFMA, whose sums then have their results' size, and the mantissas' product onto those.  The
// bits are the ones that one factor gives where it is in range.  Exponents are kept within
// 2^±100, the rest left to the mantissa: zeros, infinities, NaN and subnormal scales pass through
// it, and values times 2^(exponent − 127) are normal numbers in bf16 too.
struct Apart {
    uint32_t exponent;
    float mantissa;
};
__device__ __forceinline__ Apart apart(float s) {
    const float within = __builtin_amdgcn_fmed3f(__builtin_fabsf(s), 0x1p-100f, 0x1p100f);
    const uint32_t e = __float_as_uint(within) >> 23;
    return {e, __builtin_amdgcn_ldexpf(s, 127 - static_cast<int>(e))};
}
// Scales whose products with each other stay in range whatever pairs meet: 2^-63 to 2^63, by
// their bits.  Any other (a negative one too) has its step take them apart.
constexpr uint32_t kNearLow = (127u - 63) << 23, kNearHigh = (127u + 63) << 23;
__device__ __forceinline__ bool far(float s) {
    return __float_as_uint(s) - kNearLow > kNearHigh - kNearLow;
}

using MatmulArgs = muon_train_fp8_matmul_args;

// The fp8 MFMAs do not keep 32 bits of the products they add: of each eight (consecutive k) what
// lies below 2^-13 of the largest is cut off, the eights are added in full (one product 2^-k of
// another beside it: whole at k = 10, gone at k = 14; eight places further whole at k = 18).
// Against 64 bits results are off by 1.5e-5 (normal values) to 7e-5 (log-uniform ones) of their
// 2-norm, in chains of 16x16x32 as in single 16x16x128 instructions, at most 7·2^-13 of the sum
// of magnitudes.  bf16's rounding is 2^-8, the values' own 2^-4: results that leave as bf16 take
// them.  Results kept in fp32 (kExact) take the bf16 MFMA on the same values, which bf16 holds
// exactly: 1e-7, at half the rate.
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using muon_polar::bf16x8;
__device__ __forceinline__ bf16x8 to_bf16(uint32_t lo, uint32_t hi, float power) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, false);
    const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, power, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, false);
    const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, power, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// 16 rows of 128 K-values of an operand as a lane holds them, times 2^(e − 127) of its row's
// exponent: `exponent` is e as the instruction at hand takes it, kNone that of 1.
template <bool kExact>
struct Frag {
    i32x8 v;
    uint32_t e;
    static constexpr uint32_t kNone = 127;
    __device__ __forceinline__ static uint32_t exponent(uint32_t e) { return e; }
    __device__ __forceinline__ void set(i32x8 x, uint32_t exponent) { v = x, e = exponent; }
};
template <>
struct Frag<true> {
    bf16x8 v[4];
    static constexpr uint32_t kNone = 127u << 23;
    __device__ __forceinline__ static uint32_t exponent(uint32_t e) { return e << 23; }
    __device__ __forceinline__ void set(i32x8 x, uint32_t exponent) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_bf16(x[2 * i], x[2 * i + 1], __uint_as_float(exponent));
    }
};
__device__ __forceinline__ f32x4 multiply(const Frag<false> &a, const Frag<false> &b) {
    return mfma_fp8(a.v, a.e, b.v, b.e);
}
__device__ __forceinline__ f32x4 multiply(const Frag<true> &a, const Frag<true> &b) {
    f32x4 t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < 4; ++i) t = muon_polar::mfma_16x16x32(a.v[i], b.v[i], t);
    return t;
}

// 16 B per lane from rsrc + voffset + soffset into LDS at lds_base (wave-uniform) + 16·lane
// (see dma_16B for the wait state).  The step goes into soffset, a scalar: added to the
// lanes' offsets it took two vector instructions a DMA instruction from the multiply-adds.
__device__ __forceinline__ void dma_16B_step(muon_polar::i32x4 rsrc, uint32_t lds_base,
                                             uint32_t voffset, uint32_t soffset) {
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voffset), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(soffset)),
                   "{m0}"(__builtin_amdgcn_readfirstlane(lds_base))
                 : "memory");
}
// The same with 4 B per lane.
__device__ __forceinline__ void dma_4B_step(muon_polar::i32x4 rsrc, uint32_t lds_base,
                                            uint32_t voffset, uint32_t soffset) {
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                 :
                 : "v"(voffset), "s"(rsrc), "s"(__builtin_amdgcn_readfirstlane(soffset)),
                   "{m0}"(__builtin_amdgcn_readfirstlane(lds_base))
                 : "memory");
}

// Waits for the oldest of this wave's memory instructions, the kLate behind them left under
// way if `behind` says that there are so many, and meets the workgroup's other waves.  (Branching
// inside one statement: a branch of the program's own splits the schedule around it, and the
// registers spill, 5.6 times the time.)
template <int kLate>
__device__ __forceinline__ void wait_dma_barrier(int behind) {
    static_assert(kLate <= 63, "vmcnt range");
    asm volatile("s_cmp_lg_u32 %0, 0\n\t"
                 "s_cbranch_scc1 .Ldma%=\n\t"
                 "s_waitcnt vmcnt(0)\n"
                 ".Ldma%=:\n\t"
                 "s_waitcnt vmcnt(%1) lgkmcnt(0)\n\t"
                 "s_barrier"
                 :
                 : "s"(behind), "n"(kLate)
                 : "memory", "scc");
}

// Of a pipelined step's scales, a's blocks' f and b's sb: if one of them is far, mantissas in their
// place and the exponents, one a byte; otherwise exponents of 127, which change nothing.  What
// apart() does, in one statement: where 8192 x 14336 x 4096 took 389 us with products of scales it
// took 407 with a branch of the program's own, and where it took 434, 440 with this one.
#define MUON_TRAIN_APART(scale, into)                    \
    "v_max_f32 " into ", |" scale "|, %[low]\n\t"        \
    "v_min_f32 " into ", %[high], " into "\n\t"          \
    "v_lshrrev_b32 " into ", 23, " into "\n\t"           \
    "v_sub_u32 %[t], 0x7f, " into "\n\t"                 \
    "v_ldexp_f32 " scale ", " scale ", %[t]\n\t"
#define MUON_TRAIN_APART4(f0, f1, f2, f3, exponents)                                           \
    MUON_TRAIN_APART(f0, exponents)                                                           \
    MUON_TRAIN_APART(f1, "%[eb]") "v_lshl_or_b32 " exponents ", %[eb], 8, " exponents "\n\t"  \
    MUON_TRAIN_APART(f2, "%[eb]") "v_lshl_or_b32 " exponents ", %[eb], 16, " exponents "\n\t" \
    MUON_TRAIN_APART(f3, "%[eb]") "v_lshl_or_b32 " exponents ", %[eb], 24, " exponents "\n\t"
// The two wait states at the end are for an MFMA that reads the exponents next.
#define MUON_TRAIN_APART_END MUON_TRAIN_APART("%[sb]", "%[eb]") ".Lnear%=:\n\ts_nop 1"
__device__ __forceinline__ void take_scales_apart(int any_far, float (&f)[8], float &sb, uint32_t (&ea)[2],
                                                  uint32_t &eb) {
    uint32_t t;
    asm volatile("v_mov_b32 %[ea0], 0x7f7f7f7f\n\t"
                 "v_mov_b32 %[ea1], 0x7f7f7f7f\n\t"
                 "v_mov_b32 %[eb], 0x7f\n\t"
                 "s_cmp_eq_u32 %[far], 0\n\t"
                 "s_cbranch_scc1 .Lnear%=\n\t"
                 MUON_TRAIN_APART4("%[f0]", "%[f1]", "%[f2]", "%[f3]", "%[ea0]")
                 MUON_TRAIN_APART4("%[f4]", "%[f5]", "%[f6]", "%[f7]", "%[ea1]")
                 MUON_TRAIN_APART_END
                 : [ea0] "=&v"(ea[0]), [ea1] "=&v"(ea[1]), [eb] "=&v"(eb), [t] "=&v"(t), [f0] "+v"(f[0]),
                   [f1] "+v"(f[1]), [f2] "+v"(f[2]), [f3] "+v"(f[3]), [f4] "+v"(f[4]), [f5] "+v"(f[5]),
                   [f6] "+v"(f[6]), [f7] "+v"(f[7]), [sb] "+v"(sb)
                 : [far] "s"(__builtin_amdgcn_readfirstlane(any_far)), [low] "s"(0x1p-100f), [high] "s"(0x1p100f)
                 : "scc");
}
__device__ __forceinline__ void take_scales_apart(int any_far, float (&f)[4], float &sb, uint32_t (&ea)[1],
                                                  uint32_t &eb) {
    uint32_t t;
    asm volatile("v_mov_b32 %[ea0], 0x7f7f7f7f\n\t"
                 "v_mov_b32 %[eb], 0x7f\n\t"
                 "s_cmp_eq_u32 %[far], 0\n\t"
                 "s_cbranch_scc1 .Lnear%=\n\t"
                 MUON_TRAIN_APART4("%[f0]", "%[f1]", "%[f2]", "%[f3]", "%[ea0]")
                 MUON_TRAIN_APART_END
                 : [ea0] "=&v"(ea[0]), [eb] "=&v"(eb), [t] "=&v"(t), [f0] "+v"(f[0]), [f1] "+v"(f[1]),
                   [f2] "+v"(f[2]), [f3] "+v"(f[3]), [sb] "+v"(sb)
                 : [far] "s"(__builtin_amdgcn_readfirstlane(any_far)), [low] "s"(0x1p-100f), [high] "s"(0x1p100f)
                 : "scc");
}
#undef MUON_TRAIN_APART
#undef MUON_TRAIN_APART4
#undef MUON_TRAIN_APART_END

// Four consecutive results of a row, the first `count` of them inside the matrix.
__device__ __forceinline__ void store4(void *c, int64_t at, int count, int dtype, f32x4 v) {
    if (dtype == MUON_TRAIN_BF16) {
        uint16_t *p = static_cast<uint16_t *>(c) + at;
        const u32x2 w{f32_to_bf16_bits(v[0]) | uint32_t(f32_to_bf16_bits(v[1])) << 16,
                      f32_to_bf16_bits(v[2]) | uint32_t(f32_to_bf16_bits(v[3])) << 16};
        if (count >= 4) {
            __builtin_memcpy(p, &w, 8);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < count) p[e] = static_cast<uint16_t>(w[e / 2] >> (16 * (e & 1)));
        }
    } else {
        float *p = static_cast<float *>(c) + at;
        if (count >= 4) {
            __builtin_memcpy(p, &v, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < count) p[e] = v[e];
        }
    }
}

// Exchanges that turn a wave's results into whole lines of 128 bytes.  A lane (r, p) = (l %
// 16, l / 16) holds four columns 16·j + 4·p of row r for each j.  Stored as they are, a line
// is written in four instructions of 32 bytes each, and the stores of 256 tiles that end
// together took 12 us (33.5 MB; whole lines fill memory at 6.9 TB/s).
//
// (a, b) <- parts (a0 b0 a2 b2, a1 b1 a3 b3) of (a0 a1 b0 b1, a2 a3 b2 b3) of (a, b): from
// columns 16·j and 16·(j + 1) to the low and high four of the eight columns 8·p.
__device__ __forceinline__ void turn_parts(uint32_t &a, uint32_t &b) {
    const auto x = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    const auto y = __builtin_amdgcn_permlane16_swap(x[0], x[1], false, false);
    a = y[0];
    b = y[1];
}
// Rows r and r ^ 8 swap pieces: a lane's pieces a and b, 64 bytes apart in its row, become
// pieces of rows r % 8 and 8 + r % 8, piece p + 4·(r / 8) of their line.
__device__ __forceinline__ void turn_rows(u32x4 &a, u32x4 &b, int r) {
    constexpr int kRowRotate8 = 0x128;
    const bool high = r >= 8;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint32_t give = high ? a[e] : b[e];
        const uint32_t got = __builtin_amdgcn_update_dpp(give, give, kRowRotate8, 0xf, 0xf, false);
        const uint32_t mine = high ? b[e] : a[e];
        a[e] = high ? got : mine;
        b[e] = high ? mine : got;
    }
}

// Tile of a launch: workgroup w runs on XCD w % 8, and each XCD takes a run of tiles next
// to each other (columns of kGroup row tiles, walked column by column), which share operand
// panels in its L2.
constexpr int kGroup = 8;
__device__ __forceinline__ void tile_of(int w, int tiles_m, int tiles_n, int &tm, int &tn) {
    const int total = tiles_m * tiles_n, each = total / 8, more = total % 8;
    const int xcd = w % 8, first = xcd * each + (xcd < more ? xcd : more);
    const int t = first + w / 8;
    const int group = t / (kGroup * tiles_n), in = t % (kGroup * tiles_n);
    const int high = tiles_m - group * kGroup < kGroup ? tiles_m - group * kGroup : kGroup;
    tm = group * kGroup + in % high;
    tn = in / high;
}

// A tile of BM x BN outputs, waves of WM x WN.  K runs in steps of one block of 128: the
// step's panels (rows of 128 bytes) and scales come to LDS by DMA, D steps in a ring, so
// that step k + D - 1 streams in while step k is multiplied.  A row's 16-byte chunk c lies
// at place c ^ ((row >> 1) & 7), and a lane of k-part p reads chunks p and p + 4 (both
// operands in the same order, which is all that the MFMA asks for): the 16 lanes that LDS
// serves at once then meet 16 different places of the 256-byte bank window.  (Chunks 2p and
// 2p + 1 met half as many.)
//
// The operand b, whose rows are output columns, is the MFMA's A side: a lane then holds
// four consecutive columns of one output row, and a's scale is one number a lane.  Each
// step's product starts from zero and is added to the fp32 sums times a_scale·b_scale: four
// fused multiply-adds a lane beside each MFMA (16 against its 32 clocks).
template <int BM, int BN, int WM, int WN, int D>
struct Geometry {
    static constexpr int kWaves = (BM / WM) * (BN / WN), kThreads = 64 * kWaves;
    static constexpr int kPanels = (BM + BN) * kBlock;  // bytes of a step
    static constexpr int kSlot = kPanels + (BM + BN) * 4;
    static constexpr int kLoads = kPanels / 1024 / kWaves;  // 1 KiB DMA instructions of a wave
    static constexpr int kScaleLoads = (BM + BN) / 64;      // 256 B ones of the workgroup
    static_assert(kPanels % (1024 * kWaves) == 0 && BM % 64 == 0 && BN % 64 == 0, "whole DMA blocks");
    static_assert(kScaleLoads <= kWaves, "one scale load a wave");
    static_assert(BM % (8 * kLoads) == 0, "a wave loads from one panel");
    static_assert((D - 1) * (kLoads + 1) <= 63, "vmcnt range");
    static_assert(D * kSlot <= 160 * 1024, "LDS");
    static constexpr bool kTwoSlots = D == 2;
};

template <int BM, int BN, int WM, int WN, int D, bool kExact, bool kRowB>
__global__ __launch_bounds__((Geometry<BM, BN, WM, WN, D>::kThreads)) void matmul_kernel(
    MatmulArgs g, int tiles_m, int tiles_n, int parts) {
    using Geo = Geometry<BM, BN, WM, WN, D>;
    constexpr int SM = WM / 16, SN = WN / 16, kLoads = Geo::kLoads;
    // The pipeline's registers leave no room for bf16 fragments (kExact) or a scale for each
    // column (kRowB: 60 spilled, 8192 x 14336 x 8192 in 1275 us against 1004 without; with scales
    // taken apart it takes 1017 to 1050).
    constexpr bool kPipelined = Geo::kTwoSlots && !kExact && !kRowB;
    __shared__ __attribute__((aligned(1024))) uint8_t smem[D * Geo::kSlot];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    // Workgroup blockIdx.x takes part blockIdx.x % parts of K, steps [first, steps), and leaves its
    // sums in that part's matrix.  (Pipelined kernels take all of K.)
    int steps = static_cast<int>(g.k / kBlock), first = 0, at_tile = blockIdx.x;
    if constexpr (!Geo::kTwoSlots)
        if (parts > 1) {
            const int part = at_tile % parts, each = (steps + parts - 1) / parts;
            at_tile /= parts;
            first = part * each;
            steps = first + each < steps ? first + each : steps;
            g.c = static_cast<float *>(g.c) + part * g.m * g.ldc;
        }

    // DMA: instruction d of this wave moves rows 8·(wave·kLoads + d) .. + 7 of a step's
    // BM + BN panel rows; rows outside the matrices read as zeros.  Behind them the scales:
    // 64 rows' worth a wave, one each (rows past the end: the last's).
    const int sblock = wave % Geo::kScaleLoads;
    const bool scale_a = sblock * 64 < BM;
    const muon_train_fp8_operand &so = scale_a ? g.a : g.b;
    const bool load_a = 8 * wave * kLoads < BM;  // a wave's rows are all a's or all b's
    const muon_train_fp8_operand &lo = load_a ? g.a : g.b;
    i32x4 rs, rs_scale;
    uint32_t off[kLoads], soff;
    const uint32_t sstep = static_cast<uint32_t>(4 * so.scale_col);
    auto aim = [&](int tile) {  // at a tile's first step
        int tm, tn;
        tile_of(tile, tiles_m, tiles_n, tm, tn);
        const int64_t m0 = int64_t(tm) * BM, n0 = int64_t(tn) * BN;
        const int rows_m = g.m - m0 < BM ? int(g.m - m0) : BM;
        const int rows_n = g.n - n0 < BN ? int(g.n - n0) : BN;
        const int rows = load_a ? rows_m : rows_n;
        rs = muon_polar::make_buffer_rsrc(static_cast<const uint8_t *>(lo.values) + (load_a ? m0 : n0) * lo.ld,
                                          static_cast<uint32_t>(rows * lo.ld));
#pragma unroll
        for (int d = 0; d < kLoads; ++d) {
            const int row = 8 * (wave * kLoads + d) + (lane >> 3);
            const int chunk = (lane & 7) ^ ((row >> 1) & 7);
            const int at = load_a ? row : row - BM;
            off[d] = at < rows ? static_cast<uint32_t>(at * lo.ld + 16 * chunk) : muon_polar::kOob;
        }
        const int srow = (scale_a ? sblock * 64 : sblock * 64 - BM) + lane;
        const int64_t sfirst = scale_a ? m0 : n0;
        const int slast = (scale_a ? rows_m : rows_n) - 1;
        const int64_t sat = sfirst + (srow < slast ? srow : slast);
        const int64_t from = so.block_rows == 1 ? sfirst : sfirst / kBlock;
        soff = static_cast<uint32_t>(4 * ((so.block_rows == 1 ? sat : sat / kBlock) - from) * so.scale_row);
        rs_scale = muon_polar::make_buffer_rsrc(so.scales + from * so.scale_row, 0x7ffffffcu);
    };
    const uint32_t lds0 = muon_polar::lds_addr(smem);
    auto issue = [&](int d, int step, int slot) {
        const uint32_t base = lds0 + slot * Geo::kSlot;
        const int s = step < steps ? step : steps - 1;  // past the end: the last step once more
        if (d < kLoads) {
            const int row0 = 8 * (wave * kLoads + d);
            dma_16B_step(rs, base + row0 * kBlock, off[d], s * kBlock);
        } else {
            dma_4B_step(rs_scale, base + Geo::kPanels + sblock * 256, soff, s * sstep);
        }
    };

    const int wm = (wave % (BM / WM)) * WM, wn = (wave / (BM / WM)) * WN;
    const int r = lane & 15, part = lane >> 4;
    const int lane_at = r * kBlock + ((part ^ ((r >> 1) & 7)) << 4);
    auto fragment = [&](const uint8_t *panel) {
        const i32x4 lo = *reinterpret_cast<const i32x4 *>(panel + lane_at);
        const i32x4 hi = *reinterpret_cast<const i32x4 *>(panel + (lane_at ^ 64));
        return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };

    f32x4 acc[SM][SN] = {};
    // True if each lane's results went out in 2·SM·(kExact ? 2 : 1) whole stores.
    auto store = [&](int tile) {
        int tm, tn;
        tile_of(tile, tiles_m, tiles_n, tm, tn);
        const int64_t m0 = int64_t(tm) * BM + wm, n0 = int64_t(tn) * BN + wn;
        const bool whole = m0 + WM <= g.m;
        if (SN == 4 && n0 + WN <= g.n) {  // lines of 128 bytes: 64 columns of bf16, 32 of fp32
            auto put = [&](int i, u32x4 v, int half, int64_t bytes) {
                const int64_t m = m0 + 16 * i + 8 * half + (r & 7);
                if (!whole && m >= g.m) return;
                uint8_t *row = static_cast<uint8_t *>(g.c) + (m * g.ldc + n0) * (kExact ? 4 : 2);
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any *>(row + bytes + 16 * part + 64 * (r >> 3)));
            };
#pragma unroll
            for (int i = 0; i < SM; ++i) {
                if constexpr (kExact) {
#pragma unroll
                    for (int j = 0; j < SN; j += 2) {
                        u32x4 a = __builtin_bit_cast(u32x4, acc[i][j]);
                        u32x4 b = __builtin_bit_cast(u32x4, acc[i][j + 1]);
                        turn_rows(a, b, r);
                        put(i, a, 0, 64 * j);
                        put(i, b, 1, 64 * j);
                    }
                } else {
                    uint32_t w[4][2];  // bf16 pairs of the four j
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            w[j][h] = f32_to_bf16_bits(acc[i][j % SN][2 * h]) |
                                      uint32_t(f32_to_bf16_bits(acc[i][j % SN][2 * h + 1])) << 16;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        turn_parts(w[0][h], w[1][h]);
                        turn_parts(w[2][h], w[3][h]);
                    }
                    u32x4 a{w[0][0], w[0][1], w[1][0], w[1][1]}, b{w[2][0], w[2][1], w[3][0], w[3][1]};
                    turn_rows(a, b, r);
                    put(i, a, 0, 0);
                    put(i, b, 1, 0);
                }
            }
            return whole;
        }
#pragma unroll
        for (int i = 0; i < SM; ++i) {
            const int64_t m = m0 + 16 * i + r;
            if (m >= g.m) continue;
#pragma unroll
            for (int j = 0; j < SN; ++j) {
                const int64_t n = n0 + 16 * j + 4 * part;
                if (n < g.n) store4(g.c, m * g.ldc + n, g.n - n < 4 ? int(g.n - n) : 4, g.c_dtype, acc[i][j]);
            }
        }
        return false;
    };
    if (steps == 0) {
        for (int tile = blockIdx.x; tile < tiles_m * tiles_n; tile += gridDim.x) store(tile);
        return;
    }
    if constexpr (kPipelined) {
        // Software pipeline over the step's MFMAs q = 0 .. SM·SN - 1 (block i = q / SN of a's
        // rows, j = q % SN of b's): each is followed by the multiply-adds of the one kLag
        // before it, and the fragments of a's block i + 3 are read while block i is
        // multiplied.  The barrier of the next step comes before the last two blocks, when
        // this wave has all of the step's fragments in registers: the next step's first
        // fragments are read, and the slot refilled, beside those blocks' MFMAs.  (MFMA, wait,
        // multiply-add in turn, the two waves of a SIMD covering for each other: 530 us at
        // 8192 x 14336 x 4096.)
        //
        // The workgroup's tiles are one stream of steps: in the last two of a tile the DMA
        // fetches the first two of the next, and a tile's results are stored beside the next
        // one's first loads.  (A workgroup a tile: 12 us between one tile's last step and the
        // next one's first, 84 of 439 us there.)  The first barrier then waits for the DMA
        // before the stores, not for the stores (418 -> 412 us there); the second one, behind
        // which the DMA was issued, for both.
        constexpr int kQ = SM * SN, kLag = 2, kBar = (SM - 2) * SN, kLast = (SM - 1) * SN;
        static_assert(D == 2 && SM % 4 == 0 && kQ % 4 == 0 && kLag < SN, "schedule");
        i32x8 fa[4], fb[SN];
        f32x4 t[4];
        float f[SM], sb = 0.0f;  // a's scales and b's
        // exponents, four blocks of a's to a register, and the scales' product for the block that
        // is multiplied and the one that is added up
        uint32_t ea[SM / 4], eb = 127;
        float next_factor = 0.0f, factor = 0.0f;
        int any_far = 0;
        auto base_of = [&](int s) { return smem + s * Geo::kSlot; };
        auto read_a = [&](const uint8_t *base, auto ic) {
            constexpr int i = decltype(ic)::value;
            fa[i % 4] = fragment(base + (wm + 16 * i) * kBlock);
        };
        auto read_b = [&](const uint8_t *base, auto jc) {
            constexpr int j = decltype(jc)::value;
            fb[j] = fragment(base + (BM + wn + 16 * j) * kBlock);
        };
        auto read_scales = [&](const uint8_t *base) {
            const float *scale_m = reinterpret_cast<const float *>(base + Geo::kPanels) + wm + r;
            static_for<SM>([&](auto ic) { f[ic] = scale_m[16 * ic]; });
            sb = *(reinterpret_cast<const float *>(base + Geo::kPanels) + BM + wn);
        };
        auto look = [&] {  // whether one of the scales at hand is far
            uint32_t low = __float_as_uint(sb), high = low;
            static_for<SM>([&](auto ic) {
                const uint32_t bits = __float_as_uint(f[ic]);
                low = bits < low ? bits : low;
                high = umax(high, bits);
            });
            any_far = __builtin_amdgcn_ballot_w64(low < kNearLow || high > kNearHigh) != 0 ? 1 : 0;
        };
        auto add = [&](auto qc) {
            constexpr int q = decltype(qc)::value, i = q / SN, j = q % SN;
            if constexpr (j == 0) factor = next_factor;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(t[q % 4][e], factor, acc[i][j][e]);
        };
        auto clear = [&] {  // nothing summed, nothing left to add
            factor = 0.0f;
            static_for<4>([&](auto c) { t[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; });
#pragma unroll
            for (int i = 0; i < SM; ++i)
#pragma unroll
                for (int j = 0; j < SN; ++j) acc[i][j] = t[0];
        };
        const int total = tiles_m * tiles_n;
        aim(blockIdx.x);
        static_for<kLoads + 1>([&](auto d) { issue(d, 0, 0); });
        static_for<kLoads + 1>([&](auto d) { issue(d, 1, 1); });
        muon_polar::wait_vm_barrier<kLoads + 1>();
        read_scales(base_of(0));
        look();
        static_for<3>([&](auto ic) { read_a(base_of(0), ic); });
        static_for<SN>([&](auto jc) { read_b(base_of(0), jc); });
        clear();
        int slot = 0, stored = 0;
        for (int tile = blockIdx.x; tile < total; tile += gridDim.x) {
            // the steps whose slots take the tile's own steps, then those whose slots take the
            // next tile's (with none left, this one's once more)
            for (int phase = 0; phase < 2; ++phase) {
                if (phase == 1 && tile + static_cast<int>(gridDim.x) < total) aim(tile + gridDim.x);
                const int from = phase == 0 ? 2 : 0, to = phase == 0 ? steps : 2;
                for (int ahead = from; ahead < to; ++ahead, slot ^= 1) {
                    const uint8_t *base = base_of(slot), *after = base_of(slot ^ 1);
                    take_scales_apart(any_far, f, sb, ea, eb);
                    static_for<kQ>([&](auto qc) {
                        constexpr int q = decltype(qc)::value, i = q / SN, j = q % SN;
                        if constexpr (q == kBar) {
                            wait_dma_barrier<2 * SM>(stored);
                            stored = 0;
                        }
                        if constexpr (j == 0) next_factor = f[i] * sb;
                        t[q % 4] = mfma_fp8<i % 4>(fb[j], eb, fa[i % 4], ea[i / 4]);
                        __builtin_amdgcn_sched_barrier(0);
                        if constexpr (q == kQ - 1) look();
                        // that of kLag before, at first the last step's
                        add(std::integral_constant<int, (q + kQ - kLag) % kQ>{});
                        if constexpr (j == 0 && i + 3 < SM)
                            read_a(base, std::integral_constant<int, i + 3>{});
                        if constexpr (q >= kBar) {
                            constexpr int n = q - kBar;
                            if constexpr (n < 2) read_a(after, std::integral_constant<int, n>{});
                            if constexpr (q == kLast) read_a(after, std::integral_constant<int, 2>{});
                            if constexpr (q >= kLast) read_b(after, std::integral_constant<int, j>{});
                            // the last block's factor is formed: the scales give way
                            if constexpr (q == kLast) read_scales(after);
                            // kLoads + 1 DMA instructions over the 2·SN MFMAs
                            static_for<kLoads + 1>([&](auto dc) {
                                constexpr int d = decltype(dc)::value;
                                if constexpr (d * 2 * SN / (kLoads + 1) == n) issue(d, ahead, slot);
                            });
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    });
                }
            }
            static_for<kLag>([&](auto c) {
                add(std::integral_constant<int, kQ - kLag + decltype(c)::value>{});
            });
            stored = __builtin_amdgcn_readfirstlane(store(tile));
            clear();
        }
    } else {
        aim(at_tile);
        for (int s = 0; s < D - 1; ++s)
#pragma unroll
            for (int d = 0; d <= kLoads; ++d) issue(d, first + s, s);
        int slot = 0;
        for (int k = first; k < steps; ++k) {
            muon_polar::wait_vm_barrier<(D - 2) * (kLoads + 1)>();
            using Operand = Frag<kExact>;
            const int next = slot == 0 ? D - 1 : slot - 1;  // the slot that step k - 1 left
            const uint8_t *base = smem + slot * Geo::kSlot;
            const float *scale_m = reinterpret_cast<const float *>(base + Geo::kPanels) + wm + r;
            const float *scale_n = reinterpret_cast<const float *>(base + Geo::kPanels) + BM + wn;
            // Scales are taken apart in every step, or (kLook) only where one of the wave's rows has a
            // far one.  With a scale a row on both sides that is 16 mantissas a lane of b's: 8192 x
            // 14336 x 8192 978 us with products of scales, 1166 with all apart, 1017 looking first;
            // 64 x 64 tiles, whose steps are short, lose more by looking (32 x 4096 x 14336 15.0 us,
            // 15.4, 18.5).  fp32 results have no registers left for a's exponents beside the rest.
            constexpr bool kLook = kRowB && Geo::kTwoSlots, kLookA = kLook && !kExact;
            uint32_t ea[SM], eb[SN];
            float sm[SM], sb = 1.0f;
            f32x4 sn[SN];
            if constexpr (kLookA)
#pragma unroll
                for (int i = 0; i < SM; ++i) ea[i] = Operand::kNone, sm[i] = scale_m[16 * i];
            if constexpr (kRowB)
#pragma unroll
                for (int j = 0; j < SN; ++j) {
                    eb[j] = Operand::kNone;
                    sn[j] = *reinterpret_cast<const f32x4 *>(scale_n + 16 * j + 4 * part);
                }
            bool any_far = !kLook || far(scale_n[lane % WN]);
            if constexpr (kLookA)
#pragma unroll
                for (int m = 0; m < WM; m += 64) any_far |= far(scale_m[(m + lane) % WM - r]);
            if (!kLook || __builtin_amdgcn_ballot_w64(any_far)) {
                if constexpr (kLookA)
#pragma unroll
                    for (int i = 0; i < SM; ++i) {
                        const Apart p = apart(sm[i]);
                        ea[i] = Operand::exponent(p.exponent), sm[i] = p.mantissa;
                    }
#pragma unroll
                for (int j = 0; j < SN; ++j) {
                    // kRowB: of the row of b that a lane supplies the exponent, of the four that it
                    // receives the mantissas
                    const Apart p = apart(scale_n[kRowB ? 16 * j + r : 0]);
                    eb[j] = Operand::exponent(p.exponent);
                    if constexpr (kRowB)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sn[j][e] = apart(sn[j][e]).mantissa;
                    else
                        sb = p.mantissa;
                }
            }
            Operand fb[SN];
#pragma unroll
            for (int j = 0; j < SN; ++j) fb[j].set(fragment(base + (BM + wn + 16 * j) * kBlock), eb[j]);
#pragma unroll
            for (int i = 0; i < SM; ++i) {
                Operand fa;
                if constexpr (!kLookA) {
                    const Apart p = apart(scale_m[16 * i]);
                    ea[i] = Operand::exponent(p.exponent), sm[i] = p.mantissa;
                }
                fa.set(fragment(base + (wm + 16 * i) * kBlock), ea[i]);
                const float f = kRowB ? sm[i] : sm[i] * sb;
#pragma unroll
                for (int j = 0; j < SN; ++j) {
                    const f32x4 t = multiply(fb[j], fa);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        acc[i][j][e] = fmaf(t[e], kRowB ? f * sn[j][e] : f, acc[i][j][e]);
                }
#pragma unroll
                for (int d = i * (kLoads + 1) / SM; d < (i + 1) * (kLoads + 1) / SM; ++d)
                    issue(d, k + D - 1, next);
            }
            slot = slot + 1 == D ? 0 : slot + 1;
        }
        store(at_tile);
    }
    muon_polar::wait_vm<0>();  // no DMA into LDS outlives the workgroup
}

// ------------------------------------------------------------------ few rows (decoding)
// Up to 16 rows of a: the weight's bytes bound the product, and each crosses once.  A
// workgroup of eight waves takes 16·NT output columns; the waves split K, so that one launch
// has all of a 14336 x 4096 weight's loads under way at once, and their sums meet in LDS in
// wave order.  A lane supplies row l % 16 of each operand, bytes 16·p .. + 15 and 64 + 16·p
// .. + 15 of each block (p = l / 16): an instruction reads 64 bytes of a row in a line.
//
// X: the rows of a as they come (bf16 or fp32), or already held.  A wave quantises its own
// part of K: a lane takes eight elements, 16 lanes a block, and the values pass through a
// corner of LDS of the wave's own into the MFMA's order.  Loads return in order, so x is
// asked for before the weight: quantising then runs beside the weight's loads.  (With each
// lane quantising the 32 values that it feeds to the MFMA, behind the weight's loads: one
// token through 14336 x 4096 took 17.3 us.)
constexpr int kFewRows = 16;
constexpr int kFewWaves = 8;

struct Held {};
struct DecodeArgs {
    int64_t n, ld_x;
    int m, cols, blocks;
    const void *x;
    const float *x_scales;  // held: element (row, block) at row + block·x_scale_col
    int64_t x_scale_col;
    muon_train_fp8_operand w;
    void *c;
    int64_t ldc;
    int c_dtype;
};

constexpr int kFewBlocks = 4;                               // blocks of K a wave takes at a time
constexpr int kFewPitch = kFewBlocks * kBlock + 16;         // bytes from row to row of held x in LDS
constexpr int kFewCorner = kFewRows * (kFewPitch + 4 * kFewBlocks);  // of a wave

// Quantises rows [t0, t0 + T) of x in the wave's blocks from kb on.
template <class X, int T>
struct FewRowsInput {
    Piece<X> p[T];
    __device__ __forceinline__ void load(const DecodeArgs &a, int t0, int kb, int end) {
        const int lane = threadIdx.x & 63;
        const int k = kb * kBlock + 8 * lane;
        const int valid = k < end * kBlock ? a.cols - k : 0;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            p[t].zero();
            if (t0 + t < a.m)
                p[t].load(static_cast<const typename X::Raw *>(a.x) + (t0 + t) * a.ld_x + k, valid);
        }
    }
    __device__ __forceinline__ void store(const DecodeArgs &a, int t0, uint8_t *values, float *scales) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < T; ++t) {
            if (t0 + t >= a.m) break;
            float f[8], inv[8];
            p[t].get(f);
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) m = umax(m, magnitude(f[e]));
            const float s = scale_of(row_umax(m)), r = 1.0f / s;
#pragma unroll
            for (int e = 0; e < 8; ++e) inv[e] = r;
            *reinterpret_cast<u32x2 *>(values + (t0 + t) * kFewPitch + 8 * lane) = to_fp8(f, inv);
            if ((lane & 15) == 0) scales[(t0 + t) * kFewBlocks + (lane >> 4)] = s;
        }
    }
};

template <class X, bool kExact, int NT>
__global__ __launch_bounds__(64 * kFewWaves) void few_rows_kernel(DecodeArgs a) {
    constexpr int U = kFewBlocks, kFirst = 4;  // rows of x whose loads go ahead of the weight's
    constexpr bool kHeld = std::is_same_v<X, Held>;
    constexpr int kSums = kFewWaves * NT * 64 * 16;
    constexpr int kLds = kHeld || kFewWaves * kFewCorner < kSums ? kSums : kFewWaves * kFewCorner;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
    const int r = lane & 15, part = lane >> 4;
    const int token = r < a.m ? r : a.m - 1;  // columns past the rows of x are dropped
    const int64_t n0 = int64_t(blockIdx.x) * (16 * NT);
    const int each = (a.blocks + kFewWaves - 1) / kFewWaves;
    const int first = wave * each, end = first + each < a.blocks ? first + each : a.blocks;
    const uint8_t *pw[NT];
    const float *sw[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {  // rows past the end read the last one and are dropped
        const int64_t n = n0 + 16 * t + r < a.n ? n0 + 16 * t + r : a.n - 1;
        const int64_t block = (n0 + 16 * t < a.n ? n0 + 16 * t : a.n - 1) / kBlock;
        pw[t] = static_cast<const uint8_t *>(a.w.values) + n * a.w.ld + 16 * part;
        sw[t] = a.w.scales + block * a.w.scale_row;
    }
    uint8_t *const values = lds + wave * kFewCorner;
    float *const scales = reinterpret_cast<float *>(values + kFewRows * kFewPitch);
    f32x4 acc[NT] = {};
    for (int kb = first; kb < end; kb += U) {
        i32x4 xlo[U], xhi[U], lo[U][NT], hi[U][NT];
        float sx[U];
        auto weight = [&] {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (kb + u < end) {
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        lo[u][t] = *reinterpret_cast<const i32x4 *>(pw[t] + (kb + u) * kBlock);
                        hi[u][t] = *reinterpret_cast<const i32x4 *>(pw[t] + (kb + u) * kBlock + 64);
                    }
                }
        };
        if constexpr (kHeld) {
            const uint8_t *p = static_cast<const uint8_t *>(a.x) + token * a.ld_x + 16 * part;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (kb + u < end) {
                    xlo[u] = *reinterpret_cast<const i32x4 *>(p + (kb + u) * kBlock);
                    xhi[u] = *reinterpret_cast<const i32x4 *>(p + (kb + u) * kBlock + 64);
                    sx[u] = a.x_scales[token + (kb + u) * a.x_scale_col];
                }
            weight();
        } else {
            for (int t0 = kFirst; t0 < a.m; t0 += kFirst) {
                FewRowsInput<X, kFirst> x;
                x.load(a, t0, kb, end);
                x.store(a, t0, values, scales);
            }
            FewRowsInput<X, kFirst> x;
            x.load(a, 0, kb, end);
            __builtin_amdgcn_sched_barrier(0);
            weight();
            __builtin_amdgcn_sched_barrier(0);
            x.store(a, 0, values, scales);
            const uint8_t *p = values + token * kFewPitch + 16 * part;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                xlo[u] = *reinterpret_cast<const i32x4 *>(p + u * kBlock);
                xhi[u] = *reinterpret_cast<const i32x4 *>(p + u * kBlock + 64);
                sx[u] = scales[token * kFewBlocks + u];
            }
        }
        auto whole = [](i32x4 l, i32x4 h) {
            return i32x8{l[0], l[1], l[2], l[3], h[0], h[1], h[2], h[3]};
        };
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (kb + u < end) {
                const Apart x_scale = apart(sx[u]);
                Frag<kExact> fx;
                fx.set(whole(xlo[u], xhi[u]), Frag<kExact>::exponent(x_scale.exponent));
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const Apart w_scale = apart(sw[t][(kb + u) * a.w.scale_col]);
                    Frag<kExact> fw;
                    fw.set(whole(lo[u][t], hi[u][t]), Frag<kExact>::exponent(w_scale.exponent));
                    const f32x4 p = multiply(fw, fx);
                    const float s = x_scale.mantissa * w_scale.mantissa;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(p[e], s, acc[t][e]);
                }
            }
    }
    f32x4 *const sums = reinterpret_cast<f32x4 *>(lds);
    __syncthreads();  // every wave is done with its corner
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[(wave * NT + t) * 64 + lane] = acc[t];
    __syncthreads();
    if (wave >= NT) return;
    f32x4 total = sums[wave * 64 + lane];
#pragma unroll
    for (int w = 1; w < kFewWaves; ++w) total += sums[(w * NT + wave) * 64 + lane];
    const int64_t n = n0 + 16 * wave + 4 * part;
    if (r < a.m && n < a.n) store4(a.c, r * a.ldc + n, a.n - n < 4 ? int(a.n - n) : 4, a.c_dtype, total);
}

// 32 columns a workgroup where that still fills the card (a lane's work on x then serves
// twice the weight), else 16.
template <class X>
void launch_few_rows(const DecodeArgs &a, int cus, Launches &launch) {
    const bool exact = a.c_dtype == MUON_TRAIN_F32;
    const int threads = 64 * kFewWaves;
    if (a.n >= 32 * int64_t(cus)) {
        const dim3 grid(static_cast<uint32_t>((a.n + 31) / 32));
        if (exact) launch(few_rows_kernel<X, true, 2>, grid, threads, a);
        else launch(few_rows_kernel<X, false, 2>, grid, threads, a);
    } else {
        const dim3 grid(static_cast<uint32_t>((a.n + 15) / 16));
        if (exact) launch(few_rows_kernel<X, true, 1>, grid, threads, a);
        else launch(few_rows_kernel<X, false, 1>, grid, threads, a);
    }
}

template <int BM, int BN, int WM, int WN, int D>
void launch_tiles(const MatmulArgs &g, bool exact, int parts, int cus, Launches &launch) {
    using Geo = Geometry<BM, BN, WM, WN, D>;
    const int tm = static_cast<int>((g.m + BM - 1) / BM), tn = static_cast<int>((g.n + BN - 1) / BN);
    const bool row_b = g.b.block_rows == 1;
    // pipelined kernels walk their tiles: as many workgroups as stay resident
    const int64_t tiles = int64_t(tm) * tn;
    const int64_t resident = int64_t(cus) * (160 * 1024 / (D * Geo::kSlot));
    const dim3 grid(static_cast<uint32_t>(Geo::kTwoSlots && !exact && !row_b && tiles > resident ? resident : tiles * parts));
    auto go = [&](auto e, auto r) {
        launch(matmul_kernel<BM, BN, WM, WN, D, decltype(e)::value, decltype(r)::value>, grid, Geo::kThreads,
               g, tm, tn, parts);
    };
    using std::bool_constant;
    if (exact && row_b) go(bool_constant<true>{}, bool_constant<true>{});
    else if (exact) go(bool_constant<true>{}, bool_constant<false>{});
    else if (row_b) go(bool_constant<false>{}, bool_constant<true>{});
    else go(bool_constant<false>{}, bool_constant<false>{});
}

bool dtype_ok(int t) { return t == MUON_TRAIN_F32 || t == MUON_TRAIN_BF16; }

constexpr int64_t kMaxExtent = int64_t(1) << 30;

int check(const muon_train_fp8_operand &o, int64_t k) {
    if (!o.values || !o.scales) return invalid("fp8: null pointer");
    if (reinterpret_cast<uintptr_t>(o.values) % 16 != 0 || o.ld % 16 != 0)
        return invalid("fp8: values must be 16-byte aligned, row by row");
    if (o.ld < k) return invalid("fp8: rows of values must not overlap");
    // the rows of a tile are reached by 31-bit offsets
    if (o.ld > MUON_TRAIN_FP8_MAX_LD) return invalid("fp8: rows of values lie too far apart");
    if (o.block_rows != 1 && o.block_rows != kBlock) return invalid("fp8: block_rows must be 1 or 128");
    // so are the scales of a tile
    if (o.scale_row < 0 || o.scale_row > (1 << 26) || o.scale_col < 0 ||
        o.scale_col > MUON_TRAIN_FP8_MAX_SCALES / (k / kBlock + 1))
        return invalid("fp8: scales lie too far apart");
    if (o.block_rows == 1 && o.scale_row != 1)
        return invalid("fp8: scales of single rows must lie next to each other");
    return MUON_POLAR_OK;
}

}  // namespace

}  // namespace muon_train

using namespace muon_train;

extern "C" int muon_train_fp8_quantize(const muon_train_fp8_quantize_args *args, hipStream_t stream) {
    if (!args) return invalid("fp8: args is null");
    const QuantArgs a = *args;
    if (a.rows < 0 || a.cols < 0 || a.rows > kMaxExtent || a.cols > kMaxExtent)
        return invalid("fp8: rows and cols must be 0 to 2^30");
    if (!dtype_ok(a.x_dtype)) return invalid("fp8: dtype must be float32 or bfloat16");
    if (a.block_rows != 1 && a.block_rows != kBlock) return invalid("fp8: block_rows must be 1 or 128");
    if (a.rows == 0 || a.cols == 0) return MUON_POLAR_OK;
    if (!a.x || (!a.values && !a.values_t)) return invalid("fp8: null pointer");
    if ((a.values || a.block_rows == kBlock) && !a.scales) return invalid("fp8: null pointer");
    if (a.values_t && a.block_rows == 1 && !a.scales_t) return invalid("fp8: null pointer");
    if (a.ld_x < a.cols) return invalid("fp8: rows of x must not overlap");
    if (reinterpret_cast<uintptr_t>(a.values) % 16 != 0 || reinterpret_cast<uintptr_t>(a.values_t) % 16 != 0)
        return invalid("fp8: values must be 16-byte aligned");
    const int64_t tr = (a.rows + kBlock - 1) / kBlock, tc = (a.cols + kBlock - 1) / kBlock;
    if (tr * tc > INT32_MAX) return invalid("fp8: matrix too large");
    const int64_t x_bytes = ((a.rows - 1) * a.ld_x + a.cols) * (a.x_dtype == MUON_TRAIN_BF16 ? 2 : 4);
    const int64_t v_bytes = a.rows * tc * kBlock, t_bytes = a.cols * tr * kBlock;
    if (meet(a.x, x_bytes, a.values, v_bytes) || meet(a.x, x_bytes, a.values_t, t_bytes) ||
        meet(a.values, v_bytes, a.values_t, t_bytes))
        return invalid("fp8: x and values must not overlap");
    const int t = static_cast<int>(tc);
    Launches launch{stream};
    if (a.block_rows == 1 && !a.values_t && tr * tc < 512) {
        const dim3 few(static_cast<uint32_t>((a.rows + 15) / 16 * tc));
        if (a.x_dtype == MUON_TRAIN_BF16) launch(quantize_rows_kernel<Bf16>, few, kQuantThreads, a, t);
        else launch(quantize_rows_kernel<F32>, few, kQuantThreads, a, t);
        return launch.result("fp8_quantize");
    }
    const dim3 grid(static_cast<uint32_t>(tr * tc));
    if (a.x_dtype == MUON_TRAIN_BF16) {
        if (a.block_rows == 1) launch(quantize_kernel<Bf16, 1>, grid, kQuantThreads, a, t);
        else launch(quantize_kernel<Bf16, kBlock>, grid, kQuantThreads, a, t);
    } else {
        if (a.block_rows == 1) launch(quantize_kernel<F32, 1>, grid, kQuantThreads, a, t);
        else launch(quantize_kernel<F32, kBlock>, grid, kQuantThreads, a, t);
    }
    return launch.result("fp8_quantize");
}

namespace muon_train {
namespace {

int check(const MatmulArgs &g) {
    if (g.m < 0 || g.n < 0 || g.k < 0 || g.m > kMaxExtent || g.n > kMaxExtent || g.k > kMaxExtent)
        return invalid("fp8: m, n and k must be 0 to 2^30");
    if (g.k % kBlock != 0) return invalid("fp8: k must be a multiple of 128");
    if (!dtype_ok(g.c_dtype)) return invalid("fp8: dtype must be float32 or bfloat16");
    if (g.m == 0 || g.n == 0) return MUON_POLAR_OK;
    if (!g.c) return invalid("fp8: null pointer");
    if (g.ldc < g.n) return invalid("fp8: rows of c must not overlap");
    if (g.k > 0) {
        int st = check(g.a, g.k);
        if (st == MUON_POLAR_OK) st = check(g.b, g.k);
        if (st != MUON_POLAR_OK) return st;
    }
    const int64_t c_bytes = ((g.m - 1) * g.ldc + g.n) * (g.c_dtype == MUON_TRAIN_BF16 ? 2 : 4);
    if (g.k > 0 && (meet(g.c, c_bytes, g.a.values, (g.m - 1) * g.a.ld + g.k) ||
                    meet(g.c, c_bytes, g.b.values, (g.n - 1) * g.b.ld + g.k)))
        return invalid("fp8: c must not overlap its operands");
    return MUON_POLAR_OK;
}

int64_t tiles(const MatmulArgs &g, int64_t t) { return ((g.m + t - 1) / t) * ((g.n + t - 1) / t); }

bool few_rows(const MatmulArgs &g) {
    return g.k > 0 && g.m <= kFewRows && g.a.block_rows == 1 && g.b.block_rows == kBlock;
}

// Side of a product's tiles.  A tile takes a compute unit's share of the tiles in turn: the
// tile whose turns, at the time of one of its own size, end first.  Times as shares of a 256 x
// 256 tile's: at 8192 x 4096 x 4096 a turn of 256s takes 62 us, of 128s 20.5, of 64s 7.4 (fp32
// 113, 32 and 11.3), the smaller ones' more where there are few (64s at 1024 x 2048 10.6).  On
// both sides of the borders, K = 4096: 1024 x 2048 in 64s 21.1 us, in 128s 28.0; 1024 x 4096
// 37.1 and 31.0; 2048 x 4096 in 128s 48.3, in 256s 52.3; 3000 x 4096 64.8 and 58.7 (fp32 104.9
// and 107.0); 4096 x 6144 124 and 107 (fp32 198 and 211).
int tile_side(const MatmulArgs &g, int cus) {
    if (g.k <= kBlock) return 64;  // a single block of K leaves nothing to pipeline
    const bool exact = g.c_dtype == MUON_TRAIN_F32;
    auto cost = [&](int64_t t, int share) { return (tiles(g, t) + cus - 1) / cus * share; };
    const int64_t cost64 = cost(64, exact ? 12 : 14), cost128 = cost(128, exact ? 29 : 35);
    if (cost64 <= cost128 && cost64 <= cost(256, 100)) return 64;
    return cost128 <= cost(256, 100) ? 128 : 256;
}

// Parts of K that 64 x 64 tiles are split into where they leave compute units idle.  A tile's
// unit takes in no more than 58 GB/s (29 bytes a clock) however many loads are under way: two
// rings of half the steps each, in one workgroup, took 31.7 us against 33.6 at 32 x 4096 x
// 14336, the parts on other units 15.6 with their joining (fp32 51 -> 20).  One workgroup a
// unit: two took 17.4.  A part keeps enough steps to fill its ring, and the join costs what
// some 16 steps do: 128 x 4096 x 4096 saves 16 of 32 steps, 12.7 and 12.6 us (fp32 17.8 and
// 15.1); 64 x 4096 x 4096 saves 24, 12.7 and 10.4; 512 x 768 x 2048 would save 8, 8.1 and 9.5.
int split_parts(const MatmulArgs &g, int cus) {
    constexpr int kSplitSteps = 4, kSplitGain = 16;
    if (few_rows(g) || tile_side(g, cus) != 64) return 1;
    const int64_t steps = g.k / kBlock;
    int64_t parts = cus / tiles(g, 64);
    if (parts > steps / kSplitSteps) parts = steps / kSplitSteps;
    if (parts < 2 || steps - steps / parts < kSplitGain) return 1;
    const int64_t each = (steps + parts - 1) / parts;
    return static_cast<int>((steps + each - 1) / each);
}

int64_t split_pitch(const MatmulArgs &g) { return (g.n + 3) / 4 * 4; }
int64_t split_bytes(const MatmulArgs &g, int parts) { return parts < 2 ? 0 : 4 * parts * g.m * split_pitch(g); }

// c = the parts' sums in the parts' order, four columns a thread.
__global__ __launch_bounds__(256) void join_kernel(MatmulArgs g, const float *sums, int64_t pitch, int parts) {
    const int64_t at = int64_t(blockIdx.x) * 256 + threadIdx.x, quads = pitch / 4;
    if (at >= g.m * quads) return;
    const f32x4 *p = reinterpret_cast<const f32x4 *>(sums) + at;
    f32x4 total = p[0];
    for (int i = 1; i < parts; ++i) total += p[i * g.m * quads];
    const int64_t m = at / quads, n = at % quads * 4;
    store4(g.c, m * g.ldc + n, g.n - n < 4 ? int(g.n - n) : 4, g.c_dtype, total);
}

int matmul(const MatmulArgs &g, float *workspace, size_t bytes, hipStream_t stream) {
    const int st = check(g);
    if (st != MUON_POLAR_OK || g.m == 0 || g.n == 0) return st;
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "fp8: no device");
    Launches launch{stream};
    if (few_rows(g)) {
        const DecodeArgs d{g.n, g.a.ld, int(g.m), int(g.k), int(g.k / kBlock), g.a.values, g.a.scales,
                           g.a.scale_col, g.b, g.c, g.ldc, g.c_dtype};
        launch_few_rows<Held>(d, cus, launch);
        return launch.result("fp8_matmul");
    }
    if (tiles(g, 64) > INT32_MAX) return invalid("fp8: matrix too large");
    const bool exact = g.c_dtype == MUON_TRAIN_F32;
    const int side = tile_side(g, cus), parts = workspace ? split_parts(g, cus) : 1;
    if (parts > 1) {
        if (bytes < static_cast<size_t>(split_bytes(g, parts))) return invalid("fp8: workspace too small");
        MatmulArgs part = g;
        part.c = workspace;
        part.ldc = split_pitch(g);
        part.c_dtype = MUON_TRAIN_F32;
        launch_tiles<64, 64, 32, 32, 4>(part, exact, parts, cus, launch);
        const int64_t quads = g.m * (split_pitch(g) / 4);
        launch(join_kernel, dim3(static_cast<uint32_t>((quads + 255) / 256)), 256, g, workspace, split_pitch(g), parts);
    } else if (side == 64) {
        launch_tiles<64, 64, 32, 32, 4>(g, exact, 1, cus, launch);
    } else if (side == 128) {
        launch_tiles<128, 128, 64, 64, 2>(g, exact, 1, cus, launch);
    } else {
        launch_tiles<256, 256, 128, 64, 2>(g, exact, 1, cus, launch);
    }
    return launch.result("fp8_matmul");
}

}  // namespace
}  // namespace muon_train

extern "C" int muon_train_fp8_matmul(const muon_train_fp8_matmul_args *args, hipStream_t stream) {
    if (!args) return invalid("fp8: args is null");
    return matmul(*args, nullptr, 0, stream);
}

extern "C" int muon_train_fp8_matmul_workspace(const muon_train_fp8_matmul_args *args, size_t *bytes) {
    if (!args || !bytes) return invalid("fp8: args is null");
    *bytes = 0;
    const int st = check(*args);
    if (st != MUON_POLAR_OK || args->m == 0 || args->n == 0) return st;
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "fp8: no device");
    *bytes = static_cast<size_t>(split_bytes(*args, split_parts(*args, cus)));
    return MUON_POLAR_OK;
}

extern "C" int muon_train_fp8_matmul_in(const muon_train_fp8_matmul_args *args, void *workspace,
                                        size_t workspace_bytes, hipStream_t stream) {
    if (!args) return invalid("fp8: args is null");
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return invalid("fp8: workspace must be 16-byte aligned");
    return matmul(*args, static_cast<float *>(workspace), workspace_bytes, stream);
}

extern "C" int muon_train_fp8_decode(const muon_train_fp8_decode_args *args, hipStream_t stream) {
    if (!args) return invalid("fp8: args is null");
    const muon_train_fp8_decode_args &g = *args;
    if (g.m < 0 || g.m > kFewRows) return invalid("fp8: m must be 0 to 16");
    if (g.n < 0 || g.n > kMaxExtent || g.cols < 1 || g.cols > kMaxExtent)
        return invalid("fp8: n must be 0 to 2^30 and cols 1 to 2^30");
    if (!dtype_ok(g.x_dtype) || !dtype_ok(g.c_dtype)) return invalid("fp8: dtype must be float32 or bfloat16");
    if (g.m == 0 || g.n == 0) return MUON_POLAR_OK;
    if (!g.x || !g.c) return invalid("fp8: null pointer");
    if (g.ld_x < g.cols) return invalid("fp8: rows of x must not overlap");
    if (g.ldc < g.n) return invalid("fp8: rows of c must not overlap");
    const int64_t blocks = (g.cols + kBlock - 1) / kBlock;
    const int st = check(g.w, blocks * kBlock);
    if (st != MUON_POLAR_OK) return st;
    if (g.w.block_rows != kBlock) return invalid("fp8: block_rows of w must be 128");
    const int64_t c_bytes = ((g.m - 1) * g.ldc + g.n) * (g.c_dtype == MUON_TRAIN_BF16 ? 2 : 4);
    const int64_t x_bytes = ((g.m - 1) * g.ld_x + g.cols) * (g.x_dtype == MUON_TRAIN_BF16 ? 2 : 4);
    if (meet(g.c, c_bytes, g.x, x_bytes) ||
        meet(g.c, c_bytes, g.w.values, (g.n - 1) * g.w.ld + blocks * kBlock))
        return invalid("fp8: c must not overlap its operands");
    const int cus = compute_units();
    if (cus <= 0) return muon_polar::report(MUON_POLAR_ERR_HIP, "fp8: no device");
    const DecodeArgs d{g.n, g.ld_x, int(g.m), int(g.cols), int(blocks), g.x, nullptr, 0,
                       g.w, g.c, g.ldc, g.c_dtype};
    Launches launch{stream};
    if (g.x_dtype == MUON_TRAIN_BF16) launch_few_rows<Bf16>(d, cus, launch);
    else launch_few_rows<F32>(d, cus, launch);
    return launch.result("fp8_decode");
}

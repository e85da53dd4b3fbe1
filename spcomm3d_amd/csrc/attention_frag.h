// Fragments of the attention kernels (attention.hip, cache.hip): what one lane of a 64-wide
// wavefront holds of a 16 x 32 operand of the matrix instructions, and how it gets it.
//
// One layout serves every type.  Lane l stands for row (left operand) or column (right operand)
// l % 16 and group g = l / 16; its eight elements are k = 8 g .. 8 g + 7 of the 32 that the
// product runs over.  A result is 16 x 16: lane l holds column l % 16, rows 4 g .. 4 g + 3.  The
// k numbering is free as long as both operands agree, so the rows of two results (4 g + i of the
// first, 16 + 4 g + i of the second) are used as the eight k of the next product as they are:
// probabilities never leave their lanes.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace spc3d {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> struct FragOf;
template <> struct FragOf<float> { typedef f32x8 type; typedef f32x4 half; };
template <> struct FragOf<bf16_t> { typedef bf16x8 type; typedef bf16x4 half; };
template <> struct FragOf<f16_t> { typedef f16x8 type; typedef f16x4 half; };
template <typename T> using Frag = typename FragOf<T>::type;
template <typename T> using HalfFrag = typename FragOf<T>::half;

// acc += a b over the 32 k of the fragments.
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 acc)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 acc)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
}
// 32 bits: eight products of four k each; group g's element j is the k that both sides call (g, j).
__device__ __forceinline__ f32x4 mma(f32x8 a, f32x8 b, f32x4 acc)
{
#pragma unroll
    for (int j = 0; j < 8; ++j)
        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], acc, 0, 0, 0);
    return acc;
}

template <typename T> __device__ __forceinline__ Frag<T> zero_frag()
{
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        f[j] = (T)0.0f;
    return f;
}

// Four results rounded to T; two such are the k of the next product.
template <typename T> __device__ __forceinline__ HalfFrag<T> rounded(f32x4 x)
{
    HalfFrag<T> f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        f[i] = (T)x[i];
    return f;
}
template <typename T> __device__ __forceinline__ Frag<T> join(HalfFrag<T> lo, HalfFrag<T> hi)
{
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// Eight elements of a row in global memory, 16-byte aligned.
template <typename T> __device__ __forceinline__ Frag<T> load_frag(const T *p)
{
    if constexpr (sizeof(T) == 4) {
        const f32x4 lo = *reinterpret_cast<const f32x4 *>(p), hi = *reinterpret_cast<const f32x4 *>(p + 4);
        return f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    } else {
        return *reinterpret_cast<const Frag<T> *>(p);
    }
}
template <typename T> __device__ __forceinline__ void store_half(T *p, f32x4 v)
{
    *reinterpret_cast<HalfFrag<T> *>(p) = rounded<T>(v);
}

// A tile of rows in LDS, DP elements of each, cut into chunks of 16 bytes; chunk c of row r lies
// at place c ^ mix(r) of its row.  Two kinds of reads have to be free of bank conflicts: row by row
// (16 lanes take the same chunk of 16 rows) and transposed (32 lanes take 8 bytes each of two
// neighbouring chunks of 8 rows), hence the rotation of the row's low bits: neighbouring rows
// differ in the chunk's second bit, not its first.
template <typename T, int DP> struct Tile {
    static constexpr int kVec = 16 / (int)sizeof(T);                 // elements of a chunk
    static constexpr int kUsed = DP / kVec;                          // chunks of a row in use
    static constexpr int kChunks = DP > 64 ? 128 / kVec : 64 / kVec; // chunks of a row's place
    static constexpr int kRowBytes = kChunks * 16;

    static __device__ __forceinline__ int mix(int r)
    {
        if constexpr (sizeof(T) == 4)
            return r & 15;
        else if constexpr (kChunks == 16)
            return ((r & 7) << 1) | ((r >> 3) & 1);
        else
            return ((r & 6) | ((r >> 3) & 1)); // 128 bytes: two rows share the banks of one place
    }
    static __device__ __forceinline__ uint32_t at(int r, int c) { return r * kRowBytes + ((c ^ mix(r)) << 4); }

    // Left operand from rows: lane l holds row r0 + l % 16, elements 32 s + 8 g ..
    static __device__ __forceinline__ Frag<T> rows(const char *tile, int r0, int s, int lane)
    {
        const int r = r0 + (lane & 15), g = lane >> 4;
        if constexpr (sizeof(T) == 4) {
            const f32x4 lo = *reinterpret_cast<const f32x4 *>(tile + at(r, 8 * s + 2 * g));
            const f32x4 hi = *reinterpret_cast<const f32x4 *>(tile + at(r, 8 * s + 2 * g + 1));
            return f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        } else {
            return *reinterpret_cast<const Frag<T> *>(tile + at(r, 4 * s + g));
        }
    }
    // Transposed: lane l holds column 16 n + l % 16 of rows r0 + 4 g + i and r0 + 16 + 4 g + i.
    static __device__ __forceinline__ Frag<T> columns(char *tile, int r0, int n, int lane)
    {
        const int l = lane & 15, g = lane >> 4;
        if constexpr (sizeof(T) == 4) {
            f32x8 f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                f[j] = *reinterpret_cast<const float *>(
                    tile + at(r0 + 16 * (j >> 2) + 4 * g + (j & 3), 4 * n + (l >> 2)) + ((l & 3) << 2));
            return f;
        } else {
            // each group of 16 lanes reads 4 rows of 16 elements, 8 bytes a lane, and gets them by column
            const int r = r0 + 4 * g + (l >> 2), c = 2 * n + ((l & 3) >> 1);
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            union { s16x4 h[2]; Frag<T> f; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + at(r, c) + ((l & 1) << 3)));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + at(r + 16, c) + ((l & 1) << 3)));
            return u.f;
        }
    }
};

// ROWS rows of a panel straight into an LDS tile, without registers between: a wavefront's load
// fills 1 KiB in lane order, so each lane asks for the chunk whose place is its own.  Rows from nrow on
// repeat row nrow - 1 (nrow >= 1; their scores are masked); chunks from dim on are left alone
// (clear_tile).  The loads are under way when this returns: loads_done(), then a barrier.
typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) const void global_void;

template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void load_tile(char *tile, const T *src, uint64_t stride, int nrow, int dim, int tid)
{
    typedef Tile<T, DP> L;
    constexpr int kLoads = ROWS * L::kChunks / THREADS, kStep = THREADS / L::kChunks; // rows of a load
    static_assert(ROWS % kStep == 0, "whole loads");
    const int first = __builtin_amdgcn_readfirstlane(tid & ~63), r0 = tid / L::kChunks;
    const uint32_t row_bytes = (uint32_t)stride * sizeof(T); // rows are at most 2^22 elements long
    auto load = [&](int i, uint32_t r, const char *from) {
        const int c = (tid % L::kChunks) ^ L::mix(r0 + i * kStep);
        if (c * L::kVec < dim)
            __builtin_amdgcn_global_load_lds((global_void *)(from + (r * row_bytes + c * 16)),
                                             (lds_void *)(tile + (i * THREADS + first) * 16), 16, 0, 0);
    };
    if (nrow >= ROWS) { // one offset for every load, from a base of its own
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            load(i, r0, (const char *)src + (uint64_t)(i * kStep) * row_bytes);
    } else {
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            load(i, min(r0 + i * kStep, nrow - 1), (const char *)src);
    }
}
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); } // vmcnt(0)

template <int BYTES, int THREADS> __device__ __forceinline__ void clear_tile(char *tile, int tid)
{
    for (int i = tid * 16; i < BYTES; i += THREADS * 16)
        *reinterpret_cast<u32x4 *>(tile + i) = u32x4{0, 0, 0, 0};
}

// e4m3, to nearest even; what is too large for it becomes the largest (448), NaN stays NaN.
constexpr float kF8Most = 448.0f;
__device__ __forceinline__ float f8_range(float x) { return fabsf(x) > kF8Most ? copysignf(kF8Most, x) : x; }
__device__ __forceinline__ uint8_t to_f8(float x)
{
    const float y = f8_range(x);
    return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false);
}

// Weights are exp2(score - base) with a base that follows the running maximum only when a score is
// more than kSlack above it: most steps then leave the sums so far as they are.  Half keeps its bits only down to 2^-14, so
// weights are 2^value times themselves on their way through the matrix instructions (and so are
// the sums that divide them): 2^(8 + 7) at most.
constexpr float kSlack = 7.0f;
template <typename T> struct WeightShift { static constexpr float value = 0.0f; };
template <> struct WeightShift<f16_t> { static constexpr float value = 8.0f; };

// The same number, of which the compiler knows nothing more: addresses made from it inside a loop
// are made there again instead of being kept in registers that the accumulators need.
template <typename T> __device__ __forceinline__ T fresh(T x)
{
    asm volatile("" : "+v"(x));
    return x;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNegInf = -__builtin_inff();

// Over the four lanes that hold the same column of a result: each exchange leaves one number of
// either half in every lane.
template <typename F> __device__ __forceinline__ float over_column(float x, F f)
{
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float column_max(float x)
{
    return over_column(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float column_sum(float x)
{
    return over_column(x, [](float a, float b) { return a + b; });
}

} // namespace spc3d

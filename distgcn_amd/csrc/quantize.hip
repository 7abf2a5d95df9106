// Dynamic 8-bit quantisation of matrix rows: q[r][k] = x[r][k] / s[r] rounded half to even, s[r] = max_k |x[r][k]| / 127.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace dgcn {

constexpr float kScaleFloor = 1.17549435e-38f;  // 2^-126: below it the scale itself would lose bits (an all-zero row gets it too)

template <class T> __device__ __forceinline__ float to_f32(T x);
template <> __device__ __forceinline__ float to_f32(float x) { return x; }
template <> __device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f32(__hip_bfloat16 x) { return __bfloat162float(x); }

constexpr int kUnit = 8;  // elements a lane takes at a time: 8 bytes of result

// t = x * (1 / s) in float32 is within 127.01 * 2^-23 of x / s: where no half lies within 2^-15 of t, t rounds as the quotient does.
// Elsewhere the quotient itself decides, in float64: a quotient of two 24-bit numbers that is not a half differs from one by more than
// 2^-25 of its size, far beyond float64's rounding.  Neither exceeds 127: s is at least max|x| / 127 less half its last bit.
constexpr float kNear = 3.0517578125e-05f;
constexpr float kToInt = 12582912.f;  // 1.5 * 2^23: adding it rounds to an integer (half to even), left in the low bits

template <class T> struct Unit { T v[kUnit]; };
template <class T> __device__ __forceinline__ Unit<T> load_unit(const T* x, int64_t at, int cols) {
    Unit<T> u;
    if (at + kUnit <= cols) {
        __builtin_memcpy(&u, x + at, sizeof(u));
    } else {
        __builtin_memset(&u, 0, sizeof(u));
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
            if (at + i < cols) u.v[i] = x[at + i];
    }
    return u;
}

template <class T> __device__ __forceinline__ void store_unit(const Unit<T>& u, float inv, float s, bool bad, int8_t* q, int64_t at, int cols) {
    uint32_t r[kUnit];
    float gap = 1.f;  // the smallest distance of a product from a half
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        const float t = to_f32(u.v[i]) * inv, f = t + kToInt;
        gap = fminf(gap, fabsf(fabsf(t - (f - kToInt)) - 0.5f));
        r[i] = __float_as_uint(f);
    }
    if (bad) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) r[i] = 0;
    } else if (gap < kNear) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) r[i] = (uint32_t)(int)rint((double)to_f32(u.v[i]) / (double)s);
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t lo = __builtin_amdgcn_perm(r[4 * i + 1], r[4 * i], 0x0c0c0400), hi = __builtin_amdgcn_perm(r[4 * i + 3], r[4 * i + 2], 0x04000c0c);
        w[i] = lo | hi;
    }
    if (at + kUnit <= cols) {
        __builtin_memcpy(q + at, w, kUnit);
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i)
            if (at + i < cols) q[at + i] = (int8_t)(uint8_t)r[i];
    }
}

// LPR lanes per row: part of a wave, or (LPR > 64) a whole workgroup.  A lane keeps its UN units in registers between the maximum and
// the rounding, so that a row is read once; LOOP: what lies behind LPR * UN units is read twice.  The bytes are the bound: 16 384 x 4 096
// bf16 in 46.5 us (201 MB, 0.92 of a copy's rate).
template <class T, int LPR, int UN, bool LOOP>
__global__ __launch_bounds__(LPR > 256 ? LPR : 256) void k_quantize_rows(const T* __restrict__ X, int64_t ldx, int rows, int cols,
                                                                         int8_t* __restrict__ Q, int64_t ldq, float* __restrict__ scale) {
    constexpr int BLOCK = LPR > 256 ? LPR : 256, RPB = BLOCK / LPR;
    static_assert(LPR <= 64 || RPB == 1, "a row is a part of a wave or a workgroup");
    __shared__ uint32_t part[BLOCK / 64];
    const int lane = threadIdx.x % LPR;
    for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < rows; r0 += (int64_t)gridDim.x * RPB) {
        const int64_t r = r0 + threadIdx.x / LPR;
        const bool live = r < rows;
        const T* x = X + (live ? r : rows - 1) * ldx;
        Unit<T> u[UN];
#pragma unroll
        for (int j = 0; j < UN; ++j) u[j] = load_unit(x, (int64_t)(lane + j * LPR) * kUnit, cols);
        uint32_t m = 0;  // the bits of |x|: ordered like the values, infinities and NaNs on top
        auto grow = [&](const Unit<T>& v) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) m = max(m, __float_as_uint(to_f32(v.v[i])) & 0x7fffffffu);
        };
#pragma unroll
        for (int j = 0; j < UN; ++j) grow(u[j]);
        if constexpr (LOOP)
            for (int64_t at = (int64_t)(lane + UN * LPR) * kUnit; at < cols; at += (int64_t)LPR * kUnit) grow(load_unit(x, at, cols));
#pragma unroll
        for (int off = (LPR > 64 ? 64 : LPR) / 2; off > 0; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off));
        if constexpr (LPR > 64) {
            __syncthreads();  // (the row before this one has been read)
            if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < BLOCK / 64; ++w) m = max(m, part[w]);
        }
        const bool bad = m >= 0x7f800000u;
        const float s = fmaxf(__uint_as_float(m) / 127.f, kScaleFloor), inv = 1.f / s;
        if (!live) continue;
        if (lane == 0) scale[r] = bad ? NAN : s;
        int8_t* q = Q + r * ldq;
#pragma unroll
        for (int j = 0; j < UN; ++j) {
            const int64_t at = (int64_t)(lane + j * LPR) * kUnit;
            if (at < cols) store_unit(u[j], inv, s, bad, q, at, cols);
        }
        if constexpr (LOOP)
            for (int64_t at = (int64_t)(lane + UN * LPR) * kUnit; at < cols; at += (int64_t)LPR * kUnit)
                store_unit(load_unit(x, at, cols), inv, s, bad, q, at, cols);
    }
}

template <class T, int LPR, int UN, bool LOOP>
static int launch_quantize_as(const void* X, int64_t ldx, int rows, int cols, int8_t* Q, int64_t ldq, float* scale, hipStream_t s) {
    constexpr int BLOCK = LPR > 256 ? LPR : 256, RPB = BLOCK / LPR;
    TimedLaunch t("quantize", s);
    DGCN_LAUNCH(t, (k_quantize_rows<T, LPR, UN, LOOP>), dim3((unsigned)min(((int64_t)rows + RPB - 1) / RPB, (int64_t)1 << 20)), dim3(BLOCK), 0, s,
                (const T*)X, ldx, rows, cols, Q, ldq, scale);
    return check_launch("k_quantize_rows");
}

template <class T> static int launch_quantize(const void* X, int64_t ldx, int rows, int cols, int8_t* Q, int64_t ldq, float* scale, hipStream_t s) {
#define DGCN_Q_CASE(LPR, UN, LOOP) return launch_quantize_as<T, LPR, UN, LOOP>(X, ldx, rows, cols, Q, ldq, scale, s)
    // The fewest lanes that hold a row in four units each: several rows' loads are in flight per wave and less of it idles behind a
    // row's end (100 000 rows of 500 float32: 51 us, a wave per row with one unit 61; 333 bf16: 32 against 54; 16 384 rows of 1 000 fp16: 12
    // against 25 with a workgroup per row, 2 048 bf16: 26 against 35).  From 2 049 columns on a workgroup per row: 4 096 bf16 47 us, a
    // wave with eight units 64.
    const int units = (cols - 1) / kUnit + 1;
    if (units <= 1) DGCN_Q_CASE(1, 1, false);
    if (units <= 2) DGCN_Q_CASE(2, 1, false);
    if (units <= 4) DGCN_Q_CASE(4, 1, false);
    if (units <= 8) DGCN_Q_CASE(4, 2, false);
    if (units <= 16) DGCN_Q_CASE(4, 4, false);
    if (units <= 32) DGCN_Q_CASE(8, 4, false);
    if (units <= 64) DGCN_Q_CASE(16, 4, false);
    if (units <= 128) DGCN_Q_CASE(64, 2, false);
    if (units <= 256) DGCN_Q_CASE(64, 4, false);
    if (units <= 512) DGCN_Q_CASE(256, 2, false);
    if (units <= 1024) DGCN_Q_CASE(256, 4, false);
    DGCN_Q_CASE(1024, 4, true);
#undef DGCN_Q_CASE
}

}  // namespace dgcn

using namespace dgcn;

extern "C" int dgcn_quantize_rows_batch(const void* X, int32_t dtype, int64_t ldx, int32_t rows, int32_t cols, int8_t* Q, int64_t ldq,
                                        float* scale, void* stream) {
    if (dtype != DGCN_F32 && dtype != DGCN_BF16 && dtype != DGCN_F16) return fail(DGCN_ERR_ARG, "dgcn_quantize_rows_batch: unknown dtype %d", dtype);
    if (rows < 0 || cols <= 0 || ldx < cols || ldq < cols) return fail(DGCN_ERR_ARG, "dgcn_quantize_rows_batch: bad sizes");
    if (rows == 0) return DGCN_OK;
    if (!X || !Q || !scale) return fail(DGCN_ERR_ARG, "dgcn_quantize_rows_batch: null argument");
    hipStream_t s = (hipStream_t)stream;
    if (dtype == DGCN_F32) return launch_quantize<float>(X, ldx, rows, cols, Q, ldq, scale, s);
    if (dtype == DGCN_BF16) return launch_quantize<__hip_bfloat16>(X, ldx, rows, cols, Q, ldq, scale, s);
    return launch_quantize<__half>(X, ldx, rows, cols, Q, ldq, scale, s);
}

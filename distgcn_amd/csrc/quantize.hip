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

// x / s rounded half to even, exactly.  The float32 product with 1 / s is within 127 * 2^-22 of the quotient; only where a
// half lies that near does the quotient itself have to decide, and in float64 it always does: a quotient of two 24-bit
// numbers that is not a half is at least 2^-25 away from one (relative), far beyond float64's rounding.
__device__ __forceinline__ int quantize_one(float x, float inv, float s) {
    const float t = x * inv;
    float q = rintf(t);
    if (fabsf(fabsf(t - q) - 0.5f) < 1e-4f) q = (float)rint((double)x / (double)s);
    q = fminf(fmaxf(q, -127.f), 127.f);
    return (int)q;
}

// One wave per row.
template <class T>
__global__ __launch_bounds__(256) void k_quantize_rows(const T* __restrict__ X, int64_t ldx, int rows, int cols, int8_t* __restrict__ Q,
                                                       int64_t ldq, float* __restrict__ scale) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
        const T* x = X + r * ldx;
        float m = 0.f;
        bool bad = false;
        for (int k = lane; k < cols; k += 64) {
            const float a = fabsf(to_f32(x[k]));
            bad |= !(a < INFINITY);
            m = fmaxf(m, a);
        }
        for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
        bad = __any(bad);
        const float s = fmaxf(m / 127.f, kScaleFloor);
        const float inv = 1.f / s;
        if (lane == 0) scale[r] = bad ? NAN : s;
        for (int k = lane; k < cols; k += 64) Q[r * ldq + k] = bad ? 0 : (int8_t)quantize_one(to_f32(x[k]), inv, s);
    }
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
    TimedLaunch t("quantize", s);
    const dim3 grid(min(ceil_div(rows, 4), 256 * 16)), block(256);
    if (dtype == DGCN_F32) DGCN_LAUNCH(t, (k_quantize_rows<float>), grid, block, 0, s, (const float*)X, ldx, rows, cols, Q, ldq, scale);
    else if (dtype == DGCN_BF16) DGCN_LAUNCH(t, (k_quantize_rows<__hip_bfloat16>), grid, block, 0, s, (const __hip_bfloat16*)X, ldx, rows, cols, Q, ldq, scale);
    else DGCN_LAUNCH(t, (k_quantize_rows<__half>), grid, block, 0, s, (const __half*)X, ldx, rows, cols, Q, ldq, scale);
    return check_launch("k_quantize_rows");
}

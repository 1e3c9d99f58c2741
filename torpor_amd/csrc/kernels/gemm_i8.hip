// Matrix product of int8 rows with a scale for each row of x and each row of w, gfx950.
//
//   y[r][c] = act( sx[r] * sw[c] * sum_k x[r][k] * w[c][k] + bias[c] + residual[r][c] )
//
// The sum is in int32 and exact, whatever its order; it is rounded to float once and scaled in float.
//
// v_mfma_i32_16x16x64_i8: lane l holds 16 consecutive k of row l % 16 of each operand, the k group given by l / 16; the result
// register i of a lane is row 4 * (l / 16) + i, column l % 16.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kernels.hpp"
#include "mfma_tile.hpp"

namespace tpk {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(1)));

// Codes k .. k+15 of a row, 0 past its end; no byte past the end is read.
__device__ __forceinline__ i32x4 load16(const int8_t* __restrict__ row, int k, int K) {
    i32x4 v = {0, 0, 0, 0};
    if (k + 16 <= K) {
        v = *reinterpret_cast<const i32x4_any*>(row + k);
    } else {
#pragma unroll
        for (int b = 0; b < 16; ++b)
            if (k + b < K) v[b >> 2] |= (int)(uint8_t)row[k + b] << (8 * (b & 3));
    }
    return v;
}

// As apply_act, except that a NaN -- the mark of a row that could not be quantised -- stays one.
__device__ __forceinline__ float act_keep_nan(float v, int act) {
    if (act == ACT_RELU) return v < 0.f ? 0.f : v;
    if (act == ACT_RELU6) return v < 0.f ? 0.f : v > 6.f ? 6.f : v;
    return apply_act(v, act);
}

__device__ __forceinline__ void store_one(const GemmI8Args& a, int r, int c, int sum) {
    float v = (float)sum * a.sx[r] * a.sw[c];
    if (a.bias) v += a.bias[c];
    if (a.residual) v += a.residual[(long)r * a.ldr + c];
    a.y[(long)r * a.ldy + c] = act_keep_nan(v, a.act);
}

// A wavefront per 16 x 16 outputs, operands straight from memory: right for every size and alignment.
__global__ __launch_bounds__(256) void gemm_i8_plain_kernel(const GemmI8Args a) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int tiles_n = (a.n + 31) / 32;
    const int r0 = ((int)(blockIdx.x / tiles_n) * 2 + (w >> 1)) * 16, c0 = ((int)(blockIdx.x % tiles_n) * 2 + (w & 1)) * 16;
    if (r0 >= a.m || c0 >= a.n) return;
    // rows past the end read the last one; their results are not stored
    const int r = min(r0 + (lane & 15), a.m - 1), c = min(c0 + (lane & 15), a.n - 1);
    const int8_t* xp = a.x + (long)r * a.ldx;
    const int8_t* wp = a.w + (long)c * a.ldw;
    i32x4 acc = {0, 0, 0, 0};
    for (int k = 0; k < a.k; k += 64) {
        const int kk = k + 16 * (lane >> 4);
        acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(load16(xp, kk, a.k), load16(wp, kk, a.k), acc, 0, 0, 0);
    }
    const int col = c0 + (lane & 15);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = r0 + 4 * (lane >> 4) + i;
        if (row < a.m && col < a.n) store_one(a, row, col, acc[i]);
    }
}

}  // namespace

int launch_gemm_i8(const GemmI8Args& a, hipStream_t s) {
    if (!a.x || !a.sx || !a.w || !a.sw || !a.y || a.m < 0 || a.n < 0 || a.k < 0) return K_EINVAL;
    if (a.act < ACT_NONE || a.act > ACT_SIGMOID) return K_EINVAL;
    if (a.k > kGemmI8MaxK) return K_EUNSUPPORTED;
    if (a.m == 0 || a.n == 0) return K_OK;
    const long grid = (((long)a.m + 31) / 32) * (((long)a.n + 31) / 32);
    if (grid * 256 > 0xffffffffl) return K_EUNSUPPORTED;
    hipLaunchKernelGGL(gemm_i8_plain_kernel, dim3((unsigned)grid), dim3(256), 0, s, a);
    set_last_kernel("gemm_i8_plain");
    return (int)hipGetLastError();
}

}  // namespace tpk

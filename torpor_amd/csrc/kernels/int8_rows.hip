// Row operators of the 8-bit encoder layer, gfx950: quantisation of rows to int8 codes with a scale, and the norms
// around a block with its gate, the residual stream and the quantisation of the result.
//
// Both read a row once, keep it in the registers of the lanes that share it and write each output once, so they are bound by
// memory.  A lane holds ITEMS groups of four neighbouring floats; TPR lanes share a row: a wavefront (four rows a workgroup,
// no barrier) or a whole workgroup.  Which of the two goes by the width alone, so a row's result does not depend on how many
// rows there are.
//
// 128-bit accesses of floats need only the floats' own alignment on this hardware, and 32-bit stores of four codes none, so
// there is one path for every pitch and only a row's last, incomplete group goes element by element.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kernels.hpp"

#pragma clang fp contract(off)  // every fused multiply-add below is written out: one arithmetic in all variants

namespace tpk {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// Elements e .. e+3 of a row, 0 past its end.
__device__ __forceinline__ f32x4 load4(const float* __restrict__ row, int e, int width) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (e + 4 <= width) {
        v = *reinterpret_cast<const f32x4_any*>(row + e);
    } else if (e < width) {
        v[0] = row[e];
        if (e + 1 < width) v[1] = row[e + 1];
        if (e + 2 < width) v[2] = row[e + 2];
    }
    return v;
}

__device__ __forceinline__ void store4(float* __restrict__ row, int e, int width, f32x4 v) {
    if (e + 4 <= width) {
        *reinterpret_cast<f32x4_any*>(row + e) = v;
    } else if (e < width) {
        row[e] = v[0];
        if (e + 1 < width) row[e + 1] = v[1];
        if (e + 2 < width) row[e + 2] = v[2];
    }
}

__device__ __forceinline__ void store4(int8_t* __restrict__ row, int e, int width, uint32_t codes) {
    if (e + 4 <= width) {
        *reinterpret_cast<u32_any*>(row + e) = codes;
    } else if (e < width) {
        row[e] = (int8_t)codes;
        if (e + 1 < width) row[e + 1] = (int8_t)(codes >> 8);
        if (e + 2 < width) row[e + 2] = (int8_t)(codes >> 16);
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)v, d);
        v = o > v ? o : v;
    }
    return v;
}

// Largest value over the lanes that share a row.  Magnitudes are compared as the integers their bits spell: the order is the
// same and infinities and NaNs come out on top.
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* lds) {
    v = wave_max(v);
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) lds[w] = v;
        __syncthreads();
        v = lds[0];
#pragma unroll
        for (int k = 1; k < TPR / 64; ++k) v = lds[k] > v ? lds[k] : v;
    }
    return v;
}

// The scale of a row from the bits of its largest magnitude.  At least 2^-126, so that its reciprocal is finite and a row of
// zeros needs no case of its own; NaN if the row holds an infinity or a NaN.
__device__ __forceinline__ float row_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    return fmaxf(__uint_as_float(amax_bits) / 127.0f, 1.17549435e-38f);
}

// The integer nearest to the true quotient x / s, halves to even.  x * (1/s) is a few rounding steps off, which moves a
// quotient that lies next to a half to the wrong side of it; the remainder x - q*s is exact in one fused multiply-add (q*s and x
// are multiples of one another's last place and nearly equal), so comparing it with s/2 sets that right.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
    float q = rintf(x * inv);
    const float r = fmaf(-q, s, x), r2 = 2.0f * fabsf(r);
    if (r2 > s || (r2 == s && ((int)q & 1))) q += copysignf(1.0f, r);
    return (int)q;
}

__device__ __forceinline__ uint32_t codes_of(f32x4 v, float s, float inv) {
    uint32_t c = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) c |= ((uint32_t)code_of(v[k], s, inv) & 255u) << (8 * k);
    return c;
}

template <int ITEMS>
__device__ __forceinline__ uint32_t lane_amax(const f32x4 (&v)[ITEMS]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t b = __float_as_uint(v[i][k]) & 0x7fffffffu;
            m = b > m ? b : m;
        }
    return m;
}

// Writes the codes and the scale of a row whose values the lanes hold.
template <int TPR, int ITEMS>
__device__ __forceinline__ void quantise_row(const f32x4 (&v)[ITEMS], int lane, int width, int8_t* __restrict__ q,
                                             float* __restrict__ scale, uint32_t* lds) {
    const uint32_t top = row_max<TPR>(lane_amax(v), lds);
    const float s = row_scale(top);
    const bool bad = top >= 0x7f800000u;
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) store4(q, 4 * (lane + TPR * i), width, bad ? 0u : codes_of(v[i], s, inv));
    if (lane == 0) *scale = s;
}

template <int TPR, int ITEMS>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void quant_rows_kernel(const QuantRowsArgs a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
    __shared__ uint32_t lds[2][16];
    const int lane = threadIdx.x % TPR;
    int turn = 0;
    for (long row = (long)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (long)gridDim.x * RPB, turn ^= 1) {
        f32x4 v[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] = load4(a.x + row * a.ldx, 4 * (lane + TPR * i), a.width);
        quantise_row<TPR, ITEMS>(v, lane, a.width, a.q + row * a.ldq, a.scale + row, lds[turn]);
    }
}

// Mean and 1 / deviation of a row, in double.  One pass over values that the lanes already hold: sums of v - c and (v - c)^2 with c
// an element of the wavefront's own share, then brought to the common mean.  An element is at most sqrt(width) deviations
// from the mean, so no more than a factor `width` of the 53 bits cancels, whatever the row's offset.
struct Moments {
    double mean, rstd;
};

template <int TPR, int ITEMS>
__device__ __forceinline__ Moments row_moments(const f32x4 (&v)[ITEMS], int lane, int width, int kind, float eps, double (*lds)[4]) {
    Moments m;
    double s1 = 0.0, s2 = 0.0;
    if (kind == 2) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // zeros past the end add nothing
                const double d = (double)v[i][k];
                s2 = fma(d, d, s2);
            }
        s2 = wave_sum(s2);
        if constexpr (TPR > 64) {
            if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6][0] = s2;
            __syncthreads();
            s2 = 0.0;
#pragma unroll
            for (int k = 0; k < TPR / 64; ++k) s2 += lds[k][0];
        }
        m.mean = 0.0;
        m.rstd = 1.0 / sqrt(s2 / (double)width + (double)eps);
        return m;
    }
    const double c = (double)__shfl(v[0][0], 0);
    int n = 0;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (4 * (lane + TPR * i) + k < width) {
                const double d = (double)v[i][k] - c;
                s1 += d;
                s2 = fma(d, d, s2);
            }
        }
    s1 = wave_sum(s1);
    s2 = wave_sum(s2);
    double mean, var;
    if constexpr (TPR > 64) {
        const int w = threadIdx.x >> 6;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {  // elements of this wavefront's share
            const int left = width - 4 * (TPR * i + 64 * w);
            n += left < 0 ? 0 : left > 256 ? 256 : left;
        }
        if ((threadIdx.x & 63) == 0) {
            lds[w][0] = s1;
            lds[w][1] = s2;
            lds[w][2] = c;
            lds[w][3] = (double)n;
        }
        __syncthreads();
        double total = 0.0;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) total += fma(lds[k][3], lds[k][2] - lds[0][2], lds[k][0]);
        mean = total / (double)width;  // about the first wavefront's c
        var = 0.0;
#pragma unroll
        for (int k = 0; k < TPR / 64; ++k) {
            const double d = mean - (lds[k][2] - lds[0][2]);
            var += fma(d, fma(lds[k][3], d, -2.0 * lds[k][0]), lds[k][1]);
        }
        mean += lds[0][2];
    } else {
        const double d = s1 / (double)width;
        mean = c + d;
        var = fma(-d, s1, s2);
    }
    var = var / (double)width;
    if (var < 0.0) var = 0.0;  // a rounding step below zero; NaN stays NaN
    m.mean = mean;
    m.rstd = 1.0 / sqrt(var + (double)eps);
    return m;
}

// t = norm(v) of four elements: (v - mean) * rstd * gamma + beta
__device__ __forceinline__ double normed(float v, const Moments& m, float gamma, float beta) {
    return fma(((double)v - m.mean) * m.rstd, (double)gamma, (double)beta);
}

template <int TPR, int ITEMS>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_block_kernel(const NormBlockArgs a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
    __shared__ double sums[2][2][16][4];
    __shared__ uint32_t tops[2][16];
    const int lane = threadIdx.x % TPR, width = a.width;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    int turn = 0;  // the next row's sums lie beside this row's, which a slower wavefront may still be reading
    for (long row = (long)blockIdx.x * RPB + threadIdx.x / TPR; row < a.rows; row += (long)gridDim.x * RPB, turn ^= 1) {
        f32x4 v[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] = load4(a.x + row * a.ldx, 4 * (lane + TPR * i), width);
        Moments post = {0.0, 1.0};
        if (a.post) post = row_moments<TPR, ITEMS>(v, lane, width, a.post, a.post_eps, sums[turn][0]);
        const float* gate = nullptr;
        if (a.gate) gate = a.gate + (a.rows_per_gate ? row / a.rows_per_gate : 0) * (long)width;
        // the residual stream, rounded to float
        const double b = (double)a.block_scale, c = (double)a.residual_scale;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int e = 4 * (lane + TPR * i);
            const f32x4 pg = a.post ? load4(a.post_gamma, e, width) : zero, pb = a.post_beta ? load4(a.post_beta, e, width) : zero;
            const f32x4 gt = gate ? load4(gate, e, width) : zero;
            const f32x4 rs = a.residual ? load4(a.residual + row * a.ldr, e, width) : zero;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                double t = a.post ? normed(v[i][k], post, pg[k], pb[k]) : (double)v[i][k];
                if (gate) t *= (double)gt[k];
                t *= b;
                if (a.residual) t = fma(c, (double)rs[k], t);
                v[i][k] = e + k < width ? (float)t : 0.f;
            }
            if (a.h) store4(a.h + row * a.ldh, e, width, v[i]);
        }
        if (a.pre) {
            const Moments pre = row_moments<TPR, ITEMS>(v, lane, width, a.pre, a.pre_eps, sums[turn][1]);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int e = 4 * (lane + TPR * i);
                const f32x4 g = load4(a.pre_gamma, e, width), bt = a.pre_beta ? load4(a.pre_beta, e, width) : zero;
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = e + k < width ? (float)normed(v[i][k], pre, g[k], bt[k]) : 0.f;
            }
        }
        if (a.y) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) store4(a.y + row * a.ldy, 4 * (lane + TPR * i), width, v[i]);
        }
        if (a.q) quantise_row<TPR, ITEMS>(v, lane, width, a.q + row * a.ldq, a.scale + row, tops[turn]);
    }
}

// The grid's threads have to fit 32 bits; more rows than that go round the loop.
constexpr long kMaxGrid = 1l << 20;

template <int TPR>
unsigned row_grid(long rows) {
    constexpr int RPB = (TPR > 256 ? TPR : 256) / TPR;
    const long blocks = (rows + RPB - 1) / RPB;
    return (unsigned)(blocks < kMaxGrid ? blocks : kMaxGrid);
}

}  // namespace

int launch_quant_rows(const QuantRowsArgs& a, hipStream_t s) {
    if (!a.x || !a.q || !a.scale || a.rows < 0 || a.width < 1) return K_EINVAL;
    if (a.width > kRowOpMaxWidth) return K_EUNSUPPORTED;
    if (a.rows == 0) return K_OK;
#define QUANT(TPR, ITEMS)                                                                                            \
    hipLaunchKernelGGL((quant_rows_kernel<TPR, ITEMS>), dim3(row_grid<TPR>(a.rows)), dim3(TPR > 256 ? TPR : 256), 0, s, a)
    if (a.width <= 1024) QUANT(64, 4);
    else if (a.width <= 4096) QUANT(256, 4);
    else if (a.width <= 16384) QUANT(1024, 4);
    else QUANT(1024, 16);
#undef QUANT
    set_last_kernel("quant_rows");
    return (int)hipGetLastError();
}

int launch_norm_block(const NormBlockArgs& a, hipStream_t s) {
    if (!a.x || a.rows < 0 || a.width < 1 || (!a.h && !a.y && !a.q) || (a.q && !a.scale)) return K_EINVAL;
    if ((a.post && !a.post_gamma) || (a.pre && !a.pre_gamma)) return K_EINVAL;
    if (a.width > kRowOpMaxWidth) return K_EUNSUPPORTED;
    if (a.rows == 0) return K_OK;
#define NORM(TPR, ITEMS)                                                                                             \
    hipLaunchKernelGGL((norm_block_kernel<TPR, ITEMS>), dim3(row_grid<TPR>(a.rows)), dim3(TPR > 256 ? TPR : 256), 0, s, a)
    if (a.width <= 1024) NORM(64, 4);
    else if (a.width <= 4096) NORM(256, 4);
    else if (a.width <= 16384) NORM(1024, 4);
    else NORM(1024, 16);
#undef NORM
    set_last_kernel("norm_block");
    return (int)hipGetLastError();
}

}  // namespace tpk

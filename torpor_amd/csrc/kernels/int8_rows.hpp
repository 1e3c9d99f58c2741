// Part of ops.hip: row operators of the 8-bit encoder layer, gfx950: quantisation of rows to int8 codes with a scale, and the norms
// around a block with its gate, the residual stream and the quantisation of the result.
//
// Both read a row once, keep it in the registers of the lanes that share it and write each output once.  Many rows are bound by memory
// (16384x4096: codes 5.8 TB/s, norms on both sides 5.1) with the vector units busy for 83 and 72 % of it; a batch of an encoder is bound by
// the vector units' issue (norm of 1536x1024, 6.9 us: 373 instructions a wavefront, of them the statistics and scaling in double, 69 % busy).
// A lane holds ITEMS groups of four neighbouring floats; TPR lanes share a row: a wavefront (four rows a workgroup, no barrier) or a whole
// workgroup.  For the norms that goes by the width alone, so that a row's sums, and with them its bits, do not depend on how many rows there
// are; the largest magnitude has no order, so the quantisation may go by the rows as well.
//
// 128-bit accesses of floats need only the floats' own alignment on this hardware, and 32-bit stores of four codes none, so
// there is one path for every pitch and only a row's last, incomplete group goes element by element.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "kernels.hpp"

#pragma clang fp contract(off)  // every fused multiply-add below is written out: one arithmetic in all variants

namespace tpk {

namespace i8 {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// Group e .. e+3 of a row, 0 past its end.  FOURS: the width is a multiple of 4, so that no group ends inside.  Rows start at an address
// that is the same for a whole wavefront, so that a lane keeps one 32-bit offset a group for all of a row's tensors.
template <bool FOURS>
__device__ __forceinline__ f32x4 load4(const float* __restrict__ row, uint32_t e, uint32_t width) {
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (FOURS ? e < width : e + 4 <= width) {
        v = *reinterpret_cast<const f32x4_any*>(row + e);
    } else if (!FOURS && e < width) {
        v[0] = row[e];
        if (e + 1 < width) v[1] = row[e + 1];
        if (e + 2 < width) v[2] = row[e + 2];
    }
    return v;
}

// AROUND: past the caches.  A norm's outputs go so (16384x4096: 237 -> 227 us alone; a layer of 1536 rows 49.5 -> 48.8, others alike);
// codes that the product reads next do not (the layer 49.5 -> 51.2).
template <bool FOURS, bool AROUND>
__device__ __forceinline__ void store4(float* __restrict__ row, uint32_t e, uint32_t width, f32x4 v) {
    if (FOURS ? e < width : e + 4 <= width) {
        if (AROUND) __builtin_nontemporal_store(v, reinterpret_cast<f32x4_any*>(row + e));
        else *reinterpret_cast<f32x4_any*>(row + e) = v;
    } else if (!FOURS && e < width) {
        row[e] = v[0];
        if (e + 1 < width) row[e + 1] = v[1];
        if (e + 2 < width) row[e + 2] = v[2];
    }
}

template <bool FOURS, bool AROUND>
__device__ __forceinline__ void store4(int8_t* __restrict__ row, uint32_t e, uint32_t width, uint32_t codes) {
    if (FOURS ? e < width : e + 4 <= width) {
        if (AROUND) __builtin_nontemporal_store(codes, reinterpret_cast<u32_any*>(row + e));
        else *reinterpret_cast<u32_any*>(row + e) = codes;
    } else if (!FOURS && e < width) {
        row[e] = (int8_t)codes;
        if (e + 1 < width) row[e + 1] = (int8_t)(codes >> 8);
        if (e + 2 < width) row[e + 2] = (int8_t)(codes >> 16);
    }
}

// Reductions over a wavefront whose result every lane gets: neighbours, pairs, quads and eights by moves within 16 lanes (a mirrored
// order serves as well as a swap once the lanes on either side agree), then the 16s and the halves by gfx950's row swaps.
// A tenth of the latency of the same through LDS permutes.
template <int CTRL>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ double moved(double v) {
    return __hiloint2double((int)moved<CTRL>((uint32_t)__double2hiint(v)), (int)moved<CTRL>((uint32_t)__double2loint(v)));
}
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kMirror8 = 0x141, kMirror16 = 0x140;

// The two values that a lane's row (16 lanes) and the row beside it hold, and those of the wavefront's halves.
struct Two {
    uint32_t a, b;
};
__device__ __forceinline__ Two rows16(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return {r[0], r[1]};
}
__device__ __forceinline__ Two rows32(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return {r[0], r[1]};
}

// Sum over groups of N lanes (a power of two).
template <int N = 64>
__device__ __forceinline__ double lanes_sum(double v) {
    if constexpr (N > 1) v += moved<kSwap1>(v);
    if constexpr (N > 2) v += moved<kSwap2>(v);
    if constexpr (N > 4) v += moved<kMirror8>(v);
    if constexpr (N > 8) v += moved<kMirror16>(v);
    if constexpr (N > 16) {
        const Two lo = rows16((uint32_t)__double2loint(v)), hi = rows16((uint32_t)__double2hiint(v));
        v = __hiloint2double((int)hi.a, (int)lo.a) + __hiloint2double((int)hi.b, (int)lo.b);
    }
    if constexpr (N > 32) {
        const Two lo = rows32((uint32_t)__double2loint(v)), hi = rows32((uint32_t)__double2hiint(v));
        v = __hiloint2double((int)hi.a, (int)lo.a) + __hiloint2double((int)hi.b, (int)lo.b);
    }
    return v;
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

template <int N = 64>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    if constexpr (N > 1) v = umax(v, moved<kSwap1>(v));
    if constexpr (N > 2) v = umax(v, moved<kSwap2>(v));
    if constexpr (N > 4) v = umax(v, moved<kMirror8>(v));
    if constexpr (N > 8) v = umax(v, moved<kMirror16>(v));
    if constexpr (N > 16) {
        const Two r = rows16(v);
        v = umax(r.a, r.b);
    }
    if constexpr (N > 32) {
        const Two r = rows32(v);
        v = umax(r.a, r.b);
    }
    return v;
}

// Largest value over the lanes that share a row.  Magnitudes are compared as the integers their bits spell: the order is the
// same and infinities and NaNs come out on top.
template <int TPR>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* lds) {
    v = lanes_max(v);
    if constexpr (TPR > 64) {
        constexpr int NW = TPR / 64;
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
        __syncthreads();
        v = lanes_max<NW>(lds[threadIdx.x % NW]);
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
template <int TPR, int ITEMS, bool FOURS, bool AROUND>
__device__ __forceinline__ void quantise_row(const f32x4 (&v)[ITEMS], int lane, int width, int8_t* __restrict__ q,
                                             float* __restrict__ scale, uint32_t* lds) {
    const uint32_t top = row_max<TPR>(lane_amax(v), lds);
    const float s = row_scale(top);
    const bool bad = top >= 0x7f800000u;
    const float inv = 1.0f / s;
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) store4<FOURS, AROUND>(q, 4 * (lane + TPR * i), width, bad ? 0u : codes_of(v[i], s, inv));
    if (lane == 0) *scale = s;
}

// The wavefront's place in its workgroup, as a scalar.
__device__ __forceinline__ int wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

template <int TPR, int ITEMS, bool FOURS>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void quant_rows_kernel(const QuantRowsArgs a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR;
    __shared__ uint32_t lds[2][16];
    const int lane = threadIdx.x % TPR;
    int turn = 0;  // the next row's largest values lie beside this row's, which a slower wavefront may still be reading
    for (long row = (long)blockIdx.x * RPB + (RPB > 1 ? wave() : 0); row < a.rows; row += (long)gridDim.x * RPB, turn ^= 1) {
        f32x4 v[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] = load4<FOURS>(a.x + row * a.ldx, 4 * (lane + TPR * i), a.width);
        quantise_row<TPR, ITEMS, FOURS, false>(v, lane, a.width, a.q + row * a.ldq, a.scale + row, lds[turn]);
    }
}

// Keeps the compiler from carrying values derived from v (their conversions to double) over this point in registers.
template <int ITEMS>
__device__ __forceinline__ void settle(f32x4 (&v)[ITEMS]) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) asm volatile("" : "+v"(v[i]));
}

// Keeps a lane's groups apart where it holds four or sixteen of them: side by side, which is how one or two are taken, their doubles,
// addresses and vectors need more than the 128 registers of a lane of 1024, and what is spilled takes scratch memory, which the callers
// were promised not to need.  Everything that depends on `at` is worked out behind this point, not ahead of the loop over rows.
// With spilled registers 512x65536 with both norms, gate and stream took 371 us, 512x65535 544, 4096x12001 430; without 120 to 130, 120 to 135, 215 to 220.
template <int ITEMS>
__device__ __forceinline__ void one_by_one(int& at) {
    if constexpr (ITEMS > 2) {
        asm volatile("" : "+v"(at));
        __builtin_amdgcn_sched_barrier(0);
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
    constexpr int NW = TPR / 64;
    const int w = threadIdx.x >> 6;
    double s1 = 0.0, s2 = 0.0, mean = 0.0, var;
    if (kind == 2) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            one_by_one<ITEMS>(lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {  // zeros past the end add nothing
                const double d = (double)v[i][k];
                s2 = fma(d, d, s2);
            }
        }
        var = lanes_sum(s2);
        if constexpr (NW > 1) {
            if ((threadIdx.x & 63) == 0) lds[w][0] = var;
            __syncthreads();
            var = lanes_sum<NW>(lds[threadIdx.x % NW][0]);
        }
    } else {
        const float first = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v[0][0])));
        const double c = (double)first;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            one_by_one<ITEMS>(lane);
            f32x4 g = v[i];
            if constexpr (ITEMS > 2) asm volatile("" : "+v"(g));  // or all doubles of both branches are made before them
            const int left = width - 4 * (lane + TPR * i);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double d = (double)(k < left ? g[k] : first) - c;
                s1 += d;
                s2 = fma(d, d, s2);
            }
        }
        s1 = lanes_sum(s1);
        s2 = lanes_sum(s2);
        if constexpr (NW > 1) {
            int n = 0;
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
            // a lane for each wavefront's share; the mean is counted from the first one's c
            const double* share = lds[threadIdx.x % NW];
            const double from = share[2] - lds[0][2], count = share[3], sum = share[0];
            const double off = lanes_sum<NW>(fma(count, from, sum)) / (double)width, d = off - from;
            var = lanes_sum<NW>(fma(d, fma(count, d, -2.0 * sum), share[1]));
            mean = lds[0][2] + off;
        } else {
            const double off = s1 / (double)width;
            mean = c + off;
            var = fma(-off, s1, s2);
        }
    }
    var = var / (double)width;
    if (var < 0.0) var = 0.0;  // a rounding step below zero; NaN stays NaN
    return {mean, 1.0 / sqrt(var + (double)eps)};
}

// A lane's groups of a vector; a constant where there is none, so that the arithmetic needs no branches.
template <bool FOURS, int ITEMS>
__device__ __forceinline__ void load_groups(f32x4 (&v)[ITEMS], const float* __restrict__ row, int first, int step, int width, float absent) {
    if (row) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] = load4<FOURS>(row, first + step * i, width);
    } else {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] = f32x4{absent, absent, absent, absent};
    }
}

template <int TPR, int ITEMS, bool POST, bool PRE, bool FOURS>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256, TPR > 256 ? TPR / 256 : 4) void norm_block_kernel(const NormBlockArgs a) {
    constexpr int THREADS = TPR > 256 ? TPR : 256, RPB = THREADS / TPR, STEP = 4 * TPR;
    constexpr int PART = ITEMS > 2 ? 1 : ITEMS;  // groups whose gamma, beta and gate are in registers at a time
    // The residual is fetched with x where there is room for both.  Of sixteen groups the two fill all registers of a lane, so there a
    // group's residual is fetched when its turn comes (with four groups that costs: 2048x16384 without a post norm 81 -> 86 us).
    constexpr int HELD = ITEMS > 4 ? 1 : ITEMS;
    __shared__ double sums[2][2][16][4];
    __shared__ uint32_t tops[2][16];
    const int width = a.width;
    int turn = 0;  // the next row's sums lie beside this row's, which a slower wavefront may still be reading
    for (long row = (long)blockIdx.x * RPB + (RPB > 1 ? wave() : 0); row < a.rows; row += (long)gridDim.x * RPB, turn ^= 1) {
        int lane = threadIdx.x % TPR;
        one_by_one<ITEMS>(lane);
        int e0 = 4 * lane;
        const float* res = a.residual ? a.residual + row * a.ldr : nullptr;
        f32x4 v[ITEMS], rs[HELD];
        load_groups<FOURS>(v, a.x + row * a.ldx, e0, STEP, width, 0.f);
        if constexpr (HELD == ITEMS) load_groups<FOURS>(rs, res, e0, STEP, width, 0.f);
        Moments post = {0.0, 1.0};
        if constexpr (POST) post = row_moments<TPR, ITEMS>(v, lane, width, a.post, a.post_eps, sums[turn][0]);
        settle(v);
        const float* gate = a.gate;
        if (gate && a.rows_per_gate)
            gate += (row >> 32 || a.rows_per_gate >> 32 ? row / a.rows_per_gate : (long)((uint32_t)row / (uint32_t)a.rows_per_gate)) * (long)width;
        // the residual stream, rounded to float
        const double b = (double)a.block_scale, c = (double)a.residual_scale;
#pragma unroll
        for (int j = 0; j < ITEMS; j += PART) {
            one_by_one<ITEMS>(e0);
            f32x4 pg[PART], pb[PART], gt[PART];
            if constexpr (HELD < ITEMS) load_groups<FOURS>(rs, res, e0 + j * STEP, STEP, width, 0.f);
            if constexpr (POST) {
                load_groups<FOURS>(pg, a.post_gamma, e0 + j * STEP, STEP, width, 1.f);
                load_groups<FOURS>(pb, a.post_beta, e0 + j * STEP, STEP, width, 0.f);
            }
            load_groups<FOURS>(gt, gate, e0 + j * STEP, STEP, width, 1.f);
#pragma unroll
            for (int i = 0; i < PART; ++i) {
                const int e = e0 + (j + i) * STEP;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    double t = (double)v[j + i][k];
                    if constexpr (POST) t = fma((t - post.mean) * post.rstd, (double)pg[i][k], (double)pb[i][k]);
                    t *= (double)gt[i][k];
                    t *= b;
                    t = fma(c, (double)rs[HELD == ITEMS ? j + i : 0][k], t);
                    v[j + i][k] = (float)t;  // 0 past the end, where all factors are
                }
                if (a.h) store4<FOURS, true>(a.h + row * a.ldh, e, width, v[j + i]);
            }
        }
        if constexpr (PRE) {
            settle(v);
            const Moments pre = row_moments<TPR, ITEMS>(v, lane, width, a.pre, a.pre_eps, sums[turn][1]);
            settle(v);
#pragma unroll
            for (int j = 0; j < ITEMS; j += PART) {
                one_by_one<ITEMS>(e0);
                f32x4 g[PART], bt[PART];
                load_groups<FOURS>(g, a.pre_gamma, e0 + j * STEP, STEP, width, 1.f);
                load_groups<FOURS>(bt, a.pre_beta, e0 + j * STEP, STEP, width, 0.f);
#pragma unroll
                for (int i = 0; i < PART; ++i) {
                    const int e = e0 + (j + i) * STEP;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        v[j + i][k] = (float)fma(((double)v[j + i][k] - pre.mean) * pre.rstd, (double)g[i][k], (double)bt[i][k]);
                    if (a.y) store4<FOURS, true>(a.y + row * a.ldy, e, width, v[j + i]);
                }
            }
        } else if (a.y) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) store4<FOURS, true>(a.y + row * a.ldy, e0 + i * STEP, width, v[i]);
        }
        if (a.q) quantise_row<TPR, ITEMS, FOURS, true>(v, lane, width, a.q + row * a.ldq, a.scale + row, tops[turn]);
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

template <int TPR, int ITEMS>
void launch_norm(const NormBlockArgs& a, hipStream_t s) {
    const dim3 grid(row_grid<TPR>(a.rows)), threads(TPR > 256 ? TPR : 256);
    const auto go = [&](auto fours) {
        constexpr bool F = decltype(fours)::value;
        if (a.post && a.pre) hipLaunchKernelGGL((norm_block_kernel<TPR, ITEMS, true, true, F>), grid, threads, 0, s, a);
        else if (a.post) hipLaunchKernelGGL((norm_block_kernel<TPR, ITEMS, true, false, F>), grid, threads, 0, s, a);
        else if (a.pre) hipLaunchKernelGGL((norm_block_kernel<TPR, ITEMS, false, true, F>), grid, threads, 0, s, a);
        else hipLaunchKernelGGL((norm_block_kernel<TPR, ITEMS, false, false, F>), grid, threads, 0, s, a);
    };
    if (a.width % 4 == 0) go(std::true_type{});
    else go(std::false_type{});
}

template <int TPR, int ITEMS>
void launch_quant(const QuantRowsArgs& a, hipStream_t s) {
    const dim3 grid(row_grid<TPR>(a.rows)), threads(TPR > 256 ? TPR : 256);
    if (a.width % 4 == 0) hipLaunchKernelGGL((quant_rows_kernel<TPR, ITEMS, true>), grid, threads, 0, s, a);
    else hipLaunchKernelGGL((quant_rows_kernel<TPR, ITEMS, false>), grid, threads, 0, s, a);
}

}  // namespace
}  // namespace i8

int launch_quant_rows(const QuantRowsArgs& a, hipStream_t s) {
    using namespace i8;
    if (!a.x || !a.q || !a.scale || a.rows < 0 || a.width < 1) return K_EINVAL;
    if (a.width > kRowOpMaxWidth) return K_EUNSUPPORTED;
    if (a.rows == 0) return K_OK;
#define QUANT(TPR, ITEMS) launch_quant<TPR, ITEMS>(a, s)
    // the widest row that each takes; of 513 to 1024 elements a row is a wavefront's where there are enough rows to fill the chip
    // (8192x1024 7.9 us against a workgroup's 9.4, 16384x600 11.3 against 14.6; 1536x1024 3.9 against 3.5, 16x768 3.3 against 2.5)
    if (a.width <= 256) QUANT(64, 1);
    else if (a.width <= 512) QUANT(64, 2);
    else if (a.width <= 1024 && a.rows >= 8192) QUANT(64, 4);
    else if (a.width <= 1024) QUANT(256, 1);
    else if (a.width <= 2048) QUANT(256, 2);
    else if (a.width <= 4096) QUANT(512, 2);
    else if (a.width <= 8192) QUANT(1024, 2);
    else if (a.width <= 16384) QUANT(1024, 4);
    else QUANT(1024, 16);
#undef QUANT
    set_last_kernel("quant_rows");
    return (int)hipGetLastError();
}

int launch_norm_block(const NormBlockArgs& a, hipStream_t s) {
    using namespace i8;
    if (!a.x || a.rows < 0 || a.width < 1 || (!a.h && !a.y && !a.q) || (a.q && !a.scale)) return K_EINVAL;
    if ((a.post && !a.post_gamma) || (a.pre && !a.pre_gamma)) return K_EINVAL;
    if (a.width > kRowOpMaxWidth) return K_EUNSUPPORTED;
    if (a.rows == 0) return K_OK;
#define NORM(TPR, ITEMS) launch_norm<TPR, ITEMS>(a, s)
    if (a.width <= 256) NORM(64, 1);
    else if (a.width <= 512) NORM(64, 2);
    else if (a.width <= 1024) NORM(256, 1);
    else if (a.width <= 2048) NORM(256, 2);
    else if (a.width <= 4096) NORM(512, 2);
    else if (a.width <= 8192) NORM(1024, 2);
    else if (a.width <= 16384) NORM(1024, 4);
    else NORM(1024, 16);
#undef NORM
    set_last_kernel("norm_block");
    return (int)hipGetLastError();
}

}  // namespace tpk

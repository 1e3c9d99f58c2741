// Matrix product of int8 rows with a scale for each row of x and each row of w, gfx950.
//
//   y[r][c] = act( sx[r] * sw[c] * sum_k x[r][k] * w[c][k] + bias[c] + residual[r][c] )
//
// The sum is in int32 and exact, whatever its order; it is rounded to float once and scaled in float.
//
// Operand layout of v_mfma_i32_16x16x64_i8 / v_mfma_i32_32x32x32_i8: a lane holds 16 consecutive k of row (lane % 16 / 32) of
// each operand, the group of k given by (lane / 16 / 32).  Result register v of a lane: column lane % 16 / 32, row
// 4 * (lane / 16) + v, or 8 * (v / 4) + 4 * (lane / 32) + v % 4.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "kernels.hpp"
#include "mfma_tile.hpp"

namespace tpk {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4_any __attribute__((ext_vector_type(4), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// 16 codes at any address.
__device__ __forceinline__ i32x4 load16(const int8_t* __restrict__ p) { return *reinterpret_cast<const i32x4_any*>(p); }

// The first `left` of 16 codes, 0 behind them; nothing behind them is read.
__device__ __forceinline__ i32x4 load16(const int8_t* __restrict__ p, int left) {
    if (left >= 16) return load16(p);
    i32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 15; ++b)
        if (b < left) v[b >> 2] |= (int)(uint8_t)p[b] << (8 * (b & 3));
    return v;
}

// As apply_act, except that a NaN -- the mark of a row that could not be quantised -- stays one.
__device__ __forceinline__ float act_keep_nan(float v, int act) {
    if (act == ACT_RELU) return v < 0.f ? 0.f : v;
    if (act == ACT_RELU6) return v < 0.f ? 0.f : v > 6.f ? 6.f : v;
    return apply_act(v, act);
}

// ------------------------------------------------------------------------------------------------ few outputs
// Outputs for less than the whole chip as tiles of their own: a workgroup takes 16 FM x 16 FN outputs, its wavefronts split K
// and add up through LDS.  Every code is used by one wavefront only, so operands go from memory to registers, U groups of 64
// codes a row at a time.
template <int FM, int FN, int W, int U>
__global__ __launch_bounds__(64 * W) void gemm_i8_split_kernel(const GemmI8Args a) {
    constexpr int OUT = 256 * FM * FN;
    __shared__ int sums[W][OUT];
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int tiles_n = (a.n + 16 * FN - 1) / (16 * FN);
    const int r0 = (int)(blockIdx.x / tiles_n) * 16 * FM, c0 = (int)(blockIdx.x % tiles_n) * 16 * FN;
    const int row = lane & 15, kl = 16 * (lane >> 4);
    const int8_t *xp[FM], *wp[FN];
    // rows past the end read the last one; their results are not stored
#pragma unroll
    for (int i = 0; i < FM; ++i) xp[i] = a.x + (long)min(r0 + 16 * i + row, a.m - 1) * a.ldx + kl;
#pragma unroll
    for (int j = 0; j < FN; ++j) wp[j] = a.w + (long)min(c0 + 16 * j + row, a.n - 1) * a.ldw + kl;

    i32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    const int groups = (a.k + 63) >> 6, whole = a.k >> 6, per = (groups + W - 1) / W;
    int g = w * per;
    const int end = min(g + per, groups), fast = min(end, whole);
    for (; g + U <= fast; g += U) {
        i32x4 xf[FM][U], wf[FN][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < FN; ++j) wf[j][u] = load16(wp[j] + ((long)(g + u) << 6));
#pragma unroll
            for (int i = 0; i < FM; ++i) xf[i][u] = load16(xp[i] + ((long)(g + u) << 6));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[i][u], wf[j][u], acc[i][j], 0, 0, 0);
    }
    for (; g < end; ++g) {
        i32x4 xf[FM], wf[FN];
        const int left = a.k - (g << 6) - kl;
#pragma unroll
        for (int j = 0; j < FN; ++j) wf[j] = load16(wp[j] + ((long)g << 6), left);
#pragma unroll
        for (int i = 0; i < FM; ++i) xf[i] = load16(xp[i] + ((long)g << 6), left);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[i], wf[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) sums[w][(16 * i + 4 * (lane >> 4) + v) * 16 * FN + 16 * j + row] = acc[i][j][v];
    __syncthreads();
    for (int o = t; o < OUT; o += 64 * W) {
        const int r = r0 + o / (16 * FN), c = c0 + o % (16 * FN);
        if (r >= a.m || c >= a.n) continue;
        int sum = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) sum += sums[k][o];
        float v = (float)sum * a.sx[r] * a.sw[c];
        if (a.bias) v += a.bias[c];
        if (a.residual) v += a.residual[(long)r * a.ldr + c];
        a.y[(long)r * a.ldy + c] = act_keep_nan(v, a.act);
    }
}

// ------------------------------------------------------------------------------------------------ many outputs
typedef __attribute__((address_space(1))) const void gmem_t;
typedef __attribute__((address_space(3))) void lmem_t;

__device__ const i32x4 kZeros = {0, 0, 0, 0};

struct TileDev {
    GemmI8Args a;
    int tiles_m, tiles_n;
};

// BM x BN outputs a workgroup, WGM x WGN wavefronts, K in blocks of 128 codes through LDS.
template <int BM, int BN, int WGM, int WGN, bool DIRECT>
__global__ __launch_bounds__(64 * WGM * WGN) void gemm_i8_tile_kernel(const TileDev p) {
    constexpr int T = 64 * WGM * WGN, NX = BM * 8 / T, NW = BN * 8 / T, NL = NX + NW;
    constexpr int TM = BM / WGM / 32, TN = BN / WGN / 32, STAGE = (BM + BN) * 128;
    constexpr int WN = 32 * TN, OP = WN + 8;  // columns of a wavefront, pitch of its output rows in LDS
    static_assert(BM * 8 % T == 0 && BN * 8 % T == 0 && T / 8 % 16 == 0, "staging in whole rows");
    static_assert(WGM * WGN * 32 * OP * 4 <= 2 * STAGE, "output rows fit the operands' LDS");
    __shared__ __attribute__((aligned(128))) int8_t lds[2][STAGE];
    const GemmI8Args& a = p.a;
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);

    // workgroup -> tile
    const int total = p.tiles_m * p.tiles_n;
    int id = blockIdx.x;
    {
        const int q = total >> 3, rem = total & 7, xcd = id & 7, local = id >> 3;
        id = xcd * q + min(xcd, rem) + local;
    }
    constexpr int GROUP = 8;
    const int per = GROUP * p.tiles_n, g = id / per, in = id - g * per;
    const int rows_g = min(GROUP, p.tiles_m - g * GROUP);
    const int tm = g * GROUP + in % rows_g, tn = in / rows_g;
    const int r0 = tm * BM, c0 = tn * BN;

    const int K = a.k, steps = (K + 127) >> 7;
    const int koff = (((t & 7) ^ ((t >> 4) & 7)) << 4);
    const int8_t* src[NL];
#pragma unroll
    for (int j = 0; j < NX; ++j) src[j] = a.x + (long)min(r0 + j * (T / 8) + (t >> 3), a.m - 1) * a.ldx + koff;
#pragma unroll
    for (int j = 0; j < NW; ++j) src[NX + j] = a.w + (long)min(c0 + j * (T / 8) + (t >> 3), a.n - 1) * a.ldw + koff;

    i32x4 reg[DIRECT ? 1 : NL];
    auto fetch = [&](int s, int stage) {
        const int left = K - (s << 7) - koff;  // codes of the row from this lane's chunk on
        if constexpr (DIRECT) {
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                const int8_t* q = src[j] + ((long)s << 7);
                if (left <= 0) q = reinterpret_cast<const int8_t*>(&kZeros);
                __builtin_amdgcn_global_load_lds((gmem_t*)q, (lmem_t*)(&lds[stage][(j * T + w * 64) * 16]), 16, 0, 0);
            }
        } else if (K - (s << 7) >= 128) {
#pragma unroll
            for (int j = 0; j < NL; ++j) reg[j] = load16(src[j] + ((long)s << 7));
        } else {
#pragma unroll
            for (int j = 0; j < NL; ++j) reg[j] = load16(src[j] + ((long)s << 7), left);
        }
    };
    auto put = [&](int stage) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int j = 0; j < NL; ++j) *reinterpret_cast<i32x4*>(&lds[stage][(j * T + t) * 16]) = reg[j];
        }
    };

    i32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) acc[i][j][v] = 0;

    const int wr = (w / WGN) * (BM / WGM), wc = (w % WGN) * (BN / WGN);
    const int frow = lane & 31, half = lane >> 5, sw = (frow >> 1) & 7;
    if (steps > 0) {
        fetch(0, 0);
        put(0);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        const int cur = s & 1;
        if (s + 1 < steps) fetch(s + 1, cur ^ 1);
        const int8_t* xb = &lds[cur][(wr + frow) * 128];
        const int8_t* wb = &lds[cur][(BM + wc + frow) * 128];
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            const int off = ((2 * kk + half) ^ sw) << 4;
            i32x4 xf[TM], wf[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) xf[i] = *reinterpret_cast<const i32x4*>(xb + i * 32 * 128 + off);
#pragma unroll
            for (int j = 0; j < TN; ++j) wf[j] = *reinterpret_cast<const i32x4*>(wb + j * 32 * 128 + off);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xf[i], wf[j], acc[i][j], 0, 0, 0);
        }
        if (s + 1 < steps) put(cur ^ 1);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }

    // 32 rows of a wavefront at a time through its share of LDS, so that lanes store four neighbours
    int* out = reinterpret_cast<int*>(&lds[0][0]) + w * 32 * OP;
    constexpr int LPR = WN / 4, RPI = 64 / LPR;  // lanes a row, rows an instruction
    const int oc = 4 * (lane % LPR), col = c0 + wc + oc;
    float csw[4], cb[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int c = min(col + e, a.n - 1);
        csw[e] = a.sw[c];
        cb[e] = a.bias ? a.bias[c] : 0.f;
    }
    const bool whole = col + 4 <= a.n;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int v = 0; v < 16; ++v) out[(8 * (v >> 2) + 4 * half + (v & 3)) * OP + 32 * j + frow] = acc[i][j][v];
        __builtin_amdgcn_wave_barrier();
#pragma unroll 2
        for (int q = 0; q < 32 / RPI; ++q) {
            const int rl = q * RPI + lane / LPR, row = r0 + wr + 32 * i + rl;
            if (row >= a.m || col >= a.n) continue;
            const i32x4 sum = *reinterpret_cast<const i32x4*>(out + rl * OP + oc);
            const float s = a.sx[row];
            f32x4_any v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)sum[e] * s * csw[e] + cb[e];
            if (a.residual) {
                const float* rp = a.residual + (long)row * a.ldr + col;
                if (whole) {
                    const f32x4_any r = *reinterpret_cast<const f32x4_any*>(rp);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += r[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (col + e < a.n) v[e] += rp[e];
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = act_keep_nan(v[e], a.act);
            float* yp = a.y + (long)row * a.ldy + col;
            if (whole) {
                *reinterpret_cast<f32x4_any*>(yp) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (col + e < a.n) yp[e] = v[e];
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <int BM, int BN, int WGM, int WGN>
int launch_tile(const GemmI8Args& a, hipStream_t s, const char* name) {
    TileDev p;
    p.a = a;
    p.tiles_m = (a.m + BM - 1) / BM;
    p.tiles_n = (a.n + BN - 1) / BN;
    const long grid = (long)p.tiles_m * p.tiles_n;
    if (grid * 64 * WGM * WGN > 0xffffffffl) return K_EUNSUPPORTED;
    const bool direct = ((reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | (uintptr_t)a.ldx | (uintptr_t)a.ldw |
                          (uintptr_t)a.k) & 15) == 0;
    if (direct)
        hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WGM, WGN, true>), dim3((unsigned)grid), dim3(64 * WGM * WGN), 0, s, p);
    else
        hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WGM, WGN, false>), dim3((unsigned)grid), dim3(64 * WGM * WGN), 0, s, p);
    set_last_kernel(name);
    return (int)hipGetLastError();
}

template <int FM, int FN, int W, int U>
int launch_split(const GemmI8Args& a, hipStream_t s, const char* name) {
    const long grid = ((a.m + 16l * FM - 1) / (16 * FM)) * ((a.n + 16l * FN - 1) / (16 * FN));
    if (grid * 64 * W > 0xffffffffl) return K_EUNSUPPORTED;
    hipLaunchKernelGGL((gemm_i8_split_kernel<FM, FN, W, U>), dim3((unsigned)grid), dim3(64 * W), 0, s, a);
    set_last_kernel(name);
    return (int)hipGetLastError();
}

}  // namespace

int launch_gemm_i8(const GemmI8Args& a, hipStream_t s) {
    if (!a.x || !a.sx || !a.w || !a.sw || !a.y || a.m < 0 || a.n < 0 || a.k < 0) return K_EINVAL;
    if (a.act < ACT_NONE || a.act > ACT_SIGMOID) return K_EINVAL;
    if (a.k > kGemmI8MaxK) return K_EUNSUPPORTED;
    if (a.m == 0 || a.n == 0) return K_OK;
    const auto tiles = [&](long bm, long bn) { return ((a.m + bm - 1) / bm) * ((a.n + bn - 1) / bn); };
    if (a.m <= 16) return launch_split<1, 1, 8, 4>(a, s, "gemm_i8_split");
    if (tiles(64, 64) < 128) return launch_split<2, 2, 8, 4>(a, s, "gemm_i8_split");
    if (tiles(256, 256) >= 192) return launch_tile<256, 256, 2, 4>(a, s, "gemm_i8_256x256");
    if (tiles(64, 64) <= 2048) return launch_tile<64, 64, 2, 2>(a, s, "gemm_i8_64x64");
    return launch_tile<128, 128, 2, 4>(a, s, "gemm_i8_128x128");
}

}  // namespace tpk

// Part of gemm.hip: matrix product of int8 rows with a scale for each row of x and each row of w, gfx950.
//
//   y[r][c] = act( sx[r] * sw[c] * sum_k x[r][k] * w[c][k] + bias[c] + residual[r][c] )
//
// The sum is in int32 and exact, whatever its order; it is rounded to float once and scaled in float.
//
// Operand layout of v_mfma_i32_16x16x64_i8 / v_mfma_i32_32x32x32_i8: a lane holds 16 consecutive k of row (lane % 16 / 32) of
// each operand, the group of k given by (lane / 16 / 32).  Result register v of a lane: column lane % 16 / 32, row
// 4 * (lane / 16) + v, or 8 * (v / 4) + 4 * (lane / 32) + v % 4.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "kernels.hpp"
#include "mfma_tile.hpp"

#pragma clang fp contract(off)  // fused multiply-adds are written out: the same bits from every variant

namespace tpk {

int num_cu();

namespace i8 {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4_words __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

// A lane's run of 16 codes in a row that is walked in steps.  128-bit loads need an address that is a multiple of 4 and take more
// than twice the time at others (8x4096x4096 with a pitch of 4097: 13.9 us, of 4100: 5.9), so rows that do not lie so are read
// as the five whole words around the run and shifted into place; bytes of the outer two words that belong to a neighbour are
// read but not used.  ANY = false: every row starts at a multiple of 4.
template <bool ANY>
struct Run {
    const int8_t* p;  // the run's first code, rounded down to a word
    uint32_t shift;   // bytes between the two
    __device__ __forceinline__ void set(const int8_t* first) {
        shift = ANY ? (uint32_t)reinterpret_cast<uintptr_t>(first) & 3 : 0;
        p = first - shift;
    }
    struct Words {
        i32x4 w;
        int next;
    };
    __device__ __forceinline__ Words load(long at) const {
        Words v;
        v.w = *reinterpret_cast<const i32x4_words*>(p + at);
        // an aligned run has no fifth word: its last one again, so that nothing behind the run is read
        if constexpr (ANY) v.next = *reinterpret_cast<const int*>(p + at + (shift ? 16 : 12));
        return v;
    }
    __device__ __forceinline__ i32x4 codes(const Words& v) const {
        if constexpr (!ANY) return v.w;
        i32x4 r;
#pragma unroll
        for (int k = 0; k < 4; ++k) r[k] = (int)__builtin_amdgcn_alignbyte((uint32_t)(k < 3 ? v.w[k + 1] : v.next), (uint32_t)v.w[k], shift);
        return r;
    }
    // as load, where a row ends inside the run: only words that hold some of its `left` codes are read, what is behind them is 0
    __device__ __forceinline__ Words load_part(long at, int left) const {
        if (left >= 16) return load(at);
        const int end = left > 0 ? left + (int)shift : 0;  // valid bytes from p + at on
        auto word = [&](int i) {
            const int n = end - 4 * i;
            if (n <= 0) return 0;
            const int v = *reinterpret_cast<const int*>(p + at + 4 * i);
            return n >= 4 ? v : v & ((1 << (8 * n)) - 1);
        };
        return Words{i32x4{word(0), word(1), word(2), word(3)}, ANY ? word(4) : 0};
    }
    // the first `left` of the 16 codes, 0 behind them
    __device__ __forceinline__ i32x4 part(long at, int left) const { return codes(load_part(at, left)); }
};

// The epilogue's activations.  A NaN -- the mark of a row that could not be quantised -- stays one under all of them.
//
// gelu(v) = v Phi(v) = max(v, 0) - |v| erfc(|v| / sqrt 2) / 2, where nothing cancels, and erfc(a / sqrt 2) = 2^Q(a).  Q is a polynomial of
// degree 12 without constant term, so that what little it is around zero is exact in proportion, fitted to log2 erfc for the least error
// over 0 <= a <= 8 (7e-9 of erfc up to 3.5, 3e-6 at 6, 1e-4 at 8; beyond, where gelu is below 1e-14, it goes on falling).
// Relative 2-norm of the error over -0.1..0.1 / 0.1..1 / -1..-0.1 / 1..3 / -2..-1: 3.1 / 2.7 / 4.5 / 2.6 / 8.0 e-8; of v/2 (1 + erf) with a
// rounded erf 3.7 / 3.9 / 5.6 / 3.5 / 15 e-8.  One exponential and a dozen multiply-adds, where erff takes fifty instructions.
__device__ __forceinline__ float fast_gelu(float v) {
    const float m = fabsf(v), a = m > 30.f ? 30.f : m;  // not fminf, which would drop a NaN; 2^Q is 0 there
    float q = fmaf(-1.863773709e-10f, a, 8.821156422e-09f);
    q = fmaf(q, a, -1.871114413e-07f);
    q = fmaf(q, a, 2.34651501e-06f);
    q = fmaf(q, a, -1.919724094e-05f);
    q = fmaf(q, a, 0.0001044538097f);
    q = fmaf(q, a, -0.000338407291f);
    q = fmaf(q, a, 7.366945954e-05f);
    q = fmaf(q, a, 0.006895748203f);
    q = fmaf(q, a, -0.05242477477f);
    q = fmaf(q, a, -0.4592220994f);
    q = fmaf(q, a, -1.151104364f);
    return fmaf(-0.5f * a, __builtin_amdgcn_exp2f(q * a), fmaxf(v, 0.f));
}
// 1 / (1 + e) with e = exp(-v).  What the exponent h loses to its rounding, -v - h ln 2, is multiplied onto e again; without that the error
// grows with |v| (2e-7 at -7, 6e-7 at -20; with it the relative 2-norm is 4.6e-8 of the sigmoid and 5.5e-8 of silu or less, for 0.4 us of
// 1536x4096x1024).  Beyond 100 e is 0; below -87.3, where the result is less than the smallest normal float, h stays at 126 and the
// correction, as it grows, drives e to infinity.
__device__ __forceinline__ float fast_sigmoid(float v) {
    const float z = v > 100.f ? 100.f : v, h = fminf(-1.44269504f * z, 126.f);
    const float e = __builtin_amdgcn_exp2f(h);
    return __builtin_amdgcn_rcpf(1.f + fmaf(e, fmaf(-0.69314718f, h, -z), e));
}
__device__ __forceinline__ float act_keep_nan(float v, int act) {
    if (act == ACT_RELU) return v < 0.f ? 0.f : v;
    if (act == ACT_GELU) return fast_gelu(v);
    if (act == ACT_TANH) return tanhf(v);
    if (act == ACT_RELU6) return v < 0.f ? 0.f : v > 6.f ? 6.f : v;
    if (act == ACT_SILU) return v * fast_sigmoid(v);
    if (act == ACT_SIGMOID) return fast_sigmoid(v);
    return v;
}

template <int ACT>
__device__ __forceinline__ void act4(f32x4_any& v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = act_keep_nan(v[e], ACT);
}

// An exact sum as a float (one rounding), scaled (two more, the second shared with the bias).
__device__ __forceinline__ float scaled(int sum, float sx, float sw, float bias) { return fmaf((float)sum * sx, sw, bias); }

// The same for rows of any size.  From a scale of 2^96 on, that of a row with values beyond 1e31, sum * sx may pass the largest float where the
// result does not; 2^64 of it then goes over to sw, which changes no bit of any other result.
constexpr float kFarScale = 0x1p96f;
__device__ __forceinline__ float scaled_far(int sum, float sx, float sw, float bias) {
    if (!(sx >= kFarScale)) return scaled(sum, sx, sw, bias);
    const float w = sw * 0x1p64f;
    return scaled(sum, sx * 0x1p-64f, sum == 0 && w > 3.40282347e38f ? 0.f : w, bias);
}

// One output from its sum.
__device__ __forceinline__ void finish_one(const GemmI8Args& a, int r, int c, int sum) {
    if (r >= a.m || c >= a.n) return;
    float v = scaled_far(sum, a.sx[r], a.sw[c], a.bias ? a.bias[c] : 0.f);
    if (a.residual) v += a.residual[(long)r * a.ldr + c];
    a.y[(long)r * a.ldy + c] = act_keep_nan(v, a.act);
}

// ------------------------------------------------------------------------------------------------ few outputs
// Too few outputs to fill the chip with larger tiles, a decoding step above all: a workgroup takes 16 FM x 16 FN outputs, its W
// wavefronts split K and add up through LDS.  Every code is used by one wavefront only, so operands go from memory to registers, U
// groups of 64 codes a row at a time.  Bound by the weights' bytes: 8x16384x4096 takes 13.0 us with the operands in the
// last-level cache, 16.6 us from memory (4.1 TB/s); 1x16384x16384 50 us (5.4 TB/s).  With eight rows or fewer half the matrix
// unit's work is on repeated rows, which costs nothing next to the loads.  Small calls end at the latency of two trips to memory:
// 1x768x768 takes 2.6 us back to back, of which 2.2 is what an empty launch takes.
template <int FM, int FN, int W, int U, bool ANY>
__global__ __launch_bounds__(64 * W) void gemm_i8_split_kernel(const GemmI8Args a) {
    constexpr int OUT = 256 * FM * FN;
    __shared__ int sums[W][OUT];
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int tiles_n = (a.n + 16 * FN - 1) / (16 * FN);
    const int r0 = (int)(blockIdx.x / tiles_n) * 16 * FM, c0 = (int)(blockIdx.x % tiles_n) * 16 * FN;
    const int row = lane & 15, kl = 16 * (lane >> 4);
    Run<ANY> xp[FM], wp[FN];
    // rows past the end read the last one; their results are not stored
#pragma unroll
    for (int i = 0; i < FM; ++i) xp[i].set(a.x + (long)min(r0 + 16 * i + row, a.m - 1) * a.ldx + kl);
#pragma unroll
    for (int j = 0; j < FN; ++j) wp[j].set(a.w + (long)min(c0 + 16 * j + row, a.n - 1) * a.ldw + kl);

    i32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    const int groups = (a.k + 63) >> 6, whole = a.k >> 6, per = (groups + W - 1) / W;
    int g = w * per;
    const int end = min(g + per, groups), fast = min(end, whole);
    for (; g + U <= fast; g += U) {
        typename Run<ANY>::Words xf[FM][U], wf[FN][U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int j = 0; j < FN; ++j) wf[j][u] = wp[j].load((long)(g + u) << 6);
#pragma unroll
            for (int i = 0; i < FM; ++i) xf[i][u] = xp[i].load((long)(g + u) << 6);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < FM; ++i)
#pragma unroll
                for (int j = 0; j < FN; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xp[i].codes(xf[i][u]), wp[j].codes(wf[j][u]), acc[i][j], 0, 0, 0);
    }
    for (; g < end; ++g) {
        i32x4 xf[FM], wf[FN];
        const int left = a.k - (g << 6) - kl;
#pragma unroll
        for (int j = 0; j < FN; ++j) wf[j] = wp[j].part((long)g << 6, left);
#pragma unroll
        for (int i = 0; i < FM; ++i) xf[i] = xp[i].part((long)g << 6, left);
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
        int sum = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) sum += sums[k][o];
        finish_one(a, r0 + o / (16 * FN), c0 + o % (16 * FN), sum);
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

enum Fetch { DIRECT, WORDS, BYTES };  // chunks of 16 codes straight to LDS; through registers, rows at multiples of 4; at any address

enum Rest { NOTHING, GELU, ANYTHING };  // what an epilogue does beyond scaling

// BM x BN outputs a workgroup, WGM x WGN wavefronts, K in blocks of BK codes through two LDS buffers.
//
// A row's 16-code chunks lie in LDS in an order turned by the row (koff / sw below), so that the 16 lanes that read one chunk of 16
// rows touch all 64 banks; the direct loads, which write LDS in lane order, turn the addresses they read instead.  Fragments of the
// next 64 codes are read while one group multiplies.  The loads that refill a buffer leave one at a time between the products
// behind the barrier that frees it: sent off together they held up every wavefront for a thousand cycles of each block
// (8192^3 with the loads in a burst 572 us, spread 516).  16x16 products rather than 32x32: half the accumulator traffic, which shows
// because the chip runs at its power limit here (8192^3 of random codes 516 -> 467 us; of zeros, 417 -> 435).  Stores go past the
// caches, or y drives the operands out of them (467 -> 434 us; 4096^3 74 -> 63; 1536x4096x1024 with gelu 17.2 -> 14.6), also where the next
// kernel reads y at once: the products, norms and codes of a BERT-large layer take 79.1 us (81.4 through the caches) at 1536 rows, 151.7 (158.0)
// at 4096, 51.0 (51.1) at 512; only 128 rows of BERT-base have it the other way, 33.6 (33.3).  At 434 us, 2.5 POP/s, the product is as fast as
// the matrix unit's clock under that limit allows a library's to be (445 us for the same size, without scales).
template <int BM, int BN, int WGM, int WGN, int BK, Fetch HOW>
__global__ __launch_bounds__(64 * WGM * WGN) void gemm_i8_tile_kernel(const TileDev p) {
    constexpr bool ANY = HOW == BYTES;
    constexpr int T = 64 * WGM * WGN, CH = BK / 16, NX = BM * CH / T, NW = BN * CH / T, NL = NX + NW;
    constexpr int TM = BM / WGM / 16, TN = BN / WGN / 16, BLOCK = (BM + BN) * BK, KK = BK / 64;
    constexpr int WN = 16 * TN, OP = WN + 4;  // columns of a wavefront, pitch of its output rows in LDS
    constexpr int SPAN = 16 / CH;             // rows that lie side by side in the 64 LDS banks
    constexpr int OUT = WGM * WGN * 16 * OP * 4, LDS = 2 * BLOCK > OUT ? 2 * BLOCK : OUT;
    static_assert(BM * CH % T == 0 && BN * CH % T == 0 && T / CH % 16 == 0, "staging in whole rows");
    __shared__ __attribute__((aligned(256))) int8_t lds[LDS];
    const GemmI8Args& a = p.a;
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);

    // workgroup -> tile: each XCD (workgroup id mod 8) takes a run of tiles, eight tile rows deep, whose operands share its L2
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

    const int wr = (w / WGN) * (BM / WGM), wc = (w % WGN) * (BN / WGN);
    const int frow = lane & 15, part = lane >> 4, sw = (frow / SPAN) % CH;
    // whether a wavefront has a row for finish_one; asked for ahead of the operands (behind the products a small call waits for it: 128x3072x768 with
    // gelu 4.60 -> 4.75 us; a test for every row in the epilogue took 2 % of 1536x4096x1024)
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < TM; ++i) most = fmaxf(most, a.sx[min(r0 + wr + 16 * i + frow, a.m - 1)]);

    const int K = a.k, steps = (K + BK - 1) / BK;
    const int koff = ((t % CH) ^ ((t / CH / SPAN) % CH)) * 16;
    Run<ANY> src[NL];
#pragma unroll
    for (int j = 0; j < NX; ++j) src[j].set(a.x + (long)min(r0 + j * (T / CH) + t / CH, a.m - 1) * a.ldx + koff);
#pragma unroll
    for (int j = 0; j < NW; ++j) src[NX + j].set(a.w + (long)min(c0 + j * (T / CH) + t / CH, a.n - 1) * a.ldw + koff);

    typename Run<ANY>::Words reg[HOW == DIRECT ? 1 : NL];
    // loads j0 .. j1-1 of block s, on their way to LDS or to registers
    auto fetch = [&](int s, int j0, int j1) {
        const int left = K - s * BK - koff;  // codes of the row from this lane's chunk on
        if constexpr (HOW == DIRECT) {
            int8_t* const to = lds + (s & 1) * BLOCK + w * 1024;
            if (K - s * BK >= BK) {
#pragma unroll
                for (int j = j0; j < j1; ++j)
                    __builtin_amdgcn_global_load_lds((gmem_t*)(src[j].p + (long)s * BK), (lmem_t*)(to + j * T * 16), 16, 0, 0);
            } else {  // the last block ends inside: chunks behind the end are zeros
#pragma unroll
                for (int j = j0; j < j1; ++j) {
                    const int8_t* q = left > 0 ? src[j].p + (long)s * BK : reinterpret_cast<const int8_t*>(&kZeros);
                    __builtin_amdgcn_global_load_lds((gmem_t*)q, (lmem_t*)(to + j * T * 16), 16, 0, 0);
                }
            }
        } else if (K - s * BK >= BK) {
#pragma unroll
            for (int j = j0; j < j1; ++j) reg[j] = src[j].load((long)s * BK);
        } else {
#pragma unroll
            for (int j = j0; j < j1; ++j) reg[j] = src[j].load_part((long)s * BK, left);
        }
    };
    auto put = [&](int s, int j0, int j1) {
        if constexpr (HOW != DIRECT) {
#pragma unroll
            for (int j = j0; j < j1; ++j) *reinterpret_cast<i32x4*>(lds + (s & 1) * BLOCK + (j * T + t) * 16) = src[j].codes(reg[j]);
        }
    };
    // Behind it every wavefront has done with what it read or wrote in LDS so far and, if direct, its loads have arrived.
    auto meet = [&]() {
        if constexpr (HOW == DIRECT) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // Direct loads bring whole chunks; where the last one of x ends inside (K no multiple of 16) what lies behind the end becomes 0,
    // so that it does not matter what w has there.
    auto cut = [&](int s) {
        if constexpr (HOW == DIRECT) {
            if ((K & 15) == 0 || s != steps - 1) return;
            const int c = (K - s * BK) >> 4, n = K & 15;
            for (int r = t; r < BM; r += T) {
                i32x4* const at = reinterpret_cast<i32x4*>(lds + (s & 1) * BLOCK + r * BK + ((c ^ ((r / SPAN) % CH)) << 4));
                i32x4 v = *at;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = n >= 4 * i + 4 ? v[i] : n > 4 * i ? v[i] & ((1 << (8 * (n - 4 * i))) - 1) : 0;
                *at = v;
            }
            meet();
        }
    };

    i32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = i32x4{0, 0, 0, 0};

    i32x4 xf[2][TM], wf[2][TN];
    auto frags = [&](int s, int kk, int to) {
        const int8_t* base = lds + (s & 1) * BLOCK + frow * BK + (((4 * kk + part) ^ sw) << 4);
#pragma unroll
        for (int i = 0; i < TM; ++i) xf[to][i] = *reinterpret_cast<const i32x4*>(base + (wr + i * 16) * BK);
#pragma unroll
        for (int j = 0; j < TN; ++j) wf[to][j] = *reinterpret_cast<const i32x4*>(base + (BM + wc + j * 16) * BK);
    };
    // products q0 .. q1-1 of a group
    auto multiply = [&](int from, int q0, int q1) {
#pragma unroll
        for (int q = q0; q < q1; ++q)
            // w first: a lane's four results are neighbours in a row of y
            acc[q / TN][q % TN] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[from][q % TN], xf[from][q / TN], acc[q / TN][q % TN], 0, 0, 0);
    };

    if (steps > 0) {
        constexpr int Q = TM * TN;
        static_assert(KK % 2 == 0, "fragment buffers alternate");
        fetch(0, 0, NL);
        if constexpr (HOW == DIRECT) {
            if (steps > 1) {
                fetch(1, 0, NL);
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
                __builtin_amdgcn_s_barrier();
                asm volatile("" ::: "memory");
            } else {
                meet();
            }
        } else {
            put(0, 0, NL);
            if (steps > 1) fetch(1, 0, NL);
            meet();
        }
        cut(0);
        frags(0, 0, 0);
        for (int s = 0; s < steps; ++s) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                if (kk + 1 < KK) {
                    frags(s, kk + 1, (kk + 1) & 1);
                } else if (s + 1 < steps) {
                    // this wavefront has read all of block s; behind the barrier every wavefront has, and block s + 1 is there
                    put(s + 1, 0, NL);
                    meet();
                    cut(s + 1);
                    frags(s + 1, 0, 0);
                }
                // Loads into the place of a block go out behind the barrier that frees it, one at a time between the products of the
                // block's last group.
                constexpr int n = NL + 1;
                __builtin_amdgcn_sched_barrier(0);
                if (kk == KK - 1) {
#pragma unroll
                    for (int j = 0; j < NL; ++j) {
                        multiply(kk & 1, Q * j / n, Q * (j + 1) / n);
                        __builtin_amdgcn_sched_barrier(0);
                        if (s + 2 < steps) fetch(s + 2, j, j + 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    multiply(kk & 1, Q * NL / n, Q);
                } else {
                    multiply(kk & 1, 0, Q);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    __syncthreads();

    // four columns of a row
    auto finish = [&](int row, int col, const i32x4& sum, float s, const float (&csw)[4], const float (&cb)[4], auto what) {
        constexpr Rest rest = decltype(what)::value;
        if (row >= a.m || col >= a.n) return;
        const bool whole = col + 4 <= a.n;
        f32x4_any v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = scaled(sum[e], s, csw[e], cb[e]);
        if constexpr (rest != NOTHING) {
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
            if constexpr (rest == GELU) act4<ACT_GELU>(v);
            else if (a.act == ACT_RELU) act4<ACT_RELU>(v);
            else if (a.act == ACT_TANH) act4<ACT_TANH>(v);
            else if (a.act == ACT_RELU6) act4<ACT_RELU6>(v);
            else if (a.act == ACT_SILU) act4<ACT_SILU>(v);
            else if (a.act == ACT_SIGMOID) act4<ACT_SIGMOID>(v);
        }
        float* yp = a.y + (long)row * a.ldy + col;
        if (whole) {
            __builtin_nontemporal_store(v, reinterpret_cast<f32x4_any*>(yp));
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (col + e < a.n) yp[e] = v[e];
        }
    };
    auto column = [&](int col, float (&csw)[4], float (&cb)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int c = min(col + e, a.n - 1);
            csw[e] = a.sw[c];
            cb[e] = a.bias ? a.bias[c] : 0.f;
        }
    };
    // 16 rows of a wavefront at a time through its share of LDS, so that a store covers whole lines of y
    int* out = reinterpret_cast<int*>(lds) + w * 16 * OP;
    constexpr int LPR = WN / 4, RPI = 64 / LPR;  // lanes a row, rows an instruction
    const int oc = 4 * (lane % LPR), col = c0 + wc + oc;
    float csw[4], cb[4];
    column(col, csw, cb);
    const bool far = __builtin_amdgcn_ballot_w64(most >= kFarScale) != 0;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) *reinterpret_cast<i32x4*>(out + frow * OP + 16 * j + 4 * part) = acc[i][j];
        __builtin_amdgcn_wave_barrier();
        const int rl = lane / LPR, row = r0 + wr + 16 * i + rl;
        const auto rows = [&](auto what) {
            // at most four times: 256x256 has eight, with which the whole is more than the compiler unrolls, and accumulators that it has
            // to index lie in scratch memory
            constexpr int times = 16 / RPI < 4 ? 16 / RPI : 4;
#pragma unroll times
            for (int q = 0; q < 16; q += RPI)
                finish(row + q, col, *reinterpret_cast<const i32x4*>(out + (rl + q) * OP + oc), a.sx[min(row + q, a.m - 1)], csw, cb, what);
        };
        if (__builtin_expect(far, 0)) {
#pragma unroll 1
            for (int o = lane; o < 16 * WN; o += 64) finish_one(a, r0 + wr + 16 * i + o / WN, c0 + wc + o % WN, out[o / WN * OP + o % WN]);
        } else if (a.act == ACT_GELU) rows(std::integral_constant<Rest, GELU>{});
        else if (a.residual || a.act != ACT_NONE) rows(std::integral_constant<Rest, ANYTHING>{});
        else rows(std::integral_constant<Rest, NOTHING>{});
        __builtin_amdgcn_wave_barrier();
    }
}

// How the operands lie: every row at a multiple of 16, at a multiple of 4, or anywhere.
Fetch fetch_of(const GemmI8Args& a) {
    const uintptr_t rows = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.w) | (uintptr_t)a.ldx | (uintptr_t)a.ldw;
    return (rows & 15) == 0 ? DIRECT : (rows & 3) == 0 ? WORDS : BYTES;
}

using Launch = void (*)(const GemmI8Args& a, Fetch how, unsigned grid, hipStream_t s);

template <int FM, int FN, int W, int U>
void launch_split(const GemmI8Args& a, Fetch how, unsigned grid, hipStream_t s) {
    if (how == BYTES) hipLaunchKernelGGL((gemm_i8_split_kernel<FM, FN, W, U, true>), dim3(grid), dim3(64 * W), 0, s, a);
    else hipLaunchKernelGGL((gemm_i8_split_kernel<FM, FN, W, U, false>), dim3(grid), dim3(64 * W), 0, s, a);
}

template <int BM, int BN, int WGM, int WGN, int BK, bool REG>
void launch_tile(const GemmI8Args& a, Fetch how, unsigned grid, hipStream_t s) {
    const TileDev p = {a, (a.m + BM - 1) / BM, (a.n + BN - 1) / BN};
    const dim3 g(grid), t(64 * WGM * WGN);
    if constexpr (REG) {
        if (how == WORDS) hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WGM, WGN, BK, WORDS>), g, t, 0, s, p);
        else hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WGM, WGN, BK, BYTES>), g, t, 0, s, p);
    } else {
        hipLaunchKernelGGL((gemm_i8_tile_kernel<BM, BN, WGM, WGN, BK, DIRECT>), g, t, 0, s, p);
    }
}

// What a call takes with one tile or another:  2 us + sqrt((bytes / 5.6 TB/s)^2 + work^2), so the tile with the least work is taken:
//   work = tile * (1 + more * (rounds - 1)),  next for more from a CU's tile number `held` + 1 on,
//   tile = first + codes * k / 1024 + act us, what one tile takes (act: with gelu, silu, sigmoid or tanh in the epilogue),
//   rounds = tiles for each CU, rounded up by the share `last`,
//   held = tiles that a CU's LDS and wavefronts hold at once (second table: not told apart), more = what one beside others adds.
// The numbers are fitted to timings of all tiles at 870 shapes, most of them random (m 1 to 16384, n 128 to 32768, k 64 to 16384, with
// gelu and without): the tile taken is on average within 1 % of the fastest, at most 26 %, and within 1.1 % at 120 random shapes that
// the fit has not seen.  What they reflect: a CU fetches about 27 bytes a cycle of what lies in L2, so (m + n) * k of a tile counts until
// its products do; small tiles win as long as there are too few to go round; 256x256 is alone on its CU, so its epilogue has nothing to
// hide behind and it needs a long k.  At 8192^3 256x256 takes 438 us, 192x128 500; at 8192x8192x1024 with gelu 256x256 takes 112, 192x128
// 113 to 116, 64x128 127; at 1536x4096x1024 with gelu 64x128 takes 14.6, 192x128 15.5, 64x64 18.9; at 256x1024x4096 32x32 takes 9.7 us, 64x64
// 10.6, 16x16 16.5.  The activations have changed since the fit: at 120 other random shapes, a quarter of them at odd addresses, the tile taken
// is now within 1.5 % of the fastest on average and 25 % at most.  Rows at other addresses than multiples of 16 go through registers (second
// table, 260 shapes, within 0.9 %, at most 20 %): 3000x4096x4091 with a pitch of 4096 takes 56 us, of 4091 102.
struct Tile {
    int m, n, threads;
    float first, codes, act, more;
    int held;
    float next, last;
    Launch launch;
    const char* name;
};
const Tile kDirect[] = {
    {16, 16, 512, 0.26f, 0.67f, 0.01f, 0.96f, 4, 1.25f, 0.81f, launch_split<1, 1, 8, 4>, "gemm_i8_16x16"},
    {16, 32, 512, 0.55f, 1.06f, 0.05f, 0.98f, 4, 0.99f, 1.f, launch_split<1, 2, 8, 4>, "gemm_i8_16x32"},
    {32, 32, 1024, 0.87f, 1.38f, 0.f, 1.54f, 2, 1.39f, 0.91f, launch_split<2, 2, 16, 2>, "gemm_i8_32x32"},
    {32, 64, 512, 1.11f, 2.13f, 0.24f, 0.36f, 3, 0.57f, 1.f, launch_tile<32, 64, 2, 4, 256, false>, "gemm_i8_32x64"},
    {64, 64, 512, 1.47f, 2.58f, 0.23f, 0.37f, 2, 0.87f, 0.93f, launch_tile<64, 64, 4, 2, 256, false>, "gemm_i8_64x64"},
    {96, 64, 512, 1.89f, 2.72f, 0.43f, 0.64f, 2, 0.8f, 0.58f, launch_tile<96, 64, 2, 4, 256, false>, "gemm_i8_96x64"},
    {64, 128, 512, 1.49f, 4.45f, 0.68f, 0.38f, 3, 0.83f, 1.f, launch_tile<64, 128, 2, 4, 128, false>, "gemm_i8_64x128"},
    {192, 128, 512, 2.74f, 6.62f, 2.44f, 0.98f, 2, 0.86f, 0.43f, launch_tile<192, 128, 4, 2, 128, false>, "gemm_i8_192x128"},
    {256, 256, 512, 8.66f, 12.55f, 5.71f, 0.f, 1, 1.13f, 0.97f, launch_tile<256, 256, 4, 2, 128, false>, "gemm_i8_256x256"},
};
const Tile kThroughRegisters[] = {
    {16, 16, 512, 0.36f, 1.12f, 0.f, 0.95f, 1, 0.95f, 0.83f, launch_split<1, 1, 8, 4>, "gemm_i8_16x16"},
    {16, 32, 512, 0.7f, 1.72f, 0.f, 0.95f, 1, 0.95f, 0.85f, launch_split<1, 2, 8, 4>, "gemm_i8_16x32"},
    {32, 32, 1024, 1.56f, 2.03f, 0.1f, 1.2f, 1, 1.2f, 1.f, launch_split<2, 2, 16, 2>, "gemm_i8_32x32"},
    {64, 64, 1024, 1.97f, 3.82f, 0.4f, 0.75f, 1, 0.75f, 0.66f, launch_tile<64, 64, 4, 4, 256, true>, "gemm_i8_64x64"},
    {64, 64, 512, 1.15f, 5.44f, 0.4f, 0.49f, 1, 0.49f, 0.23f, launch_tile<64, 64, 4, 2, 128, true>, "gemm_i8_64x64"},
    {128, 128, 1024, 2.2f, 7.99f, 1.9f, 1.2f, 1, 1.2f, 1.f, launch_tile<128, 128, 4, 4, 128, true>, "gemm_i8_128x128"},
    {192, 128, 512, 4.9f, 9.5f, 2.8f, 1.2f, 1, 1.2f, 1.f, launch_tile<192, 128, 4, 2, 128, true>, "gemm_i8_192x128"},
    {256, 128, 1024, 3.65f, 11.08f, 3.8f, 1.2f, 1, 1.2f, 1.f, launch_tile<256, 128, 4, 4, 128, true>, "gemm_i8_256x128"},
};

}  // namespace
}  // namespace i8

int launch_gemm_i8(const GemmI8Args& a, hipStream_t s) {
    using namespace i8;
    if (((!a.x || !a.w) && a.k) || !a.sx || !a.sw || !a.y || a.m < 0 || a.n < 0 || a.k < 0) return K_EINVAL;
    if (a.act < ACT_NONE || a.act > ACT_SIGMOID) return K_EINVAL;
    if (a.k > kGemmI8MaxK) return K_EUNSUPPORTED;
    if (a.m == 0 || a.n == 0) return K_OK;
    const Fetch how = fetch_of(a);
    const Tile *table = how == DIRECT ? kDirect : kThroughRegisters, *best = nullptr;
    const int count = how == DIRECT ? (int)(sizeof(kDirect) / sizeof(Tile)) : (int)(sizeof(kThroughRegisters) / sizeof(Tile));
    const bool act = a.act != ACT_NONE && a.act != ACT_RELU && a.act != ACT_RELU6;
    float least = 0.f;
    long grid = 0;
    for (int k = 0; k < count; ++k) {
        const Tile& t = table[k];
        const long tiles = (((long)a.m + t.m - 1) / t.m) * (((long)a.n + t.n - 1) / t.n);
        if (tiles * t.threads > 0xffffffffl) continue;  // the grid's threads have to fit 32 bits
        const int cus = num_cu();
        const float full = (float)((tiles + cus - 1) / cus), part = tiles > cus ? (float)tiles / (float)cus : 1.f;
        const float rounds = t.last * full + (1.f - t.last) * part;
        const float tile = t.first + t.codes * (float)a.k / 1024.f + (act ? t.act : 0.f);
        const float work = tile * (1.f + t.more * (fminf(rounds, (float)t.held) - 1.f) + t.next * fmaxf(rounds - (float)t.held, 0.f));
        if (!best || work < least) best = &t, least = work, grid = tiles;
    }
    if (!best) return K_EUNSUPPORTED;
    best->launch(a, how, (unsigned)grid, s);
    set_last_kernel(best->name);
    return (int)hipGetLastError();
}

}  // namespace tpk

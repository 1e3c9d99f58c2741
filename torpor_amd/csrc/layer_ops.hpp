// Argument lists of the 8-bit encoder-layer operators (TP_OP_QUANT_ROWS, TP_OP_GEMM_I8, TP_OP_NORM_BLOCK): checked,
// turned into operand rectangles and into the kernels' arguments.  Shared by the engine, which knows virtual addresses
// and how large every block is, and by the entry point on raw addresses.  Host logic only.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/torpor_amd.h"
#include "kernels/kernels.hpp"

namespace tp {

// `rows` rows of `width` elements, `pitch` elements apart.
struct Operand {
    int slot = 0;       // index in the pointer list
    uint64_t addr = 0;  // 0: not given
    int64_t rows = 1, width = 0, pitch = 0;
    int elem = 4;  // bytes of an element
    bool output = false;
    bool in_place = false;  // output: may be an operand marked `reused`;  input: `reused`

    __int128 span() const { return (__int128)(rows - 1) * pitch + width; }  // elements from first to last
};

struct Operands {
    Operand v[12];
    int n = 0;
    bool empty = false;  // no rows: the call does nothing
};

// Whether two operands share a byte.  Rows of one pitch whose columns lie side by side (slices of one wider tensor) do not.
inline bool share_bytes(const Operand& a, const Operand& b) {
    const __int128 a0 = a.addr, a1 = a0 + a.span() * a.elem, b0 = b.addr, b1 = b0 + b.span() * b.elem;
    if (a1 <= b0 || b1 <= a0) return false;
    const __int128 pitch = (__int128)a.pitch * a.elem;
    if (a.rows == 1 || b.rows == 1 || pitch != (__int128)b.pitch * b.elem) return true;
    const __int128 d = (((b0 - a0) % pitch) + pitch) % pitch;  // where b's columns start in a's row
    return d < (__int128)a.width * a.elem || d + (__int128)b.width * b.elem > pitch;
}

// Checks an argument list and lists its operands.  `p` may be virtual or raw addresses.
inline int layer_op_operands(int op_id, const uint64_t* p, int np, const int64_t* i, int ni, int nf, Operands* out) {
    constexpr int64_t kIntMax = 0x7fffffff, kLongMax = ((int64_t)1 << 46) - 1;
    auto P = [&](int k) { return k < np ? p[k] : (uint64_t)0; };
    auto I = [&](int k) { return k < ni ? i[k] : (int64_t)0; };
    auto pitch = [&](int k, int64_t dense) { return I(k) ? I(k) : dense; };
    bool ok = true;
    // one operand of the list; `rows` rows at least `width` apart
    auto add = [&](int slot, bool optional, int64_t rows, int64_t width, int64_t ld, int elem, bool output, bool in_place) {
        if (rows > 1 && ld < width) ok = false;
        if (!P(slot)) {  // an operand without elements has no address
            if (!optional && !out->empty && width > 0) ok = false;
            return;
        }
        if (P(slot) % (uint64_t)elem) ok = false;
        Operand& o = out->v[out->n++];
        o.slot = slot;
        o.addr = P(slot);
        o.rows = rows;
        o.width = width;
        o.pitch = ld;
        o.elem = elem;
        o.output = output;
        o.in_place = in_place;
    };
    for (int k = 0; k < ni; ++k)
        if (i[k] < 0 || i[k] > kLongMax) return TP_EINVAL;
    out->n = 0;
    out->empty = false;
    switch (op_id) {
        case TP_OP_QUANT_ROWS: {
            if (np < 3 || ni < 2) return TP_EINVAL;
            const int64_t rows = I(0), width = I(1);
            if (width < 1) return TP_EINVAL;
            if (width > tpk::kRowOpMaxWidth) return TP_EUNSUPPORTED;
            out->empty = rows == 0;
            const int64_t r = rows ? rows : 1;
            add(0, false, r, width, pitch(2, width), 4, false, false);
            add(1, false, r, width, pitch(3, width), 1, true, false);
            add(2, false, 1, r, r, 4, true, false);
            break;
        }
        case TP_OP_GEMM_I8: {
            if (np < 5 || ni < 3) return TP_EINVAL;
            const int64_t m = I(0), n = I(1), k = I(2);
            if (m > kIntMax || n > kIntMax || k > kIntMax || I(7) > TP_ACT_SIGMOID) return TP_EINVAL;
            if (k > tpk::kGemmI8MaxK) return TP_EUNSUPPORTED;
            out->empty = m == 0 || n == 0;
            const int64_t M = m ? m : 1, N = n ? n : 1;
            add(0, false, M, k, pitch(3, k), 1, false, false);
            add(1, false, 1, M, M, 4, false, false);
            add(2, false, N, k, pitch(4, k), 1, false, false);
            add(3, false, 1, N, N, 4, false, false);
            add(4, false, M, N, pitch(5, N), 4, true, true);
            add(5, true, 1, N, N, 4, false, false);
            add(6, true, M, N, pitch(6, N), 4, false, true);
            break;
        }
        case TP_OP_NORM_BLOCK: {
            if (np < 9 || ni < 4 || nf < 4) return TP_EINVAL;
            const int64_t rows = I(0), width = I(1), group = I(4);
            if (width < 1 || I(2) > 2 || I(3) > 2) return TP_EINVAL;
            if (width > tpk::kRowOpMaxWidth) return TP_EUNSUPPORTED;
            // a norm has its gamma, no norm has neither vector
            if ((I(2) != 0) != (P(3) != 0) || (!I(2) && P(4)) || (I(3) != 0) != (P(5) != 0) || (!I(3) && P(6))) return TP_EINVAL;
            out->empty = rows == 0;
            if ((P(9) != 0) != (P(10) != 0) || (!P(7) && !P(8) && !P(9) && rows)) return TP_EINVAL;
            const int64_t r = rows ? rows : 1;
            add(0, false, r, width, pitch(5, width), 4, false, true);
            add(1, true, r, width, pitch(6, width), 4, false, true);
            add(2, true, group ? (r - 1) / group + 1 : 1, width, width, 4, false, false);
            for (int k = 3; k < 7; ++k) add(k, true, 1, width, width, 4, false, false);
            add(7, true, r, width, pitch(7, width), 4, true, true);
            add(8, true, r, width, pitch(8, width), 4, true, true);
            add(9, true, r, width, pitch(9, width), 1, true, false);
            add(10, true, 1, r, r, 4, true, false);
            break;
        }
        default:
            return TP_EUNSUPPORTED;
    }
    if (!ok) return TP_EINVAL;
    for (int a = 0; a < out->n; ++a) {
        const Operand& o = out->v[a];
        if (o.span() * o.elem > (__int128)kLongMax) return TP_EFAULT;  // no memory is that large
    }
    return TP_OK;
}

// Whether an output lies over another operand in a way that the kernels do not allow.
inline bool layer_op_overlap(const Operands& list) {
    if (list.empty) return false;
    for (int a = 0; a < list.n; ++a) {
        const Operand& o = list.v[a];
        if (!o.output) continue;
        for (int b = 0; b < list.n; ++b) {
            const Operand& u = list.v[b];
            if (a == b || u.width == 0) continue;
            const bool same = o.in_place && u.in_place && !u.output && o.addr == u.addr && (o.pitch == u.pitch || o.rows == 1);
            if (!same && share_bytes(o, u)) return true;
        }
    }
    return false;
}

// Launches a checked call; q[slot] are device addresses.
inline int layer_op_launch(int op_id, void* const* q, const int64_t* i, int ni, const float* f, hipStream_t s) {
    auto I = [&](int k) { return k < ni ? i[k] : (int64_t)0; };
    auto pitch = [&](int k, int64_t dense) { return (long)(I(k) ? I(k) : dense); };
    auto F = [&](int k) { return static_cast<const float*>(q[k]); };
    auto Fm = [&](int k) { return static_cast<float*>(q[k]); };
    switch (op_id) {
        case TP_OP_QUANT_ROWS: {
            tpk::QuantRowsArgs a;
            a.x = F(0);
            a.q = static_cast<int8_t*>(q[1]);
            a.scale = Fm(2);
            a.rows = (long)I(0);
            a.width = (int)I(1);
            a.ldx = pitch(2, a.width);
            a.ldq = pitch(3, a.width);
            return tpk::launch_quant_rows(a, s);
        }
        case TP_OP_GEMM_I8: {
            tpk::GemmI8Args a;
            a.x = static_cast<const int8_t*>(q[0]);
            a.sx = F(1);
            a.w = static_cast<const int8_t*>(q[2]);
            a.sw = F(3);
            a.y = Fm(4);
            a.bias = F(5);
            a.residual = F(6);
            a.m = (int)I(0);
            a.n = (int)I(1);
            a.k = (int)I(2);
            a.ldx = pitch(3, a.k);
            a.ldw = pitch(4, a.k);
            a.ldy = pitch(5, a.n);
            a.ldr = pitch(6, a.n);
            a.act = (int)I(7);
            return tpk::launch_gemm_i8(a, s);
        }
        case TP_OP_NORM_BLOCK: {
            tpk::NormBlockArgs a;
            a.x = F(0);
            a.residual = F(1);
            a.gate = F(2);
            a.post_gamma = F(3);
            a.post_beta = F(4);
            a.pre_gamma = F(5);
            a.pre_beta = F(6);
            a.h = Fm(7);
            a.y = Fm(8);
            a.q = static_cast<int8_t*>(q[9]);
            a.scale = Fm(10);
            a.rows = (long)I(0);
            a.width = (int)I(1);
            a.post = (int)I(2);
            a.pre = (int)I(3);
            a.rows_per_gate = (long)I(4);
            a.ldx = pitch(5, a.width);
            a.ldr = pitch(6, a.width);
            a.ldh = pitch(7, a.width);
            a.ldy = pitch(8, a.width);
            a.ldq = pitch(9, a.width);
            a.residual_scale = a.residual ? f[0] : 0.f;  // not given: no term, whatever its scale
            a.block_scale = f[1];
            a.post_eps = f[2];
            a.pre_eps = f[3];
            return tpk::launch_norm_block(a, s);
        }
        default:
            return TP_EUNSUPPORTED;
    }
}

}  // namespace tp

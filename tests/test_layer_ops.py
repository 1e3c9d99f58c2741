"""The 8-bit encoder-layer operators without a GPU: what their argument checks take and refuse (through a host-only engine
and through the entry point on raw addresses, which refuses before it touches the device), and the oracle's forms against
closed forms and torch."""
import numpy as np
import pytest
import torch

from oracle import ops as ref
from torpor_amd.server import (ACK_OK, NORM_LAYER, NORM_NONE, NORM_RMS, OP_GEMM_I8, OP_NORM_BLOCK, OP_QUANT_ROWS, OP_RELU,
                               REQ_EXECUTE_AFTER_LOAD, Server, TorporError, launch_noalloc)

EINVAL, EUNSUPPORTED, EFAULT = -22, -38, -14
BASE = 1 << 40      # raw addresses that no refused call reads


def A(mib, off=0):
    return BASE + (mib << 20) + off


@pytest.fixture(scope="module")
def host_server():
    with Server(host_only=True, mem_limit_bytes=256 << 20, pool_bytes=512 << 20) as s:
        yield s


# ------------------------------------------------------------------------------- refusals, raw addresses
QUANT_REFUSED = [
    ("no list", [], [], EINVAL),
    ("two pointers", [A(0), A(1)], [4, 8], EINVAL),
    ("no width", [A(0), A(1), A(2)], [4], EINVAL),
    ("width 0", [A(0), A(1), A(2)], [4, 0], EINVAL),
    ("rows below 0", [A(0), A(1), A(2)], [-1, 8], EINVAL),
    ("null x", [0, A(1), A(2)], [4, 8], EINVAL),
    ("null codes", [A(0), 0, A(2)], [4, 8], EINVAL),
    ("null scale", [A(0), A(1), 0], [4, 8], EINVAL),
    ("pitch of x below the width", [A(0), A(1), A(2)], [4, 8, 7, 8], EINVAL),
    ("pitch of the codes below the width", [A(0), A(1), A(2)], [4, 8, 8, 7], EINVAL),
    ("a float at an odd address", [A(0, 2), A(1), A(2)], [4, 8], EINVAL),
    ("a row too long", [A(0), A(1), A(2)], [4, 65537], EUNSUPPORTED),
    ("a size that wraps", [A(0), A(1), A(2)], [(1 << 46) - 1, 8], EFAULT),
    ("a number above every address", [A(0), A(1), A(2)], [1 << 60, 8], EINVAL),
    ("codes over x", [A(0), A(0), A(2)], [4, 8], EINVAL),
    ("scales inside the codes", [A(0), A(1), A(1, 8)], [4, 8], EINVAL),
]
GEMM = [A(0), A(1), A(2), A(3), A(4), A(5), A(6)]
GEMM_REFUSED = [
    ("four pointers", GEMM[:4], [4, 8, 16], EINVAL),
    ("two sizes", GEMM, [4, 8], EINVAL),
    ("null scale", [A(0), 0] + GEMM[2:], [4, 8, 16], EINVAL),
    ("null output", GEMM[:4] + [0, 0, 0], [4, 8, 16], EINVAL),
    ("m below 0", GEMM, [-4, 8, 16], EINVAL),
    ("m above int", GEMM, [1 << 31, 8, 16], EINVAL),
    ("k whose sum could leave 32 bits", GEMM, [4, 8, 131072], EUNSUPPORTED),
    ("pitch of x below k", GEMM, [4, 8, 16, 15], EINVAL),
    ("pitch of w below k", GEMM, [4, 8, 16, 16, 15], EINVAL),
    ("pitch of y below n", GEMM, [4, 8, 16, 16, 16, 7], EINVAL),
    ("pitch of the residual below n", GEMM, [4, 8, 16, 16, 16, 8, 7], EINVAL),
    ("unknown activation", GEMM, [4, 8, 16, 16, 16, 8, 8, 7], EINVAL),
    ("y over w", [A(0), A(1), A(2), A(3), A(2), 0, 0], [4, 8, 16], EINVAL),
    ("y over the bias", [A(0), A(1), A(2), A(3), A(4), A(4, 64), 0], [4, 8, 16], EINVAL),
    ("y one row behind the residual", [A(0), A(1), A(2), A(3), A(4), 0, A(4, 32)], [4, 8, 16], EINVAL),
    ("y over a residual of another pitch", [A(0), A(1), A(2), A(3), A(4), 0, A(4)], [4, 8, 16, 0, 0, 8, 9], EINVAL),
    ("bias at an odd address", [A(0), A(1), A(2), A(3), A(4), A(5, 1), 0], [4, 8, 16], EINVAL),
]
NORM = [A(0), A(1), A(2), A(3), A(4), A(5), A(6), A(7), A(8), A(9), A(10)]


def _norm(**at):
    return [at.get(str(i), at.get("p%d" % i, v)) for i, v in enumerate(NORM)]


BOTH = [4, 8, NORM_RMS, NORM_LAYER]
NORM_REFUSED = [
    ("eight pointers", NORM[:8], BOTH, EINVAL),
    ("three sizes", NORM, BOTH[:3], EINVAL),
    ("unknown norm", NORM, [4, 8, 3, 1], EINVAL),
    ("norm without gamma", _norm(p5=0), BOTH, EINVAL),
    ("gamma without norm", NORM, [4, 8, NORM_NONE, NORM_LAYER], EINVAL),
    ("beta without norm", _norm(p3=0), [4, 8, NORM_NONE, NORM_LAYER], EINVAL),
    ("codes without scale", _norm(p10=0), BOTH, EINVAL),
    ("scale without codes", _norm(p9=0), BOTH, EINVAL),
    ("no output", _norm(p7=0, p8=0, p9=0, p10=0), BOTH, EINVAL),
    ("a row too long", NORM, [4, 65537, 2, 1], EUNSUPPORTED),
    ("pitch below the width", NORM, BOTH + [0, 7], EINVAL),
    ("codes' pitch below the width", NORM, BOTH + [0, 0, 0, 0, 0, 7], EINVAL),
    ("h and y in one place", _norm(p8=NORM[7]), BOTH, EINVAL),
    ("codes over x", _norm(p9=NORM[0]), BOTH, EINVAL),
    ("y over gamma", _norm(p8=NORM[5]), BOTH, EINVAL),
    ("y over the gate", _norm(p8=NORM[2]), BOTH, EINVAL),
    ("y in x's place at another pitch", _norm(p8=NORM[0]), BOTH + [0, 8, 0, 0, 9], EINVAL),
    ("h one element into x", _norm(p7=NORM[0] + 4), BOTH, EINVAL),
    ("null x", _norm(p0=0), BOTH, EINVAL),
]


@pytest.mark.parametrize("op,case", [(OP_QUANT_ROWS, c) for c in QUANT_REFUSED] + [(OP_GEMM_I8, c) for c in GEMM_REFUSED] +
                         [(OP_NORM_BLOCK, c) for c in NORM_REFUSED], ids=lambda v: v[0] if isinstance(v, tuple) else str(v))
def test_refusals_on_raw_addresses(op, case):
    _, ptrs, ints, code = case
    assert launch_noalloc(op, ptrs, ints, [1.0, 1.0, 1e-5, 1e-5] if op == OP_NORM_BLOCK else ()) == code


def test_raw_entry_point_refuses_other_operators_and_missing_floats():
    assert launch_noalloc(OP_RELU, [A(0), A(1)], [4]) == EUNSUPPORTED
    assert launch_noalloc(0, [], []) == EUNSUPPORTED
    assert launch_noalloc(OP_NORM_BLOCK, NORM, BOTH, [1.0, 1.0, 1e-5]) == EINVAL
    assert launch_noalloc(OP_QUANT_ROWS, [A(0)] * 13, [4, 8]) == EINVAL
    assert launch_noalloc(OP_QUANT_ROWS, [A(0), A(1), A(2)], [4] * 21) == EINVAL


def test_calls_without_rows_do_nothing():
    assert launch_noalloc(OP_QUANT_ROWS, [A(0), A(1), A(2)], [0, 8]) == 0
    assert launch_noalloc(OP_GEMM_I8, GEMM, [0, 8, 16]) == 0
    assert launch_noalloc(OP_GEMM_I8, GEMM, [4, 0, 16]) == 0
    assert launch_noalloc(OP_NORM_BLOCK, NORM, [0, 8, 2, 1], [1.0, 1.0, 1e-5, 1e-5]) == 0


# ------------------------------------------------------------------------------- through an engine without a device
def test_engine_checks_spans_and_overlap(host_server):
    s, f = host_server, 30
    assert s.signal(REQ_EXECUTE_AFTER_LOAD, f, "1")[0] == ACK_OK
    w, sw = s.malloc(f, 32 * 64), s.malloc(f, 32 * 4)
    s.h2d(f, w, np.zeros((32, 64), np.int8))
    s.h2d(f, sw, np.zeros(32, np.float32))
    s.device_synchronize(f)
    x, q, sc = s.malloc(f, 8 * 64 * 4), s.malloc(f, 8 * 64), s.malloc(f, 8 * 4)
    y = s.malloc(f, 8 * 32 * 4)
    wide = s.malloc(f, 8 * 128 * 4)

    def refused(op, ptrs, ints, floats=(), codes=(EINVAL,)):
        with pytest.raises(TorporError) as e:
            s.launch(f, op, ptrs, ints, floats)
        assert e.value.code in codes, e.value.code

    s.launch(f, OP_QUANT_ROWS, [x, q, sc], [8, 64])
    s.launch(f, OP_QUANT_ROWS, [x, q, sc], [0, 64])
    s.launch(f, OP_QUANT_ROWS, [wide + 4 * 64, q, sc], [8, 64, 128])   # the right half of a wider tensor: ends with it
    refused(OP_QUANT_ROWS, [x, q, sc], [9, 64], codes=(EFAULT,))
    refused(OP_QUANT_ROWS, [x, q, sc], [8, 65], codes=(EFAULT,))
    refused(OP_QUANT_ROWS, [wide + 4 * 65, q, sc], [8, 64, 128], codes=(EFAULT,))
    refused(OP_QUANT_ROWS, [x, x, sc], [8, 64])
    s.launch(f, OP_GEMM_I8, [q, sc, w, sw, y], [8, 32, 64])
    s.launch(f, OP_GEMM_I8, [q, sc, w, sw, y, sw, y], [8, 32, 64, 0, 0, 0, 0, 2])   # into its residual
    refused(OP_GEMM_I8, [q, sc, w, sw, y], [9, 32, 64], codes=(EFAULT,))
    refused(OP_GEMM_I8, [q, sc, w, sw, y], [8, 33, 64], codes=(EFAULT,))
    refused(OP_GEMM_I8, [q, sc, w, sw, y], [8, 32, 65], codes=(EFAULT,))
    refused(OP_GEMM_I8, [q, sc, w, sw, y, 0, y + 4], [7, 32, 64])
    # one tensor's left half is the residual, its right half the output: side by side, not over each other
    s.launch(f, OP_GEMM_I8, [q, sc, w, sw, wide, 0, wide + 4 * 32], [8, 32, 64, 0, 0, 128, 128])
    refused(OP_GEMM_I8, [q, sc, w, sw, wide, 0, wide + 4 * 31], [8, 32, 64, 0, 0, 128, 128])
    g = s.malloc(f, 64 * 4)
    h = s.malloc(f, 8 * 64 * 4)
    fl = [1.0, 1.0, 1e-5, 1e-5]
    s.launch(f, OP_NORM_BLOCK, [x, h, 0, 0, 0, g, 0, h, x], [8, 64, 0, 2], fl)     # h into the residual, y into x
    s.launch(f, OP_NORM_BLOCK, [x, 0, g, 0, 0, 0, 0, 0, 0, q, sc], [8, 64, 0, 0], fl)
    refused(OP_NORM_BLOCK, [x, 0, g, 0, 0, 0, 0, 0, 0, q, sc], [8, 64, 0, 0, 4], fl, codes=(EFAULT,))   # two gate rows
    refused(OP_NORM_BLOCK, [x, h, 0, 0, 0, g, 0, h, h], [8, 64, 0, 2], fl)
    with pytest.raises(TorporError):
        s.stream_synchronize(f)     # refused ops are reported once more at the next sync


# ------------------------------------------------------------------------------- the oracle's forms
def test_oracle_quant_rows_by_hand():
    x = np.array([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5], [0, 0, 0, 0, 0, 0], [1e-44, 0, -1e-44, 0, 0, 0],
                  [np.inf, 1, 2, 3, 4, 5], [np.nan, 1, 2, 3, 4, 5], [-254, 1, 3, 5, 253, 254]], np.float32)
    q, s = ref.quant_rows(x)
    np.testing.assert_array_equal(s, np.array([1, 2.0 ** -126, 2.0 ** -126, np.nan, np.nan, 2], np.float32))
    np.testing.assert_array_equal(q, [[127, 0, 2, 2, 0, -2], [0] * 6, [0] * 6, [0] * 6, [0] * 6, [-127, 0, 2, 2, 126, 127]])


def test_oracle_gemm_and_norm_against_torch():
    rng = np.random.default_rng(0)
    xq, wq = rng.integers(-127, 128, (5, 33)), rng.integers(-127, 128, (7, 33))
    sx, sw = rng.random(5).astype(np.float32), rng.random(7).astype(np.float32)
    b, r = rng.standard_normal(7), rng.standard_normal((5, 7))
    y, _ = ref.gemm_i8(xq, sx, wq, sw, b, r, "gelu")
    t = torch.from_numpy(xq * sx[:, None].astype(np.float64)) @ torch.from_numpy(wq * sw[:, None].astype(np.float64)).T
    want = torch.nn.functional.gelu(t + torch.from_numpy(b) + torch.from_numpy(r))
    np.testing.assert_allclose(y, want.numpy(), rtol=1e-12, atol=1e-14)
    x = rng.standard_normal((6, 20)).astype(np.float32)
    g, be = rng.standard_normal(20).astype(np.float32), rng.standard_normal(20).astype(np.float32)
    h, y = ref.norm_block(x, pre=("layer", g, be, 1e-5))
    np.testing.assert_array_equal(h, x.astype(np.float64))
    want = torch.nn.functional.layer_norm(torch.from_numpy(x).double(), (20,), torch.from_numpy(g).double(),
                                          torch.from_numpy(be).double(), 1e-5)
    np.testing.assert_allclose(y, want.numpy(), rtol=1e-12, atol=1e-13)
    res, gate = rng.standard_normal((6, 20)), rng.standard_normal((2, 20))
    h, _ = ref.norm_block(x, res, gate, 4, post=("rms", g, None, 1e-6), a=0.5, b=2.0)
    rms = torch.nn.functional.rms_norm(torch.from_numpy(x).double(), (20,), torch.from_numpy(g).double(), 1e-6).numpy()
    np.testing.assert_allclose(h, 0.5 * res + 2.0 * gate[[0, 0, 0, 0, 1, 1]] * rms, rtol=1e-12, atol=1e-13)


# ------------------------------------------------------------------------------- the served encoder's weights
def test_quantize_rows_agrees_with_the_operators_definition():
    from torpor_amd.functions.base import quantize_rows

    rng = np.random.default_rng(1)
    w = (rng.standard_normal((40, 33)) * np.exp(rng.standard_normal((40, 1)) * 4)).astype(np.float32)
    w[0] = 0
    w[1] = np.float32(1e-44)
    w[2, :] = np.arange(33) - 16.5      # halves of the scale below
    w[2, 0] = 127
    for got, want in zip(quantize_rows(w), ref.quant_rows(w)):
        np.testing.assert_array_equal(got, want)
    w[3, 5] = np.nan
    with pytest.raises(ValueError):
        quantize_rows(w)


def test_quantized_bert_uploads_codes_and_scales_for_the_encoder_only():
    from torpor_amd.functions import bert

    cfg = dict(layers=2, hidden=75, heads=3, ffn=50)
    weights = bert.init_weights(seed=3, vocab=40, max_pos=16, cfg=cfg)
    plain = bert.Bert(None, 1, weights=weights, cfg=cfg).weights()
    mixed = bert.Bert(None, 1, weights=weights, cfg=cfg, quantized=True).weights()
    matrices = [k for k in plain if k.startswith("encoder.") and plain[k].ndim == 2]
    assert len(matrices) == 8 and set(mixed) == set(plain) | {k + "_scale" for k in matrices}
    for k, v in plain.items():
        if k in matrices:
            assert mixed[k].dtype == np.int8 and mixed[k].shape == v.shape and mixed[k + "_scale"].shape == v.shape[:1]
            # half a step of a channel's scale at most (the scale itself is rounded: 1 + 2^-23 covers it)
            assert (np.abs(mixed[k] * mixed[k + "_scale"][:, None].astype(np.float64) - v) <=
                    mixed[k + "_scale"][:, None] * 0.5 * (1 + 2.0 ** -16)).all()
        else:
            np.testing.assert_array_equal(mixed[k], v)


# ------------------------------------------------------------------------------- the compiled kernels
def _kernels_of(library, tmp_path):
    """{mangled name: (bytes of scratch memory a lane, registers spilled)} of every gfx950 kernel in a library that was built here: the
    code objects lie in bundles, each a list of (offset, size, target) behind its magic number."""
    import os
    import re
    import struct
    import subprocess

    readelf = "/opt/rocm/llvm/bin/llvm-readelf"
    if not os.path.exists(readelf):
        pytest.skip("llvm-readelf not installed")
    blob, found = open(library, "rb").read(), {}
    for m in re.finditer(b"__CLANG_OFFLOAD_BUNDLE__", blob):
        at = m.start()
        (count,), pos = struct.unpack_from("<Q", blob, at + 24), at + 32
        for _ in range(count):
            off, size, n = struct.unpack_from("<QQQ", blob, pos)
            target = blob[pos + 24:pos + 24 + n]
            pos += 24 + n
            if b"gfx950" not in target or not size:
                continue
            elf = tmp_path / "code.o"
            elf.write_bytes(blob[at + off:at + off + size])
            notes = subprocess.run([readelf, "--notes", str(elf)], capture_output=True, text=True, check=True).stdout
            for part in notes.split("- .agpr_count:")[1:]:
                get = {k: v for k, v in re.findall(r"\.(name|private_segment_fixed_size|vgpr_spill_count|sgpr_spill_count): +(\S+)", part)
                       if k != "name" or v.startswith("_Z")}
                found[get["name"]] = (int(get["private_segment_fixed_size"]), int(get["vgpr_spill_count"]))
    return found


def test_the_operators_kernels_use_no_scratch_memory(tmp_path):
    """What tp_launch_noalloc promises: nothing of a row is spilled, or the runtime would have to provide memory for it."""
    from torpor_amd import _lib

    kernels = {k: v for k, v in _kernels_of(_lib.LIB_PATH, tmp_path).items()
               if any(n in k for n in ("quant_rows_kernel", "norm_block_kernel", "gemm_i8_"))}
    assert sum("norm_block" in k for k in kernels) >= 40 and sum("gemm_i8" in k for k in kernels) >= 15 and \
        sum("quant_rows" in k for k in kernels) >= 10
    bad = {k: v for k, v in kernels.items() if v != (0, 0)}
    assert not bad, bad


# ------------------------------------------------------------------------------- operands without elements
EMPTY_CALLS = [(OP_QUANT_ROWS, 3, [0, 8], ()), (OP_GEMM_I8, 7, [0, 8, 16], ()), (OP_GEMM_I8, 7, [4, 0, 16], ()), (OP_GEMM_I8, 5, [0, 0, 0], ())]
FL = [1.0, 1.0, 1e-5, 1e-5]


def test_calls_without_rows_need_no_addresses():
    """An empty tensor has no address (torch's data_ptr() is 0): the call does nothing all the same."""
    f = 31
    with Server(host_only=True, mem_limit_bytes=256 << 20, pool_bytes=512 << 20) as s:
        assert s.signal(REQ_EXECUTE_AFTER_LOAD, f, "1")[0] == ACK_OK
        g = s.malloc(f, 64)
        s.h2d(f, g, np.zeros(16, np.float32))
        s.device_synchronize(f)
        for op, np_, ints, floats in EMPTY_CALLS:
            assert launch_noalloc(op, [0] * np_, ints, floats) == 0, (op, ints)
            s.launch(f, op, [0] * np_, ints, floats)
        for run in (lambda *a: launch_noalloc(OP_NORM_BLOCK, *a), lambda *a: s.launch(f, OP_NORM_BLOCK, *a) or 0):
            assert run([0, 0, 0, 0, 0, g, 0, 0, 0, 0, 0], [0, 8, NORM_NONE, NORM_RMS], FL) == 0
            assert run([0, 0, 0, 0, 0, 0, 0, 0, 0], [0, 8, NORM_NONE, NORM_NONE], FL) == 0
    # with rows every address is needed, and what else is wrong stays wrong without rows
    assert launch_noalloc(OP_GEMM_I8, [0] * 5, [4, 8, 0]) == EINVAL          # k = 0: scales and output have elements
    assert launch_noalloc(OP_GEMM_I8, [0, A(1), 0, A(3), A(4)], [4, 8, 1]) == EINVAL
    assert launch_noalloc(OP_QUANT_ROWS, [0] * 3, [0, 65537]) == EUNSUPPORTED
    assert launch_noalloc(OP_QUANT_ROWS, [0] * 3, [1, 8]) == EINVAL
    assert launch_noalloc(OP_NORM_BLOCK, [A(0)] + [0] * 8, [4, 8, 0, 0], FL) == EINVAL
    assert launch_noalloc(OP_NORM_BLOCK, [0] * 9, [0, 8, NORM_NONE, NORM_RMS], FL) == EINVAL      # a norm has its gamma

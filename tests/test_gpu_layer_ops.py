"""The 8-bit encoder-layer operators (OP_QUANT_ROWS, OP_GEMM_I8, OP_NORM_BLOCK) on the GPU against their float64 forms, on raw
addresses and through the engine.

Tolerances.  U = 2^-24 is the largest relative rounding error of a float32 operation.  Codes and scales have a definition
without slack and are equal.  The product's integer sum is exact; rounding it to float, two scalings and up to two additions
cost at most 3U|p| + U|p + bias| + U|p + bias + residual|.  The norms are worked out in float64 and rounded once: U of the
value, and 1e-13 of the largest terms for the float64 arithmetic itself (rows of up to 65536 terms, 53 bits)."""
import numpy as np
import pytest
import torch  # before anything initialises the system's HIP runtime: see tests/conftest.py

from oracle import ops as ref
from tests.harness import OpSession
from torpor_amd.server import (ACT_GELU, ACT_NONE, ACT_RELU, ACT_RELU6, ACT_SIGMOID, ACT_SILU, ACT_TANH, NORM_LAYER, NORM_NONE,
                               NORM_RMS, OP_GEMM_I8, OP_NORM_BLOCK, OP_QUANT_ROWS, launch_noalloc)

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = {"none": ACT_NONE, "relu": ACT_RELU, "gelu": ACT_GELU, "tanh": ACT_TANH, "relu6": ACT_RELU6, "silu": ACT_SILU,
        "sigmoid": ACT_SIGMOID}
NORMS = {None: NORM_NONE, "layer": NORM_LAYER, "rms": NORM_RMS}


def _launch(op, ptrs, ints, floats=(), stream=None):
    s = torch.cuda.current_stream() if stream is None else stream
    r = launch_noalloc(op, ptrs, ints, floats, stream=s.cuda_stream)
    assert r == 0, r


def _dev(a, pitch=None, shift=0):
    """`a` [rows, width] on the GPU with rows `pitch` elements apart, `shift` elements into an allocation, marker values between and
    behind the rows.  Returns (base tensor, address of the first element)."""
    a = np.ascontiguousarray(a)
    rows, width = a.shape
    pitch = pitch or width
    base = np.full(shift + rows * pitch + 64, 77, a.dtype)
    view = base[shift:shift + rows * pitch].reshape(rows, pitch)
    view[:, :width] = a
    t = torch.from_numpy(base).cuda()
    return t, t.data_ptr() + shift * a.itemsize


def _back(t, rows, width, pitch=None, shift=0):
    """The [rows, width] values of a buffer laid out by _dev, after checking that the markers around them are untouched."""
    pitch = pitch or width
    host = t.cpu().numpy()
    view = host[shift:shift + rows * pitch].reshape(rows, pitch)
    assert (host[:shift] == 77).all() and (host[shift + rows * pitch:] == 77).all() and (view[:, width:] == 77).all()
    return np.ascontiguousarray(view[:, :width])


# ------------------------------------------------------------------------------- quantisation
def _quant(x, px=None, pq=None, sx=0, sq=0):
    rows, width = x.shape
    _keep, xp = _dev(x, px, sx)
    q, qp = _dev(np.full((rows, width), 77, np.int8), pq, sq)
    s, sp = _dev(np.full((1, rows), 77, np.float32))
    _launch(OP_QUANT_ROWS, [xp, qp, sp], [rows, width, px or width, pq or width])
    torch.cuda.synchronize()
    return _back(q, rows, width, pq, sq), _back(s, 1, rows)[0]


@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (5, 3), (2, 63), (7, 64), (4, 65), (9, 255), (1, 256), (6, 257), (33, 768),
                                        (16, 1021), (5, 1024), (5, 1025), (3, 4095), (2, 4096), (2, 4097), (2, 16384), (2, 16385),
                                        (1, 65535), (2, 65536), (5000, 40)])
def test_quant_rows(rows, width):
    rng = np.random.default_rng(rows * 7 + width)
    x = (rng.standard_normal((rows, width)) * np.exp(rng.standard_normal((rows, 1)) * 3)).astype(np.float32)
    q, s = _quant(x)
    wq, ws = ref.quant_rows(x)
    np.testing.assert_array_equal(s, ws)
    np.testing.assert_array_equal(q, wq)


@pytest.mark.parametrize("px,pq,sx,sq", [(130, 128, 0, 0), (128, 131, 1, 3), (129, 133, 3, 1), (140, 144, 2, 2)])
def test_quant_rows_pitches_and_odd_addresses(px, pq, sx, sq):
    x = np.random.default_rng(px).standard_normal((11, 127)).astype(np.float32)
    q, s = _quant(x, px, pq, sx, sq)
    wq, ws = ref.quant_rows(x)
    np.testing.assert_array_equal(s, ws)
    np.testing.assert_array_equal(q, wq)


@pytest.mark.parametrize("width", [6, 1021, 5000])
def test_quant_rows_borders_and_special_rows(width):
    """Halves, values one step beside a half, zeros, denormals, the largest floats, an infinity and NaNs in one place of a row."""
    rng = np.random.default_rng(width)
    rows = []
    for s in (1.0, 0.7, 3e-37, 1e30, 2.0 ** -126):
        s = np.float32(s)
        top = np.float32(127) * s
        x = np.full(width, top, np.float32)
        h = ((rng.integers(-127, 127, width - 1) + 0.5) * np.float64(s)).astype(np.float32)   # next to a half, or on it
        step = rng.integers(-1, 2, width - 1)
        x[1:] = np.where(step == 0, h, np.nextafter(h, np.where(step > 0, np.float32(np.inf), np.float32(-np.inf)).astype(np.float32)))
        rows.append(x)
    rows.append(np.zeros(width, np.float32))
    rows.append((rng.integers(-60, 60, width) * 1e-45).astype(np.float32))
    rows.append(np.where(rng.random(width) < 0.5, -1, 1).astype(np.float32) * np.finfo(np.float32).max)
    for bad in (np.inf, -np.inf, np.nan):
        for at in (0, width - 1):
            x = rng.standard_normal(width).astype(np.float32)
            x[at] = bad
            rows.append(x)
    x = np.stack(rows)
    q, s = _quant(x)
    wq, ws = ref.quant_rows(x)
    np.testing.assert_array_equal(s, ws)
    np.testing.assert_array_equal(q, wq)


# ------------------------------------------------------------------------------- the product
def _gemm_error(xq, sx, wq, sw, bias, res, act, y):
    """|y - exact| and its bound, element by element."""
    want, v = ref.gemm_i8(xq, sx, wq, sw, bias, res, act)
    p = np.abs(ref.gemm_i8(xq, sx, wq, sw)[0])
    pb = np.abs(ref.gemm_i8(xq, sx, wq, sw, bias)[0]) if bias is not None else 0
    err_v = (3 * U * p + U * pb + (U * np.abs(v) if res is not None else 0)) * (1 + 1e-6)
    # slope of the activation at most 1.13 (gelu); its own arithmetic: erff / expf / tanhf within 2 ulp, three more roundings
    bound = err_v if act in ("none", "relu", "relu6") else 1.13 * err_v + 6 * U * (np.abs(v) + 1)
    return np.abs(y.astype(np.float64) - want), bound


def _gemm(xq, sx, wq, sw, bias=None, res=None, act="none", px=None, pw=None, py=None, pr=None, shift=0, in_place=False):
    m, k = xq.shape
    n = wq.shape[0]
    a, ap = _dev(xq, px, shift) if k else _dev(np.zeros((m, 1), np.int8))
    b, bp = _dev(wq, pw, shift) if k else _dev(np.zeros((n, 1), np.int8))
    s1, s1p = _dev(sx[None])
    s2, s2p = _dev(sw[None])
    bb, bbp = _dev(bias[None]) if bias is not None else (None, 0)
    r, rp = _dev(res, pr) if res is not None else (None, 0)
    if in_place:
        y, yp, py = r, rp, pr
    else:
        y, yp = _dev(np.full((m, n), 77, np.float32), py)
    _launch(OP_GEMM_I8, [ap, s1p, bp, s2p, yp, bbp, rp], [m, n, k, px or k, pw or k, py or n, pr or n, ACTS[act]])
    torch.cuda.synchronize()
    return _back(y, m, n, py)


def _operands(rng, m, n, k, lowest=False):
    xq = rng.integers(-128 if lowest else -127, 128, (m, k)).astype(np.int8)
    wq = rng.integers(-128 if lowest else -127, 128, (n, k)).astype(np.int8)
    sx = np.exp(rng.standard_normal(m)).astype(np.float32) * np.float32(0.02)
    sw = np.exp(rng.standard_normal(n)).astype(np.float32) * np.float32(0.001)
    return xq, sx, wq, sw


SHAPES = [(1, 1, 1), (1, 768, 768), (2, 3, 5), (1, 17, 4096), (3, 1000, 63), (8, 64, 64), (15, 33, 65), (16, 256, 1024), (17, 130, 1000),
          (31, 31, 31), (32, 512, 128), (33, 127, 129), (64, 64, 2048), (65, 192, 320), (100, 300, 200), (127, 129, 511), (128, 128, 128),
          (129, 257, 1021), (200, 2048, 256), (255, 255, 255), (256, 256, 512), (257, 513, 384), (333, 1003, 1021), (512, 512, 96),
          (1000, 40, 640), (40, 5000, 80), (1300, 1290, 72), (520, 2050, 1040), (2049, 260, 2048)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemm_i8(m, n, k):
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    ops = _operands(rng, m, n, k)
    bias = rng.standard_normal(n).astype(np.float32)
    res = rng.standard_normal((m, n)).astype(np.float32)
    for bi, re in ((None, None), (bias, None), (bias, res)):
        err, bound = _gemm_error(*ops, bi, re, "none", _gemm(*ops, bi, re))
        assert (err <= bound).all(), (m, n, k, float((err - bound).max()))


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,n,k", [(1, 100, 64), (33, 130, 200), (300, 400, 128)])
def test_gemm_i8_activations(act, m, n, k):
    rng = np.random.default_rng(k)
    ops = _operands(rng, m, n, k)
    bias = (rng.standard_normal(n) * 3).astype(np.float32)
    err, bound = _gemm_error(*ops, bias, None, act, _gemm(*ops, bias, None, act))
    assert (err <= bound).all(), float((err / bound).max())


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,n,k,pitch", [(9, 77, 130, 144), (300, 901, 272, 272), (300, 901, 272, 273), (700, 1502, 144, 144),
                                         (1500, 1003, 400, 401), (1030, 1100, 96, 96)])
def test_gemm_i8_activations_behind_a_residual(act, m, n, k, pitch):
    """Every activation on top of bias and residual, in the epilogues that store four columns at a time and at a row's end."""
    rng = np.random.default_rng(m + n)
    ops = _operands(rng, m, n, k)
    bias = (rng.standard_normal(n) * 2).astype(np.float32)
    res = (rng.standard_normal((m, n)) * 2).astype(np.float32)
    for in_place in (False, True):
        err, bound = _gemm_error(*ops, bias, res, act, _gemm(*ops, bias, res.copy(), act, px=pitch, pw=pitch, in_place=in_place))
        assert (err <= bound).all(), (in_place, float((err / bound).max()))


@pytest.mark.parametrize("m,n,k", [(1, 70, 100), (20, 70, 100), (150, 260, 160), (300, 300, 257)])
@pytest.mark.parametrize("dx,dw,dy,dr,shift", [(0, 0, 3, 1, 0), (1, 2, 0, 0, 0), (16, 32, 4, 4, 0), (4, 12, 1, 0, 5), (28, 28, 0, 8, 16)])
def test_gemm_i8_pitches_and_odd_addresses(m, n, k, dx, dw, dy, dr, shift):
    rng = np.random.default_rng(m + dx)
    ops = _operands(rng, m, n, k)
    res = rng.standard_normal((m, n)).astype(np.float32)
    y = _gemm(*ops, None, res, px=k + dx, pw=k + dw, py=n + dy, pr=n + dr, shift=shift)
    err, bound = _gemm_error(*ops, None, res, "none", y)
    assert (err <= bound).all()


@pytest.mark.parametrize("m,n", [(1, 40), (40, 200), (200, 300)])
def test_gemm_i8_empty_inner_length_and_residual_in_place(m, n):
    rng = np.random.default_rng(n)
    bias, res = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n)).astype(np.float32)
    z = (np.zeros((m, 0), np.int8), np.ones(m, np.float32), np.zeros((n, 0), np.int8), np.ones(n, np.float32))
    np.testing.assert_array_equal(_gemm(*z, bias, res), bias + res)
    ops = _operands(rng, m, n, 96)
    want = _gemm(*ops, bias, res, pr=n + 4)
    np.testing.assert_array_equal(_gemm(*ops, bias, res, pr=n + 4, in_place=True), want)


@pytest.mark.parametrize("m", [1, 20, 130])
def test_gemm_i8_largest_sums(m):
    """The longest rows of the lowest code: 131071 * 2^14 is just below 2^31."""
    k, n = 131071, 20
    xq, wq = np.full((m, k), -128, np.int8), np.full((n, k), -128, np.int8)
    wq[1] = 127
    y = _gemm(xq, np.ones(m, np.float32), wq, np.ones(n, np.float32))
    want = np.tile(np.float32(131071 * 16384.0), (m, n))
    want[:, 1] = np.float32(-131071 * 128.0 * 127.0)
    np.testing.assert_array_equal(y, want)


@pytest.mark.parametrize("m,n,k", [(4, 96, 200), (150, 96, 200), (150, 300, 256)])
def test_gemm_i8_marks_of_bad_rows_reach_the_output(m, n, k):
    """A row that could not be quantised has a NaN for its scale: that row of the product is NaN under every activation, no other is."""
    rng = np.random.default_rng(3)
    xq, sx, wq, sw = _operands(rng, m, n, k, lowest=True)
    sx[2] = np.nan
    for act in sorted(ACTS):
        y = _gemm(xq, sx, wq, sw, act=act)
        assert np.isnan(y[2]).all() and np.isfinite(np.delete(y, 2, 0)).all(), act


@pytest.mark.parametrize("m,n,k", [(1, 768, 768), (50, 1024, 1024), (600, 1024, 512)])
def test_gemm_i8_through_the_engine_gives_the_same_bits(gpu_server, m, n, k):
    rng = np.random.default_rng(k)
    xq, sx, wq, sw = _operands(rng, m, n, k)
    bias = rng.standard_normal(n).astype(np.float32)
    with OpSession(gpu_server, [wq, sw, bias]) as t:
        x, s, y = t.act(xq), t.act(sx), t.empty(m * n * 4)
        t.s.launch(t.fid, OP_GEMM_I8, [x, s, t.w[0], t.w[1], y, t.w[2]], [m, n, k, 0, 0, 0, 0, ACT_GELU])
        assert t.s.last_kernel().startswith("gemm_i8")
        got = t.read(y, (m, n))
    np.testing.assert_array_equal(got, _gemm(xq, sx, wq, sw, bias, None, "gelu"))


# ------------------------------------------------------------------------------- norms around a block
class _Norm:
    """One case of OP_NORM_BLOCK: inputs on the host, the call, and the float64 outcome."""

    def __init__(self, rng, rows, width, post, pre, gate=None, group=0, residual=True, beta=True, a=1.0, b=1.0, eps=1e-5, offset=0.5):
        f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.rows, self.width, self.post, self.pre, self.group, self.a, self.b, self.eps = rows, width, post, pre, group, a, b, eps
        self.x = f(rows, width) * 3 + np.float32(offset)
        self.res = f(rows, width) if residual else None
        self.gate = None if gate is None else f(-(-rows // group) if group else 1, width)
        self.pg, self.pb = (f(width) if post else None), (f(width) if post and beta else None)
        self.g, self.be = (f(width) if pre else None), (f(width) if pre and beta else None)

    def run(self, h=True, y=True, q=True, dx=0, dr=0, dh=0, dy=0, dq=0, shift=0, h_over=None, y_over=None):
        R, W = self.rows, self.width
        x, xp = _dev(self.x, W + dx, shift)
        r, rp = _dev(self.res, W + dr, shift) if self.res is not None else (None, 0)
        vec = [_dev(v.reshape(1, -1), shift=shift) if v is not None else (None, 0) for v in
               (self.gate, self.pg, self.pb, self.g, self.be)]
        outs, ptrs, pitches = {}, [], []
        for name, want, extra, over, kind in (("h", h, dh, h_over, np.float32), ("y", y, dy, y_over, np.float32),
                                              ("q", q, dq, None, np.int8)):
            if over:
                t, p, extra = (x, xp, dx) if over == "x" else (r, rp, dr)
            else:
                t, p = _dev(np.full((R, W), 77, kind), W + extra, shift) if want else (None, 0)
            outs[name] = (t, W + extra)
            ptrs.append(p)
            pitches.append(W + extra)
        s, sp = _dev(np.full((1, R), 77, np.float32)) if q else (None, 0)
        _launch(OP_NORM_BLOCK, [xp, rp] + [v[1] for v in vec] + ptrs + [sp],
                [R, W, NORMS[self.post], NORMS[self.pre], self.group, W + dx, W + dr] + pitches, [self.a, self.b, self.eps, self.eps])
        torch.cuda.synchronize()
        got = {n: _back(t, R, W, p, shift) for n, (t, p) in outs.items() if t is not None}
        if s is not None:
            got["scale"] = _back(s, 1, R)[0]
        return got

    def check(self, got):
        # eps is a float32 argument: 1e-5 as the kernel sees it
        eps = float(np.float32(self.eps))
        post = (self.post, self.pg, self.pb, eps) if self.post else None
        pre = (self.pre, self.g, self.be, eps) if self.pre else None
        h, y = ref.norm_block(self.x, self.res, self.gate, self.group, post, pre, float(np.float32(self.a)), float(np.float32(self.b)))
        big = np.abs(h).max(1, keepdims=True)
        if "h" in got:
            err = np.abs(got["h"] - h)
            assert (err <= U * np.abs(h) * (1 + 1e-6) + 1e-13 * (big + np.abs(self.x).max())).all(), float(err.max())
            if pre is not None:      # judged on the kernel's own h, so that a last place of h is not counted again
                _, y = ref.norm_block(got["h"], pre=pre)
            else:
                y = got["h"].astype(np.float64)
        if "y" in got and ("h" in got or pre is None):
            hh = got["h"].astype(np.float64) if "h" in got else h
            spread = np.sqrt(hh.var(1, keepdims=True) + eps) if self.pre == "layer" else np.sqrt((hh * hh).mean(1, keepdims=True) + eps)
            term = 1e-13 * np.abs(hh).max(1, keepdims=True) / spread * (np.abs(self.g) if self.g is not None else 1)
            err = np.abs(got["y"] - y)
            slack = U * np.abs(y) * (1 + 1e-6) + term + 1e-13 * (np.abs(self.be) if self.be is not None else 0)
            assert (err <= slack).all(), float((err - slack).max())
        if "q" in got and "y" in got:
            wq, ws = ref.quant_rows(got["y"])
            np.testing.assert_array_equal(got["scale"], ws)
            np.testing.assert_array_equal(got["q"], wq)


WIDTHS = [1, 2, 3, 5, 63, 64, 65, 255, 256, 257, 768, 1021, 1024, 1025, 1531, 4096, 4097, 16384, 16385, 65536]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("post,pre", [(None, "layer"), ("rms", "rms"), ("layer", None)])
def test_norm_block(width, post, pre):
    rng = np.random.default_rng(width)
    for rows in ((1, 7) if width > 5000 else (1, 3, 37)):
        c = _Norm(rng, rows, width, post, pre)
        c.check(c.run())


@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("pre", [None, "layer", "rms"])
@pytest.mark.parametrize("gate,group", [(None, 0), ("one", 0), ("each", 1), ("some", 5)])
@pytest.mark.parametrize("residual,beta", [(True, True), (False, False)])
def test_norm_block_every_combination(post, pre, gate, group, residual, beta):
    rng = np.random.default_rng(group + 3)
    for width in (77, 1200):
        c = _Norm(rng, 13, width, post, pre, gate, group, residual, beta, a=0.75, b=-0.3)
        full = c.run()
        c.check(full)
        # every choice of outputs gives the same bits
        for want in (dict(h=False), dict(y=False), dict(q=False), dict(h=False, y=False), dict(h=False, q=False), dict(y=False, q=False)):
            for name, value in c.run(**want).items():
                np.testing.assert_array_equal(value, full[name], err_msg=str((want, name)))


@pytest.mark.parametrize("width", [127, 1021, 2050])
@pytest.mark.parametrize("over", [("res", "x"), ("x", "res"), (None, "x"), ("res", None)])
def test_norm_block_in_place(width, over):
    c = _Norm(np.random.default_rng(width), 21, width, "rms", "layer", "one")
    want = c.run()
    got = c.run(h_over=over[0], y_over=over[1], dx=3, dr=6)
    for name in want:
        np.testing.assert_array_equal(got[name], want[name], err_msg=name)


@pytest.mark.parametrize("dx,dr,dh,dy,dq,shift", [(1, 2, 3, 1, 1, 0), (4, 8, 4, 4, 4, 1), (0, 0, 0, 0, 3, 3), (5, 0, 5, 0, 0, 2)])
def test_norm_block_pitches_and_odd_addresses(dx, dr, dh, dy, dq, shift):
    c = _Norm(np.random.default_rng(dx), 9, 515, "layer", "rms", "some", 4)
    want = c.run()
    got = c.run(dx=dx, dr=dr, dh=dh, dy=dy, dq=dq, shift=shift)
    for name in want:
        np.testing.assert_array_equal(got[name], want[name], err_msg=name)


@pytest.mark.parametrize("width", [700, 3000])
def test_norm_block_splits_into_separate_calls_with_the_same_bits(width):
    """Residual stream, norm and codes in one call, and as three."""
    rng = np.random.default_rng(5)
    c = _Norm(rng, 19, width, "rms", "layer", "one", a=0.5, b=2.0)
    want = c.run()
    first = _Norm(rng, 19, width, "rms", None, "one", a=0.5, b=2.0)
    first.x, first.res, first.gate, first.pg, first.pb = c.x, c.res, c.gate, c.pg, c.pb
    h = first.run(y=False, q=False)["h"]
    np.testing.assert_array_equal(h, want["h"])
    second = _Norm(rng, 19, width, None, "layer", residual=False)
    second.x, second.g, second.be = h, c.g, c.be
    y = second.run(h=False, q=False)["y"]
    np.testing.assert_array_equal(y, want["y"])
    q, s = _quant(y)
    np.testing.assert_array_equal(q, want["q"])
    np.testing.assert_array_equal(s, want["scale"])


@pytest.mark.parametrize("width", [64, 1021, 4099])
def test_norm_block_rows_that_are_hard_on_the_statistics(width):
    """Constant rows (variance 0 under eps 1e-12), rows far from zero, one far element, infinities, NaNs, zeros, the largest floats."""
    rng = np.random.default_rng(width)
    c = _Norm(rng, 9, width, None, "layer", residual=False, eps=1e-12)
    c.x[0] = 1234.567
    c.x[1] = 0
    c.x[2] = rng.standard_normal(width) * 1e-3 + 1e4
    c.x[3, 0] = 1e6
    c.x[4, -1] = -3e7
    c.x[5] = rng.choice([-1, 1], width) * np.float32(3e38)
    c.x[6] = c.x[6] * np.float32(1e-30)
    c.x[7, width // 2] = np.inf
    c.x[8, 3] = np.nan
    got = c.run()
    np.testing.assert_array_equal(got["y"][0], c.be)
    np.testing.assert_array_equal(got["y"][1], c.be)
    assert np.isnan(got["y"][7:]).all() and np.isnan(got["scale"][7:]).all() and (got["q"][7:] == 0).all()
    for k in ("x", "rows"):
        setattr(c, k, c.x[:7] if k == "x" else 7)
    c.check({k: v[:7] for k, v in got.items()})
    for kind in ("layer", "rms"):
        d = _Norm(rng, 4, width, kind, "rms", residual=False)
        d.x[0] = 0
        d.x[1] = np.float32(-3e38)
        d.x[2, 0] = np.float32(1e-40)
        d.check(d.run())


# ------------------------------------------------------------------------------- offsets, streams, graphs
def test_offsets_past_32_bits():
    """Rows whose distance times their number passes 2^32 elements and bytes."""
    rng = np.random.default_rng(0)
    width, pitch = 130, (1 << 31) + 24
    x = rng.standard_normal((3, width)).astype(np.float32)
    big = torch.empty(2 * pitch + width, device="cuda")
    for r in range(3):
        big[r * pitch:r * pitch + width] = torch.from_numpy(x[r])
    q = torch.zeros(2 * pitch + width, dtype=torch.int8, device="cuda")
    s = torch.zeros(3, device="cuda")
    _launch(OP_QUANT_ROWS, [big.data_ptr(), q.data_ptr(), s.data_ptr()], [3, width, pitch, pitch])
    wq, ws = ref.quant_rows(x)
    got = torch.stack([q[r * pitch:r * pitch + width] for r in range(3)]).cpu().numpy()
    np.testing.assert_array_equal(got, wq)
    np.testing.assert_array_equal(s.cpu().numpy(), ws)
    # the codes as the weights and as the rows of a product, its result with the same pitch
    y = big
    for m in (1, 3):
        one = torch.ones(3, device="cuda")
        _launch(OP_GEMM_I8, [q.data_ptr(), one.data_ptr(), q.data_ptr(), one.data_ptr(), y.data_ptr()], [m, 3, width, pitch, pitch, pitch])
        got = torch.stack([y[r * pitch:r * pitch + 3] for r in range(m)]).cpu().numpy()
        np.testing.assert_array_equal(got, (wq.astype(np.int64) @ wq.astype(np.int64).T)[:m])
    g = torch.ones(width, device="cuda")
    for r in range(3):
        big[r * pitch:r * pitch + width] = torch.from_numpy(x[r])
    _launch(OP_NORM_BLOCK, [big.data_ptr(), 0, 0, 0, 0, g.data_ptr(), 0, 0, big.data_ptr()],
            [3, width, NORM_NONE, NORM_RMS, 0, pitch, 0, 0, pitch], [1.0, 1.0, 0.0, 1e-6])
    got = torch.stack([big[r * pitch:r * pitch + width] for r in range(3)]).cpu().numpy()
    _, want = ref.norm_block(x, pre=("rms", np.ones(width), None, float(np.float32(1e-6))))
    assert (np.abs(got - want) <= U * np.abs(want) * 1.001 + 1e-12).all()


class _Layer:
    """Half an encoder layer on raw addresses: norm and codes, product with gelu, codes, product with the stream added."""

    def __init__(self, seed, rows=70, hidden=256, ffn=520):
        g = torch.Generator(device="cuda").manual_seed(seed)
        f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
        self.rows, self.hidden, self.ffn = rows, hidden, ffn
        self.x, self.g, self.be = f(rows, hidden), f(hidden), f(hidden)
        self.w1, self.s1 = torch.randint(-127, 128, (ffn, hidden), generator=g, device="cuda", dtype=torch.int8), f(ffn).abs() * 1e-3
        self.w2, self.s2 = torch.randint(-127, 128, (hidden, ffn), generator=g, device="cuda", dtype=torch.int8), f(hidden).abs() * 1e-3
        self.b1 = f(ffn)
        e = lambda *s, t=torch.float32: torch.empty(*s, device="cuda", dtype=t)  # noqa: E731
        self.y, self.q, self.s = e(rows, hidden), e(rows, hidden, t=torch.int8), e(rows)
        self.mid, self.q2, self.sq2 = e(rows, ffn), e(rows, ffn, t=torch.int8), e(rows)
        self.out = e(rows, hidden)

    def run(self, stream):
        p = lambda t: t.data_ptr()  # noqa: E731
        R, H, F = self.rows, self.hidden, self.ffn
        _launch(OP_NORM_BLOCK, [p(self.x), 0, 0, 0, 0, p(self.g), p(self.be), 0, p(self.y), p(self.q), p(self.s)],
                [R, H, NORM_NONE, NORM_LAYER], [1.0, 1.0, 0.0, 1e-5], stream)
        _launch(OP_GEMM_I8, [p(self.q), p(self.s), p(self.w1), p(self.s1), p(self.mid), p(self.b1)], [R, F, H, 0, 0, 0, 0, ACT_GELU], (), stream)
        _launch(OP_QUANT_ROWS, [p(self.mid), p(self.q2), p(self.sq2)], [R, F], (), stream)
        _launch(OP_GEMM_I8, [p(self.q2), p(self.sq2), p(self.w2), p(self.s2), p(self.out), 0, p(self.y)], [R, H, F], (), stream)

    def want(self):
        """Step by step on the kernels' own intermediate values: (error, bound) of the result."""
        n = lambda t: t.cpu().numpy()  # noqa: E731
        wq, ws = ref.quant_rows(n(self.y))
        np.testing.assert_array_equal(n(self.q), wq)
        np.testing.assert_array_equal(n(self.s), ws)
        err, bound = _gemm_error(n(self.q), n(self.s), n(self.w1), n(self.s1), n(self.b1), None, "gelu", n(self.mid))
        assert (err <= bound).all()
        wq, ws = ref.quant_rows(n(self.mid))
        np.testing.assert_array_equal(n(self.q2), wq)
        np.testing.assert_array_equal(n(self.sq2), ws)
        err, bound = _gemm_error(n(self.q2), n(self.sq2), n(self.w2), n(self.s2), None, n(self.y), "none", n(self.out))
        assert (err <= bound).all()
        return n(self.out)


def test_a_layer_in_sequence_on_other_streams_and_in_graphs():
    """The operators as a layer calls them: eager, two at once on two streams, and captured into two graphs that are replayed
    side by side with new inputs between the replays."""
    a, b = _Layer(1), _Layer(2, rows=3)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    a.run(torch.cuda.current_stream())
    b.run(torch.cuda.current_stream())
    torch.cuda.synchronize()
    want = [a.want(), b.want()]
    for l in (a, b):
        l.out.zero_()
    torch.cuda.synchronize()
    for _ in range(3):
        a.run(s1)
        b.run(s2)
    torch.cuda.synchronize()
    for l, w in zip((a, b), want):
        np.testing.assert_array_equal(l.out.cpu().numpy(), w)
    graphs = []
    for l, s in ((a, s1), (b, s2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            l.run(torch.cuda.current_stream())
        graphs.append(g)
    for turn in range(4):
        for l in (a, b):
            l.x.normal_(generator=torch.Generator(device="cuda").manual_seed(turn))
            l.out.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, (s1, s2)):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        replayed = [l.out.cpu().numpy() for l in (a, b)]
        for l, r in zip((a, b), replayed):
            l.run(torch.cuda.current_stream())
            torch.cuda.synchronize()
            np.testing.assert_array_equal(r, l.want())


def test_calls_without_rows_launch_nothing():
    t = torch.full((64,), 7.0, device="cuda")
    p = t.data_ptr()
    _launch(OP_QUANT_ROWS, [p, p + 64, p + 128], [0, 4])
    _launch(OP_GEMM_I8, [p, p, p, p, p + 64], [0, 4, 4])
    _launch(OP_NORM_BLOCK, [p, 0, 0, 0, 0, p, 0, 0, p + 64], [0, 4, 0, 2], [1.0, 1.0, 0.0, 1e-6])
    torch.cuda.synchronize()
    assert (t == 7).all()


@pytest.mark.parametrize("n,k", [(768, 768), (1000, 333), (4096, 1024), (300, 4100)])
def test_gemm_i8_row_results_do_not_depend_on_the_batch(n, k):
    """The first row of every batch size, computed by whatever tile the size leads to, has the same bits."""
    rng = np.random.default_rng(n)
    xq, sx, wq, sw = _operands(rng, 2100, n, k)
    bias = rng.standard_normal(n).astype(np.float32)
    res = rng.standard_normal((2100, n)).astype(np.float32)
    want = _gemm(xq[:1], sx[:1], wq, sw, bias, res[:1], "gelu")
    for m in (2, 17, 40, 100, 200, 520, 1100, 2100):
        got = _gemm(xq[:m], sx[:m], wq, sw, bias, res[:m], "gelu")
        np.testing.assert_array_equal(got[:1], want, err_msg=str(m))


@pytest.mark.parametrize("width", [100, 400, 1000, 1531, 3000, 6000])
def test_row_operators_do_not_depend_on_the_batch(width):
    rng = np.random.default_rng(width)
    big = _Norm(rng, 9000 if width < 2000 else 500, width, "layer", "rms", "one")
    want = big.run()
    one = _Norm(rng, 1, width, "layer", "rms", "one")
    one.x, one.res, one.gate, one.pg, one.pb, one.g, one.be = big.x[7:8], big.res[7:8], big.gate, big.pg, big.pb, big.g, big.be
    for name, v in one.run().items():
        np.testing.assert_array_equal(v[0], want[name][7], err_msg=name)
    q, s = _quant(big.x)
    q1, s1 = _quant(big.x[7:8])
    np.testing.assert_array_equal(q1[0], q[7])
    assert s1[0] == s[7]


# sizes whose costs lead to each of the tiles in turn, K over several blocks with a last one that ends inside a chunk
TILE_SHAPES = [(5, 300, 1037), (40, 600, 333), (200, 300, 521), (300, 900, 777), (500, 1100, 1037), (1500, 1000, 1100), (1500, 2200, 300),
               (1900, 2000, 1037), (1500, 4000, 900), (4000, 4100, 700), (96, 760, 1037), (190, 760, 1037), (4090, 4090, 1037)]


@pytest.mark.parametrize("pad", ["16", "4", "odd"])
def test_gemm_i8_every_tile_with_rows_of_every_kind(pad):
    """Rows at multiples of 16, of 4 and at odd addresses, through every tile that the choice knows for them."""
    from torpor_amd import _lib

    seen = set()
    for m, n, k in TILE_SHAPES:
        rng = np.random.default_rng(m + n)
        pitch = {"16": (k + 15) // 16 * 16, "4": (k + 3) // 4 * 4 | 4, "odd": k | 1}[pad]
        ops = _operands(rng, m, n, k)
        bias = rng.standard_normal(n).astype(np.float32)
        y = _gemm(*ops, bias, px=pitch, pw=pitch)
        name = _lib.lib().tp_last_kernel().decode()
        seen.add(name)
        # float64 products of float64 numbers below 2^53 are exact here too, and quicker than integer ones
        p = (ops[0].astype(np.float64) @ ops[2].astype(np.float64).T) * ops[1].astype(np.float64)[:, None] * ops[3].astype(np.float64)
        assert (np.abs(y - (p + bias)) <= (3 * U * np.abs(p) + U * np.abs(p + bias)) * (1 + 1e-6)).all(), (m, n, k, name)
    tiles = "16x16 16x32 32x32 64x64 192x128 " + ("32x64 96x64 64x128 256x256" if pad == "16" else "128x128 256x128")
    assert seen == {"gemm_i8_" + t for t in tiles.split()}


def test_more_rows_than_a_grid_has_workgroups():
    """Rows beyond the largest grid go round the kernels' loop (4 rows a workgroup, 2^20 workgroups)."""
    rows, width = (1 << 22) + 77, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, width, generator=g, device="cuda")
    q, s = torch.empty(rows, width, dtype=torch.int8, device="cuda"), torch.empty(rows, device="cuda")
    _launch(OP_QUANT_ROWS, [x.data_ptr(), q.data_ptr(), s.data_ptr()], [rows, width])
    y, q2, s2 = torch.empty_like(x), torch.empty_like(q), torch.empty_like(s)
    gamma = torch.ones(width, device="cuda")
    _launch(OP_NORM_BLOCK, [x.data_ptr(), 0, 0, 0, 0, gamma.data_ptr(), 0, 0, y.data_ptr(), q2.data_ptr(), s2.data_ptr()],
            [rows, width, NORM_NONE, NORM_RMS], [1.0, 1.0, 0.0, 1e-6])
    part = np.r_[0:5, 1000000:1000005, (1 << 22) - 5:(1 << 22) + 77]
    at = torch.from_numpy(part).cuda()
    for src, codes, scale in ((x, q, s), (y, q2, s2)):
        wq, ws = ref.quant_rows(src[at].cpu().numpy())
        np.testing.assert_array_equal(codes[at].cpu().numpy(), wq)
        np.testing.assert_array_equal(scale[at].cpu().numpy(), ws)
    _, want = ref.norm_block(x[at].cpu().numpy(), pre=("rms", np.ones(width), None, float(np.float32(1e-6))))
    assert (np.abs(y[at].cpu().numpy() - want) <= U * np.abs(want) * 1.001 + 1e-12).all()
    # every row: codes times scale is within half a step of the value (and a rounding of the scale) everywhere
    assert bool(((q.float() * s[:, None] - x).abs() <= s[:, None] * 0.5001).all())


def test_gemm_i8_very_many_rows():
    """Nine million rows of five codes: tiles are counted and rows addressed past what 16-row tiles have in a grid's 2^32 threads."""
    m, n, k = 9_000_001, 3, 5
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randint(-127, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    sx, sw = torch.rand(m, generator=g, device="cuda"), torch.ones(n, device="cuda")
    y = torch.empty(m, n, device="cuda")
    _launch(OP_GEMM_I8, [x.data_ptr(), sx.data_ptr(), w.data_ptr(), sw.data_ptr(), y.data_ptr()], [m, n, k])
    want = (x.float() @ w.float().t()) * sx[:, None]      # sums below 2^24: exact; one rounding on either side
    assert bool((y == want).all())


# rows that are worked on one group after the other: both widths of them, every ending of a row's last group, few and all groups full
LONG_WIDTHS = [8193, 8196, 12002, 16383, 16384, 16387, 20000, 33333, 65533, 65536]


@pytest.mark.parametrize("width", LONG_WIDTHS)
@pytest.mark.parametrize("post,pre", [("rms", "layer"), ("layer", "rms"), ("layer", None), (None, "rms"), (None, None)])
def test_norm_block_long_rows(width, post, pre):
    """Gate, residual, stream and codes, also in place: the residual of a long row is read while its stream is written."""
    rng = np.random.default_rng(width)
    c = _Norm(rng, 5, width, post, pre, "some", 2, a=0.75, b=-0.3)
    want = c.run()
    c.check(want)
    for over in (("res", "x"), ("x", "res"), (None, "res")):
        got = c.run(h_over=over[0], y_over=over[1], dx=3, dr=6)
        for name in want:
            np.testing.assert_array_equal(got[name], want[name], err_msg=str((over, name)))
    one = _Norm(rng, 5, width, post, pre, residual=False, beta=False)
    one.check(one.run())


# The activations by themselves: with k = 0 and a residual alone, y = act(residual) of exactly these numbers.  Relative bounds from the
# formulas, a rounding U each, the hardware's exponential and reciprocal within 2U:
#   gelu: max(v, 0) less a term |v| 2^Q(|v|) / 2.  The term: its product U, 2^ 2U, and ln 2 times the error of Q, whose Horner steps and
#     coefficients sum up to 2 (a + a^2) U at a = |v| <= 4 and to 4 (a + a^2) U up to 6, the fit of Q 1.2e-8 of the term up to 4 and 4e-7 up
#     to 6; above, where the term is below 6e-9, 14 (a + a^2) U and 1e-4 of what is left of it at 6, 7 and 8: 3e-13.  One rounding of the difference.
#   sigmoid: e within 3U, 1 + e U, its reciprocal 2U, the product U: 7U; silu one more.
#   tanh: within 5 units in the last place by its documentation, 10U.
# Results below 2^-126 come as 0: 2^-118 absolute.
def _activation_bound(act, v):
    from scipy.special import erfc, expit

    a = np.abs(v)
    if act == "gelu":
        want = v * erfc(-v / np.sqrt(2.0)) / 2
        half = a * erfc(a / np.sqrt(2.0)) / 2
        term = np.where(a <= 4, (3 + 2 * (a + a * a)) * U + 1.2e-8, (3 + 4 * (a + a * a)) * U + 4e-7) * half
        term = np.where(a <= 6, term, 3e-13)
        return want, U * np.abs(want) * (1 + 1e-6) + term + 2.0 ** -118
    want = {"sigmoid": expit(v), "silu": v * expit(v), "tanh": np.tanh(v)}[act]
    return want, {"sigmoid": 7, "silu": 8, "tanh": 10}[act] * U * np.abs(want) + 2.0 ** -118


@pytest.mark.parametrize("act", ["gelu", "silu", "sigmoid", "tanh"])
@pytest.mark.parametrize("m,n", [(3, 501), (40, 200), (300, 900), (1500, 2000)])
def test_gemm_i8_activations_are_exact_relative_to_their_value(act, m, n):
    """Values of all sizes: next to zero, where a fit has to meet the function's slope, and far out."""
    rng = np.random.default_rng(m)
    scale = rng.choice([1e-30, 1e-4, 0.05, 0.3, 1.0, 1.0, 3.0, 8.0, 30.0], (m, n))
    v = (rng.standard_normal((m, n)) * scale).astype(np.float32)
    v[0, :8] = [0.0, 6.0, -6.0, 8.5, -8.5, -12.9, 31.0, -31.0]
    z = (np.zeros((m, 0), np.int8), np.ones(m, np.float32), np.zeros((n, 0), np.int8), np.ones(n, np.float32))
    y = _gemm(*z, None, v, act=act)
    want, bound = _activation_bound(act, v.astype(np.float64))
    err = np.abs(y - want)
    at = np.unravel_index(np.argmax(err / bound), err.shape)
    assert (err <= bound).all(), (float((err / bound).max()), float(v[at]), float(y[at]), float(want[at]))
    # on average far less than the bound: a relative 2-norm of two roundings or less wherever values are of ordinary size
    for lo, hi in ((-1, -0.1), (-0.1, 0.1), (0.1, 1), (1, 3)) if act != "tanh" else ():
        at = (v > lo) & (v < hi) & (np.abs(v) > 1e-20)
        norm = np.sqrt((err[at] ** 2).sum() / (want[at] ** 2).sum())
        assert norm <= 2 * U, (lo, hi, norm)


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,n", [(3, 40), (300, 900)])
def test_gemm_i8_activations_of_infinities_and_nans(act, m, n):
    """The limits; silu of minus infinity is infinity over infinity, a NaN, as v / (1 + exp(-v)) has it."""
    v = np.tile(np.array([np.inf, -np.inf, np.nan, 3e38, -3e38], np.float32), (m, n // 5))
    z = (np.zeros((m, 0), np.int8), np.ones(m, np.float32), np.zeros((n, 0), np.int8), np.ones(n, np.float32))
    y = _gemm(*z, None, v, act=act)
    big = np.float32(3e38)
    want = {"none": [np.inf, -np.inf, np.nan, big, -big], "relu": [np.inf, 0, np.nan, big, 0], "relu6": [6, 0, np.nan, 6, 0],
            "gelu": [np.inf, 0, np.nan, big, 0], "tanh": [1, -1, np.nan, 1, -1], "silu": [np.inf, np.nan, np.nan, big, 0],
            "sigmoid": [1, 0, np.nan, 1, 0]}[act]
    np.testing.assert_array_equal(y, np.tile(np.array(want, np.float32), (m, n // 5)))


@pytest.mark.parametrize("m,n,k,pitch", [(4, 96, 200, 200), (40, 70, 200, 201), (150, 300, 256, 256), (300, 901, 272, 273), (1500, 2200, 320, 320)])
def test_gemm_i8_rows_near_the_largest_float(m, n, k, pitch):
    """Rows whose sum times their scale is beyond the largest float while the result is an ordinary one, between rows of every other size."""
    rng = np.random.default_rng(m)
    xq, sx, wq, sw = _operands(rng, m, n, k)
    sx[:] = rng.choice(np.float32([2.0 ** -126, 1e-20, 0.02, 2.0 ** 96, 1.5 * 2.0 ** 95, 1e31, 1e33, 2.6e36]), m)
    sx[1] = 2.6e36
    sw[:] = np.exp(rng.standard_normal(n)).astype(np.float32) * np.float32(1e-9)
    sw[3], sw[5] = np.float32(2.0 ** -126), np.float32(1e30)
    wq[5] = 0                                   # no sum at all: the bias, whatever the scales
    bias = rng.standard_normal(n).astype(np.float32)
    res = rng.standard_normal((m, n)).astype(np.float32)
    for b, r in ((None, None), (bias, res)):
        y = _gemm(xq, sx, wq, sw, b, r, px=pitch, pw=pitch)
        err, bound = _gemm_error(xq, sx, wq, sw, b, r, "none", y)
        assert np.isfinite(y).all() and (err <= bound + 2.0 ** -148).all(), float((err - bound).max())
    # beyond the largest float the result is infinite
    sw[7], wq[7], xq[1, 0], wq[7, 0] = 1.0, 0, 127, 127
    y = _gemm(xq, sx, wq, sw, px=pitch, pw=pitch)
    assert np.isinf(y[1, 7]) and y[1, 7] > 0


@pytest.mark.parametrize("m,n", [(1, 40), (40, 200), (300, 900)])
def test_gemm_i8_without_an_inner_length_needs_no_codes(m, n):
    """Codes of k = 0 have no elements and, as an empty tensor, no address."""
    x = torch.empty(m, 0, dtype=torch.int8, device="cuda")
    w = torch.empty(n, 0, dtype=torch.int8, device="cuda")
    assert x.data_ptr() == 0 and w.data_ptr() == 0
    s, bias, y = torch.ones(max(m, n), device="cuda"), torch.randn(n, device="cuda"), torch.zeros(m, n, device="cuda")
    _launch(OP_GEMM_I8, [0, s.data_ptr(), 0, s.data_ptr(), y.data_ptr(), bias.data_ptr()], [m, n, 0])
    assert bool((y == bias).all())


@pytest.mark.parametrize("width", [7, 600, 20000])
@pytest.mark.parametrize("scale", [float("nan"), float("inf"), 1.0])
def test_norm_block_without_a_residual_has_no_use_for_its_scale(width, scale):
    c = _Norm(np.random.default_rng(width), 3, width, None, "rms", residual=False)
    want = c.run()
    c.check(want)
    c.a = scale
    for name, v in c.run().items():
        np.testing.assert_array_equal(v, want[name], err_msg=name)


@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("m,n,k,pitch", [(4, 96, 200, 200), (300, 901, 272, 273), (600, 1003, 400, 400)])
def test_gemm_i8_a_row_near_the_largest_float_leaves_its_neighbours_their_bits(act, m, n, k, pitch):
    """Rows that share a wavefront with such a row are finished by other code than without it, with and without a residual in place."""
    rng = np.random.default_rng(n)
    xq, sx, wq, sw = _operands(rng, m, n, k)
    bias = rng.standard_normal(n).astype(np.float32)
    res = rng.standard_normal((m, n)).astype(np.float32)
    far = sx.copy()
    far[1::37] = 1e33
    others = np.delete(np.arange(m), np.arange(1, m, 37))
    for r in (None, res):
        one, two = (_gemm(xq, s, wq, sw, bias, None if r is None else r.copy(), act, px=pitch, pw=pitch, in_place=r is not None)
                    for s in (sx, far))
        np.testing.assert_array_equal(one[others], two[others])

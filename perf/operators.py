"""Workloads of the 8-bit transformer-layer operators: the row quantisation, the int8 matrix product and the norms
around a block, at the sizes of the served encoders and over the general range.

Where `own` is false `run` computes them in plain torch operations, else by the library's kernels.  The codes of a
quantised row are whole numbers and come as they are, beside the row's scale.  Where a case has codes among its
outputs the plain form works in 64 bits: a value next to the border between two codes has to fall on the right side.
"""
import math

import torch

own = False

DEV = "cuda"
MIN_SCALE = 2.0 ** -126
ACTS = {"none": 0, "gelu": 2, "silu": 5}
NORMS = {"none": 0, "layer": 1, "rms": 2}
EPS = {"layer": 1e-12, "rms": 1e-6}


# ------------------------------------------------------------------------------------------------- the cases
def quant(rows, width, pitch=0, **kw):
    return dict(op="quant", rows=rows, width=width, pitch=pitch or width, **kw)


def gemm(m, n, k, act="none", bias=True, residual=False, pitch=0, **kw):
    return dict(op="gemm", m=m, n=n, k=k, act=act, bias=bias, residual=residual, pitch=pitch or k, **kw)


def norm(rows, width, post="none", pre="layer", gate="none", group=1, residual=True, h=False, codes=True, **kw):
    return dict(op="norm", rows=rows, width=width, post=post, pre=pre, gate=gate, group=group, residual=residual, h=h,
                codes=codes, **kw)


def listed():
    return [
        # the context rows of one BERT-base request of a few tokens, before the attention output projection
        quant(16, 768, name="quantise few rows"),
        # a ragged batch with an odd width, rows packed without padding
        quant(391, 1021, name="quantise odd rows"),
        # the inner activations of a long prompt batch
        quant(16384, 4096, name="quantise many rows"),
        # one token through a BERT-base projection: the smallest product, a launch and little else
        gemm(1, 768, 768, name="product one token"),
        # a decoding step of eight sequences through a wide layer: the weights' bytes
        gemm(8, 16384, 4096, bias=False, name="product eight tokens"),
        # the first half of BERT-large's feed-forward block, batch 4 of 384 tokens
        gemm(1536, 4096, 1024, act="gelu", name="product feed-forward"),
        # nothing divides anything: rows of odd length at odd addresses, a residual added
        gemm(333, 1003, 1021, residual=True, name="product odd"),
        # a long prompt batch through a wide layer: the matrix rate
        gemm(8192, 8192, 8192, bias=False, name="product large"),
        # a step of four sequences between two blocks of BERT-large
        norm(4, 1024, name="norm few rows"),
        # BERT-large between two blocks, batch 4 of 384 tokens: the stream for the residual and codes for the product
        norm(1536, 1024, name="norm encoder batch"),
        # norms on both sides, a gate for each sequence of 111 tokens, an odd width
        norm(777, 1531, post="rms", pre="rms", gate="group", group=111, h=True, codes=False, name="norm odd gated"),
        # a long prompt batch: norms on both sides of the block, a learned gate for each channel, stream and codes out
        norm(16384, 4096, post="rms", pre="rms", gate="channel", h=True, name="norm many rows"),
    ]


def _size(rng, lo, hi):
    """Spread over the logarithm; every other one as it falls, the rest a multiple of 16 or 64 as layer widths are."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    step = rng.choice([1, 1, 16, 64])
    return max(lo, min(hi, v // step * step if v >= step else v))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gemm", "norm"])
    if op == "gemm":
        while True:
            m, n, k = _size(rng, 1, 8192), _size(rng, 64, 16384), _size(rng, 64, 16384)
            if m * n * k <= 8192 ** 3 and m * n <= 8192 ** 2 and n * k <= 8192 ** 2 and m * k <= 8192 ** 2:
                break
        return gemm(m, n, k, act=rng.choice(sorted(ACTS)), bias=rng.random() < 0.5, residual=rng.random() < 0.3,
                    pitch=rng.choice([k, k, (k + 15) // 16 * 16, k + rng.randrange(1, 40)]))
    while True:
        rows, width = _size(rng, 1, 16384), _size(rng, 16, 16384)
        if rows * width <= 16384 * 4096:
            break
    if op == "quant":
        return quant(rows, width, pitch=rng.choice([width, width, (width + 3) // 4 * 4, width + rng.randrange(1, 40)]))
    return norm(rows, width, post=rng.choice(["none", "layer", "rms"]), pre=rng.choice(["layer", "rms"]),
                gate=rng.choice(["none", "channel", "group"]), group=rng.randrange(1, max(2, rows)),
                residual=rng.random() < 0.8, h=rng.random() < 0.5, codes=rng.random() < 0.6)


# ------------------------------------------------------------------------------------------------- inputs
def _codes(rows, width, g, std):
    """Codes and scales as a program holds them: normal values, quantised by row."""
    x = torch.randn(rows, width, generator=g, device=DEV)
    amax = x.abs().amax(1, keepdim=True)
    return torch.round(x * (127.0 / amax)).to(torch.int8), (amax[:, 0] * (std / 127.0)).contiguous()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(case)
    if case["op"] == "quant":
        # activations: every row of its own size, a few channels much larger than the rest
        wide = torch.where(torch.rand(case["pitch"], generator=g, device=DEV) < 0.01, 20.0, 1.0)
        s["x"] = randn(case["rows"], case["pitch"]) * wide * torch.exp(randn(case["rows"], 1))
    elif case["op"] == "gemm":
        m, n, k, p = case["m"], case["n"], case["k"], case["pitch"]
        s["x"], s["sx"] = _codes(m, p, g, 1.0)
        s["w"], s["sw"] = _codes(n, p, g, 1.0 / math.sqrt(k))
        s["bias"] = randn(n) * 0.1 if case["bias"] else None
        s["res"] = randn(m, n) if case["residual"] else None
    else:
        rows, width = case["rows"], case["width"]
        s["x"] = randn(rows, width) * 3 + 0.5
        s["res"] = randn(rows, width) * 2 if case["residual"] else None
        for side in ("post", "pre"):
            s[side + "_g"] = 1 + 0.1 * randn(width) if case[side] != "none" else None
            s[side + "_b"] = 0.1 * randn(width) if case[side] == "layer" else None
        groups = -(-rows // case["group"])
        s["gate_v"] = (0.5 * randn(width) if case["gate"] == "channel" else
                       0.5 * randn(groups, width) if case["gate"] == "group" else None)
        s["a"], s["b"] = 1.0, 0.5
    return s


# ------------------------------------------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)[s["op"]](s)


def _plain_quantise(x64):
    amax = x64.abs().amax(1)
    scale = (amax / 127).float().clamp_min(MIN_SCALE)
    return torch.round(x64 / scale.double()[:, None]).to(torch.int8), scale


def _plain_quant(s):
    q, scale = _plain_quantise(s["x"][:, :s["width"]].double())
    return {"q": q, "scale": scale}


def _plain_gemm(s):
    k = s["k"]
    y = s["x"][:, :k].float() @ s["w"][:, :k].float().t()
    y = y * s["sx"][:, None] * s["sw"][None, :]
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["res"] is not None:
        y = y + s["res"]
    if s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    return {"y": y}


def _plain_norm_of(t, kind, gamma, beta):
    if kind == "layer":
        t = t - t.mean(1, keepdim=True)
    t = t / torch.sqrt((t * t).mean(1, keepdim=True) + EPS[kind]) * gamma
    return t if beta is None else t + beta


def _plain_norm(s):
    to = torch.float64 if s["codes"] else torch.float32
    t = s["x"].to(to)
    if s["post"] != "none":
        t = _plain_norm_of(t, s["post"], s["post_g"], s["post_b"])
    if s["gate"] == "channel":
        t = t * s["gate_v"]
    elif s["gate"] == "group":
        t = t * s["gate_v"][torch.arange(s["rows"], device=DEV) // s["group"]]
    t = t * s["b"]
    if s["res"] is not None:
        t = t + s["a"] * s["res"].to(to)
    h = t.float()
    y = _plain_norm_of(h.to(to), s["pre"], s["pre_g"], s["pre_b"]).float()
    out = {"y": y}
    if s["h"]:
        out["h"] = h
    if s["codes"]:
        out["q"], out["scale"] = _plain_quantise(y.to(to))
    return out


_plain = {"quant": _plain_quant, "gemm": _plain_gemm, "norm": _plain_norm}


# ------------------------------------------------------------------------------------------------- the framework's calls
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _launch(op, ptrs, ints, floats=()):
    from torpor_amd.server import launch_noalloc

    r = launch_noalloc(op, ptrs, ints, floats, stream=torch.cuda.current_stream().cuda_stream)
    if r:
        raise RuntimeError("launch_noalloc: %d" % r)


def _own_quant(s):
    from torpor_amd.server import OP_QUANT_ROWS

    rows, width = s["rows"], s["width"]
    q = torch.empty(rows, width, dtype=torch.int8, device=DEV)
    scale = torch.empty(rows, device=DEV)
    _launch(OP_QUANT_ROWS, [s["x"].data_ptr(), q.data_ptr(), scale.data_ptr()], [rows, width, s["pitch"], width])
    return {"q": q, "scale": scale}


def _own_gemm(s):
    from torpor_amd.server import OP_GEMM_I8

    m, n, k, p = s["m"], s["n"], s["k"], s["pitch"]
    y = torch.empty(m, n, device=DEV)
    _launch(OP_GEMM_I8, [s["x"].data_ptr(), s["sx"].data_ptr(), s["w"].data_ptr(), s["sw"].data_ptr(), y.data_ptr(),
                         _ptr(s["bias"]), _ptr(s["res"])], [m, n, k, p, p, n, n, ACTS[s["act"]]])
    return {"y": y}


def _own_norm(s):
    from torpor_amd.server import OP_NORM_BLOCK

    rows, width = s["rows"], s["width"]
    out = {"y": torch.empty(rows, width, device=DEV)}
    if s["h"]:
        out["h"] = torch.empty(rows, width, device=DEV)
    if s["codes"]:
        out["q"] = torch.empty(rows, width, dtype=torch.int8, device=DEV)
        out["scale"] = torch.empty(rows, device=DEV)
    _launch(OP_NORM_BLOCK,
            [s["x"].data_ptr(), _ptr(s["res"]), _ptr(s["gate_v"]), _ptr(s["post_g"]), _ptr(s["post_b"]), _ptr(s["pre_g"]),
             _ptr(s["pre_b"]), _ptr(out.get("h")), out["y"].data_ptr(), _ptr(out.get("q")), _ptr(out.get("scale"))],
            [rows, width, NORMS[s["post"]], NORMS[s["pre"]], s["group"] if s["gate"] == "group" else 0],
            [s["a"], s["b"], EPS.get(s["post"], 0.0), EPS[s["pre"]]])
    return out


_own = {"quant": _own_quant, "gemm": _own_gemm, "norm": _own_norm}


# ------------------------------------------------------------------------------------------------- work and truth
def work(case):
    if case["op"] == "quant":
        n = case["rows"] * case["width"]
        return {"bytes": 5 * n + 4 * case["rows"], "flops": 4 * n}
    if case["op"] == "gemm":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": (m + n) * (k + 4) + 4 * m * n * (2 if case["residual"] else 1) + 4 * n * case["bias"],
                "flops": 2 * m * n * k}
    rows, width = case["rows"], case["width"]
    n = rows * width
    each = 4 + 4 * case["residual"] + 4 + 4 * case["h"] + case["codes"]
    gates = {"none": 0, "channel": 1, "group": -(-rows // case["group"])}[case["gate"]]
    vectors = sum({"none": 0, "layer": 2, "rms": 1}[case[side]] for side in ("post", "pre")) + gates
    return {"bytes": each * n + 4 * vectors * width + 4 * rows * case["codes"], "flops": 16 * n}


def _exact_codes(y):
    """Of values that are held in 32 bits: the code of a value goes by the scale as it is stored."""
    top = torch.maximum(y.max(1).values, -y.min(1).values)
    scale = torch.maximum(top / 127.0, torch.full_like(top, MIN_SCALE))
    ratio = y / scale.float().double().unsqueeze(1)
    low = torch.floor(ratio)
    part = ratio - low
    up = (part > 0.5) | ((part == 0.5) & (low.remainder(2) == 1))
    return (low + up.double()).to(torch.int8), scale


def _exact_norm(t, kind, gamma, beta):
    width = t.shape[1]
    ones = torch.full((width,), 1.0 / width, dtype=torch.float64, device=DEV)
    mean = (t @ ones if kind == "layer" else torch.zeros_like(t[:, 0])).unsqueeze(1)
    var = ((t - mean).square() @ ones).unsqueeze(1)
    out = (t - mean) * torch.rsqrt(var + EPS[kind]) * gamma.double()
    return out if beta is None else out + beta.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        q, scale = _exact_codes(s["x"].double()[:, :case["width"]])
        return {"q": q, "scale": scale}
    if case["op"] == "gemm":
        k = case["k"]
        x = s["x"][:, :k].double() * s["sx"].double()[:, None]
        w = s["w"][:, :k].double() * s["sw"].double()[:, None]
        y = torch.mm(x, w.t().contiguous())
        for more in (s["bias"], s["res"]):
            if more is not None:
                y += more.double()
        if case["act"] == "gelu":
            y = y * (torch.erfc(-y / math.sqrt(2.0)) / 2)
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        return {"y": y}
    t = s["x"].double()
    if case["post"] != "none":
        t = _exact_norm(t, case["post"], s["post_g"], s["post_b"])
    if case["gate"] == "channel":
        t = torch.einsum("rc,c->rc", t, s["gate_v"].double())
    elif case["gate"] == "group":
        t = t * s["gate_v"].double().repeat_interleave(case["group"], 0)[:case["rows"]]
    h = s["b"] * t if s["res"] is None else torch.add(s["b"] * t, s["res"].double(), alpha=s["a"])
    y = _exact_norm(h.float().double(), case["pre"], s["pre_g"], s["pre_b"])  # the stream is held in 32 bits between the two
    out = {"y": y}
    if case["h"]:
        out["h"] = h
    if case["codes"]:
        out["q"], out["scale"] = _exact_codes(y.float().double())
    return out

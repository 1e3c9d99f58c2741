"""BERT with its encoder in 8 bits: every 8-bit operator that a request launches is checked on the buffers it actually ran on
against the float64 forms (tolerances as in test_gpu_layer_ops), requests are bit-identical warm, cold, replayed and over fewer
rows, and a swapped-out model moves about a quarter of the encoder's bytes."""
import numpy as np
import pytest
import torch

from oracle import models as om
from oracle import ops as ref
from tests.test_gpu_layer_ops import U, _gemm_error
from tests.test_gpu_models import _check_swap_identity, _cycle
from tests.test_gpu_wire import gpu_wire_server  # noqa: F401  (a server process, as a fixture)
from torpor_amd import client as wire
from torpor_amd.functions import bert
from torpor_amd.server import ACT_GELU, OP_GEMM_I8, OP_NORM_BLOCK, OP_QUANT_ROWS, Server

pytestmark = pytest.mark.gpu


class _Checking(bert.Bert):
    """Reads an operator's inputs and outputs back right after its launch."""

    def __init__(self, *a, **kw):
        super().__init__(*a, **kw)
        self.seen = {}

    def forward(self, inputs):
        inner = self.s

        class Spy:
            def __getattr__(_, name):
                return getattr(inner, name)

            def launch(_, fid, op, ptrs, ints=(), floats=()):
                inner.launch(fid, op, ptrs, ints, floats)
                if op in (OP_GEMM_I8, OP_QUANT_ROWS, OP_NORM_BLOCK):
                    self.seen[op] = self.seen.get(op, 0) + 1
                    self._check(inner, op, ptrs, ints, floats)

        self.s = Spy()
        try:
            return super().forward(inputs)
        finally:
            self.s = inner

    def _check(self, s, op, ptrs, ints, floats):
        def read(va, shape, dtype=np.float32):
            out = np.empty(shape, dtype)
            s.d2h(self.fid, out, va)
            return out

        if op == OP_QUANT_ROWS:
            rows, width = ints
            wq, ws = ref.quant_rows(read(ptrs[0], (rows, width)))
            np.testing.assert_array_equal(read(ptrs[1], (rows, width), np.int8), wq)
            np.testing.assert_array_equal(read(ptrs[2], (rows,)), ws)
        elif op == OP_GEMM_I8:
            m, n, k = ints[:3]
            err, bound = _gemm_error(read(ptrs[0], (m, k), np.int8), read(ptrs[1], (m,)), read(ptrs[2], (n, k), np.int8),
                                     read(ptrs[3], (n,)), read(ptrs[5], (n,)), None, "gelu" if ints[7] == ACT_GELU else "none",
                                     read(ptrs[4], (m, n)))
            assert (err <= bound).all()
        else:
            rows, width = ints[:2]
            x, g, b = read(ptrs[0], (rows, width)), read(ptrs[5], (width,)), read(ptrs[6], (width,))
            res = read(ptrs[1], (rows, width)) if ptrs[1] else None
            y = read(ptrs[8], (rows, width))
            h, want = ref.norm_block(x, res, pre=("layer", g, b, float(np.float32(floats[3]))))
            # y is rounded once; h before it is too, and a last place of h more or less (its float64 sum may lie next to a border
            # between two floats) moves y by U |h| gamma / deviation
            dev = np.sqrt(h.var(1, keepdims=True) + floats[3])
            assert (np.abs(y - want) <= U * np.abs(want) * 1.001 + 2 * U * np.abs(h).max(1, keepdims=True) / dev * np.abs(g) + 1e-12).all()
            if len(ptrs) > 9:
                wq, ws = ref.quant_rows(y)
                np.testing.assert_array_equal(read(ptrs[9], (rows, width), np.int8), wq)
                np.testing.assert_array_equal(read(ptrs[10], (rows,)), ws)


@pytest.mark.parametrize("hidden,heads,ffn,qa", [(128, 2, 256, True), (75, 3, 50, False), (256, 4, 1000, False)])
def test_quantized_bert(gpu_server, hidden, heads, ffn, qa):
    """Head widths 64 (fused attention) and 25, rows of whole 16s and odd ones, with token types and a padding mask."""
    cfg = dict(layers=2, hidden=hidden, heads=heads, ffn=ffn)
    B, S = 3, 40
    weights = bert.init_weights(seed=5, vocab=300, max_pos=64, cfg=cfg, qa_head=qa)
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 300, (B, S), generator=g).numpy()
    tt = torch.randint(0, 2, (B, S), generator=g).numpy()
    am = np.ones((B, S), np.int64)
    am[0, 29:] = 0
    am[2, 8:] = 0
    fn = _Checking(gpu_server, 40 + hidden % 7, batch=B, seq=S, weights=weights, cfg=cfg, token_types=True, masked=True, quantized=True)
    inputs = [ids, tt, bert.Bert.additive_mask(am)]
    first = fn.register(inputs)
    assert fn.seen == {OP_NORM_BLOCK: 5, OP_GEMM_I8: 8, OP_QUANT_ROWS: 4}
    fn.forward = bert.Bert.forward.__get__(fn)      # from here on as a user runs it
    _check_swap_identity(gpu_server, fn, fn.weights())
    _cycle(gpu_server, fn, inputs, first)
    # fewer sequences than registered: each sequence's rows are its own, so the answers are the same bits
    some = fn.invoke_rows([a[:2] for a in inputs], 2)
    for a, b in zip(some, first):
        np.testing.assert_array_equal(a, b[:2])
    fn.unload()
    # Distance from the float model.  A code is off by at most half a step of 1/127 of its row's largest element; with rows of normal
    # values (largest about 3.5 deviations) that is an error of 3.5 / 127 / sqrt(12) = 0.8 % of the row on each side of a product,
    # 1.1 % of a product's result, and eight products in a row, were their errors all to add up in full, come to 9 %.
    model = om.load_numpy_state(om.Bert(vocab=300, max_pos=64, qa_head=qa, **cfg), weights)
    with torch.no_grad():
        want = model(torch.from_numpy(ids), torch.from_numpy(tt), torch.from_numpy(am))
    for got, w in zip(first, want):
        w = w.numpy()
        rel = np.linalg.norm(got - w) / np.linalg.norm(w)
        assert rel < 0.09, rel


def test_quantized_bert_base_moves_fewer_bytes(gpu_server):
    """BERT-base, one sequence of 128: cold requests give the bits of the first one; the weight image is smaller by three quarters of
    the encoder matrices' bytes (85.0 million elements; a scale for each of 6912 channels a layer comes on top)."""
    weights = bert.init_weights("bert-base", seed=0)
    ids = torch.randint(0, 30522, (1, 128), generator=torch.Generator().manual_seed(0)).numpy()
    sizes = {}
    for fid, quantized in ((50, False), (51, True)):
        fn = bert.Bert(gpu_server, fid, "bert-base", batch=1, seq=128, weights=weights, quantized=quantized)
        first = fn.register([ids])
        _cycle(gpu_server, fn, [ids], first)
        sizes[quantized] = gpu_server.model_info(fid)["param_bytes"]
        fn.unload()
    elements = 12 * (4 * 768 * 768 + 2 * 768 * 3072)
    assert sizes[False] - sizes[True] == 3 * elements - 12 * 4 * (3 * 768 + 768 + 3072 + 768)


def _small():
    cfg = dict(layers=2, hidden=128, heads=2, ffn=200)
    weights = bert.init_weights(seed=2, vocab=500, max_pos=64, cfg=cfg)
    ids = torch.randint(0, 500, (2, 48), generator=torch.Generator().manual_seed(1)).numpy()
    return cfg, weights, ids


def test_quantized_bert_over_the_wire(gpu_wire_server):  # noqa: F811
    """int8 weights and the three operators through the message protocol: the same bits as in process, warm, cold and replayed."""
    cfg, weights, ids = _small()
    with Server(mem_limit_bytes=1 << 30, pool_bytes=2 << 30) as local:
        want = bert.Bert(local, 0, batch=2, seq=48, weights=weights, cfg=cfg, quantized=True).register([ids])
    with wire.RemoteServer(gpu_wire_server, client_id=21) as rs:
        fn = bert.Bert(rs, 21, batch=2, seq=48, weights=weights, cfg=cfg, quantized=True)
        got = [fn.register([ids]), fn.invoke([ids], replay=False)]
        fn.unload()
        got.append(fn.invoke([ids]))
        fn.unload()
    for answer in got:
        for a, b in zip(answer, want):
            np.testing.assert_array_equal(a, b)


def test_quantized_bert_as_a_captured_graph(monkeypatch):
    """Warm requests launch the operators as one graph; other inputs between them, every answer that of the op-by-op path."""
    monkeypatch.setenv("TORPOR_GRAPH_MIN_OPS", "4")
    cfg, weights, ids = _small()
    other = np.ascontiguousarray(ids[:, ::-1])
    with Server(mem_limit_bytes=1 << 30, pool_bytes=2 << 30) as s:
        fn = bert.Bert(s, 3, batch=2, seq=48, weights=weights, cfg=cfg, quantized=True)
        first = fn.register([ids])
        second = [a.copy() for a in fn.invoke([other], replay=False)]
        for turn in range(6):
            for x, want in ((ids, first), (other, second)):
                for a, b in zip(fn.invoke([x]), want):
                    np.testing.assert_array_equal(a, b, err_msg=str(turn))
        fn.unload()
        for a, b in zip(fn.invoke([ids]), first):
            np.testing.assert_array_equal(a, b)

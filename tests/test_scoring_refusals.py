"""Calls of the 8-bit floating point operators and of token scoring that are
refused, and those that have nothing to do. All of it is decided before the GPU is
touched, so it runs without one: the context is a stand-in of zero bytes that no
refused call reads."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import uocr_moe as um  # noqa: E402

BF16, F16, F32, I64 = 0, 1, 2, 3
CTX = ctypes.create_string_buffer(4096)
P = ctypes.cast(ctypes.create_string_buffer(256), ctypes.c_void_p)  # some address


def call(name, *args):
    results = {um._operator(name, sync)(*args)
               for sync in ((True,) if name == "uocr_fp8_quantize_weight" else (True, False))}
    assert len(results) == 1  # both forms
    return results.pop()


def scores(tokens=P, n_top=0, logprobs=P, entropy=P, top_ids=None, top_logprobs=None):
    return ctypes.byref(um.TokenScores(tokens, n_top, logprobs, entropy, top_ids, top_logprobs))


@pytest.mark.parametrize("name", ["uocr_fp8_quantize", "uocr_fp8_quantize_weight"])
def test_quantize(name):
    ok = [CTX, P, F32, 3, 200, 200, P, P]

    def with_(i, v):
        return call(name, *[v if j == i else a for j, a in enumerate(ok)])
    assert with_(0, None) == um.SHAPE
    for i in (1, 6, 7):
        assert with_(i, None) == um.SHAPE
    for t in (F16, I64, 9):
        assert with_(2, t) == um.UNSUPPORTED
    assert with_(4, 0) == um.SHAPE
    assert with_(5, 199) == um.SHAPE
    assert with_(3, 0) == um.OK
    assert with_(3, (1 << 22) + 1) == um.RESOURCE
    assert call(name, CTX, P, F32, 1 << 22, 1 << 20, 1 << 20, P, P) == um.RESOURCE
    assert call(name, CTX, P, F32, 1, (1 << 22) + 1, 1 << 30, P, P) == um.RESOURCE


def test_linear():
    ok = [CTX, P, P, 3, 200, P, P, 50, P, F32]

    def with_(i, v):
        return call("uocr_fp8_linear", *[v if j == i else a for j, a in enumerate(ok)])
    assert with_(0, None) == um.SHAPE
    for i in (1, 2, 5, 6, 8):
        assert with_(i, None) == um.SHAPE
    assert with_(4, 0) == um.SHAPE
    assert with_(7, 0) == um.SHAPE
    for t in (F16, I64, -1):
        assert with_(9, t) == um.UNSUPPORTED
    for i in (3, 4, 7):
        assert with_(i, (1 << 22) + 1) == um.RESOURCE
    assert with_(3, 0) == um.OK


def test_token_logprobs():
    def go(type_=F32, rows=2, vocab=30, ld=30, logits=P, ctx=CTX, s=None):
        return call("uocr_token_logprobs", ctx, logits, type_, rows, vocab, ld, s or scores())
    assert go(ctx=None) == um.SHAPE
    assert go(logits=None) == um.SHAPE
    assert go(type_=I64) == um.UNSUPPORTED
    assert go(vocab=0) == um.SHAPE
    assert go(ld=29) == um.SHAPE
    assert call("uocr_token_logprobs", CTX, P, F32, 2, 30, 30, None) == um.SHAPE
    assert go(s=scores(tokens=None)) == um.SHAPE  # log probabilities of nothing
    assert go(s=scores(logprobs=None, entropy=None)) == um.SHAPE
    assert go(s=scores(n_top=31, top_ids=P, top_logprobs=P)) == um.SHAPE
    assert go(vocab=100, ld=100, s=scores(n_top=65, top_ids=P, top_logprobs=P)) == um.UNSUPPORTED
    assert go(s=scores(n_top=3, top_ids=P)) == um.SHAPE
    assert go(s=scores(n_top=3, top_logprobs=P)) == um.SHAPE
    assert go(rows=(1 << 22) + 1) == um.RESOURCE
    assert go(vocab=1 << 30, ld=1 << 30) == um.RESOURCE
    assert go(rows=0) == um.OK
    assert go(rows=0, s=scores(tokens=None, logprobs=None, entropy=None)) == um.OK


def test_linear_logprobs():
    def go(m=2, n=30, s=None, **kw):
        a = dict(ctx=CTX, x=P, xs=P, w=P, ws=P, k=64) | kw
        return call("uocr_fp8_linear_logprobs", a["ctx"], a["x"], a["xs"], m, a["k"], a["w"],
                    a["ws"], n, s or scores())
    for name in ("ctx", "x", "xs", "w", "ws"):
        assert go(**{name: None}) == um.SHAPE
    assert go(k=0) == um.SHAPE
    assert go(n=0) == um.SHAPE
    assert go(s=scores(tokens=None)) == um.SHAPE
    assert go(s=scores(n_top=31, top_ids=P, top_logprobs=P)) == um.SHAPE
    assert go(m=(1 << 22) + 1) == um.RESOURCE
    assert go(m=0) == um.OK


def test_head_logprobs():
    assert call("uocr_lm_head_logprobs", CTX, None, P, 1, scores()) == um.SHAPE
    assert call("uocr_lm_head_logprobs", None, P, P, 1, scores()) == um.SHAPE


class FakeContext:
    handle = None
    device = -1  # where host tensors are


def refused(fn, *args, **kw):
    with pytest.raises(um.UocrError) as e:
        fn(FakeContext, *args, **kw)
    return e.value.status


def test_binding_checks_shapes():
    """The binding refuses tensors whose shapes do not fit before it hands their
    addresses on (one that fits reaches the library, which refuses the context)."""
    x, q = torch.zeros(3, 200), torch.zeros(3, 200, dtype=torch.uint8)
    s = torch.zeros(3, 2)

    def message(fn, *args, **kw):
        with pytest.raises(um.UocrError) as e:
            fn(FakeContext, *args, **kw)
        return str(e.value)
    assert "null context" in message(um.fp8_quantize, x, q, s)
    assert "null context" in message(um.fp8_quantize, torch.zeros(3, 400)[:, 100:300], q, s)
    for bad in ((x, q[:2], s), (x, q, s[:, :1]), (x.t(), q.t(), s), (x, x, s),
                (torch.zeros(3, 400)[:, ::2], q, s), (x[0], q[0], s[0])):
        assert refused(um.fp8_quantize, *bad) == um.SHAPE
        assert "null context" not in message(um.fp8_quantize, *bad)
    assert refused(um.fp8_quantize, x.double(), q, s) == um.UNSUPPORTED
    w, ws = torch.zeros(130, 200, dtype=torch.uint8), torch.zeros(2, 2)
    y = torch.zeros(3, 130)
    assert "null context" in message(um.fp8_linear, q, s, w, ws, y)
    for bad in ((q, s, w[:, :100], ws, y), (q, s[:2], w, ws, y), (q, s, w, ws[:1], y),
                (q, s, w, ws, y.t()), (q, s, w.t().contiguous().t(), ws, y)):
        assert refused(um.fp8_linear, *bad) == um.SHAPE
        assert "null context" not in message(um.fp8_linear, *bad)
    t, lp = torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    ids, tl = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4)
    assert "null context" in message(um.token_logprobs, x, t, lp, lp, ids, tl)
    for bad in ((x, t[:2], lp), (x, t.long(), lp), (x, t, lp[:1]), (x, t, lp, lp[::2]),
                (x, t, lp, lp, ids, tl[:, :3]), (x[0], t, lp)):
        assert refused(um.token_logprobs, *bad) == um.SHAPE
        assert "null context" not in message(um.token_logprobs, *bad)
    # Types of the right size, and tensors that are somewhere else than the context.
    e5m2 = torch.zeros(3, 200).to(torch.float8_e5m2)
    assert refused(um.fp8_quantize, x, e5m2, s) == um.SHAPE
    assert refused(um.fp8_quantize, x, q, s.int()) == um.SHAPE
    assert refused(um.fp8_linear, e5m2, s, w, ws, y) == um.SHAPE
    assert refused(um.fp8_linear, q, s, w, ws.int(), y) == um.SHAPE
    assert refused(um.token_logprobs, x, t.float(), lp) == um.SHAPE
    assert refused(um.token_logprobs, x, t, lp.int()) == um.SHAPE
    assert refused(um.token_logprobs, x, t, lp, lp, tl, ids) == um.SHAPE
    assert "null context" in message(um.fp8_linear_logprobs, q, s, w, ws, t, lp)

    class OnGpu:
        handle, device = None, 0
    for fn, *args in ((um.fp8_quantize, x, q, s), (um.fp8_linear, q, s, w, ws, y),
                      (um.token_logprobs, x, t, lp), (um.fp8_linear_logprobs, q, s, w, ws, t, lp)):
        with pytest.raises(um.UocrError) as e:
            fn(OnGpu, *args)
        assert e.value.status == um.SHAPE and "device" in str(e.value)


def test_head_binding():
    class Head(um.LmHead):
        def __init__(self):
            self.handle, self.width = None, 64
    hidden, t, lp = torch.zeros(3, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(3)
    head = Head()

    def message(*args):
        with pytest.raises(um.UocrError) as e:
            head.logprobs(FakeContext, *args)
        assert e.value.status == um.SHAPE
        return str(e.value)
    assert "null handle" in message(hidden, t, lp)
    for bad in (hidden[:, :60], hidden.half(), hidden[0], torch.zeros(3, 128)[:, ::2], torch.zeros(3, 60)):
        assert "null handle" not in message(bad, t, lp)
    with pytest.raises(um.UocrError) as e:
        um.LmHead(FakeContext, torch.ones(64), 1e-6, q=torch.zeros(300, 64, dtype=torch.uint8),
                  scales=torch.ones(300, 2), mode=um.QUANT_FP8_BLOCKS)
    assert e.value.status == um.SHAPE and "scales" in str(e.value)

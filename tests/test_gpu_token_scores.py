"""Token scores (uocr_token_logprobs, uocr_fp8_linear_logprobs,
uocr_lm_head_logprobs) against their definitions in 64 bits on the CPU.

Tolerances, in units u = 2^-24. d = log2(e) (x - m) carries two roundings and the
constant's, 3 |d| u; 2^d is off by that and two half steps of the instruction (a term
that counts has |d| < 20); a row's sum of
positive terms runs through fewer than 64 additions in a thread and 30 in trees, so
S is off by less than 128 u of itself, log S by 128 u, and the given token's own
distance by 8 |log p| u (the distance, its product with ln 2, the sum). For the
entropy every term carries the same relative error, and |log S| + |sum p d| <= 2 (H +
1) where the reference is the row's largest logit: 256 (1 + H) u. The reference may
be another chunk's: moving it by D multiplies a part by 2^D, off by D u <= 60 u."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

import uocr_moe as um  # noqa: E402
from test_gpu_fp8 import blocks, device_exact, device_product, exact_product, random_product, say, spread  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    c = um.Context(0, 256 << 20)
    yield c
    c.close()


class Scores:
    """Output arrays with a guard value, and rows behind the last one."""

    def __init__(self, rows, top):
        self.rows, self.top = rows, top
        self.arrays = {"logprobs": torch.full((rows + 2,), 555.0), "entropy": torch.full((rows + 2,), 555.0)}
        if top:
            self.arrays["top_ids"] = torch.full((rows + 2, top), 555, dtype=torch.int32)
            self.arrays["top_logprobs"] = torch.full((rows + 2, top), 555.0)
        self.arrays = {k: v.cuda() for k, v in self.arrays.items()}

    def views(self):
        return {k: v[:self.rows] for k, v in self.arrays.items()}

    def host(self):
        assert all(bool((v[self.rows:] == 555).all()) for v in self.arrays.values())
        return {k: v[:self.rows].cpu().numpy().astype(np.float64) for k, v in self.arrays.items()}


def reference(x, tokens, top):
    """Scores of float64 logits."""
    rows, vocab = x.shape
    m = x.max(1, keepdims=True)
    e = np.exp(x - m)
    total = e.sum(1, keepdims=True)
    logp = x - m - np.log(total)
    p = e / total
    out = {"logprobs": logp[np.arange(rows), np.maximum(tokens, 0)],
           "entropy": -np.where(p > 0, p * np.where(p > 0, logp, 0), 0).sum(1)}
    if top:
        ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
        out["top_ids"] = ids.astype(np.float64)
        out["top_logprobs"] = np.take_along_axis(logp, ids, 1)
    pad = tokens < 0
    for k, v in (("logprobs", 0), ("entropy", 0), ("top_ids", -1), ("top_logprobs", -math.inf)):
        if k in out:
            out[k][pad] = v
    return out


def compare(got, want, extra=0.0):
    """Within the bounds above; extra: how far a logit itself may be off."""
    tol = {"logprobs": lambda w: (128 + 60 + 8 * np.abs(w)) * U + 2 * extra,
           "top_logprobs": lambda w: (128 + 60 + 8 * np.abs(w)) * U + 2 * extra,
           "entropy": lambda w: 256 * (1 + w) * U + extra * 4 * (1 + w)}
    for k, w in want.items():
        g = got[k]
        if k == "top_ids":
            assert np.array_equal(g, w), np.argwhere(g != w)[:5]
            continue
        fin = np.isfinite(w)
        assert np.array_equal(g[~fin], w[~fin], equal_nan=True), k
        off, t = np.abs(g[fin] - w[fin]), tol[k](w[fin])
        if off.size:
            say(f"  {k} off {off.max():.2e}, {np.max(off / t):.3f} of the bound")
        assert (off <= t).all(), (k, np.argwhere(off > t)[:5])


def logits_of(rng, rows, vocab, dtype):
    x = 2 * rng.standard_normal((rows, vocab)) - 2
    x[rng.random((rows, vocab)) < 4 / vocab] += 9
    return torch.from_numpy(x).to(dtype)


DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# Vocabularies around a vector, a group of columns, a chunk, and the decoder's.
SIZES = [(1, 1), (3, 2), (2, 7), (5, 63), (4, 64), (3, 65), (7, 129), (2, 1023), (2, 1025), (300, 1000),
         (9, 4099), (2, 16385), (1, 129280), (40, 40001), (3, 8192), (3, 8193), (600, 200), (65, 9000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,vocab", SIZES)
def test_token_logprobs(ctx, rows, vocab, dtype):
    say(f"scores {rows}x{vocab} {dtype}")
    rng = np.random.default_rng(rows + vocab)
    x = logits_of(rng, rows, vocab, dtype)
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    for top in sorted({0, 1, min(5, vocab), min(20, vocab), min(64, vocab)}):
        want = reference(x.double().numpy(), tokens, top)
        wide = torch.full((rows, vocab + 3), float("nan"), dtype=dtype)
        wide[:, 1:1 + vocab] = x
        for form in (x.cuda(), wide.cuda()[:, 1:1 + vocab]):
            out = Scores(rows, top)
            torch.cuda.synchronize()
            um.token_logprobs(ctx, form, torch.from_numpy(tokens).cuda(), **out.views())
            compare(out.host(), want)


# Vocabularies of one launch per row, and of two.
@pytest.mark.parametrize("vocab", [3001, 20001])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_banned_ids_and_ties(ctx, dtype, vocab):
    """-inf is probability 0 (a banned given token: -inf); equal logits by rising
    id, -0 equal to 0; the lowest finite value is a logit like others."""
    rng = np.random.default_rng(5)
    rows = 12
    x = logits_of(rng, rows, vocab, dtype)
    x[:, rng.random(vocab) < 0.5] = -math.inf
    x[1] = 0.0
    x[1, ::2] = -0.0
    x[2] = -math.inf
    x[2, 1777] = 3.0  # one word left
    x[3] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[4, 2500] = 0.0
    x[11] = torch.finfo(dtype).max
    x[5] = torch.round(x[5])  # many equal ones
    x[6, :2048] = -math.inf  # whole groups and chunks banned
    x[7, 1024:] = -math.inf
    x[8] = torch.arange(vocab).to(dtype)  # rising, falling
    x[9] = -torch.arange(vocab).to(dtype)
    x[10] = -math.inf
    x[10, [5, 6, 3000]] = torch.tensor([-1.0, -1.0, -1.0], dtype=dtype)
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    tokens[2], tokens[10] = 1777, 0
    want = reference(x.double().numpy(), tokens, 64)
    assert want["logprobs"][10] == -math.inf
    out = Scores(rows, 64)
    d, t = x.cuda(), torch.from_numpy(tokens).cuda()
    torch.cuda.synchronize()
    um.token_logprobs(ctx, d, t, **out.views())
    compare(out.host(), want)


def test_far_spread_logits(ctx):
    """Logits thousands apart, in chunks and lanes of their own."""
    rng = np.random.default_rng(6)
    x = torch.from_numpy(rng.uniform(-4000, 4000, (6, 20000))).float()
    x[1, :10000] -= 1e30
    x[2, 19999] = 1e30
    x[3] = torch.linspace(-1e4, 1e4, 20000)
    tokens = x.argmax(1).int().numpy()
    want = reference(x.double().numpy(), tokens, 3)
    out = Scores(6, 3)
    d, t = x.cuda(), torch.from_numpy(tokens).cuda()
    torch.cuda.synchronize()
    um.token_logprobs(ctx, d, t, **out.views())
    compare(out.host(), want)


@pytest.mark.parametrize("vocab", [700, 12300])
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_rows_without_a_distribution(ctx, dtype, vocab):
    """NaN, +inf and rows with no finite logit raise Numerical and get NaN and ids
    -1; the rows beside them are right; padding rows may hold anything."""
    rng = np.random.default_rng(7)
    rows, top = 9, 4
    x = logits_of(rng, rows, vocab, dtype)
    good = x.clone()
    x[1, 699] = math.nan
    x[3, 0] = math.inf
    x[5] = -math.inf
    x[6] = math.nan
    x[8, 350] = -math.nan
    tokens = rng.integers(0, vocab, rows).astype(np.int32)
    want = reference(good.double().numpy(), tokens, top)
    bad = [1, 3, 5, 6, 8]
    for k, v in want.items():
        v[bad] = -1 if k == "top_ids" else math.nan
    out = Scores(rows, top)
    d, t = x.cuda(), torch.from_numpy(tokens).cuda()
    torch.cuda.synchronize()
    with pytest.raises(um.UocrError) as e:
        um.token_logprobs(ctx, d, t, **out.views())
    assert e.value.status == um.NUMERICAL
    compare(out.host(), want)
    # The same rows as padding: not looked at.
    tokens[bad] = [-1, -5, -100, -2 ** 31, -1]
    want = reference(good.double().numpy(), tokens, top)
    out = Scores(rows, top)
    t = torch.from_numpy(tokens).cuda()
    torch.cuda.synchronize()
    um.token_logprobs(ctx, d, t, **out.views())
    compare(out.host(), want)


def test_token_past_the_vocabulary(ctx):
    rng = np.random.default_rng(8)
    x = logits_of(rng, 4, 100, torch.float32)
    tokens = np.array([3, 100, 99, 2 ** 31 - 1], np.int32)
    want = reference(x.double().numpy(), np.minimum(tokens, 99), 2)
    want["logprobs"][[1, 3]] = math.nan
    out = Scores(4, 2)
    d, t = x.cuda(), torch.from_numpy(tokens).cuda()
    torch.cuda.synchronize()
    with pytest.raises(um.UocrError) as e:
        um.token_logprobs(ctx, d, t, **out.views())
    assert e.value.status == um.SHAPE and "vocabulary" in str(e.value)
    compare(out.host(), want)


def test_outputs_one_by_one(ctx):
    """Each output alone gives the bits it has among the others."""
    rng = np.random.default_rng(9)
    x = logits_of(rng, 5, 5000, torch.bfloat16).cuda()
    t = torch.from_numpy(rng.integers(0, 5000, 5).astype(np.int32)).cuda()
    all_ = Scores(5, 7)
    torch.cuda.synchronize()
    um.token_logprobs(ctx, x, t, **all_.views())
    want = all_.host()
    for names in (("logprobs",), ("entropy",), ("top_ids", "top_logprobs")):
        one = Scores(5, 7)
        torch.cuda.synchronize()
        um.token_logprobs(ctx, x, t if "logprobs" in names else None, **{n: one.views()[n] for n in names})
        got = one.host()
        for n in want:
            assert np.array_equal(got[n], want[n] if n in names else np.full_like(want[n], 555)), (names, n)


def test_small_scratch_takes_rows_in_turn():
    """A context whose scratch holds a few rows' work gives the same scores, and
    one that holds none refuses."""
    rng = np.random.default_rng(10)
    x = logits_of(rng, 50, 40000, torch.float32)
    tokens = rng.integers(0, 40000, 50).astype(np.int32)
    want = reference(x.double().numpy(), tokens, 3)
    d, t = x.cuda(), torch.from_numpy(tokens).cuda()
    small = um.Context(0, 20000)
    out = Scores(50, 3)
    torch.cuda.synchronize()
    um.token_logprobs(small, d, t, **out.views())
    compare(out.host(), want)
    small.close()
    tiny = um.Context(0, 256)
    with pytest.raises(um.UocrError) as e:
        um.token_logprobs(tiny, d, t, **out.views())
    assert e.value.status == um.RESOURCE
    tiny.close()


# -------------------------------------------------------- from the product

FUSED = [(1, 1, 16), (1, 5000, 128), (2, 63, 40), (3, 65, 1280), (7, 129, 130), (16, 1000, 256), (17, 4097, 128),
         (40, 300, 896), (64, 257, 144), (65, 2000, 272), (130, 1537, 128), (257, 700, 384), (300, 5000, 1280),
         (300, 5000, 1279), (600, 2000, 131), (40, 3001, 1)]


def fused_reference(ops, tokens, top):
    a, b = spread(*ops)
    return reference(a @ b.T, tokens, top)


def scaled(ops, factor):
    return ops[0], ops[1] * factor, ops[2], ops[3]


@pytest.mark.parametrize("m,n,k", FUSED)
def test_linear_logprobs_exact_logits(ctx, m, n, k):
    """Logits that are exact in f32 (whole numbers times a power of two), so that
    only the scoring rounds."""
    say(f"fused scores {m}x{n}x{k}")
    factor = 2.0 ** -round(math.log2(64 * math.sqrt(k)))
    ops = scaled(exact_product(m, n, k, m + n), factor)
    rng = np.random.default_rng(m)
    tokens = rng.integers(0, n, m).astype(np.int32)
    if m > 2:
        tokens[m // 2] = -1
        tokens[0], tokens[1] = 0, n - 1
    dev, t = device_product(*ops), torch.from_numpy(tokens).cuda()
    for top in (0, min(3, n)):
        want = fused_reference(ops, tokens, top)
        out = Scores(m, top)
        torch.cuda.synchronize()
        um.fp8_linear_logprobs(ctx, *dev, t, **out.views())
        compare(out.host(), want)


@pytest.mark.parametrize("m,n,k", FUSED)
def test_linear_logprobs_random(ctx, m, n, k):
    say(f"fused random scores {m}x{n}x{k}")
    ops = scaled(random_product(m, n, k, m + n + 1), 1.0)
    a, b = spread(*ops)
    ops = scaled(ops, np.float32(3.0 / np.std(a @ b.T)) if m * n > 1 else 1e-3)
    ops = (ops[0], ops[1].astype(np.float32), ops[2], ops[3])
    a, b = spread(*ops)
    extra = 2 * (k + 3 * blocks(k)) * U * float((np.abs(a) @ np.abs(b).T).max())
    tokens = np.random.default_rng(m).integers(0, n, m).astype(np.int32)
    out, again = Scores(m, 0), Scores(m, 0)
    dev, t = device_product(*ops), torch.from_numpy(tokens).cuda()
    torch.cuda.synchronize()
    um.fp8_linear_logprobs(ctx, *dev, t, **out.views())
    compare(out.host(), reference(a @ b.T, tokens, 0), extra)
    um.fp8_linear_logprobs(ctx, *dev, t, **again.views())
    assert all(np.array_equal(out.host()[x], again.host()[x]) for x in out.host())


@pytest.mark.parametrize("m,n,k", [(65, 33, 16), (100, 700, 272), (129, 2100, 1296), (200, 1, 128),
                                   (300, 130, 6848), (2049, 65, 144), (129, 1900, 1296), (600, 500, 272)])
def test_linear_logprobs_many_rows_of_small_products(ctx, m, n, k):
    say(f"small fused scores {m}x{n}x{k}")
    test_linear_logprobs_exact_logits(ctx, m, n, k)
    test_linear_logprobs_random(ctx, m, n, k)


@pytest.mark.parametrize("m,n,k", [(1, 129280, 1280), (2, 65536, 144), (19, 70001, 256), (48, 66003, 640),
                                   (64, 65700, 2400), (1100, 8200, 272), (700, 20000, 1296), (1, 66000, 1279),
                                   (48, 66003, 641), (700, 20000, 1279)])
def test_linear_logprobs_wide(ctx, m, n, k):
    say(f"wide fused scores {m}x{n}x{k}")
    (x, xs, w, ws), logits = device_exact(m, n, k, m + n)
    factor = 2.0 ** -round(math.log2(64 * math.sqrt(k)))
    tokens = np.random.default_rng(m).integers(0, n, m).astype(np.int32)
    tokens[-1] = n - 1
    want = reference((logits * factor).cpu().numpy(), tokens, 0)
    out, t, xs = Scores(m, 0), torch.from_numpy(tokens).cuda(), xs * factor
    torch.cuda.synchronize()
    um.fp8_linear_logprobs(ctx, x, xs, w, ws, t, **out.views())
    compare(out.host(), want)


@pytest.mark.parametrize("m,n", [(2, 500), (200, 3000), (600, 8000), (7, 66000)])
@pytest.mark.parametrize("offset", [2.0 ** 20, -2.0 ** 22])
def test_linear_logprobs_of_logits_far_from_zero(ctx, m, n, offset):
    """Logits offset + whole numbers of some units: the first block is a constant of
    all words, the second what tells them apart; all sums exact in f32."""
    say(f"fused scores {m}x{n} around {offset}")
    rng = np.random.default_rng(m + n)
    x, w = np.zeros((m, 256)), np.zeros((n, 256))
    x[:, 0], w[:, 0] = 1, np.sign(offset)
    x[:, 128:], w[:, 128:] = rng.integers(-1, 2, (m, 128)), rng.integers(-1, 2, (n, 128))
    scales = np.ones((m, 2), np.float32)
    scales[:, 0] = abs(offset)
    ops = [torch.from_numpy(a).to(torch.float8_e4m3fn).cuda() for a in (x, w)]
    ws = torch.ones((blocks(n), 2), device="cuda")
    tokens = rng.integers(0, n, m).astype(np.int32)
    out = Scores(m, 0)
    torch.cuda.synchronize()
    um.fp8_linear_logprobs(ctx, ops[0], torch.from_numpy(scales).cuda(), ops[1], ws,
                           torch.from_numpy(tokens).cuda(), **out.views())
    compare(out.host(), reference(offset + x[:, 128:] @ w[:, 128:].T, tokens, 0))


@pytest.mark.parametrize("m", [3, 200])
def test_linear_logprobs_errors(ctx, m):
    n, k = 300, 256
    ops = scaled(exact_product(m, n, k, 1), 2.0 ** -8)
    tokens = np.arange(m).astype(np.int32)
    tokens[1] = n
    dev, t = device_product(*ops), torch.from_numpy(tokens).cuda()
    out = Scores(m, 0)
    torch.cuda.synchronize()
    with pytest.raises(um.UocrError) as e:
        um.fp8_linear_logprobs(ctx, *dev, t, **out.views())
    assert e.value.status == um.SHAPE
    want = fused_reference(ops, np.minimum(tokens, n - 1), 0)
    want["logprobs"][1] = math.nan
    compare(out.host(), want)
    x = ops[0].copy()
    x[2, 255] = 0x7f  # a NaN byte: that row's logits are NaN
    dev = device_product(x, *ops[1:])
    out = Scores(m, 0)
    t = torch.from_numpy(np.arange(m).astype(np.int32)).cuda()
    torch.cuda.synchronize()
    with pytest.raises(um.UocrError) as e:
        um.fp8_linear_logprobs(ctx, *dev, t, **out.views())
    assert e.value.status == um.NUMERICAL
    want = fused_reference(ops, np.arange(m).astype(np.int32), 0)
    for v in want.values():
        v[2] = math.nan
    compare(out.host(), want)


def test_linear_logprobs_small_scratch():
    ops = scaled(exact_product(90, 4000, 128, 2), 2.0 ** -9)
    tokens = np.arange(90).astype(np.int32)
    dev, t = device_product(*ops), torch.from_numpy(tokens).cuda()
    for top, size in ((0, 20000), (3, 70000)):
        small = um.Context(0, size)
        out = Scores(90, top)
        torch.cuda.synchronize()
        um.fp8_linear_logprobs(small, *dev, t, **out.views())
        compare(out.host(), fused_reference(ops, tokens, top))
        small.close()
    # Ragged rows, with room for a copy of some of them at a time, and without.
    ops = scaled(exact_product(300, 700, 257, 3), 2.0 ** -9)
    tokens = np.arange(300).astype(np.int32)
    rag, tr = device_product(*ops), torch.from_numpy(tokens).cuda()
    for top, size in ((0, 100000), (0, 250000), (3, 120000), (3, 600000)):
        small = um.Context(0, size)
        out = Scores(300, top)
        torch.cuda.synchronize()
        um.fp8_linear_logprobs(small, *rag, tr, **out.views())
        compare(out.host(), fused_reference(ops, tokens, top))
        small.close()
    tiny = um.Context(0, 256)
    with pytest.raises(um.UocrError) as e:
        um.fp8_linear_logprobs(tiny, *dev, t, **Scores(90, 0).views())
    assert e.value.status == um.RESOURCE
    tiny.close()


# ----------------------------------------------------- the vocabulary head

def head_inputs(rng, T, V, H):
    hidden = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32) * 2).cuda()
    norm = torch.from_numpy((0.5 + rng.random(H)).astype(np.float32)).cuda()
    weight = torch.from_numpy(rng.standard_normal((V, H)).astype(np.float32) * 2.5 / math.sqrt(H)).to(torch.bfloat16)
    tokens = torch.from_numpy(rng.integers(0, V, T).astype(np.int32)).cuda()
    return hidden, norm, weight.cuda(), tokens


def normalized(hidden, norm, eps=1e-6):
    x = hidden.double().cpu().numpy()
    return x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * norm.double().cpu().numpy()


@pytest.mark.parametrize("T,V,H", [(1, 3000, 1280), (7, 1000, 192), (70, 5003, 1280), (5, 300, 100)])
def test_fp8_head(ctx, T, V, H):
    """The head with e4m3 weights: its scores are those of the operators it is made
    of, one after the other, bit for bit; its logits theirs of the last row; and
    all are as near the unquantised model as the quantisation allows (each factor
    off by half an e4m3 step, 2^-4 of it, or half the least step, 2^-10 times its
    scale, against sum|x w|)."""
    say(f"fp8 head T={T} V={V} H={H}")
    rng = np.random.default_rng(T + V)
    hidden, norm, weight, tokens = head_inputs(rng, T, V, H)
    wq = torch.empty((V, H), dtype=torch.uint8, device="cuda")
    ws = torch.empty((blocks(V), blocks(H)), device="cuda")
    torch.cuda.synchronize()
    um.fp8_quantize_weight(ctx, weight, wq, ws)
    head = um.LmHead(ctx, norm, 1e-6, q=wq, scales=ws, mode=um.QUANT_FP8_BLOCKS, where=um.MEMORY_DEVICE)
    assert head.precision == "fp8_weights_dynamic_activations"
    xn = torch.empty_like(hidden)
    xq = torch.empty((T, H), dtype=torch.uint8, device="cuda")
    xs = torch.empty((T, blocks(H)), device="cuda")
    um.rms_norm(ctx, hidden, norm, 1e-6, xn)
    um.fp8_quantize(ctx, xn, xq, xs)
    for top in (0, 4):
        whole, parts = Scores(T, top), Scores(T, top)
        torch.cuda.synchronize()
        head.logprobs(ctx, hidden, tokens, **whole.views())
        um.fp8_linear_logprobs(ctx, xq, xs, wq, ws, tokens, **parts.views())
        a, b = whole.host(), parts.host()
        for k in a:
            assert np.array_equal(a[k], b[k]), k
    x, w = normalized(hidden, norm), weight.double().cpu().numpy()
    sizes = np.abs(x) @ np.abs(w).T
    least = (np.repeat(xs.cpu().numpy().astype(np.float64), 128, 1)[:, :H] @ np.abs(w).T
             + np.abs(x) @ np.repeat(np.repeat(ws.cpu().numpy().astype(np.float64), 128, 0)[:V], 128, 1)[:, :H].T)
    off = (2 * 2.0 ** -4 + 2.0 ** -8) * sizes + 1.1 * 2.0 ** -10 * least
    want = reference(x @ w.T, tokens.cpu().numpy(), 0)
    assert (np.abs(a["logprobs"] - want["logprobs"]) <= 2 * off.max(1)).all()
    logits, row = torch.empty(V, device="cuda"), torch.empty((1, V), device="cuda")
    torch.cuda.synchronize()
    head.logits(ctx, hidden, logits)
    um.fp8_linear(ctx, xq[-1:], xs[-1:], wq, ws, row)
    assert torch.equal(logits, row[0])
    assert (np.abs(logits.cpu().numpy() - (x[-1] @ w.T)) <= off[-1]).all()
    head.close()


@pytest.mark.parametrize("kind", ["bf16", "int8", "w8a8"])
@pytest.mark.parametrize("T,V,H", [(1, 1000, 1280), (3, 517, 96), (37, 2000, 1280)])
def test_other_heads(ctx, kind, T, V, H):
    """BF16 and INT8 heads: logits in f32 sums of another order (H + 32 roundings of
    2^-24 against sum|x w|, and a norm that is off by some H / 64 + 16 of them), and
    one row under W8A8 as uocr_lm_head_logits has it."""
    say(f"{kind} head T={T} V={V} H={H}")
    rng = np.random.default_rng(T + V + H)
    hidden, norm, weight, tokens = head_inputs(rng, T, V, H)
    if kind == "bf16":
        head = um.LmHead(ctx, norm, 1e-6, weight=weight, where=um.MEMORY_DEVICE)
        w = weight.double().cpu().numpy()
    else:
        q = rng.integers(-127, 128, (V, H), dtype=np.int8)
        sc = (rng.random((V, H // 32)) * 6e-4 / math.sqrt(H / 1280)).astype(np.float32)
        head = um.LmHead(ctx, norm, 1e-6, q=torch.from_numpy(q).cuda(), scales=torch.from_numpy(sc).cuda(),
                         mode=um.QUANT_WEIGHTS_ONLY if kind == "int8" else um.QUANT_DYNAMIC,
                         where=um.MEMORY_DEVICE)
        w = q.astype(np.float64) * np.repeat(sc.astype(np.float64), 32, 1)
    out = Scores(T, 0)
    torch.cuda.synchronize()
    head.logprobs(ctx, hidden, tokens, **out.views())
    if kind == "w8a8" and T == 1:
        logits = torch.empty(V, device="cuda")
        torch.cuda.synchronize()
        head.logits(ctx, hidden, logits)
        # The fused head normalises in another order of sums: one int8 step of a
        # value (1/127 of its block's largest) may differ, times its weight.
        x = normalized(hidden, norm)
        extra = float(np.abs(x).max() / 127 * np.abs(w).max())
        compare(out.host(), reference(logits.double().cpu().numpy()[None], tokens.cpu().numpy(), 0), extra)
    else:
        x = normalized(hidden, norm)
        extra = (H + 32 + H / 64 + 16) * U * float((np.abs(x) @ np.abs(w).T).max())
        compare(out.host(), reference(x @ w.T, tokens.cpu().numpy(), 0), extra)
    head.close()


def fp8_head(ctx, norm, weight):
    V, H = weight.shape
    wq = torch.empty((V, H), dtype=torch.uint8, device="cuda")
    ws = torch.empty((blocks(V), blocks(H)), device="cuda")
    torch.cuda.synchronize()
    um.fp8_quantize_weight(ctx, weight, wq, ws)
    return um.LmHead(ctx, norm, 1e-6, q=wq, scales=ws, mode=um.QUANT_FP8_BLOCKS, where=um.MEMORY_DEVICE)


@pytest.mark.parametrize("kind", ["bf16", "fp8"])
@pytest.mark.parametrize("H", [100, 1280, 2000, 2102])
@pytest.mark.parametrize("top", [0, 3])
def test_head_padding_rows_are_not_looked_at(ctx, kind, H, top):
    """A padded batch: what lies in the padding rows (NaN, infinities) changes
    nothing of the others and raises nothing."""
    say(f"{kind} head with padding, H={H} top={top}")
    rng = np.random.default_rng(H)
    hidden, norm, weight, tokens = head_inputs(rng, 9, 700, H)
    pad = [0, 4, 5, 8]
    tokens[pad] = -1
    head = fp8_head(ctx, norm, weight) if kind == "fp8" else \
        um.LmHead(ctx, norm, 1e-6, weight=weight, where=um.MEMORY_DEVICE)
    want, got = Scores(9, top), Scores(9, top)
    torch.cuda.synchronize()
    head.logprobs(ctx, hidden, tokens, **want.views())
    hidden[0], hidden[4], hidden[5, 3], hidden[8, H - 1] = math.nan, math.inf, -math.inf, 3e38
    torch.cuda.synchronize()
    head.logprobs(ctx, hidden, tokens, **got.views())
    a, b = want.host(), got.host()
    for k in a:
        assert np.array_equal(a[k], b[k]), k
    assert (b["logprobs"][pad] == 0).all() and (b["entropy"][pad] == 0).all()
    assert (b["logprobs"][[1, 2, 3, 6, 7]] < 0).all()
    head.close()


def test_head_of_many_logits_and_ragged_width():
    """More outputs than one launch of the plain linear operator has waves for, in a
    scratch that would hold them all: the rows are taken in turn."""
    big = um.Context(0, 1 << 30)
    T, V, H = 3500, 20000, 20
    say(f"bf16 head T={T} V={V} H={H}")
    hidden, norm, weight, tokens = head_inputs(np.random.default_rng(5), T, V, H)
    head = um.LmHead(big, norm, 1e-6, weight=weight, where=um.MEMORY_DEVICE)
    out = Scores(T, 0)
    torch.cuda.synchronize()
    head.logprobs(big, hidden, tokens, **out.views())
    x, w = normalized(hidden, norm), weight.double().cpu().numpy()
    rows = [0, 1, 1700, 3354, 3355, 3356, 3499]
    extra = (H + 32 + H / 64 + 16) * U * float((np.abs(x[rows]) @ np.abs(w).T).max())
    got = {k: v[rows] for k, v in out.host().items()}
    compare(got, reference(x[rows] @ w.T, tokens.cpu().numpy()[rows], 0), extra)
    head.close()
    big.close()


def test_head_refusals(ctx):
    rng = np.random.default_rng(1)
    hidden, norm, weight, tokens = head_inputs(rng, 4, 300, 256)
    wq = torch.zeros((300, 256), dtype=torch.uint8, device="cuda")
    ws = torch.ones((3, 2), device="cuda")

    def status(q, s):
        torch.cuda.synchronize()
        with pytest.raises(um.UocrError) as e:
            um.LmHead(ctx, norm, 1e-6, q=q, scales=s, mode=um.QUANT_FP8_BLOCKS, where=um.MEMORY_DEVICE)
        return e.value.status
    bad = wq.clone()
    bad[299, 255] = 0xff
    assert status(bad, ws) == um.FORMAT
    for v in (float("nan"), float("inf"), -1.0):
        s = ws.clone()
        s[2, 1] = v
        assert status(wq, s) == um.NUMERICAL
    assert status(wq, None) == um.FORMAT
    head = um.LmHead(ctx, norm, 1e-6, q=wq, scales=ws, mode=um.QUANT_FP8_BLOCKS, where=um.MEMORY_DEVICE)
    out = Scores(4, 2)
    hidden[2, 7] = float("nan")
    torch.cuda.synchronize()
    with pytest.raises(um.UocrError) as e:
        head.logprobs(ctx, hidden, tokens, **out.views())
    assert e.value.status == um.NUMERICAL
    with pytest.raises(um.UocrError) as e:
        head.logprobs(ctx, hidden, None, logprobs=out.views()["logprobs"])
    assert e.value.status == um.SHAPE
    head.logprobs(ctx, hidden[:0], tokens[:0], logprobs=out.views()["logprobs"][:0])
    head.close()


@pytest.mark.parametrize("vocab", [4000, 20000])
def test_scores_in_a_graph(ctx, vocab):
    """Captured scoring replays with the eager bits, eager work in between; the
    logits change between replays."""
    rng = np.random.default_rng(11)
    hidden, norm, weight, tokens = head_inputs(rng, 33, 4000, 640)
    wq = torch.empty((4000, 640), dtype=torch.uint8, device="cuda")
    ws = torch.empty((blocks(4000), 5), device="cuda")
    torch.cuda.synchronize()
    um.fp8_quantize_weight(ctx, weight, wq, ws)
    head = um.LmHead(ctx, norm, 1e-6, q=wq, scales=ws, mode=um.QUANT_FP8_BLOCKS, where=um.MEMORY_DEVICE)
    x = logits_of(rng, 33, vocab, torch.bfloat16).cuda()
    got, want = [Scores(33, 0), Scores(33, 5), Scores(33, 5)], [Scores(33, 0), Scores(33, 5), Scores(33, 5)]

    def work(out, sync):
        head.logprobs(ctx, hidden, tokens, **out[0].views(), sync=sync)
        head.logprobs(ctx, hidden, tokens, **out[1].views(), sync=sync)
        um.token_logprobs(ctx, x, tokens, **out[2].views(), sync=sync)
    torch.cuda.synchronize()
    work(want, True)
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(ctx.stream)):
        work(got, False)
    for rep in range(4):
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            a, b = a.host(), b.host()
            assert all(np.array_equal(a[k], b[k]) for k in a), rep
        hidden.mul_(-1.25)
        x.neg_()
        torch.cuda.synchronize()
        work(want, True)
    ctx.synchronize()
    head.close()

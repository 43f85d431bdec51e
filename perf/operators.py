"""Workloads of the 8-bit floating point operators and of token scoring.

Four operators, each with cases of its own; `op` says which:

* "quantize": rows in e4m3 with one scale per 128 columns of a row;
* "linear": the product of such rows with an e4m3 matrix that has one scale per
  128 x 128 tile;
* "score": log probabilities of given tokens, entropy and the most probable
  alternatives, from logits;
* "linear_score": log probabilities and entropy straight from the product, without
  logits in memory.

Sizes are the decoder's: hidden 1280, expert width 896, the dense layer's width
6848, vocabulary 129280.
"""
import functools
import math
import os
import sys

import torch

own = False

H, I, DENSE, V = 1280, 896, 6848, 129280
BLOCK = 128
MOST = 448.0  # the largest e4m3
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _quantize(name, rows, cols, dtype):
    return {"name": name, "op": "quantize", "rows": rows, "cols": cols, "dtype": dtype}


def _linear(name, m, n, k, dtype):
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype}


def _score(name, rows, vocab, top, dtype, padded=False, banned=False):
    return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "top": top, "dtype": dtype,
            "padded": padded, "banned": banned}


def _linear_score(name, m, n, k):
    return {"name": name, "op": "linear_score", "m": m, "n": n, "k": k}


def listed():
    return [
        # The hidden row of one generated token.
        _quantize("quantize_token", 1, H, "f32"),
        # The hidden rows of a long prompt before the dense layer's down product;
        # the last block of a row has 64 columns.
        _quantize("quantize_prompt", 4096, DENSE, "bf16"),
        # An expert's down product for one generated token.
        _linear("linear_token", 1, H, I, "f32"),
        # The dense layer's up product for sixteen sequences decoded together.
        _linear("linear_batch", 16, DENSE, H, "bf16"),
        # The dense layer's down product over the image tokens of one page: few
        # rows and columns, long sums.
        _linear("linear_page", 277, H, DENSE, "f32"),
        # The dense layer's up product over a long prompt.
        _linear("linear_prompt", 4096, DENSE, H, "bf16"),
        # Choosing the next token of one sequence from its logits.
        _score("score_token", 1, V, 5, "f32"),
        # A padded batch of sequences whose repeated words are banned.
        _score("score_batch", 61, V, 20, "bf16", padded=True, banned=True),
        # A recognised page's text scored with its alternatives.
        _score("score_page", 1517, V, 5, "f32"),
        # The confidence of each token as it is generated.
        _linear_score("linear_score_token", 1, V, H),
        # The same for a batch of sequences.
        _linear_score("linear_score_batch", 48, V, H),
        # Long recognised texts scored in one pass.
        _linear_score("linear_score_prompt", 4096, V, H),
    ]


def _spread(rng, least, most):
    return min(most, max(least, int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "score", "linear_score"])
    if op == "quantize":
        c = _quantize("", _spread(rng, 1, 4096), _spread(rng, 1, DENSE), rng.choice(["f32", "bf16"]))
    elif op == "linear":
        # Widths as layers have them, and others down to a single one.
        n = rng.choice([I, H, 2 * I, DENSE, _spread(rng, 1, DENSE)])
        k = rng.choice([I, H, 2 * I, DENSE, _spread(rng, 1, DENSE)])
        m = _spread(rng, 1, 4096)
        if m * n * k > 4096 * DENSE * H:
            m = 4096 * DENSE * H // (n * k)
        c = _linear("", m, n, k, rng.choice(["f32", "bf16"]))
    elif op == "score":
        vocab = rng.choice([V, _spread(rng, 32, V)])
        c = _score("", _spread(rng, 1, 1517), vocab, rng.randint(0, min(20, vocab)),
                   rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.5, rng.random() < 0.5)
    else:
        c = _linear_score("", _spread(rng, 1, 4096), rng.choice([V, _spread(rng, 32, V)]),
                          rng.choice([I, H, _spread(rng, 16, H)]))
    del c["name"]
    return c


# ------------------------------------------------------------------- inputs

def _blocks(n):
    return -(-n // BLOCK)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _power(e, dtype=torch.float32):
    """2^e of whole numbers e, exactly: the exponent's bits."""
    if dtype == torch.float64:
        return ((e.long() + 1023) << 52).view(torch.float64)
    return ((e.int() + 127) << 23).view(torch.float32)


def _hidden_rows(g, rows, cols):
    """Activations: Gaussian, each row with a size of its own and a few columns
    that are much larger than the others, as hidden states have them."""
    x = torch.randn((rows, cols), generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=g, device="cuda"))
    loud = torch.rand((1, cols), generator=g, device="cuda") < 0.005
    return torch.where(loud, 12 * x, x)


def _row_blocks(x):
    """[rows, cols] as [rows, blocks, 128], zeros behind the last column."""
    rows, cols = x.shape
    return torch.nn.functional.pad(x, (0, _blocks(cols) * BLOCK - cols)).view(rows, -1, BLOCK)


def _quantized_rows(x):
    """e4m3 rows and their scales, made here by any scale that fits (amax / 448,
    not a power of two): a product takes the scales that it is given."""
    b = _row_blocks(x)
    s = b.abs().amax(-1, keepdim=True).clamp_min(1e-12) / MOST
    q = (b / s).clamp(-MOST, MOST).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return q.contiguous().to(torch.float8_e4m3fn), s[..., 0].contiguous()


def _quantized_matrix(g, n, k, std):
    w = std * torch.randn((n, k), generator=g, device="cuda")
    p = torch.nn.functional.pad(w, (0, _blocks(k) * BLOCK - k, 0, _blocks(n) * BLOCK - n))
    p = p.view(_blocks(n), BLOCK, _blocks(k), BLOCK)
    s = p.abs().amax((1, 3)) / MOST
    q = (p / s[:, None, :, None]).clamp(-MOST, MOST).reshape(_blocks(n) * BLOCK, -1)[:n, :k]
    return q.contiguous().to(torch.float8_e4m3fn), s.contiguous()


def prepare(case, seed):
    g = _generator(seed)
    if case["op"] == "quantize":
        rows, cols = case["rows"], case["cols"]
        return {"case": case, "x": _hidden_rows(g, rows, cols).to(TYPES[case["dtype"]]),
                "q": torch.empty((rows, cols), dtype=torch.float8_e4m3fn, device="cuda"),
                "scales": torch.empty((rows, _blocks(cols)), device="cuda")}
    if case["op"] == "score":
        rows, vocab, top = case["rows"], case["vocab"], case["top"]
        # Logits of a language model: a broad bulk, and a few words far above it,
        # in some rows one word that is nearly certain.
        x = 2.0 * torch.randn((rows, vocab), generator=g, device="cuda") - 2.0
        best = torch.randint(vocab, (rows, 12), generator=g, device="cuda")
        lift = 6.0 + 5.0 * torch.rand((rows, 12), generator=g, device="cuda")
        x.scatter_reduce_(1, best, lift, "amax")
        tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.8, best[:, 0],
                             torch.randint(vocab, (rows,), generator=g, device="cuda"))
        if case["banned"]:
            ban = torch.randint(vocab, (rows, 1 + vocab // 200), generator=g, device="cuda")
            x.scatter_(1, ban, -math.inf)
        if case["padded"]:
            # The sequences' ends: no token was given there.
            tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.25, -1, tokens)
        s = {"case": case, "logits": x.to(TYPES[case["dtype"]]), "tokens": tokens.to(torch.int32)}
        if top:
            s["top_ids"] = torch.empty((rows, top), dtype=torch.int32, device="cuda")
            s["top_logprobs"] = torch.empty((rows, top), device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        x = _hidden_rows(g, m, k)
        if case["op"] == "linear_score":  # behind the final norm
            x *= torch.rsqrt(x.square().mean(1, keepdim=True))
        xq, xs = _quantized_rows(x)
        # Sums of the products with a spread of about 2.5 (logits) or 1.
        std = (2.5 if case["op"] == "linear_score" else 1.0) / math.sqrt(k)
        wq, ws = _quantized_matrix(g, n, k, std)
        s = {"case": case, "xq": xq, "xs": xs, "wq": wq, "ws": ws}
        if case["op"] == "linear":
            s["y"] = torch.empty((m, n), dtype=TYPES[case["dtype"]], device="cuda")
            return s
        rows = m
        s["tokens"] = torch.randint(n, (m,), generator=g, device="cuda").to(torch.int32)
    s["logprobs"] = torch.empty(rows, device="cuda")
    s["entropy"] = torch.empty(rows, device="cuda")
    return s


# ---------------------------------------------------------- the plain form

def _plain_quantize(x):
    b = _row_blocks(x.float())
    most = b.abs().amax(-1, keepdim=True)
    fraction, exponent = torch.frexp(most)  # most = fraction * 2^exponent, 1/2 <= fraction < 1
    # The least e with most / 2^e <= 448 = 0.875 * 2^9.
    e = (exponent - 9 + (fraction > 0.875).int()).clamp_min(-126)
    e = torch.where(most > 0, e, 0)
    q = (b * _power(-e)).reshape(x.shape[0], -1)[:, :x.shape[1]]
    return q.to(torch.float8_e4m3fn), _power(e)[..., 0]


def _dequantized(q, s, rows_per_scale):
    """The f32 (or, with f64 scales, f64) values of an e4m3 matrix."""
    n, k = q.shape
    s = s.repeat_interleave(BLOCK, 1)[:, :k]
    if rows_per_scale > 1:
        s = s.repeat_interleave(rows_per_scale, 0)[:n]
    return q.to(s.dtype) * s


def _plain_product(s):
    return _dequantized(s["xq"], s["xs"], 1) @ _dequantized(s["wq"], s["ws"], BLOCK).t()


def _plain_score(logits, tokens, top):
    x = logits.float()
    skipped = tokens < 0
    most = x.amax(1, keepdim=True)
    d = x - most
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    given = d.gather(1, tokens.clamp_min(0).long()[:, None])[:, 0]
    spread = torch.where(e > 0, e * d, 0.0).sum(1)
    out = {"logprobs": torch.where(skipped, 0.0, given - log_total),
           "entropy": torch.where(skipped, 0.0, log_total - spread / total)}
    if top:
        # Largest first, and of equal logits the one of the lower index: one whole
        # number of 64 bits orders both.
        bits = logits.float().view(torch.int32).long()
        bits = torch.where(bits == -2 ** 31, 0, bits)  # -0 is 0
        order = torch.where(bits < 0, -(bits + 2 ** 31), bits)
        index = torch.arange(x.shape[1], device=x.device)
        ids = ((order << 32) + (2 ** 31 - index)).topk(top, 1).indices
        out["top_ids"] = torch.where(skipped[:, None], -1, ids).to(torch.int32)
        out["top_logprobs"] = torch.where(skipped[:, None], -math.inf,
                                          d.gather(1, ids) - log_total[:, None])
    return out


def _plain(s):
    c = s["case"]
    if c["op"] == "quantize":
        q, scales = _plain_quantize(s["x"])
        return {"q": q, "scales": scales}
    if c["op"] == "linear":
        return _plain_product(s).to(TYPES[c["dtype"]])
    if c["op"] == "score":
        return _plain_score(s["logits"], s["tokens"], c["top"])
    return _plain_score(_plain_product(s), s["tokens"], 0)


# ------------------------------------------------------ the framework's form

@functools.lru_cache(maxsize=None)
def _framework():
    """The package and the context that a program makes once."""
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "unlimited-ocr-kernel_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import uocr_moe as um
    return um, um.Context(0, 256 << 20)


def _own(s):
    um, ctx = _framework()
    op = s["case"]["op"]
    if op == "quantize":
        um.fp8_quantize(ctx, s["x"], s["q"], s["scales"], sync=False)
        return {"q": s["q"], "scales": s["scales"]}
    if op == "linear":
        um.fp8_linear(ctx, s["xq"], s["xs"], s["wq"], s["ws"], s["y"], sync=False)
        return s["y"]
    out = {"logprobs": s["logprobs"], "entropy": s["entropy"]}
    if op == "score":
        if "top_ids" in s:
            out.update(top_ids=s["top_ids"], top_logprobs=s["top_logprobs"])
        um.token_logprobs(ctx, s["logits"], s["tokens"], **out, sync=False)
    else:
        um.fp8_linear_logprobs(ctx, s["xq"], s["xs"], s["wq"], s["ws"], s["tokens"], **out,
                               sync=False)
    return out


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------- work, exact

def work(case):
    c = case
    if c["op"] == "quantize":
        size = 4 if c["dtype"] == "f32" else 2
        return {"bytes": c["rows"] * (c["cols"] * (size + 1) + _blocks(c["cols"]) * 4),
                "flops": 2 * c["rows"] * c["cols"]}
    if c["op"] == "score":
        size = 4 if c["dtype"] == "f32" else 2
        # A quarter of a padded batch's rows need not be read.
        rows = c["rows"] * (0.75 if c["padded"] else 1.0)
        return {"bytes": rows * c["vocab"] * size + c["rows"] * (12 + 8 * c["top"]),
                "flops": 5 * rows * c["vocab"]}
    m, n, k = c["m"], c["n"], c["k"]
    size = m * k + n * k + 4 * _blocks(k) * (m + _blocks(n))
    if c["op"] == "linear":
        return {"bytes": size + m * n * (4 if c["dtype"] == "f32" else 2), "flops": 2 * m * n * k}
    return {"bytes": size + 12 * m, "flops": 2 * m * n * k + 5 * m * n}


def _exact_rows(x, tokens, top):
    """Scores of f64 logits, row by row of the definition."""
    p = torch.softmax(x, 1)
    logp = torch.log_softmax(x, 1)
    skipped = tokens < 0
    out = {"logprobs": logp.gather(1, tokens.clamp_min(0).long()[:, None])[:, 0],
           "entropy": -torch.where(p > 0, p * logp, 0.0).sum(1)}
    out = {k: v.masked_fill(skipped, 0.0) for k, v in out.items()}
    if top:
        ids = x.sort(dim=1, descending=True, stable=True).indices[:, :top]
        out["top_ids"] = ids.masked_fill(skipped[:, None], -1).to(torch.int32)
        out["top_logprobs"] = logp.gather(1, ids).masked_fill(skipped[:, None], -math.inf)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        x = s["x"].double()
        rows, cols = x.shape
        width = _blocks(cols) * BLOCK
        b = torch.zeros((rows, width), dtype=torch.float64, device="cuda")
        b[:, :cols] = x
        b = b.view(rows, -1, BLOCK)
        most = b.abs().amax(-1)
        e = torch.ceil(torch.log2(most / MOST)).clamp_min(-126)
        # log2 rounds: put right by the definition itself, the least e with most <= 448 * 2^e.
        e = torch.where(most <= MOST * _power(e - 1, most.dtype), e - 1, e)
        e = torch.where(most > MOST * _power(e, most.dtype), e + 1, e).clamp_min(-126)
        scale = torch.where(most > 0, _power(e, most.dtype), 1.0)
        v = b / scale[..., None]
        # Nearest e4m3, ties to even: a step of 2^(exponent - 3), no finer than 2^-9.
        step = _power(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3, v.dtype)
        q = (torch.round(v / step) * step).view(rows, -1)[:, :cols]
        return {"q": q, "scales": scale}
    if case["op"] == "linear":
        x = _dequantized(s["xq"], s["xs"].double(), 1)
        w = _dequantized(s["wq"], s["ws"].double(), BLOCK)
        return torch.mm(x, w.t())
    parts, rows = [], 256
    if case["op"] == "linear_score":
        x = _dequantized(s["xq"], s["xs"].double(), 1)
        w = _dequantized(s["wq"], s["ws"].double(), BLOCK).t().contiguous()
    for r in range(0, s["tokens"].shape[0], rows):
        part = (s["logits"][r:r + rows].double() if case["op"] == "score"
                else torch.mm(x[r:r + rows], w))
        parts.append(_exact_rows(part, s["tokens"][r:r + rows], case.get("top", 0)))
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}

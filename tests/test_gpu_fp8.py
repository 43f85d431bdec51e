"""The 8-bit floating point operators (uocr_fp8_quantize, uocr_fp8_linear) against
their definitions in 64 bits on the CPU.

The product's tolerance: x w of two e4m3 values is exact in f32, and a sum of k
terms in any order is off by at most (k - 1) roundings of partial sums, none of
which exceeds sum|x w|. A rounding to nearest is 2^-24; the matrix instruction's own
additions may cut off instead, which is twice that. Scaling a block adds a product
of the scales, a product and a sum. So |error| <= 2 (k + 3 blocks) 2^-24 sum|x w|
xs ws; a bf16 result is rounded once more, 2^-8 of it. bf16 results of more than 64
rows come from the e4m3 matrix instruction, which cuts each product of a group of eight
off 13 bits below the exponent of the group's largest one: each loses less than 2^-13
of that one, the group less than 8 times that, and the largest is at most the group's
sum|x w|, so 2^-10 sum|x w| more. Where all values and partial
sums are whole numbers below 2^24 (times one power of two) nothing is rounded, and
the result is exact."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import uocr_moe as um  # noqa: E402

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    c = um.Context(0, 256 << 20)
    yield c
    c.close()


def say(msg):
    print(msg, flush=True)


def blocks(n):
    return -(-n // 128)


# e4m3 as values: sign, 4 exponent bits (bias 7), 3 mantissa bits; no infinities,
# 0x7f NaN.
def _e4m3():
    v = []
    for b in range(128):
        e, m = b >> 3, b & 7
        v.append(m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10))
    v[127] = np.nan
    return np.array(v + [-a for a in v])


E4M3 = _e4m3()


def nearest_e4m3(v):
    """Index of the nearest e4m3 magnitude, ties to the even mantissa."""
    grid = E4M3[:127]
    a = np.abs(v)
    hi = np.clip(np.searchsorted(grid, a), 1, 126)
    lo = hi - 1
    dl, dh = a - grid[lo], grid[hi] - a
    return np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)


def scale_of(most):
    """The least power of two s with most / s <= 448, at least 2^-126; 1 for 0."""
    if most == 0:
        return 1.0
    e = -126
    m, x = np.frexp(float(most))  # most = m 2^x
    e = max(e, int(x) - 9 + (m > 0.875))
    return 2.0 ** e


def quantized(x, tile_rows=1):
    """(codes, scales) by the definition; x float64."""
    rows, cols = x.shape
    q = np.zeros(x.shape, np.uint8)
    s = np.ones((blocks(rows) if tile_rows > 1 else rows, blocks(cols)))
    for i in range(s.shape[0]):
        for b in range(s.shape[1]):
            at = (slice(i * tile_rows, (i + 1) * tile_rows), slice(128 * b, 128 * b + 128))
            s[i, b] = scale_of(np.abs(x[at]).max())
            v = x[at] / s[i, b]
            q[at] = nearest_e4m3(v) | np.where(np.signbit(v), 0x80, 0)
    return q, s


def check_codes(got, want):
    same = (got == want) | ((got & 0x7f == 0) & (want & 0x7f == 0))
    assert same.all(), np.argwhere(~same)[:5]


def rows_of(rng, rows, cols):
    x = rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1)))
    x[:, rng.random(cols) < 0.05] *= 30
    return x


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 1280), (3, 7), (5, 128), (4, 129), (2, 896), (17, 1000),
                                       (63, 2047), (300, 640)])
def test_quantize_rows(ctx, rows, cols, dtype):
    say(f"quantize {rows}x{cols} {dtype}")
    t = getattr(torch, dtype)
    rng = np.random.default_rng(rows * 7 + cols)
    x = torch.from_numpy(rows_of(rng, rows, cols)).to(t)
    want_q, want_s = quantized(x.double().numpy())
    # Contiguous; a wider row stride; a base that allows no wide loads.
    wide = torch.zeros(rows, cols + 24, dtype=t)
    wide[:, 8:8 + cols] = x
    odd = torch.zeros(rows * cols + 1, dtype=t)
    odd[1:] = x.reshape(-1)
    for form in (x.cuda(), wide.cuda()[:, 8:8 + cols], odd.cuda()[1:].view(rows, cols)):
        q = torch.full((rows, cols), 0x55, dtype=torch.uint8, device="cuda")
        s = torch.full((rows, blocks(cols)), float("nan"), device="cuda")
        torch.cuda.synchronize()
        um.fp8_quantize(ctx, form, q, s)
        assert np.array_equal(s.cpu().numpy().astype(np.float64), want_s)
        check_codes(q.cpu().numpy(), want_q)
        # What the values stand for, quantised again, is the same.
        back = torch.from_numpy(E4M3[q.cpu().numpy()] * np.repeat(want_s, 128, 1)[:, :cols]).float()
        q2, s2 = torch.empty_like(q), torch.empty_like(s)
        torch.cuda.synchronize()
        um.fp8_quantize(ctx, back.cuda(), q2, s2)
        assert np.array_equal((E4M3[q2.cpu().numpy()] * np.repeat(s2.cpu().numpy(), 128, 1)[:, :cols]),
                              back.double().numpy())


def test_quantize_special_blocks(ctx):
    """Blocks of zeros, of the smallest and largest numbers, and largest
    magnitudes on both sides of 448 times a power of two; ties."""
    f = np.float32
    most = [0.0, 448.0, np.nextafter(f(448), f(449)), 449.0, 511.99, 512.0, 1.0, 1.75, 1.7500001,
            2.0 ** -149, 2.0 ** -126, 448 * 2.0 ** -126, 448 * 2.0 ** -126 * 1.0000002, 2.0 ** -118, np.finfo(f).max,
            1e-30, 3.5, 28.0]
    x = np.zeros((len(most), 128), f)
    rng = np.random.default_rng(3)
    for i, m in enumerate(most):
        x[i] = rng.uniform(-1, 1, 128).astype(f) * f(m)
        x[i, 5] = -m
        x[i, 6] = -0.0
    x[16, :16] = np.arange(16) / 16 * 0.25 + 3.0  # ties between steps
    x[17, :8] = 28 * np.array([1.5, 2.5, 0.5, 3.5, 4.5, 1, 2, 3]) * 2.0 ** -13
    want_q, want_s = quantized(x.astype(np.float64))
    q = torch.empty((len(most), 128), dtype=torch.uint8, device="cuda")
    s = torch.empty((len(most), 1), device="cuda")
    d = torch.from_numpy(x).cuda()
    torch.cuda.synchronize()
    um.fp8_quantize(ctx, d, q, s)
    assert np.array_equal(s.cpu().numpy().astype(np.float64), want_s)
    check_codes(q.cpu().numpy(), want_q)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_quantize_refuses_nonfinite(ctx, value, dtype):
    x = torch.ones(4, 300, dtype=getattr(torch, dtype), device="cuda")
    x[2, 299] = value
    q = torch.empty((4, 300), dtype=torch.uint8, device="cuda")
    s = torch.empty((4, 3), device="cuda")
    torch.cuda.synchronize()
    for args in ((um.fp8_quantize, s), (um.fp8_quantize_weight, s[:1])):
        with pytest.raises(um.UocrError) as e:
            args[0](ctx, x, q, args[1])
        assert e.value.status == um.NUMERICAL
    um.fp8_quantize(ctx, x[:2], q[:2], s[:2])  # and the next call is fine
    assert float(s[0, 0].item()) == 2.0 ** -8


@pytest.mark.parametrize("rows,cols", [(1, 1), (128, 128), (129, 300), (200, 1280), (127, 127), (300, 100)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_quantize_weight(ctx, rows, cols, dtype):
    say(f"quantize weight {rows}x{cols} {dtype}")
    t = getattr(torch, dtype)
    x = torch.from_numpy(rows_of(np.random.default_rng(rows + cols), rows, cols)).to(t)
    want_q, want_s = quantized(x.double().numpy(), 128)
    wide = torch.zeros(rows, cols + 5, dtype=t)
    wide[:, 3:3 + cols] = x
    for form in (x.cuda(), wide.cuda()[:, 3:3 + cols]):
        q = torch.empty((rows, cols), dtype=torch.uint8, device="cuda")
        s = torch.empty((blocks(rows), blocks(cols)), device="cuda")
        torch.cuda.synchronize()
        um.fp8_quantize_weight(ctx, form, q, s)
        assert np.array_equal(s.cpu().numpy().astype(np.float64), want_s)
        check_codes(q.cpu().numpy(), want_q)


# ------------------------------------------------------------------- product

# Rows: one, few, around 16, 32, 64, 128, 256; columns and depths that end
# inside a block, rows of bytes that start at any address, and whole ones.
PRODUCTS = [(1, 1, 1), (1, 1280, 896), (2, 130, 15), (3, 50, 1280), (5, 257, 129), (1, 129, 128),
            (15, 16, 16), (16, 896, 1280), (17, 300, 100), (31, 128, 272), (32, 384, 640), (33, 129, 1000),
            (48, 1000, 1280), (63, 64, 6848), (64, 65, 2500), (65, 1280, 896), (127, 513, 384),
            (128, 128, 128), (129, 640, 127), (200, 1000, 1296), (255, 256, 1281), (256, 256, 256),
            (257, 257, 257), (277, 1280, 6848), (300, 2000, 1280), (513, 896, 400), (700, 6848, 144)]


def device_product(x, xs, w, ws, offset=0):
    """The operands on the device, the bytes from an address `offset` past an
    allocation's start."""
    def put(a):
        flat = torch.zeros(a.size + offset, dtype=torch.uint8)
        flat[offset:] = torch.from_numpy(a.reshape(-1))
        return flat.cuda()[offset:].view(a.shape)
    return (put(x), torch.from_numpy(xs.astype(np.float32)).cuda(), put(w),
            torch.from_numpy(ws.astype(np.float32)).cuda())


def spread(x, xs, w, ws):
    """The operands' values in float64."""
    k = x.shape[1]
    return (E4M3[x] * np.repeat(xs, 128, 1)[:, :k],
            E4M3[w] * np.repeat(np.repeat(ws, 128, 0)[:w.shape[0]], 128, 1)[:, :k])


def random_product(m, n, k, seed):
    rng = np.random.default_rng(seed)
    x, w = (rng.integers(0, 256, s).astype(np.uint8) for s in ((m, k), (n, k)))
    x[x & 0x7f == 0x7f] = 0x3a
    w[w & 0x7f == 0x7f] = 0xb1
    return (x, np.exp(rng.uniform(-6, 2, (m, blocks(k)))).astype(np.float32),
            w, np.exp(rng.uniform(-6, 2, (blocks(n), blocks(k)))).astype(np.float32))


def exact_product(m, n, k, seed):
    """Whole numbers whose every partial sum is below 2^24: |x|, |w| <= 4, 16 k <=
    2^17, scales 1, 2, 4 and 8 (their product up to 64)."""
    rng = np.random.default_rng(seed)
    codes = {int(v): i for i, v in enumerate(E4M3) if v == v and v == int(v) and abs(v) <= 4}
    lut = np.array([codes[v] for v in range(-4, 5)], np.uint8)
    x, w = (lut[rng.integers(0, 9, s)] for s in ((m, k), (n, k)))
    return (x, 2.0 ** rng.integers(0, 4, (m, blocks(k))), w, 2.0 ** rng.integers(0, 4, (blocks(n), blocks(k))))


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear_exact(ctx, m, n, k):
    say(f"exact product {m}x{n}x{k}")
    ops = exact_product(m, n, k, m + n + k)
    a, b = spread(*ops)
    want = a @ b.T
    assert np.abs(want).max() < 2 ** 24
    guard = torch.full((m * n + 64,), 12345.0, device="cuda")
    for offset in (0, 3) if m * n < 100000 else (0,):
        dev = device_product(*ops, offset=offset)
        guard.fill_(12345.0)
        y = guard[:m * n].view(m, n)
        torch.cuda.synchronize()
        um.fp8_linear(ctx, *dev, y)
        got = y.cpu().numpy().astype(np.float64)
        assert np.array_equal(got, want), np.argwhere(got != want)[:5]
        assert bool((guard[m * n:] == 12345.0).all())  # nothing behind the last row
        g16 = torch.full((m * n + 64,), 77.0, device="cuda", dtype=torch.bfloat16)
        torch.cuda.synchronize()
        um.fp8_linear(ctx, *dev, g16[:m * n].view(m, n))
        assert torch.equal(g16[:m * n].view(m, n).cpu(), torch.from_numpy(want).float().to(torch.bfloat16))
        assert bool((g16[m * n:] == 77.0).all())


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_linear_random(ctx, m, n, k):
    say(f"random product {m}x{n}x{k}")
    ops = random_product(m, n, k, 3 * m + n + k)
    a, b = spread(*ops)
    want, size = a @ b.T, np.abs(a) @ np.abs(b).T
    tol = 2 * (k + 3 * blocks(k)) * U * size
    dev = device_product(*ops)
    y = torch.full((m, n), float("nan"), device="cuda")
    y2, y16 = torch.empty_like(y), torch.full((m, n), float("nan"), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    um.fp8_linear(ctx, *dev, y)
    um.fp8_linear(ctx, *dev, y2)
    um.fp8_linear(ctx, *dev, y16)
    off = np.abs(y.cpu().numpy() - want)
    say(f"  rel {np.linalg.norm(off) / np.linalg.norm(want):.2e} of the bound {np.max(off / tol):.3f}")
    assert (off <= tol).all()
    assert torch.equal(y, y2)  # equal calls, equal bits
    off = np.abs(y16.double().cpu().numpy() - want)
    tol += 2.0 ** -10 * size
    assert (off <= tol + 2.0 ** -8 * (np.abs(want) + tol)).all()


# More than 64 rows of products too small for the tiles: 64 rows to a workgroup, the
# last ones with 1 to 64, and depths shared by up to sixteen waves.
MANY_SMALL = [(65, 33, 16), (65, 1300, 896), (100, 700, 272), (129, 2100, 1296), (191, 16, 640), (200, 1, 128),
              (300, 130, 6848), (1000, 17, 400), (2049, 65, 144),
              (129, 1900, 1296), (600, 500, 272)]
# At most 64 rows of a depth that is long for its columns, and of many columns.
FEW_DEEP = [(1, 256, 8192), (20, 512, 4096), (33, 129, 2080), (48, 2052, 2192), (64, 300, 6848), (17, 30001, 656)]
# Rows that end anywhere: read where they are by few rows, copied for the tiles otherwise.
RAGGED = [(1, 256, 8191), (20, 512, 4093), (48, 300, 6846), (33, 257, 1281), (100, 700, 901), (300, 1280, 2190),
          (600, 3000, 1001), (1000, 17, 399), (64, 5000, 1279), (2, 6848, 3), (500, 900, 13)]


@pytest.mark.parametrize("m,n,k", MANY_SMALL + FEW_DEEP + RAGGED)
def test_linear_many_rows_of_small_products(ctx, m, n, k):
    say(f"small product {m}x{n}x{k}")
    test_linear_exact(ctx, m, n, k)
    test_linear_random(ctx, m, n, k)


@pytest.mark.parametrize("m,n,k", [(3, 44, 272), (70, 600, 144), (300, 1280, 2192), (520, 8192, 128), (2, 66000, 144),
                                   (5, 64, 100)])
def test_linear_results_at_any_element(ctx, m, n, k):
    """Results that start one element behind an aligned address, and nothing beside them."""
    say(f"unaligned result {m}x{n}x{k}")
    ops = exact_product(m, n, k, m + n)
    a, b = spread(*ops)
    want = torch.from_numpy(a @ b.T)
    dev = device_product(*ops)
    for dtype in (torch.float32, torch.bfloat16):
        guard = torch.full((m * n + 2,), 77.0, device="cuda", dtype=dtype)
        torch.cuda.synchronize()
        um.fp8_linear(ctx, *dev, guard[1:-1].view(m, n))
        assert torch.equal(guard[1:-1].view(m, n).cpu(), want.float().to(dtype))
        assert float(guard[0]) == float(guard[-1]) == 77.0


def test_linear_most_rows(ctx):
    """As many rows as a call takes, of one column: whole numbers again."""
    m, k = 1 << 22, 16
    for rows in (m, m - 64, m - 65):
        say(f"product {rows}x1x{k}")
        x = (torch.arange(rows * k, device="cuda", dtype=torch.int64) % 9 - 4).float().view(rows, k)
        w = torch.tensor([[float(i % 5) for i in range(k)]], device="cuda")
        xq, wq = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
        xs, ws = torch.full((rows, 1), 2.0, device="cuda"), torch.ones((1, 1), device="cuda")
        y = torch.zeros((rows, 1), device="cuda")
        torch.cuda.synchronize()
        um.fp8_linear(ctx, xq, xs, wq, ws, y)
        assert torch.equal(y[:, 0], 2 * (x * w).sum(1))


def device_exact(m, n, k, seed):
    """exact_product made on the device, with its result there in float64."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    codes = {int(v): i for i, v in enumerate(E4M3) if v == v and v == int(v) and abs(v) <= 4}
    lut = torch.tensor([codes[v] for v in range(-4, 5)], dtype=torch.uint8, device="cuda")

    def operand(rows, tile):
        v = torch.randint(0, 9, (rows, k), generator=g, device="cuda")
        s = 2.0 ** torch.randint(0, 4, (blocks(rows) if tile else rows, blocks(k)), generator=g, device="cuda")
        f = s.repeat_interleave(128, 1)[:, :k]
        f = f.repeat_interleave(128, 0)[:rows] if tile else f
        return lut[v], s.float(), (v - 4).double() * f
    x, xs, a = operand(m, False)
    w, ws, b = operand(n, True)
    return (x, xs, w, ws), torch.mm(a, b.t().contiguous())


# Vocabularies: whole and ragged columns and depths, x small and too large for LDS.
@pytest.mark.parametrize("m,n,k", [(1, 65536, 1280), (1, 129280, 1280), (3, 70001, 272), (16, 65549, 128),
                                   (17, 66000, 144), (33, 129280, 640), (48, 65600, 1280), (64, 65537, 1296),
                                   (64, 65700, 2400), (1, 66000, 6848), (5, 65530, 16),
                                   # More tiles than fit the card at once; depths of one, two and
                                   # many blocks, and of more than eight.
                                   (2100, 5001, 112), (1500, 6848, 272), (1300, 8000, 1296),
                                   (130, 66000, 400), (4096, 2052, 2192),
                                   # Rows that end anywhere.
                                   (1, 66000, 1279), (33, 65600, 145), (64, 65537, 17), (5, 65530, 7),
                                   (17, 70001, 1281), (2000, 6000, 1283)])
def test_linear_wide_exact(ctx, m, n, k):
    say(f"wide product {m}x{n}x{k}")
    ops, want = device_exact(m, n, k, m + n)
    guard = torch.full((m * n + 64,), 12345.0, device="cuda")
    y = guard[:m * n].view(m, n)
    torch.cuda.synchronize()
    um.fp8_linear(ctx, *ops, y)
    assert torch.equal(y.double(), want)
    assert bool((guard[m * n:] == 12345.0).all())
    y16 = torch.empty((m, n), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    um.fp8_linear(ctx, *ops, y16)
    assert torch.equal(y16, want.float().to(torch.bfloat16))


@pytest.mark.parametrize("m", [1, 20, 150, 300])
def test_linear_nan_bytes_stay_in_their_row_and_column(ctx, m):
    n, k = 300, 400
    x, xs, w, ws = random_product(m, n, k, 9)
    x[m // 2, 399] = 0x7f
    w[200, 0] = 0xff
    y = torch.zeros((m, n), device="cuda")
    dev = device_product(x, xs, w, ws)
    torch.cuda.synchronize()
    um.fp8_linear(ctx, *dev, y)
    nan = np.zeros((m, n), bool)
    nan[m // 2] = True
    nan[:, 200] = True
    assert np.array_equal(np.isnan(y.cpu().numpy()), nan)


def test_linear_depth_ends_between_rows_with_nan(ctx):
    """Rows whose bytes end inside a block: what follows in memory (the next row,
    all NaN, and bytes behind the last one) is not taken in."""
    for m, n, k in ((3, 40, 144), (40, 300, 144), (300, 300, 130), (3, 40, 133), (40, 300, 1279), (64, 5000, 1),
                    (2, 66000, 135), (300, 1280, 2191)):
        x, xs, w, ws = exact_product(m, n, k, 5)
        x[1::2] = 0x7f
        w[1::2] = 0xff
        dev = device_product(x, xs, w, ws)
        y = torch.zeros((m, n), device="cuda")
        torch.cuda.synchronize()
        um.fp8_linear(ctx, *dev, y)
        a, b = spread(x[::2], xs[::2], w, ws)
        got = y.cpu().numpy()[::2, ::2]
        assert np.array_equal(got, a @ b.T[:, ::2])


@pytest.mark.parametrize("m,n,k", [(300, 700, 257), (700, 1000, 129), (200, 300, 1279), (65, 66000, 33)])
def test_linear_without_room_for_a_copy(m, n, k):
    """A scratch that holds neither the copy of ragged rows nor partial sums."""
    say(f"product {m}x{n}x{k} without room")
    cramped = um.Context(0, 4096)
    ops, want = device_exact(m, n, k, m + k)
    y = torch.full((m, n), float("nan"), device="cuda")
    y16 = torch.empty((m, n), device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    um.fp8_linear(cramped, *ops, y)
    um.fp8_linear(cramped, *ops, y16)
    assert torch.equal(y.double(), want) and torch.equal(y16, want.float().to(torch.bfloat16))
    cramped.close()


def test_linear_in_a_graph_and_between_streams(ctx):
    """A captured product replays with the eager bits on what its inputs hold then;
    two contexts work at once."""
    ops = [device_product(*random_product(m, 1000, k, 40 + m)) for m, k in ((1, 1280), (30, 1280), (300, 1280), (300, 1279))]
    want = []
    for d in ops:
        want.append(torch.empty((d[0].shape[0], 1000), device="cuda"))
        torch.cuda.synchronize()
        um.fp8_linear(ctx, *d, want[-1])
    got = [torch.full_like(w, float("nan")) for w in want]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=torch.cuda.ExternalStream(ctx.stream)):
        for d, y in zip(ops, got):
            um.fp8_linear(ctx, *d, y, sync=False)
    other = um.Context(0, 64 << 20)
    extra = [torch.empty_like(w) for w in want]
    for rep in range(4):
        for y in got + extra:
            y.fill_(float("nan"))
        torch.cuda.synchronize()
        g.replay()
        for d, y in zip(ops, extra):
            um.fp8_linear(other, *d, y, sync=False)
        torch.cuda.synchronize()
        for w, y, z in zip(want, got, extra):
            assert torch.equal(w, y) and torch.equal(w, z), rep
    other.close()

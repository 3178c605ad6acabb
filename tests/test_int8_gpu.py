"""Rows in 8-bit integers and their products through the C ABI, against plain computations in 64 bits: codes and scales
equal, products within the roundings of their f32 epilogue."""
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HALF_STEP = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
TYPES = ("float32", "float16", "bfloat16")


@pytest.fixture(scope="module")
def ctx():
    import needle_amd as na

    c = na.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def torch():
    import torch

    return torch


def _codes_ref(x):
    """x: numpy rows of f32 values -> (codes, scales): the quotient of two f32 numbers is far enough from every half in 64
    bits (their distance from one is at least 2^-32 of it)."""
    x = np.asarray(x, dtype=np.float32)
    top = np.abs(x).max(axis=1) if x.shape[1] else np.zeros(x.shape[0], np.float32)
    with np.errstate(all="ignore"):
        s = (top * (np.float32(1) / np.float32(127))).astype(np.float32)
        s[~np.isfinite(top)] = np.nan
        q = np.rint(x.astype(np.float64) / s.astype(np.float64)[:, None])
    q = np.where(s[:, None] > 0, np.clip(q, -127, 127), 0)
    return q.astype(np.int8), s


def _rows(rng, n, dim):
    x = (rng.standard_normal((n, dim)) * np.exp(rng.standard_normal((n, 1)))).astype(np.float32)
    return x


def _quantize(torch, ctx, t, codes=None):
    n, dim = t.shape
    codes = torch.full((n, dim), 99, dtype=torch.int8, device="cuda") if codes is None else codes
    scales = torch.full((n,), -1.0, device="cuda")
    ctx.quantize_rows_device(t, codes, scales)
    return codes, scales


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,dim", [(1, 1), (7, 3), (5, 16), (3, 63), (130, 64), (2, 129), (33, 384), (9, 768), (6, 1000), (3, 1024), (2, 1025),
                                   (5, 4096), (2, 5000), (1, 20011), (1001, 24), (70, 9), (65, 31), (9, 190), (5, 2049), (4, 4095), (3, 8191),
                                   (3, 8193), (2, 16_384), (2, 16_385)])
def test_quantize_rows(ctx, torch, dtype, n, dim):
    rng = np.random.default_rng(n * 31 + dim)
    t = torch.from_numpy(_rows(rng, n, dim)).to("cuda").to(getattr(torch, dtype))
    if n > 2:
        t[1] = 0
    codes, scales = _quantize(torch, ctx, t)
    want, s = _codes_ref(t.float().cpu().numpy())
    assert np.array_equal(scales.cpu().numpy(), s)
    assert np.array_equal(codes.cpu().numpy(), want)


def test_quantize_rows_ties_and_range(ctx, torch):
    """Quotients that are halves (to even) or lie one f32 step beside one, rows near both ends of the f32 range, rows with
    NaN and infinities."""
    rows = []
    for s in (1.0, 0.37, 3.1e-5, 1e-30, 2.0 ** -140, 1e30):
        s = np.float32(s)
        top = np.float32(127) * s
        halves = (np.arange(-127, 127) + 0.5) * np.float64(top * (np.float32(1) / np.float32(127)))
        h = halves.astype(np.float32)
        rows += [np.concatenate([[top], h]), np.concatenate([[top], np.nextafter(h, np.float32(np.inf))]),
                 np.concatenate([[top], np.nextafter(h, np.float32(-np.inf))])]
    rng = np.random.default_rng(0)
    tiny = np.zeros((4, 255), np.float32)
    tiny[0, :3] = np.array([190, 64, 1]) * np.float32(2.0 ** -149)   # the scale is one denormal step
    tiny[1, :2] = np.array([63, -1]) * np.float32(2.0 ** -149)       # the scale rounds to zero
    tiny[2] = rng.standard_normal(255).astype(np.float32) * np.float32(1e-42)
    tiny[3] = rng.uniform(-3.4e38, 3.4e38, 255).astype(np.float32)
    x = np.concatenate([np.stack(rows).astype(np.float32), tiny])
    bad = np.tile(rng.standard_normal(255).astype(np.float32), (3, 1))
    bad[0, 254], bad[1, 3], bad[2, 0] = np.nan, np.inf, -np.inf
    x = np.concatenate([x, bad])
    codes, scales = _quantize(torch, ctx, torch.from_numpy(x).cuda())
    want, s = _codes_ref(x)
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True) and np.isnan(s[-3:]).all()
    assert np.array_equal(codes.cpu().numpy(), want) and not want[-3:].any()


@pytest.mark.parametrize("dtype,dim", [("float16", 2 ** 32 - 1), ("bfloat16", 2 ** 32 - 8190), ("float32", 2 ** 31 + 5)])
def test_quantize_a_row_of_billions(ctx, torch, dtype, dim):
    """A row that ends within one step of 2^32 values, where a 32-bit place would wrap, and one longer than 2^31."""
    t = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(dim % 1000)
    x = torch.empty(1, dim, dtype=t, device="cuda")
    some = torch.randn(1 << 24, generator=g, device="cuda").clamp_(-5, 5).to(t)
    for at in range(0, dim, some.numel()):
        x[0, at:at + some.numel()] = some[:min(some.numel(), dim - at)]
    x[0, dim - 2] = -7.0
    codes, scales = _quantize(torch, ctx, x)
    s = np.float32(7) * (np.float32(1) / np.float32(127))
    assert float(scales[0]) == float(s)
    for at in (0, 2 ** 31 - 50_000, dim - 5_000_000):
        want = torch.round(x[0, at:at + 5_000_000].double() / float(s)).to(torch.int8)
        assert torch.equal(codes[0, at:at + 5_000_000], want)
    for at in range(0, dim, 1 << 28):  # the rest: every code within one of its value
        off = (codes[0, at:at + (1 << 28)].float() * float(s) - x[0, at:at + (1 << 28)].float()).abs().max()
        assert float(off) <= 0.5001 * float(s)


@pytest.mark.parametrize("dtype", ("float16", "bfloat16"))
def test_quantize_rows_of_few_bits(ctx, torch, dtype):
    """Half-precision values against every significand of the row's largest: quotients that are halves, or nearly so, are
    common."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.randn(1024, 640, generator=g, device="cuda") * 0.3).clamp(-1, 1).to(getattr(torch, dtype))
    x[:, 7] = (1.0 + torch.arange(1024, device="cuda") / 1024).to(getattr(torch, dtype))
    for rows in (x, x[:, :96].contiguous(), x[::3, 1:]):
        codes, scales = _quantize(torch, ctx, rows)
        want, s = _codes_ref(rows.float().cpu().numpy())
        assert np.array_equal(scales.cpu().numpy(), s)
        assert np.array_equal(codes.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim,x_stride,c_stride,offset", [(33, 50, 41, 1), (384, 400, 384, 0), (256, 257, 259, 3), (64, 64, 128, 0), (1100, 1111, 1101, 5)])
def test_quantize_rows_that_lie_apart(ctx, torch, dtype, dim, x_stride, c_stride, offset):
    g = torch.Generator(device="cuda").manual_seed(dim)
    n = 21
    buf = torch.randn(n * x_stride + 64, generator=g, device="cuda").to(getattr(torch, dtype))
    x = buf[offset:offset + n * x_stride].view(n, x_stride)[:, :dim]
    out = torch.full((n * c_stride + 64,), 77, dtype=torch.int8, device="cuda")
    codes = out[offset:offset + n * c_stride].view(n, c_stride)[:, :dim]
    _, scales = _quantize(torch, ctx, x, codes)
    want, s = _codes_ref(x.float().cpu().numpy())
    assert np.array_equal(codes.cpu().numpy(), want) and np.array_equal(scales.cpu().numpy(), s)
    left = torch.ones_like(out, dtype=torch.bool)
    left[offset:offset + n * c_stride].view(n, c_stride)[:, :dim] = False
    assert (out[left] == 77).all()


def test_quantize_rows_host_form(ctx):
    from needle_amd import InvalidVector

    rng = np.random.default_rng(2)
    for x in (_rows(rng, 9, 77), _rows(rng, 4, 10).astype(np.float16)):
        codes, scales = ctx.quantize_rows(x)
        want, s = _codes_ref(x)
        assert np.array_equal(codes, want) and np.array_equal(scales, s)
    for v in (np.nan, np.inf):
        x = _rows(rng, 3, 5)
        x[2, 4] = v
        with pytest.raises(InvalidVector):
            ctx.quantize_rows(x)
    codes, scales = ctx.quantize_rows(np.zeros((0, 5), np.float32))
    assert codes.shape == (0, 5) and scales.shape == (0,)
    codes, scales = ctx.quantize_rows(np.zeros((2, 0), np.float32))
    assert not scales.any()


def _table(torch, g, n, k, stride=None, offset=0, low=-128):
    stride = stride or k
    buf = torch.randint(low, 128, (n * stride + 64,), generator=g, device="cuda", dtype=torch.int8)
    codes = buf[offset:offset + n * stride].view(n, stride)[:, :k]
    return codes, torch.rand(n, generator=g, device="cuda") * 0.02 + 1e-4


def _check_product(out, a, sa, b, sb, bias, dtype):
    """out against 64 bits.  The f32 epilogue rounds the sum, two products and the sum with the bias, half a step each, the
    first three relative to the product; a half type rounds once more (fp16 by 2^-25 at least: its smallest step)."""
    exact = (a.cpu().numpy().astype(np.float64) @ b.cpu().numpy().astype(np.float64).T) * sa.double().cpu().numpy()[:, None] * \
        sb.double().cpu().numpy()[None, :]
    u = HALF_STEP["float32"]
    room = 3.01 * u * np.abs(exact)
    if bias is not None:
        exact = exact + bias.double().cpu().numpy()[None, :]
        room = room + u * (np.abs(exact) + room)
    if dtype != "float32":
        room = room + HALF_STEP[dtype] * (np.abs(exact) + room) + (2.0 ** -25 if dtype == "float16" else 0.0)
    off = np.abs(out.double().cpu().numpy() - exact)
    assert (off <= room).all(), (float((off / np.maximum(room, 1e-300)).max()), np.argwhere(off > room)[:5])


SHAPES = [(1, 1, 1), (1, 17, 16), (3, 5, 7), (16, 16, 64), (17, 33, 65), (1, 1000, 128), (4, 130, 1024), (5, 2049, 384), (64, 64, 63), (65, 127, 300),
          (128, 128, 128), (130, 257, 256), (200, 700, 80), (256, 256, 512), (257, 513, 1008), (300, 1000, 1000), (1, 300, 4096), (16, 515, 5000),
          (33, 64, 2048), (512, 768, 272), (70, 40, 16), (1000, 3, 96), (2, 9, 9999), (4112, 4097, 528), (4100, 4105, 513), (1500, 1700, 192), (1500, 1701, 67), (50, 33_000, 96),
          (20, 20_000, 33), (16, 17_000, 400), (7, 20_000, 700), (40, 50, 4097), (65, 130, 2064), (100, 90, 9000), (64, 128, 2112), (130, 1000, 2048),
          (20, 30, 131_071)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(ctx, torch, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m * 7 + n * 3 + k)
    a, sa = _table(torch, g, m, k)
    b, sb = _table(torch, g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    for dtype, t in zip(TYPES, (None, bias, bias)):
        out = torch.full((m, n), float("nan"), dtype=getattr(torch, dtype), device="cuda")
        ctx.matmul_i8_device(a, sa, b, sb, out, d_bias=t)
        _check_product(out, a, sa, b, sb, t, dtype)


@pytest.mark.parametrize("m,n,k,a_stride,b_stride,o_stride,offset", [
    (5, 70, 64, 96, 80, 70, 0), (37, 501, 301, 384, 384, 501, 0), (3, 129, 48, 49, 51, 131, 1), (70, 200, 256, 272, 257, 203, 16),
    (300, 300, 128, 144, 128, 304, 0), (260, 300, 144, 160, 176, 302, 16), (1, 65, 200, 200, 203, 65, 7), (130, 140, 33, 64, 64, 140, 0),
    (40, 50, 7, 16, 16, 50, 0), (17, 33, 1, 16, 32, 33, 0), (100, 90, 515, 528, 528, 90, 0), (60, 20_000, 255, 256, 272, 20_000, 0),
    (520, 6000, 1009, 1024, 1024, 6000, 16), (2040, 8190, 529, 544, 560, 8190, 0), (2040, 8190, 528, 544, 560, 8190, 0), (100, 90, 2500, 2512, 2528, 90, 0),
    (64, 64, 2049, 2064, 2064, 64, 0), (200, 300, 3333, 3344, 3333, 300, 0), (64, 64, 2240, 2240, 2256, 64, 16)])
def test_matmul_rows_that_lie_apart(ctx, torch, m, n, k, a_stride, b_stride, o_stride, offset):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a, sa = _table(torch, g, m, k, a_stride, offset)
    b, sb = _table(torch, g, n, k, b_stride, offset)
    for dtype in TYPES:
        buf = torch.full((m * o_stride + 64,), 5.0, dtype=getattr(torch, dtype), device="cuda")
        out = buf[offset:offset + m * o_stride].view(m, o_stride)[:, :n]
        ctx.matmul_i8_device(a, sa, b, sb, out)
        _check_product(out, a, sa, b, sb, None, dtype)
        left = torch.ones_like(buf, dtype=torch.bool)
        left[offset:offset + m * o_stride].view(m, o_stride)[:, :n] = False
        assert (buf[left] == 5.0).all()


def test_matmul_extremes(ctx, torch):
    """The longest sums of the largest products, scales that are zero, huge, infinite or NaN, an empty k."""
    k = 131071
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    b[1], b[2, ::2] = 127, 127
    one = torch.ones(3, device="cuda")
    out = torch.empty(2, 3, device="cuda")
    ctx.matmul_i8_device(a, one[:2].contiguous(), b, one, out)
    _check_product(out, a, one[:2], b, one, None, "float32")
    assert float(out[0, 0]) == float(np.float32(128 * 128 * k))
    g = torch.Generator(device="cuda").manual_seed(1)
    a, sa = _table(torch, g, 4, 32)
    b, sb = _table(torch, g, 70, 32)
    a[3] = 0
    sa[:3] = torch.tensor([0.0, float("nan"), 1e30])
    sb[:3] = torch.tensor([float("inf"), 1e30, 1e-30])
    out = torch.empty(4, 70, device="cuda")
    ctx.matmul_i8_device(a, sa, b, sb, out)
    acc = (a.cpu().float() @ b.cpu().float().T)
    want = acc * sa.cpu()[:, None] * sb.cpu()[None, :]
    assert torch.equal(out.cpu().isnan(), want.isnan()) and torch.equal(out.cpu().nan_to_num(7.0, 8.0, 9.0), want.nan_to_num(7.0, 8.0, 9.0))
    empty = torch.empty(4, 0, dtype=torch.int8, device="cuda"), torch.empty(70, 0, dtype=torch.int8, device="cuda")
    bias = torch.randn(70, generator=g, device="cuda")
    sa[1], sb[0] = 1.0, 1.0
    ctx.matmul_i8_device(empty[0], sa, empty[1], sb, out, d_bias=bias)
    assert torch.equal(out, bias.expand(4, 70))
    ctx.matmul_i8_device(empty[0], sa, empty[1], sb, out)
    assert not out.any()
    none = torch.empty(0, 70, device="cuda")
    ctx.matmul_i8_device(a[:0], sa[:0], b, sb, none)
    ctx.matmul_i8_device(a, sa, b[:0], sb[:0], torch.empty(4, 0, device="cuda"))


def test_matmul_behind_four_billion(ctx, torch):
    """Outputs and rows whose offsets pass 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(5)
    a, sa = _table(torch, g, 70_000, 16)
    b, sb = _table(torch, g, 66_048, 16)
    out = torch.empty(70_000, 66_048, dtype=torch.bfloat16, device="cuda")
    ctx.matmul_i8_device(a, sa, b, sb, out)
    for r, c in ((slice(0, 65), slice(0, 65)), (slice(69_900, 70_000), slice(65_900, 66_048)), (slice(65_100, 65_200), slice(30_000, 30_100))):
        _check_product(out[r, c], a[r], sa[r], b[c], sb[c], None, "bfloat16")
    del out
    b = torch.randint(-128, 128, (2 ** 26 + 100, 16), generator=g, device="cuda", dtype=torch.int8)  # two slabs of b
    sb = torch.rand(b.shape[0], generator=g, device="cuda")
    out = torch.empty(2, b.shape[0], device="cuda")
    ctx.matmul_i8_device(a[:2], sa[:2], b, sb, out, d_bias=sb)
    for c in (slice(0, 300), slice(2 ** 26 - 150, 2 ** 26 + 100)):
        _check_product(out[:, c], a[:2], sa[:2], b[c], sb[c], sb[c], "float32")
    rows = torch.randint(-128, 128, (2 ** 22 + 70, 33), generator=g, device="cuda", dtype=torch.int8)  # and of a
    sr = torch.rand(rows.shape[0], generator=g, device="cuda")
    out = torch.empty(rows.shape[0], 5, device="cuda")
    ctx.matmul_i8_device(rows, sr, rows[:5], sr[:5], out)
    for r in (slice(0, 300), slice(2 ** 22 - 150, 2 ** 22 + 70)):
        _check_product(out[r], rows[r], sr[r], rows[:5], sr[:5], None, "float32")
    del out, rows, b
    wide = torch.randint(-127, 128, (3, 2 ** 31 + 64), generator=g, device="cuda", dtype=torch.int8)  # rows 2 GiB apart
    x = wide[:, :100]
    out = torch.empty(3, 3, device="cuda")
    ctx.matmul_i8_device(x, sa[:3], x, sb[:3], out)
    _check_product(out, x, sa[:3], x, sb[:3], None, "float32")


def test_a_product_of_eight_million_tiles(ctx, torch):
    """An output of 275 GB, of as many 128 x 128 tiles as one launch has no grid for."""
    m, n, k = 2050, 1 << 26, 16
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < m * n * 2 + (4 << 30):
        pytest.skip("the output does not fit this device")
    g = torch.Generator(device="cuda").manual_seed(13)
    a, sa = _table(torch, g, m, k)
    b, sb = _table(torch, g, n, k)
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    rows, cols = (slice(0, 70), slice(980, 1100), slice(1990, 2050)), (slice(0, 300), slice(2 ** 25 - 100, 2 ** 25 + 100), slice(n - 300, n))
    for r in rows:
        for c in cols:
            out[r, c] = float("nan")
    ctx.matmul_i8_device(a, sa, b, sb, out)
    for r in rows:
        for c in cols:
            _check_product(out[r, c], a[r], sa[r], b[c], sb[c], None, "bfloat16")
    del out
    torch.cuda.empty_cache()


def test_a_product_without_room_for_its_copies(torch):
    """Rows that the loads cannot take as they are get copied to aligned ones where that is faster; on a device without room
    for the copies the product is made without them."""
    import needle_amd as na

    m, n, k = 7000, 12_000, 100_001  # copies of 1.9e9 bytes
    g = torch.Generator(device="cuda").manual_seed(11)
    a, sa = _table(torch, g, m, k)
    b, sb = _table(torch, g, n, k)
    out = torch.full((m, n), float("nan"), device="cuda")
    c = na.Context(0)
    try:
        c.matmul_i8_device(a[:40, :64], sa[:40], b[:40, :64], sb[:40], torch.empty(40, 40, device="cuda"))
        torch.cuda.synchronize()
        torch.cuda.empty_cache()
        left = torch.cuda.mem_get_info()[0] - (1 << 30)
        full = torch.empty(left, dtype=torch.uint8, device="cuda")
        assert torch.cuda.mem_get_info()[0] < (m + n) * k
        c.matmul_i8_device(a, sa, b, sb, out)
        del full
        torch.cuda.empty_cache()
        again = torch.full((m, n), float("nan"), device="cuda")
        c.matmul_i8_device(a, sa, b, sb, again)  # with room
    finally:
        c.close()
    assert torch.equal(out, again)
    at, bt = (torch.randint(0, r, (300,), generator=g, device="cuda") for r in (m, n))
    acc = torch.stack([(a[i].double() * b[j].double()).sum() for i, j in zip(at.tolist(), bt.tolist())])
    exact = acc * sa[at].double() * sb[bt].double()
    assert ((out[at, bt].double() - exact).abs() <= 3.01 * HALF_STEP["float32"] * exact.abs()).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 40, 33), (4, 1000, 1024), (37, 130, 301), (300, 520, 768), (2, 3, 0), (1, 8192, 8192), (16, 300, 511), (5, 17_000, 300),
                                   (13, 33_000, 630), (3, 1, 2047), (16, 70_000, 400), (2, 4099, 4096)])
def test_linear_is_quantize_then_matmul(ctx, torch, dtype, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn(m, k + 3, generator=g, device="cuda").to(getattr(torch, dtype))[:, :k]
    if m > 4:
        x[1], x[3, k // 2] = 0, float("inf")
    b, sb = _table(torch, g, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    for out_dtype in (torch.float32, x.dtype):
        out, two = (torch.empty(m, n, dtype=out_dtype, device="cuda") for _ in range(2))
        ctx.linear_i8_device(x, b, sb, out, d_bias=bias)
        codes, scales = _quantize(torch, ctx, x)
        ctx.matmul_i8_device(codes, scales, b, sb, two, d_bias=bias)
        assert torch.equal(out.isnan(), two.isnan()) and torch.equal(out.nan_to_num(7.0), two.nan_to_num(7.0))
        if m > 4:
            assert out[3].isnan().all() and torch.equal(out[1].float(), bias.to(out_dtype).float())


def test_matmul_host_form(ctx):
    rng = np.random.default_rng(3)
    a, b = rng.integers(-128, 128, (5, 130), dtype=np.int8), rng.integers(-128, 128, (77, 130), dtype=np.int8)
    sa, sb, bias = rng.random(5).astype(np.float32), rng.random(77).astype(np.float32), rng.standard_normal(77).astype(np.float32)
    acc = (a.astype(np.int64) @ b.astype(np.int64).T).astype(np.float32)
    assert np.array_equal(ctx.matmul_i8(a, sa, b, sb), acc * sa[:, None] * sb[None, :])
    assert np.array_equal(ctx.matmul_i8(a, sa, b, sb, bias), acc * sa[:, None] * sb[None, :] + bias)
    assert ctx.matmul_i8(a[:0], sa[:0], b, sb).shape == (0, 77)


def test_calls_from_threads_and_streams(ctx, torch):
    """Calls at once through one context, and inputs that a side stream is still making when the call is issued."""
    g = torch.Generator(device="cuda").manual_seed(8)
    b, sb = _table(torch, g, 900, 256)
    xs = [torch.randn(m, 256, generator=g, device="cuda") for m in (1, 40, 130, 300)]
    want = []
    for x in xs:
        out = torch.empty(x.shape[0], 900, device="cuda")
        ctx.linear_i8_device(x, b, sb, out)
        want.append(out)
    torch.cuda.synchronize()
    got, errors = [[None] * 6 for _ in xs], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for r in range(6):
                    x = xs[i] * 3.0
                    for _ in range(20):
                        x = x + 0.0
                    out = torch.empty(x.shape[0], 900, device="cuda")
                    ctx.linear_i8_device(x / 3.0, b, sb, out)
                    got[i][r] = out
        except Exception as e:  # pragma: no cover
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for i in range(len(xs)):
        x = (xs[i] * 3.0) / 3.0
        out = torch.empty(x.shape[0], 900, device="cuda")
        ctx.linear_i8_device(x, b, sb, out)
        for r in range(6):
            assert torch.equal(got[i][r], out)


def test_outputs_are_there_when_a_call_returns(ctx, torch):
    """Every call's output read at once, on another stream than any the call or its inputs used, and copied to the host."""
    g = torch.Generator(device="cuda").manual_seed(3)
    other = torch.cuda.Stream()
    for i in range(300):
        n, dim = (1, 7, 300, 20_000)[i % 4], (64, 333, 1024)[i % 3]
        x = torch.randn(n, dim, generator=g, device="cuda")
        codes, scales = torch.full((n, dim), 99, dtype=torch.int8, device="cuda"), torch.full((n,), -1.0, device="cuda")
        want = x.abs().amax(1) * torch.tensor(1.0 / 127.0, device="cuda")
        torch.cuda.synchronize()
        ctx.quantize_rows_device(x, codes, scales)
        with torch.cuda.stream(other):
            here = codes.clone(), scales.clone()
        there = scales.cpu()
        other.synchronize()
        assert torch.equal(here[1], want) and torch.equal(there, want.cpu())
        assert (here[0].abs().amax(1) == 127).all()


def test_inputs_under_way_on_another_stream(ctx, torch):
    """A call waits for torch's current stream, whichever that is."""
    side = torch.cuda.Stream()
    big = torch.randn(8192, 8192, device="cuda")
    for stream in (side, torch.cuda.default_stream()):
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            x = (big @ big)[:64].contiguous()
            codes, scales = torch.empty(64, 8192, dtype=torch.int8, device="cuda"), torch.empty(64, device="cuda")
            ctx.quantize_rows_device(x, codes, scales)
            want = x.abs().amax(1) * torch.tensor(1.0 / 127.0, device="cuda")
            assert torch.equal(scales, want)


def test_a_call_of_milliseconds(ctx, torch):
    g = torch.Generator(device="cuda").manual_seed(4)
    m, n, k = 8192, 65_536, 4096
    a, b = (torch.randint(-127, 128, (r, k), generator=g, device="cuda", dtype=torch.int8) for r in (m, n))
    sa, sb = torch.ones(m, device="cuda"), torch.ones(n, device="cuda")
    out = torch.full((m, n), float("nan"), device="cuda")
    ctx.matmul_i8_device(a, sa, b, sb, out)
    assert not out.isnan().any()
    at, bt = torch.randint(0, m, (500,), device="cuda"), torch.randint(0, n, (500,), device="cuda")
    want = (a[at].double() * b[bt].double()).sum(1)  # below 2^27: a whole number, rounded once
    assert torch.equal(out[at, bt], want.float())

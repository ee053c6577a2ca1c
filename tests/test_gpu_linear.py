"""GPU: the dense-layer operators against plain implementations in 64 bits.

Tolerances.  A rounding to type t is off by at most finfo(t).eps / 2 of the value (half a step).  8-bit products are
summed exactly, so an fp32 result passes five roundings (the sum to fp32, the two scales' product, its product with the
sum, the bias, and the result's own): 5 * 2^-24 of the terms' magnitudes bounds them.  fp32 sums of k products are off
by at most one step (2^-23, as for an adder that cuts off) of the running magnitude for each addition, k + 2 of them at
most, so (k + 2) * 2^-23 * sum |x||w| bounds those in any order.  Sigmoid has a slope of at most 1/4, and its own
arithmetic (expf to 2 steps, an addition, a division) adds less than 8 * 2^-24.
"""
import numpy as np
import pytest
import torch

from recflex_b200 import _lib, linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FLOATS = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def codes(shape, g):
    return torch.randint(-128, 128, shape, generator=g, device=DEV, dtype=torch.int32).to(torch.int8)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(out, exact, slack):
    """|out - exact| <= slack + the rounding of the result (and, near zero, half the type's smallest step)."""
    tiny = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[out.dtype]
    off = (out.double() - exact).abs()
    limit = slack + (exact.abs() + slack) * half_step(out.dtype) + tiny
    worst = (off - limit).max() if off.numel() else torch.zeros(())
    assert not torch.isnan(out.double()).any()
    assert worst <= 0, f"off by {float(off.flatten()[(off - limit).argmax()])}, {float(limit.flatten()[(off - limit).argmax()])} allowed"


def activated(y, slack, act):
    if act == "relu":
        return y.clamp(min=0), slack
    if act == "sigmoid":
        return torch.sigmoid(y), slack / 4 + 8 * 2.0 ** -24
    return y, slack


def int_product(q, w):
    """Exact integer products (float64 holds every partial sum below 2^53)."""
    return q.double() @ w.double().transpose(-1, -2)


# ---- rows in 8 bits ------------------------------------------------------------------------------------------------
def expected_codes(x):
    """The definition, evaluated by numpy: fp32 scale by an IEEE division, the quotient in 64 bits (two 24-bit
    significands: it cannot round onto a middle that it does not equal)."""
    x32 = x.float().cpu().numpy()
    top = np.abs(x32).max(axis=1) if x32.shape[1] else np.zeros(x32.shape[0], np.float32)
    scale = (top / np.float32(127)).astype(np.float32)
    step = np.where((scale > 0) & np.isfinite(scale), scale, np.float32(1)).astype(np.float64)
    with np.errstate(invalid="ignore"):
        q = np.rint(x32.astype(np.float64) / step[:, None])
    q[~np.isfinite(top)] = 0
    q[scale == 0] = 0
    return np.clip(q, -127, 127).astype(np.int8), scale, np.isfinite(top)


def check_codes(x, q, scale):
    eq, es, fine = expected_codes(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == (x.shape[0],)
    np.testing.assert_array_equal(scale.cpu().numpy()[fine], es[fine])
    assert not np.isfinite(scale.cpu().numpy()[~fine]).any()
    np.testing.assert_array_equal(q.cpu().numpy(), eq)


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, cols", [(1, 1), (3, 7), (9, 8), (33, 250), (8, 256), (70, 257), (5, 1024), (6, 1924),
                                        (2, 4097), (3, 15608), (2, 16385), (1, 24160), (2, 32769), (1, 70001)])
def test_quantize_rows(dtype, rows, cols):
    x = (torch.randn(rows, cols, generator=gen(rows * 7 + cols), device=DEV) * 0.3).to(dtype)
    check_codes(x, *linear.quantize_rows(x))


@pytest.mark.parametrize("dtype", FLOATS)
def test_quantize_rows_of_every_layout(dtype):
    base = torch.randn(40, 330, generator=gen(5), device=DEV).to(dtype)
    flat = base.flatten()
    for x in (base[:, 1:300], base[:, ::3], base.t(), base[3:4, 5:], base[:1].expand(9, 330), flat[1:1 + 31 * 41].view(31, 41),
              base[::2, :64], base[:0], base[:, :0]):
        check_codes(x, *linear.quantize_rows(x))


def test_quantize_rows_ties_and_extremes():
    """Ties (a row whose scale is a power of two holds many), zeros, subnormal and huge rows, infinities and NaN."""
    halves = torch.arange(-254, 255, device=DEV, dtype=torch.float32) / 2
    rows = [halves, halves * 2.0 ** -30, halves * 2.0 ** 60, halves * 2.0 ** -120, halves * 2.0 ** -140, halves * 0,
            torch.nextafter(halves, torch.full_like(halves, 1e9)), torch.nextafter(halves, torch.full_like(halves, -1e9)),
            halves / 127 * 3.4e38, torch.full_like(halves, 2.0 ** -149), halves * 3, halves / 3]
    x = torch.stack(rows)
    x[6:8].clamp_(-127, 127)
    bad = halves.repeat(4, 1)
    bad[0, 5], bad[1, 300], bad[2, 0], bad[3, 7] = float("inf"), float("-inf"), float("nan"), float("nan")
    bad[3, 9] = float("inf")
    x = torch.cat([x, bad])
    check_codes(x, *linear.quantize_rows(x))
    for dtype in (torch.bfloat16, torch.float16):
        check_codes(x.to(dtype), *linear.quantize_rows(x.to(dtype)))


# ---- the 8-bit product --------------------------------------------------------------------------------------------
def scales(n, g):
    return torch.rand(n, generator=g, device=DEV) * 0.01 + 1e-4


def check_int8(q, qs, w, ws, bias, act, out):
    acc = int_product(q, w)
    y = acc * (qs.double()[:, None] * ws.double())
    mag = y.abs()
    if bias is not None:
        y = y + bias.double()
        mag = mag + bias.double().abs()
    check(out, *activated(y, 5 * 2.0 ** -24 * mag, act))


@pytest.mark.parametrize("k, n", [(1, 1), (16, 8), (31, 33), (128, 1), (480, 64), (1000, 129), (1924, 256), (1025, 1024),
                                  (4096, 17), (15608, 200)])
@pytest.mark.parametrize("rows", [1, 2, 31, 64, 129, 300])
def test_int8_linear(rows, k, n):
    g = gen(rows + 31 * k + n)
    q, w = codes((rows, k), g), codes((n, k), g)
    qs, ws = scales(rows, g), scales(n, g)
    bias = torch.randn(n, generator=g, device=DEV)
    pick = rows + k + n
    act, dtype = ("none", "relu", "sigmoid")[pick % 3], FLOATS[pick // 3 % 3]
    out = linear.int8_linear(q, qs, w, ws, bias if pick % 2 else None, act, dtype)
    assert out.dtype == dtype and out.shape == (rows, n)
    check_int8(q, qs, w, ws, bias if pick % 2 else None, act, out)


@pytest.mark.parametrize("rows, k, n", [(2000, 1924, 1024), (4096, 480, 1024), (777, 15608, 128), (20000, 256, 128),
                                        (66000, 128, 1), (5, 131071, 3), (300, 131071, 300)])
def test_int8_linear_large(rows, k, n):
    """Many tiles; and the longest rows, whose extreme values reach the end of the 32-bit sums."""
    g = gen(rows)
    q, w = codes((rows, k), g), codes((n, k), g)
    if k == 131071:
        q[0], w[0], q[1], w[1] = -128, -128, 127, -128
    qs, ws, bias = scales(rows, g), scales(n, g), torch.randn(n, generator=g, device=DEV)
    out = linear.int8_linear(q, qs, w, ws, bias, "none", torch.float32)
    check_int8(q, qs, w, ws, bias, "none", out)
    again = linear.int8_linear(q, qs, w, ws, bias, "none", torch.float32)
    assert torch.equal(out, again)


# sizes that reach each of the tiles (512 and 256 columns on pairs of CTAs, 256, 128, 64 and 16 columns on one, K split
# over two and four), with columns and K that end inside them
TILES = [(16384, 15608, 1024), (16300, 15000, 1001), (9000, 6000, 1000), (4096, 1924, 1000), (4096, 1924, 333), (4096, 480, 1000),
         (2000, 1924, 777), (1000, 1030, 65), (5000, 3001, 15), (512, 15608, 700), (333, 9001, 300)]


@pytest.mark.parametrize("act", ["none", "relu", "sigmoid"])
@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, k, n", TILES)
def test_int8_linear_on_every_tile(rows, k, n, dtype, act):
    if rows * k > 1 << 26 and (dtype, act) not in ((torch.float32, "sigmoid"), (torch.bfloat16, "relu"), (torch.float16, "none")):
        pytest.skip("the largest sizes run once for each type and activation")
    g = gen(rows + k + n)
    q, w = codes((rows, k), g), codes((n, k), g)
    # results of a few units, where the sigmoid bends
    qs = scales(rows, g) * 8 / k ** 0.5
    ws, bias = scales(n, g), torch.randn(n, generator=g, device=DEV)
    wide = torch.full((rows + 1, n + 3), 7.0, dtype=dtype, device=DEV)
    out = linear.int8_linear(q, qs, w, ws, bias, act, dtype)
    check_int8(q, qs, w, ws, bias, act, out)
    linear.int8_linear(q, qs, w, ws, bias, act, dtype, out=wide[:, 1:n + 1])  # rows that take no wide stores
    assert torch.equal(wide[:rows, 1:n + 1], out)
    assert (wide[:, 0] == 7).all() and (wide[:, n + 1:] == 7).all() and (wide[rows] == 7).all()


@pytest.mark.parametrize("kind", ["bf16", "f16", "i8"])
@pytest.mark.parametrize("rows, groups, k, n", [(9000, 9, 1924, 500), (9000, 9, 1924, 1000), (12000, 9, 1924, 1000),
                                                (20000, 9, 1030, 250), (3000, 40, 1924, 1000), (700, 3, 9000, 300)])
@pytest.mark.parametrize("gather", [False, True])
def test_grouped_linear_on_every_tile(rows, groups, k, n, kind, gather):
    g = gen(rows + groups + n)
    ids = torch.randint(-1, groups, (rows,), generator=g, device=DEV) * torch.randint(0, 2, (rows,), generator=g, device=DEV)
    order, offsets = linear.group_rows(ids, groups)
    kw = {}
    if kind == "i8":
        x, w = codes((rows, k), g), codes((groups, n, k), g)
        kw = dict(x_scale=scales(rows, g), weight_scale=scales(groups * n, g).view(groups, n))
    else:
        dtype = torch.bfloat16 if kind == "bf16" else torch.float16
        x = torch.randn(rows, k, generator=g, device=DEV).to(dtype)
        w = (torch.randn(groups, n, k, generator=g, device=DEV) / k ** 0.5).to(dtype)
    bias = torch.randn(groups, n, generator=g, device=DEV)
    rows_in = order if gather else None
    got = linear.grouped_linear(x, w, offsets, bias, "relu", rows_in, order, **kw)
    exact, slack = plain_grouped(x, w, offsets, bias, "relu", rows_in, order, torch.zeros_like(got), kw.get("x_scale"), kw.get("weight_scale"))
    check(got, exact, slack)
    assert torch.equal(got, linear.grouped_linear(x, w, offsets, bias, "relu", rows_in, order, **kw))
    linear.check_status(DEV)


def test_int8_linear_layouts_and_given_out():
    g = gen(3)
    base, wbase = codes((64, 300), g), codes((50, 400), g)
    qs, ws = scales(64, g), scales(50, g)
    for q, w in ((base[:, 3:203], wbase[:, 1:201]), (base[:, ::2][:, :100], wbase[:, :200:2]),
                 (base[:1].expand(64, 300), wbase[:, :300]), (base[:, :208][::2], wbase[:, 16:224])):
        s = qs[:q.shape[0]]
        check_int8(q, s, w, ws, None, "none", linear.int8_linear(q, s, w, ws, out_dtype=torch.float32))
        wide = torch.full((q.shape[0] + 3, 77), 7.0, dtype=torch.float16, device=DEV)
        out = linear.int8_linear(q, s, w, ws, out_dtype=torch.float16, out=wide[:, 11:61])
        check_int8(q, s, w, ws, None, "none", out[:q.shape[0]])
        assert (wide[:, :11] == 7).all() and (wide[:, 61:] == 7).all() and (wide[q.shape[0]:] == 7).all()


@pytest.mark.parametrize("dtype", FLOATS)
@pytest.mark.parametrize("rows, n", [(2, 512), (40, 1), (300, 16), (900, 512), (900, 100)])
def test_sigmoid_over_its_range(rows, n, dtype):
    """Rows of zeros give sigmoid(bias) exactly as the kernel evaluates it: relative to the value, up to where it is 0."""
    bias = torch.linspace(-87, 87, n, device=DEV) if n > 1 else torch.full((1,), -40.0, device=DEV)
    if n > 4:
        bias[:4] = torch.tensor([0.0, float("inf"), -float("inf"), -1e4], device=DEV)
    zero = torch.zeros(max(rows, n), 64, dtype=torch.int8, device=DEV)
    scale = torch.ones(max(rows, n), device=DEV)
    out = linear.int8_linear(zero[:rows], scale[:rows], zero[:n], scale[:n], bias, "sigmoid", dtype)
    want = torch.sigmoid(bias.double()).expand(rows, n)
    # expf 2 units of 2^-23, the sum half a unit, the quotient 2 units; then the rounding to `dtype`, and where that type
    # ends half its smallest step (fp32: values below 2^-126 may be 0)
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}[dtype]
    assert ((out.double() - want).abs() <= want * (4.5 * 2.0 ** -23 + half_step(dtype)) * (1 + 2.0 ** -10) + tiny).all()
    assert torch.isnan(linear.int8_linear(zero[:rows], scale[:rows], zero[:n], scale[:n], bias * float("nan"), "sigmoid", dtype)).all()


@pytest.mark.parametrize("n", [1, 15, 16, 17, 20, 33, 36, 129, 250, 252, 500])
@pytest.mark.parametrize("kind", ["i8", "bf16"])
def test_results_rows_are_on_wide_boundaries_or_packed_as_given(kind, n):
    g = gen(n)
    for rows, out_dtype in ((3, None), (700, None)) + (((700, torch.float32),) if kind == "i8" else ()):
        x, w, kw = codes((rows, 40), g), codes((2, n, 40), g), dict(x_scale=scales(rows, g), weight_scale=scales(2 * n, g).view(2, n))
        if kind == "bf16":
            x, w, kw = x.bfloat16(), w.bfloat16(), {}
        order, offsets = linear.group_rows(torch.randint(0, 2, (rows,), generator=g, device=DEV), 2)
        for out_rows in (None, order):
            got = linear.grouped_linear(x, w, offsets, out_rows=out_rows, out_dtype=out_dtype, **kw)
            per = 16 // got.dtype.itemsize
            assert got.stride() == (n if n <= 16 else -(-n // per) * per, 1)
            packed = torch.full((rows, n), 7.0, dtype=got.dtype, device=DEV)
            linear.grouped_linear(x, w, offsets, out_rows=out_rows, out_dtype=out_dtype, out=packed, **kw)
            assert torch.equal(packed, got)
            exact, slack = plain_grouped(x, w, offsets, None, "none", None, out_rows, torch.zeros_like(got), kw.get("x_scale"), kw.get("weight_scale"))
            check(got, exact, slack)
        if n > 16 and out_dtype is None:
            # the next product reads such rows where they lie
            assert linear.pack_rows(got) is got


def test_rows_that_are_not_finite_give_nan_and_leave_the_others_alone():
    g = gen(4)
    x = torch.randn(40, 100, generator=g, device=DEV)
    w, bias = torch.randn(30, 100, generator=g, device=DEV), torch.randn(30, generator=g, device=DEV)
    clean = linear.Int8Linear(w, bias)(x)
    x[3, 5], x[17, 99] = float("inf"), float("nan")
    out = linear.Int8Linear(w, bias)(x)
    bad = torch.zeros(40, dtype=torch.bool, device=DEV)
    bad[[3, 17]] = True
    assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])
    zero = linear.Int8Linear(w, bias)(torch.zeros(2, 100, device=DEV))
    assert torch.equal(zero, bias.expand(2, 30))


# ---- rows by expert ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("rows, groups", [(0, 3), (1, 1), (31, 4), (33, 1), (256, 8), (1000, 1024), (16384, 64),
                                          (16385, 64), (20000, 1024), (70001, 7), (200000, 256), (1000003, 1000)])
def test_group_rows(rows, groups, dtype):
    rng = np.random.default_rng(rows + groups)
    ids = np.minimum(rng.integers(0, groups, rows), rng.integers(0, groups, rows))
    odd = rng.random(rows) < 0.05
    ids[odd] = rng.choice([-1, -2 ** 31, groups, groups + 1, 2 ** 31 - 1], int(odd.sum()))
    if dtype == torch.int64 and rows > 10:
        ids[::97] = 2 ** 32  # no expert: its low half is 0, which is one
    order, offsets = linear.group_rows(torch.from_numpy(ids).to(DEV, dtype), groups)
    key = np.where((ids < 0) | (ids >= groups), groups, ids)
    np.testing.assert_array_equal(order.cpu().numpy(), np.argsort(key, kind="stable"))
    np.testing.assert_array_equal(offsets.cpu().numpy(), np.searchsorted(np.sort(key), np.arange(groups + 1)))
    assert order.dtype == torch.int32 and offsets.dtype == torch.int32


def test_group_rows_strided_and_one_popular_expert():
    ids = torch.zeros(60000, dtype=torch.int64, device=DEV)
    ids[::1000] = 5
    for t in (ids, ids[::3], ids[1:], ids[:0]):
        order, offsets = linear.group_rows(t, 6)
        assert torch.equal(order.long(), torch.sort(t, stable=True).indices)
        assert int(offsets[6]) == t.numel() and int(offsets[5]) == int((t == 0).sum())


# ---- products by expert ------------------------------------------------------------------------------------------
def plain_grouped(x, w, offsets, bias, act, in_rows, out_rows, out, xs=None, ws=None):
    """(exact, slack) over the rows of `out` (float64), rows of no expert as they are in `out`."""
    exact, slack = out.double().clone(), torch.zeros_like(out, dtype=torch.float64)
    ends = offsets.tolist()
    k = x.shape[1]
    for g in range(w.shape[0]):
        at = torch.arange(ends[g], ends[g + 1], device=DEV)
        src = in_rows[at].long() if in_rows is not None else at
        dst = out_rows[at].long() if out_rows is not None else at
        if xs is not None:
            y = int_product(x[src], w[g]) * (xs[src].double()[:, None] * ws[g].double())
            mag, unit = y.abs(), 5 * 2.0 ** -24
        else:
            y = x[src].double() @ w[g].double().t()
            mag, unit = x[src].double().abs() @ w[g].double().abs().t(), (k + 2) * 2.0 ** -23
        if bias is not None:
            y, mag = y + bias[g].double(), mag + bias[g].double().abs()
        exact[dst], slack[dst] = activated(y, mag * unit, act)
    return exact, slack


def offsets_of(sizes, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(sizes)]), dtype=torch.int32, device=DEV)


SIZES = [[1], [0, 1, 0], [3, 0, 0, 130], [128, 64, 1, 0], [5] * 40, [0, 0, 0], [300, 2, 257], [1] * 9 + [0] * 50 + [2] * 5,
         [129, 127, 1000, 0, 31], [256, 256]]


@pytest.mark.parametrize("kind", ["bf16", "f16", "i8"])
@pytest.mark.parametrize("k, n", [(8, 1), (64, 16), (100, 33), (480, 128), (1924, 96), (1025, 300), (2048, 1024)])
@pytest.mark.parametrize("case", range(len(SIZES)))
def test_grouped_linear(kind, k, n, case):
    sizes = SIZES[case]
    if k * n > 1 << 20 and case not in (2, 6, 8):
        pytest.skip("the widest layer runs on three of the size lists")
    g = gen(case * 100 + k + n)
    E, used = len(sizes), sum(sizes)
    behind = case % 3  # positions of no expert
    P = used + behind
    gather, scatter = bool((case + k) % 2), bool((case + n // 2) % 2)
    x_rows = P + 5 if gather else P
    offsets = offsets_of(sizes)
    perm = torch.randperm(max(1, x_rows), generator=g, device=DEV).to(torch.int32)
    in_rows = perm[:P].contiguous() if gather else None
    out_rows = torch.randperm(max(1, P), generator=g, device=DEV)[:P].to(torch.int32) if scatter else None
    bias = torch.randn(E, n, generator=g, device=DEV) if (k + n + case) % 2 else None
    act = ("none", "relu", "sigmoid")[(case + k) % 3]
    kw = {}
    if kind == "i8":
        x, w = codes((x_rows, k), g), codes((E, n, k), g)
        kw = dict(x_scale=scales(x_rows, g), weight_scale=scales(E * n, g).view(E, n))
        dtype = FLOATS[(case + k) % 3]
    else:
        dtype = torch.bfloat16 if kind == "bf16" else torch.float16
        x = torch.randn(x_rows, k, generator=g, device=DEV).to(dtype)
        w = (torch.randn(E, n, k, generator=g, device=DEV) / k ** 0.5).to(dtype)
    out = torch.full((P + 2, n), 3.0, dtype=dtype, device=DEV)
    exact, slack = plain_grouped(x, w, offsets, bias, act, in_rows, out_rows, out, kw.get("x_scale"), kw.get("weight_scale"))
    got = linear.grouped_linear(x, w, offsets, bias, act, in_rows, out_rows, out_dtype=dtype, out=out, **kw)
    assert got is out
    check(out, exact, slack)
    fresh = linear.grouped_linear(x, w, offsets, bias, act, in_rows, out_rows, out_dtype=dtype, **kw)
    assert fresh.shape == (P, n) and fresh.dtype == dtype
    rest = torch.arange(used, P, device=DEV)
    rest = out_rows[rest].long() if scatter else rest
    exact[rest] = 0
    check(fresh, exact[:P], slack[:P])
    linear.check_status(DEV)


@pytest.mark.parametrize("kind", ["bf16", "i8"])
def test_grouped_linear_infinities_stay_in_their_rows(kind):
    """A row that is not finite, and what stands in memory around a run (other experts' rows, rows of no expert, the
    columns behind k), change no other row."""
    g = gen(11)
    k, n = 40, 24
    sizes = [3, 20, 1, 130]
    P = sum(sizes) + 6
    x = torch.randn(P, 64, generator=g, device=DEV).bfloat16()
    w = torch.randn(4, n, k, generator=g, device=DEV).bfloat16()
    offsets = offsets_of(sizes, 2)
    layer = linear.GroupedLinear(w)
    if kind == "i8":
        layer.quantize()
    clean = layer(x[:, :k], offsets)
    x[:, k:] = float("nan")
    for r in (0, 1, P - 1, P - 2, 2, 10):
        x[r, :] = float("inf")
    out = layer(x[:, :k], offsets)
    bad = torch.zeros(P, dtype=torch.bool, device=DEV)
    bad[[2, 10]] = True
    assert torch.equal(out[~bad], clean[~bad]) and not torch.isfinite(out[bad]).any()
    assert (out[:2] == 0).all() and (out[-4:] == 0).all()


@pytest.mark.parametrize("kind", ["f16", "i8"])
@pytest.mark.parametrize("k, n, groups", [(2048, 40, 150), (2048, 300, 60), (640, 130, 300), (8192, 600, 40)])
def test_grouped_linear_many_ragged_tiles(kind, k, n, groups):
    """Tiles of one row beside full ones, over and over: the copying warps that have nothing to copy for a tile keep
    step with the others (one that fell a ring of stages behind would wait for good)."""
    g = gen(k + n)
    rng = np.random.default_rng(n)
    sizes = rng.choice([0, 1, 2, 31, 33, 64, 65, 97, 128, 129, 200, 260], groups)
    P, offsets = int(sizes.sum()), offsets_of(sizes)
    kw = {}
    if kind == "i8":
        x, w = codes((P, k), g), codes((groups, n, k), g)
        kw = dict(x_scale=scales(P, g), weight_scale=scales(groups * n, g).view(groups, n))
    else:
        x = torch.randn(P, k, generator=g, device=DEV).half()
        w = (torch.randn(groups, n, k, generator=g, device=DEV) / k ** 0.5).half()
    order = torch.randperm(P, generator=g, device=DEV).to(torch.int32)
    for rows in (None, order):
        want = linear.grouped_linear(x, w, offsets, in_rows=rows, **kw)
        exact, slack = plain_grouped(x, w, offsets, None, "none", rows, None, want, kw.get("x_scale"), kw.get("weight_scale"))
        check(want, exact, slack)
        for _ in range(30):
            assert torch.equal(linear.grouped_linear(x, w, offsets, in_rows=rows, **kw), want)
    linear.check_status(DEV)


def test_grouped_linear_repeated_rows():
    """Two experts a sample: the same row number twice in in_rows."""
    g = gen(12)
    x = torch.randn(50, 72, generator=g, device=DEV).half()
    w = torch.randn(6, 40, 72, generator=g, device=DEV).half()
    ids = torch.randint(0, 6, (100,), generator=g, device=DEV)
    order, offsets = linear.group_rows(ids, 6)
    in_rows = order // 2
    out = linear.grouped_linear(x, w, offsets, in_rows=in_rows, out_rows=order)
    y = torch.einsum("mk,mnk->mn", x.double()[torch.arange(100, device=DEV) // 2], w.double()[ids])
    mag = torch.einsum("mk,mnk->mn", x.double().abs()[torch.arange(100, device=DEV) // 2], w.double().abs()[ids])
    check(out, y, mag * 74 * 2.0 ** -23)


def test_bad_rows_and_offsets_are_reported_and_skipped():
    g = gen(13)
    x = torch.randn(64, 32, generator=g, device=DEV).bfloat16()
    w = torch.randn(3, 16, 32, generator=g, device=DEV).bfloat16()
    good = offsets_of([20, 20, 24])
    want = linear.grouped_linear(x, w, good)
    linear.check_status(DEV)

    def reported():
        with pytest.raises(_lib.EbError) as e:
            linear.check_status(DEV)
        assert e.value.code == _lib.EB_ERR_BAD_INPUT
        linear.check_status(DEV)  # cleared by the read

    rows = torch.arange(64, dtype=torch.int32, device=DEV)
    bad = rows.clone()
    bad[[5, 41]] = torch.tensor([64, -1], dtype=torch.int32, device=DEV)
    out = linear.grouped_linear(x, w, good, in_rows=bad)
    keep = torch.ones(64, dtype=torch.bool, device=DEV)
    keep[[5, 41]] = False
    assert torch.equal(out[keep], want[keep]) and (out[~keep] == 0).all()
    reported()
    bad = rows.clone()
    bad[[7, 63]] = torch.tensor([2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=DEV)
    out = linear.grouped_linear(x, w, good, out_rows=bad)
    keep = torch.ones(64, dtype=torch.bool, device=DEV)
    keep[[7, 63]] = False
    assert torch.equal(out[keep], want[keep]) and (out[~keep] == 0).all()
    reported()
    for ends, clamped in (([0, 20, 40, 1000], [0, 20, 40, 64]), ([0, 40, 20, 64], [0, 40, 40, 64]),
                          ([-5, 20, 40, 64], [0, 20, 40, 64]), ([50, 20, 10, 0], [50, 50, 50, 50])):
        off = torch.tensor(ends, dtype=torch.int32, device=DEV)
        out = linear.grouped_linear(x, w, off)
        same = linear.grouped_linear(x, w, torch.tensor(clamped, dtype=torch.int32, device=DEV))
        assert torch.equal(out, same)
        reported()


def test_far_offsets():
    """Rows, weights and results that lie behind 2^31 elements."""
    g = gen(40)
    x = torch.empty(140000, 16000, dtype=torch.float16, device=DEV)
    for part in x.split(20000):
        part.normal_(generator=g)
    q, scale = linear.quantize_rows(x)
    for at in (slice(0, 3), slice(139990, 140000)):
        check_codes(x[at], q[at], scale[at])
    del x
    w = codes((40, 16000), g)
    ws = scales(40, g)
    out = linear.int8_linear(q, scale, w, ws, out_dtype=torch.float32)
    check_int8(q[-300:], scale[-300:], w, ws, None, "none", out[-300:])
    last = torch.arange(139999, 139000, -1, dtype=torch.int32, device=DEV)
    part = linear.grouped_linear(q, w[None], offsets_of([last.numel()]), in_rows=last, x_scale=scale, weight_scale=ws[None], out_dtype=torch.float32)
    assert torch.equal(part, out[last.long()])
    few = linear.grouped_linear(q, w[None], offsets_of([3]), in_rows=last[:3].contiguous(), x_scale=scale, weight_scale=ws[None], out_dtype=torch.float32)
    assert torch.equal(few, part[:3])  # sums of whole numbers: the same from every kernel
    del q, out
    rows, n = 2200000, 1000
    q, w = codes((rows, 16), g), codes((n, 16), g)
    qs, ws = scales(rows, g), scales(n, g)
    out = linear.int8_linear(q, qs, w, ws)
    for at in (slice(0, 200), slice(rows - 200, rows)):
        check_int8(q[at], qs[at], w, ws, None, "none", out[at])
    back = torch.arange(rows - 1, -1, -1, dtype=torch.int32, device=DEV)
    turned = linear.grouped_linear(q, w[None], offsets_of([rows]), out_rows=back, x_scale=qs, weight_scale=ws[None], out=torch.empty_like(out))
    assert torch.equal(turned[0], out[-1]) and torch.equal(turned[-1], out[0]) and torch.equal(turned[rows // 2], out[rows - 1 - rows // 2])
    del out, turned, q
    w = torch.empty(70, 1000, 32000, dtype=torch.float16, device=DEV)
    for part in w.split(10):
        part.normal_(generator=g)
    x = torch.randn(900, 32000, generator=g, device=DEV).half()
    for sizes in ([0] * 66 + [1, 0, 1, 1], [0] * 66 + [100, 0, 200, 600]):  # a few rows, and tiles
        offsets = offsets_of(sizes)
        got = linear.grouped_linear(x[:sum(sizes)], w, offsets)
        exact, slack = plain_grouped(x[:sum(sizes)], w, offsets, None, "none", None, None, torch.zeros_like(got))
        check(got, exact, slack)
    linear.check_status(DEV)


# ---- refusals ----------------------------------------------------------------------------------------------------
def test_refusals():
    x = torch.zeros(8, 32, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(2, 16, 32, dtype=torch.bfloat16, device=DEV)
    off = offsets_of([4, 4])
    q, qs = linear.quantize_rows(x)
    wq, ws = linear.quantize_rows(w[0])
    bad = [
        (TypeError, lambda: linear.quantize_rows(x.double())),
        (ValueError, lambda: linear.quantize_rows(x[0])),
        (ValueError, lambda: linear.quantize_rows(x.clone().requires_grad_())),
        (TypeError, lambda: linear.group_rows(torch.zeros(4, device=DEV), 2)),
        (_lib.EbError, lambda: linear.group_rows(torch.zeros(4, dtype=torch.int32, device=DEV), 0)),
        (_lib.EbError, lambda: linear.group_rows(torch.zeros(4, dtype=torch.int32, device=DEV), 1025)),
        (TypeError, lambda: linear.int8_linear(x, qs, wq, ws)),
        (TypeError, lambda: linear.int8_linear(q, qs, w[0], ws)),
        (ValueError, lambda: linear.int8_linear(q, qs[:7], wq, ws)),
        (ValueError, lambda: linear.int8_linear(q, qs, wq, ws[:15])),
        (TypeError, lambda: linear.int8_linear(q, qs.double(), wq, ws)),
        (ValueError, lambda: linear.int8_linear(q[:, :31], qs, wq, ws)),
        (ValueError, lambda: linear.int8_linear(q, qs, wq, ws, activation="gelu")),
        (TypeError, lambda: linear.int8_linear(q, qs, wq, ws, out_dtype=torch.int32)),
        (TypeError, lambda: linear.int8_linear(q, qs, wq, ws, bias=torch.zeros(16, device=DEV).half())),
        (ValueError, lambda: linear.int8_linear(q, qs, wq, ws, bias=torch.zeros(1, 16, device=DEV))),
        (ValueError, lambda: linear.int8_linear(q, qs, wq.cpu(), ws)),
        (ValueError, lambda: linear.int8_linear(q, qs, wq, ws, out=torch.empty(7, 16, device=DEV))),
        (ValueError, lambda: linear.int8_linear(q, qs, wq, ws, out=torch.empty(8, 17, device=DEV))),
        (ValueError, lambda: linear.int8_linear(q, qs, wq, ws, out=torch.empty(16, 8, device=DEV).t())),
        (TypeError, lambda: linear.int8_linear(q, qs, wq, ws, out_dtype=torch.float16, out=torch.empty(8, 16, device=DEV))),
        (TypeError, lambda: linear.grouped_linear(x.float(), w.float(), off)),
        (TypeError, lambda: linear.grouped_linear(x, w.half(), off)),
        (TypeError, lambda: linear.grouped_linear(x, w, off.long())),
        (ValueError, lambda: linear.grouped_linear(x, w, off[:2])),
        (ValueError, lambda: linear.grouped_linear(x, w, None)),
        (ValueError, lambda: linear.grouped_linear(x, w[0], off)),
        (ValueError, lambda: linear.grouped_linear(x, w, off, x_scale=qs)),
        (TypeError, lambda: linear.grouped_linear(x, w, off, out_dtype=torch.float32)),
        (TypeError, lambda: linear.grouped_linear(x, w, off, in_rows=torch.arange(8, device=DEV))),
        (ValueError, lambda: linear.grouped_linear(x, w, off, out_rows=torch.arange(7, device=DEV).int())),
        (ValueError, lambda: linear.grouped_linear(x, w, off, out=x[:, :16])),
        (ValueError, lambda: linear.grouped_linear(x, w.clone().requires_grad_(), off)),
        (ValueError, lambda: linear.grouped_linear(q, wq[None].expand(2, 16, 32), off)),
        (ValueError, lambda: linear.GroupedLinear(w, activation="tanh")),
        (TypeError, lambda: linear.GroupedLinear(w.float())),
    ]
    for kind, call in bad:
        with pytest.raises(kind):
            call()
    with torch.no_grad():
        linear.grouped_linear(x, w.clone().requires_grad_(), off)


def test_empty_calls():
    x = torch.zeros(0, 32, dtype=torch.bfloat16, device=DEV)
    w = torch.zeros(2, 16, 32, dtype=torch.bfloat16, device=DEV)
    assert linear.grouped_linear(x, w, offsets_of([0, 0])).shape == (0, 16)
    q, qs = linear.quantize_rows(x)
    wq, ws = linear.quantize_rows(w[0])
    assert linear.int8_linear(q, qs, wq, ws).shape == (0, 16)
    order, offsets = linear.group_rows(torch.zeros(0, dtype=torch.int64, device=DEV), 4)
    assert order.numel() == 0 and not offsets.any()
    # a list of rows into an x without rows: every entry is out of range
    rows = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert not linear.grouped_linear(x, w, offsets_of([1, 1]), in_rows=rows).any()
    with pytest.raises(_lib.EbError):
        linear.check_status(DEV)


# ---- together ------------------------------------------------------------------------------------------------------
def chain(x, ids, first, second):
    order, offsets = linear.group_rows(ids, first.weight.shape[0])
    h = first(x, offsets, in_rows=order)
    return second(h, offsets, out_rows=order)


def chain_layers(g, quantized):
    first = linear.GroupedLinear((torch.randn(5, 96, 200, generator=g, device=DEV) / 14).bfloat16(),
                                 torch.randn(5, 96, generator=g, device=DEV), "relu")
    second = linear.GroupedLinear((torch.randn(5, 1, 96, generator=g, device=DEV) / 10).bfloat16(), None, "sigmoid")
    return (first.quantize(), second.quantize()) if quantized else (first, second)


@pytest.mark.parametrize("quantized", [False, True])
def test_captured_and_replayed_beside_eager_calls_on_another_stream(quantized):
    g = gen(21)
    first, second = chain_layers(g, quantized)
    xs = [torch.randn(700, 200, generator=g, device=DEV).bfloat16() for _ in range(3)]
    ids = [torch.randint(-1, 5, (700,), generator=g, device=DEV) for _ in range(3)]
    want = [chain(x, i, first, second) for x, i in zip(xs, ids)]
    x, i = xs[0].clone(), ids[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        chain(x, i, first, second)
        for _ in range(2):  # two graphs over the same inputs and weights
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = chain(x, i, first, second)
            graphs.append((graph, out))
    torch.cuda.synchronize()
    for turn in range(3):
        x.copy_(xs[turn])
        i.copy_(ids[turn])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for graph, _ in graphs:
                graph.replay()
        eager = [chain(xs[(turn + 1) % 3], ids[(turn + 1) % 3], first, second) for _ in range(4)]
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want[turn])
        for e in eager:
            assert torch.equal(e, want[(turn + 1) % 3])
    linear.check_status(DEV)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rows", [1, 2, 3, 5, 9, 40])
def test_chain_of_few_rows(rows, quantized):
    """Group, first layer by index, last layer back in order, for one request to a handful: against float64."""
    g = gen(50 + rows)
    first, second = chain_layers(g, quantized)
    x = torch.randn(rows, 200, generator=g, device=DEV).bfloat16()
    ids = torch.randint(-1, 5, (rows,), generator=g, device=DEV)
    got = chain(x, ids, first, second)
    assert got.shape == (rows, 1)

    def layer(rows_in, l, e):  # the rows and weights that the layer multiplies, in 64 bits
        if not quantized:
            return rows_in.double() @ l.weight[e].double().t()
        q, s = linear.quantize_rows(rows_in)
        return int_product(q, l.weight[e]) * s.double()[:, None] * l.weight_scale[e].double()

    for r in range(rows):
        e = int(ids[r])
        if e < 0:
            assert got[r] == 0
            continue
        h = torch.relu(layer(x[r:r + 1], first, e) + first.bias[e].double())
        y = torch.sigmoid(layer(h.bfloat16(), second, e))
        # every hidden value may have fallen to the other side of a border of bf16: one step, at most eps of it.  In 8 bits
        # each is then off by half a unit of the scale on either side, the scale itself by one step of the largest.  All of
        # it goes through the second layer's weights, the sigmoid's slope (1/4 at most) and the result's own rounding
        # (half a step of at most 1); 2^-20 covers the fp32 sums and the sigmoid.
        w = second.weight[e].double().abs() * (second.weight_scale[e].double()[:, None] if quantized else 1)
        off = h.abs() * 2.0 ** -7 + (h.abs().max() / 127 * (1 + 2.0 ** -7) if quantized else 0)
        slack = (off @ w.t()).item() / 4 + half_step(torch.bfloat16) + 2.0 ** -20
        assert (got[r].double() - y[0]).abs() <= slack
    linear.check_status(DEV)


def test_two_threads_on_two_streams():
    """Calls of every kind at once: nothing but the status word is shared between them."""
    import threading

    g = gen(23)
    layers = [chain_layers(g, False), chain_layers(g, True)]
    x = torch.randn(3000, 200, generator=g, device=DEV).bfloat16()
    ids = torch.randint(-1, 5, (3000,), generator=g, device=DEV)
    big_q, big_w = codes((2048, 4000), g), codes((1024, 4000), g)
    qs, ws = scales(2048, g), scales(1024, g)

    def once(i):
        return (chain(x, ids, *layers[i]), linear.int8_linear(big_q, qs, big_w, ws, None, "relu"),
                linear.int8_linear(big_q[:1], qs[:1], big_w, ws), linear.int8_linear(big_q[:200], qs[:200], big_w[:64], ws[:64]))

    want = [once(0), once(1)]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(40):
                    got = once(i)
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        failed.append(i)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not failed
    linear.check_status(DEV)


def pooled_model(**kw):
    from .helpers import device_tables, small_model, to_device
    from recflex_b200.rec_modules import RecomModel

    cfg, tables, values, offsets = small_model(2, 0.01, 300)
    torch.manual_seed(0)
    model = RecomModel([128, 64], DEV, embed_tables=device_tables(tables), **kw)
    return model, to_device(values), to_device(offsets)


@pytest.mark.parametrize("mlp_dtype", FLOATS)
def test_recom_model_in_8_bits(mlp_dtype):
    """The same codes, scales and roundings by hand give the same scores."""
    model, values, offsets = pooled_model(mlp_dtype=mlp_dtype)
    with torch.no_grad():
        full = model(values, offsets)
        pooled = model.embed_layer(values, offsets)
    weights = [(m.weight.detach().clone(), m.bias.detach().clone()) for m in model.mlp if isinstance(m, torch.nn.Linear)]
    out = model.quantize_mlp()(values, offsets)
    assert out.shape == full.shape and out.dtype == mlp_dtype
    x = pooled
    for j, (w, b) in enumerate(weights):
        q, s = linear.quantize_rows(x)
        check_codes(x, q, s)
        wq, wsc = linear.quantize_rows(w)
        act = "sigmoid" if j + 1 == len(weights) else "relu"
        y = linear.int8_linear(q, s, wq, wsc, b.float(), act, mlp_dtype)
        check_int8(q, s, wq, wsc, b.float(), act, y)
        x = y
    assert torch.equal(out, x)


@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("mlp_dtype", [torch.bfloat16, torch.float16])
def test_recom_model_with_experts(mlp_dtype, quantized):
    model, values, offsets = pooled_model(mlp_dtype=mlp_dtype, num_experts=3)
    if quantized:
        model.quantize_mlp()
    ids = torch.randint(-1, 4, (300,), generator=gen(9), device=DEV)
    out = model(values, offsets, experts=ids)
    assert out.shape == (300, 1) and out.dtype == mlp_dtype
    outside = (ids < 0) | (ids >= 3)
    assert (out[outside] == 0).all()
    pooled = model.embed_layer(values, offsets)
    x = pooled
    for e in range(3):
        mine = (ids == e).nonzero().flatten()
        x = pooled[mine]
        one = torch.tensor([0, mine.numel()], dtype=torch.int32, device=DEV)
        for layer in model.mlp:  # the expert alone: its rows in a batch of their own
            if quantized:
                q, s = linear.quantize_rows(x)
                x = linear.grouped_linear(q, layer.weight[e:e + 1], one, layer.bias[e:e + 1], layer.activation, x_scale=s,
                                          weight_scale=layer.weight_scale[e:e + 1], out_dtype=x.dtype)
            else:
                x = linear.grouped_linear(x, layer.weight[e:e + 1], one, layer.bias[e:e + 1], layer.activation)
        # the same sums: which rows stand beside a row does not change it where the same kernel serves both; two
        # kernels may add in another order, which moves a score by a rounding of each of its layers
        torch.testing.assert_close(out[mine].float(), x.float(), rtol=0, atol=8 * half_step(mlp_dtype))
    with pytest.raises(ValueError):
        model(values, offsets)
    with pytest.raises(ValueError):
        model(values, offsets, experts=ids[:-1])
    linear.check_status(DEV)


def test_recom_model_refuses_what_it_cannot_do():
    from recflex_b200.rec_modules import RecomModel

    with pytest.raises(TypeError):
        RecomModel([8], DEV, table_shapes=[(4, 4)], num_experts=2)
    with pytest.raises(ValueError):
        RecomModel([8], DEV, table_shapes=[(4, 4)], mlp_dtype=torch.bfloat16, num_experts=-1)
    model = RecomModel([8], DEV, table_shapes=[(4, 4)])
    v, o = torch.zeros(2, dtype=torch.int32, device=DEV), torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        model([v], [o], experts=v)


def test_layers_keep_their_meaning_through_state_dict_and_copies():
    g = gen(30)
    w = (torch.randn(3, 20, 37, generator=g, device=DEV) / 6).bfloat16()
    a = linear.GroupedLinear(w, torch.randn(3, 20, generator=g, device=DEV), "relu")
    x = torch.randn(50, 37, generator=g, device=DEV).bfloat16()
    off = offsets_of([10, 0, 40])
    want = a(x, off)
    b = linear.GroupedLinear(torch.zeros_like(w), torch.zeros(3, 20, device=DEV), "relu")
    b.load_state_dict(a.state_dict())
    assert torch.equal(b(x, off), want)
    import copy

    assert torch.equal(copy.deepcopy(a).to(DEV)(x, off), want)

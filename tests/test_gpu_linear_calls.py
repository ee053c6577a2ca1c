"""GPU: the dense layers around the products: reports, gradients, modules that move, the sigmoid's ends, long rows."""
import copy

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from recflex_b200 import _lib, linear

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def test_no_report_is_lost_to_a_check_on_another_stream():
    """A product with bad offsets on one stream, a check on another at every distance from it: either that check or the
    next one reports it."""
    x = torch.randn(8, 32, generator=gen(1), device=DEV).bfloat16()
    w = torch.randn(2, 16, 32, generator=gen(2), device=DEV).bfloat16()
    bad = torch.tensor([0, 9, 8], dtype=torch.int32, device=DEV)
    out = torch.empty(8, 16, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    linear.grouped_linear(x, w, bad, out=out)
    torch.cuda.synchronize()

    def reported():
        try:
            linear.check_status(DEV)
        except _lib.EbError as e:
            assert e.code == _lib.EB_ERR_BAD_INPUT
            return True
        return False

    assert reported() and not reported()
    lost = 0
    for turn in range(2000):
        with torch.cuda.stream(side):
            torch.cuda._sleep(turn * 60)  # up to 60 us
            linear.grouped_linear(x, w, bad, out=out)
        first = reported()
        side.synchronize()
        lost += not (reported() or first)
    assert lost == 0


def test_forward_mode_tangents_are_refused():
    """These layers have no derivative: a dual tensor's tangent would be dropped."""
    x = torch.randn(8, 32, device=DEV)
    h = x.bfloat16()
    w = torch.randn(2, 16, 32, device=DEV).bfloat16()
    off = torch.tensor([0, 4, 8], dtype=torch.int32, device=DEV)
    bias = torch.zeros(2, 16, device=DEV)
    q, qs = linear.quantize_rows(x)
    wq, ws = linear.quantize_rows(w[0])
    layer = linear.Int8Linear(w[0].float())
    experts = linear.GroupedLinear(w)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: linear.quantize_rows(dual(x)), lambda: linear.quantize_rows(dual(x)[:, 1:]),
                 lambda: linear.int8_linear(q, dual(qs), wq, ws), lambda: linear.int8_linear(q, qs, wq, dual(ws)),
                 lambda: linear.int8_linear(q, qs, wq, ws, dual(bias[0])),
                 lambda: linear.grouped_linear(dual(h), w, off), lambda: linear.grouped_linear(h, dual(w), off),
                 lambda: linear.grouped_linear(h, w, off, dual(bias)), lambda: linear.grouped_linear(h, w, off, out=dual(h[:, :16].clone())),
                 lambda: layer(dual(x)), lambda: experts(dual(h), off)]
        for i, call in enumerate(calls):
            with pytest.raises(ValueError, match="forward only"):
                call()
                pytest.fail(f"call {i} dropped a tangent")
        want = linear.grouped_linear(h, w, off)  # arguments without one are taken
        with torch.inference_mode():  # nothing is recorded
            assert torch.equal(linear.grouped_linear(h, w, off), want)
    assert torch.equal(linear.grouped_linear(h, w, off), want)


def test_a_tile_may_take_longer_than_a_wait_may_stand_still():
    """Rows of 2^30 values: one tile's sums take more than four seconds, while a wait in which nothing moves ends after two.
    Values of +-1, whose partial sums stay far below 2^24, are summed exactly in fp32 in any order."""
    k, n = 1 << 30, 5
    g = gen(5)

    def signs():
        return torch.randint(0, 2, (k,), generator=g, device=DEV, dtype=torch.int8).mul_(2).sub_(1).bfloat16()

    x = signs()
    w = torch.empty(1, n, k, dtype=torch.bfloat16, device=DEV)
    want = torch.empty(n, dtype=torch.float64, device=DEV)
    for j in range(n):
        w[0, j] = signs()
        want[j] = (x * w[0, j]).sum(dtype=torch.float64)
    same = torch.zeros(128, dtype=torch.int32, device=DEV)  # one row, read 128 times
    off = torch.tensor([0, 128], dtype=torch.int32, device=DEV)
    start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    start.record()
    out = linear.grouped_linear(x[None], w, off, in_rows=same)
    end.record()
    linear.check_status(DEV)
    assert torch.equal(out, want.bfloat16().expand(128, n))
    print(f"{start.elapsed_time(end):.0f} ms")


def layers_of(k):
    g = gen(k)
    w, bias = torch.randn(3, 20, k, generator=g, device=DEV) / k ** 0.5, torch.randn(3, 20, generator=g, device=DEV)
    return [linear.Int8Linear(w[0], bias[0], "relu"), linear.GroupedLinear(w.bfloat16(), bias, "relu"),
            linear.GroupedLinear(w.half(), None), linear.GroupedLinear(w.bfloat16(), bias).quantize()]


def ran(layer, k, dtype):
    x = torch.randn(30, k, generator=gen(7), device=DEV).to(dtype)
    if isinstance(layer, linear.Int8Linear):
        return layer(x)
    return layer(x, torch.tensor([0, 10, 10, 30], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("k", [37, 64])
@pytest.mark.parametrize("which", range(4))
def test_layers_that_move_keep_their_layout(which, k):
    layer = layers_of(k)[which]
    dtype = torch.bfloat16 if layer.weight.dtype == torch.int8 else layer.weight.dtype
    want = ran(layer, k, dtype)
    moved = copy.deepcopy(layer).cpu().to(DEV)
    assert linear.pack_rows(moved.weight) is moved.weight  # read in place: no copy a call
    assert torch.equal(ran(moved, k, dtype), want)


@pytest.mark.parametrize("which", range(4))
def test_layers_that_change_type_keep_their_scales(which):
    k = 37
    layer = layers_of(k)[which]
    before = copy.deepcopy(layer)
    for dtype in (torch.float16, torch.bfloat16):
        layer.to(dtype)
        assert layer.bias is None or layer.bias.dtype == torch.float32 and torch.equal(layer.bias, before.bias)
        scale = getattr(layer, "weight_scale")
        assert scale is None or scale.dtype == torch.float32 and torch.equal(scale, before.weight_scale)
        assert linear.pack_rows(layer.weight) is layer.weight
        out = ran(layer, k, dtype)
        assert out.dtype == dtype
        if layer.weight.dtype == torch.int8:
            assert torch.equal(layer.weight, before.weight) and torch.equal(out, ran(before, k, dtype))


@pytest.mark.parametrize("rows, n", [(2, 512), (40, 1), (300, 16), (900, 512), (900, 100), (65536, 1), (140, 300)])
def test_fp32_sigmoid_to_its_last_places(rows, n):
    """Rows of zeros give sigmoid(bias).  expf is within 2 units of the last place (2 * 2^-23 relative), the sum and the
    quotient are rounded to nearest (2^-24 each): 3 * 2^-23 of the value, down to where fp32 itself ends (half its
    smallest step for each of the last two roundings, two of them for expf)."""
    bias = torch.linspace(-103, 103, n, device=DEV) if n > 1 else torch.full((1,), -88.25, device=DEV)
    if n > 4:
        bias[:6] = torch.tensor([0.0, float("inf"), -float("inf"), -1e4, -88.0, -87.5], device=DEV)
    zero = torch.zeros(max(rows, n), 64, dtype=torch.int8, device=DEV)
    scale = torch.ones(max(rows, n), device=DEV)
    out = linear.int8_linear(zero[:rows], scale[:rows], zero[:n], scale[:n], bias, "sigmoid", torch.float32)
    want = torch.sigmoid(bias.double()).expand(rows, n)
    assert ((out.double() - want).abs() <= want * (3 * 2.0 ** -23) * (1 + 2.0 ** -10) + 3 * 2.0 ** -149).all()


def test_a_given_out_counts_as_changed():
    """What autograd has saved of `out` is no longer what it was: a backward pass through it must say so."""
    a = torch.ones(8, 16, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    x = torch.randn(8, 32, generator=gen(3), device=DEV).bfloat16()
    w = torch.randn(1, 16, 32, generator=gen(4), device=DEV).bfloat16()
    off = torch.tensor([0, 8], dtype=torch.int32, device=DEV)
    wide = torch.ones(8, 20, device=DEV, dtype=torch.bfloat16)
    for out in (torch.ones(8, 16, device=DEV, dtype=torch.bfloat16), wide[:, :16]):
        y = (a * out).sum()
        linear.grouped_linear(x, w, off, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        out = torch.ones(8, 16, device=DEV, dtype=torch.bfloat16)
        assert linear.grouped_linear(x, w, off, out=out) is out


def test_a_check_during_a_capture_is_refused_and_leaves_the_capture_alone():
    g = gen(6)
    x, w = torch.randn(40, 32, generator=g, device=DEV).half(), torch.randn(2, 16, 32, generator=g, device=DEV).half()
    off = torch.tensor([0, 15, 40], dtype=torch.int32, device=DEV)
    want = linear.grouped_linear(x, w, off)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = linear.grouped_linear(x, w, off)
        with pytest.raises(_lib.EbError) as e:
            linear.check_status(DEV)
        second = linear.grouped_linear(x, w, off)
    assert e.value.code == _lib.EB_ERR_UNSUPPORTED
    graph.replay()
    assert torch.equal(first, want) and torch.equal(second, want)
    linear.check_status(DEV)


@pytest.mark.parametrize("kind", ["i8", "bf16"])
@pytest.mark.parametrize("n", [1, 17, 33, 100, 250, 431, 1001])
@pytest.mark.parametrize("rows, k", [(3, 200), (300, 200), (300, 9000), (9000, 1000)])
def test_nothing_is_written_beside_the_columns_of_a_wide_out(rows, k, n, kind):
    """Rows on 16-byte boundaries with columns behind the last one, and rows behind the last one, stay as they were."""
    g = gen(rows + n)
    x = torch.randn(rows, k, generator=g, device=DEV)
    w = torch.randn(n, k, generator=g, device=DEV) / k ** 0.5
    perm = torch.randperm(rows, generator=g, device=DEV).to(torch.int32)
    off = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device=DEV)
    if kind == "i8":
        (q, s), (wq, ws) = linear.quantize_rows(x), linear.quantize_rows(w)
        calls = [(dtype, lambda out, dtype=dtype: linear.int8_linear(q, s, wq, ws, None, "relu", dtype, out=out))
                 for dtype in (torch.float32, torch.bfloat16, torch.float16)]
    else:
        h, two = x.bfloat16(), torch.stack([w, -w]).bfloat16()
        calls = [(torch.bfloat16, lambda out, rows=rows: linear.grouped_linear(h, two, off, out_rows=rows, out=out)) for rows in (None, perm)]
    for dtype, call in calls:
        packed = torch.empty(rows, n, dtype=dtype, device=DEV)
        call(packed)
        for wide in (1024, 1027):
            full = torch.full((rows + 40, wide), 7.0, dtype=dtype, device=DEV)
            call(full[:, :n])
            assert torch.equal(full[:rows, :n], packed)
            assert (full[:, n:] == 7).all() and (full[rows:] == 7).all()
    linear.check_status(DEV)


# sizes that reach each of the kernels and tiles, in rows that end inside 16 bytes
SIZES = [(1, 37, 40), (3, 1001, 33), (40, 37, 1), (300, 203, 1), (200, 3001, 5), (300, 203, 17), (300, 9001, 300), (4096, 1923, 333),
         (4096, 1923, 1000), (4096, 483, 1000), (9000, 6001, 1000), (700, 15607, 700), (16300, 3003, 1001)]


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("kind", ["i8", "bf16", "f16"])
@pytest.mark.parametrize("rows, k, n", SIZES)
def test_what_stands_behind_the_columns_is_not_multiplied(rows, k, n, kind, gather):
    """Columns behind k in the storage of x and the weights: the largest codes or NaN change nothing."""
    g = gen(rows + k)
    dtype = {"i8": torch.int8, "bf16": torch.bfloat16, "f16": torch.float16}[kind]

    def made(*shape):
        t = torch.randn(*shape, generator=g, device=DEV)
        return (t * 40).clamp(-127, 127).to(dtype) if kind == "i8" else t.to(dtype)

    pitch = (k + 15) // 16 * 16 + 32
    x, w = made(rows, pitch), made(3, n, pitch)
    kw = dict(x_scale=torch.rand(rows, generator=g, device=DEV), weight_scale=torch.rand(3, n, generator=g, device=DEV)) if kind == "i8" else {}
    ids = torch.randint(0, 3, (rows,), generator=g, device=DEV)
    order, off = linear.group_rows(ids, 3)
    got = []
    for poison in (0, 127 if kind == "i8" else float("nan")):
        x[:, k:], w[:, :, k:] = poison, poison
        got.append(linear.grouped_linear(x[:, :k], w[:, :, :k], off, in_rows=order if gather else None, **kw).clone())
        if kind == "i8":
            got.append(linear.int8_linear(x[:, :k], kw["x_scale"], w[0, :, :k], kw["weight_scale"][0]).clone())
    half = len(got) // 2
    for a, b in zip(got[:half], got[half:]):
        assert torch.equal(a, b)

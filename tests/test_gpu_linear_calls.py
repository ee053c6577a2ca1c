"""GPU: the dense layers around the products: reports, gradients, modules that move, the sigmoid's ends, long rows."""
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

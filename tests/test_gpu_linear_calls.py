"""GPU: the dense layers around the products: reports, gradients, modules that move, the sigmoid's ends, long rows."""
import pytest
import torch

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

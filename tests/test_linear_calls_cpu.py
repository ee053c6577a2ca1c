"""CPU: the dense-layer entries' refusals and bookkeeping that need no device."""
import os
import subprocess
import sys

import pytest
import torch

from recflex_b200 import _lib, linear

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an aligned address that no refused call looks at


@pytest.mark.parametrize("status, device", [(P + 2, 0), (P, -1), (P, 64)])
def test_check_status_refuses(lib, status, device):
    assert lib.eb_linear_check_status(status, device, None) == _lib.EB_ERR_INVALID_ARG


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
@pytest.mark.parametrize("shape", [(5, 37), (3, 5, 37), (5, 64)])
def test_layers_that_move_keep_their_layout_and_scales(shape, dtype):
    """The bookkeeping alone, without a device: a layer as its constructor leaves it."""
    layer = linear._Layer()
    weight = torch.arange(-60, 60).repeat(8)[: torch.Size(shape).numel()].view(shape).to(dtype)
    layer.register_buffer("weight", linear.pack_rows(weight))
    layer.register_buffer("weight_scale", torch.rand(shape[:-1]) / 3 if dtype is torch.int8 else None)
    layer.register_buffer("bias", torch.rand(shape[:-1]) / 3)
    before = {name: None if t is None else t.clone() for name, t in layer._buffers.items()}
    for change in (lambda: layer.half(), lambda: layer.to(torch.bfloat16), lambda: layer._apply(torch.clone), lambda: layer.to("cpu")):
        change()
        assert linear.pack_rows(layer.weight) is layer.weight
        assert torch.equal(layer.weight.float(), before["weight"].float())
        assert torch.equal(layer.bias, before["bias"]) and layer.bias.dtype == torch.float32
        assert dtype is not torch.int8 or (layer.weight.dtype == dtype and torch.equal(layer.weight_scale, before["weight_scale"]))
    assert layer.to("meta").weight.shape == shape


def layer_with(weight, scale=None):
    layer = linear._Layer()
    layer.register_buffer("weight", linear.pack_rows(weight))
    layer.register_buffer("weight_scale", scale)
    layer.register_buffer("bias", None)
    return layer


@pytest.mark.parametrize("strict", [False, True])
def test_codes_are_not_loaded_as_weights(strict):
    """An 8-bit layer's state does not fit one of 16 bits, nor the other way round, and neither is left half loaded."""
    codes, scale = torch.arange(60, dtype=torch.int8).view(4, 15), torch.full((4,), 0.25)
    full = (torch.arange(60).view(4, 15) / 8).bfloat16()
    for state, layer in ((layer_with(codes, scale), layer_with(full)), (layer_with(full), layer_with(codes, scale))):
        before = layer.weight.clone()
        with pytest.raises(RuntimeError, match="weight is torch"):
            layer.load_state_dict(state.state_dict(), strict=strict)
        assert torch.equal(layer.weight, before)


@pytest.mark.parametrize("assign", [False, True])
def test_loaded_weights_have_the_products_layout(assign):
    codes, scale = torch.arange(60, dtype=torch.int8).view(4, 15), torch.full((4,), 0.25)
    layer = layer_with(torch.zeros_like(codes), torch.zeros(4))
    layer.load_state_dict({"weight": codes, "weight_scale": scale.half()}, assign=assign)
    assert torch.equal(layer.weight, codes) and torch.equal(layer.weight_scale, scale)
    assert layer.weight_scale.dtype == torch.float32
    assert linear.pack_rows(layer.weight) is layer.weight


@pytest.mark.parametrize("x, scale, dtype", [(P, P + 2, _lib.EB_OUT_BF16), (P, P + 1, _lib.EB_OUT_F32),
                                             (P + 1, P, _lib.EB_OUT_F16), (P + 2, P, _lib.EB_OUT_F32)])
def test_quantize_rows_refuses_addresses_off_their_elements(lib, x, scale, dtype):
    assert lib.eb_quantize_rows(x, 4, 8, 8, dtype, P, 16, scale, 0, None) == _lib.EB_ERR_INVALID_ARG


@pytest.mark.parametrize("num_groups", [2 ** 32 + 3, 2 ** 31, -2 ** 31 - 1, 2 ** 64 + 1])
def test_expert_counts_that_do_not_fit_the_entry_are_refused(lib, num_groups):
    """ctypes keeps the low half of a number, which may be a count that the entry takes."""
    with pytest.raises(ValueError, match="num_groups"):
        linear._group_workspace(16, num_groups)
    for count in (0, -1, 1025):
        with pytest.raises(_lib.EbError):
            linear._group_workspace(16, count)


def test_the_package_is_imported_without_cuda_in_torch():
    """The parsers, schedules and modules' definitions need no device, nor a torch that has one."""
    code = ("import torch\ndel torch._C._cuda_getCurrentRawStream\n"
            "import recflex_b200.rec_modules, recflex_b200.linear\n")
    res = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr[-1500:]

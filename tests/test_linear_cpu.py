"""CPU: the dense-layer entry points refuse bad arguments before anything touches a device."""
import ctypes as C

import numpy as np
import pytest
import torch

from recflex_b200 import _lib, linear

P = 1 << 20  # an aligned address that no refused call looks at


def quantize(lib, **kw):
    a = dict(x=P, rows=4, cols=8, x_ld=8, x_dtype=_lib.EB_OUT_BF16, q=P, q_ld=16, scale=P)
    a.update(kw)
    return lib.eb_quantize_rows(a["x"], a["rows"], a["cols"], a["x_ld"], a["x_dtype"], a["q"], a["q_ld"], a["scale"], 0, None)


@pytest.mark.parametrize("change, code", [
    (dict(rows=-1), _lib.EB_ERR_INVALID_ARG), (dict(cols=-1), _lib.EB_ERR_INVALID_ARG),
    (dict(x_dtype=3), _lib.EB_ERR_INVALID_ARG), (dict(x=None), _lib.EB_ERR_INVALID_ARG),
    (dict(q=None), _lib.EB_ERR_INVALID_ARG), (dict(scale=None), _lib.EB_ERR_INVALID_ARG),
    (dict(x_ld=7), _lib.EB_ERR_INVALID_ARG), (dict(q_ld=7), _lib.EB_ERR_INVALID_ARG),
    (dict(rows=1 << 31), _lib.EB_ERR_TOO_LARGE), (dict(cols=1 << 31), _lib.EB_ERR_TOO_LARGE)])
def test_quantize_rows_refuses(lib, change, code):
    assert quantize(lib, **change) == code
    assert lib.eb_last_error()


def test_quantize_no_rows_is_no_work(lib):
    assert quantize(lib, rows=0, x=None, q=None, scale=None) == _lib.EB_OK


def test_group_rows_refuses(lib):
    need = C.c_size_t()
    sizes = lib.eb_group_rows_workspace_bytes
    assert sizes(16, 4, None) == _lib.EB_ERR_INVALID_ARG
    assert sizes(-1, 4, C.byref(need)) == _lib.EB_ERR_INVALID_ARG
    assert sizes(16, 0, C.byref(need)) == _lib.EB_ERR_INVALID_ARG
    assert sizes(16, _lib.EB_MAX_GROUPS + 1, C.byref(need)) == _lib.EB_ERR_TOO_LARGE
    assert sizes(1 << 31, 4, C.byref(need)) == _lib.EB_ERR_TOO_LARGE
    assert sizes(1 << 20, 4, C.byref(need)) == _lib.EB_OK
    call = lib.eb_group_rows
    big = need.value
    assert call(P, 16, 4, 2, P, P, P, big, 0, None) == _lib.EB_ERR_INVALID_ARG
    assert call(None, 16, 4, 0, P, P, P, big, 0, None) == _lib.EB_ERR_INVALID_ARG
    assert call(P, 16, 4, 0, None, P, P, big, 0, None) == _lib.EB_ERR_INVALID_ARG
    assert call(P, 16, 4, 0, P, None, P, big, 0, None) == _lib.EB_ERR_INVALID_ARG
    assert call(P + 4, 16, 4, 1, P, P, P, big, 0, None) == _lib.EB_ERR_INVALID_ARG
    if big:
        assert call(P, 1 << 20, 4, 0, P, P, P, big - 1, 0, None) == _lib.EB_ERR_WORKSPACE_TOO_SMALL
        assert call(P, 1 << 20, 4, 0, P, P, None, big, 0, None) == _lib.EB_ERR_WORKSPACE_TOO_SMALL


def product(lib, **kw):
    a = _lib.EbLinearArgs()
    base = dict(x=P, weight=P, x_scale=P, w_scale=P, offsets=P, out=P, status=P, x_rows=8, x_ld=32, w_ld=32, w_group_ld=512,
                positions=8, out_rows_total=8, out_ld=16, n=16, k=32, num_groups=2, dtype=_lib.EB_ROW_I8,
                out_dtype=_lib.EB_OUT_BF16, activation=0, zero_rest=0)
    base.update(kw)
    for name, value in base.items():
        setattr(a, name, value)
    return lib.eb_linear(C.byref(a), 0, None)


@pytest.mark.parametrize("change, code", [
    (dict(dtype=0), _lib.EB_ERR_INVALID_ARG), (dict(dtype=4), _lib.EB_ERR_INVALID_ARG),
    (dict(out_dtype=3), _lib.EB_ERR_INVALID_ARG), (dict(out_dtype=-1), _lib.EB_ERR_INVALID_ARG),
    (dict(dtype=_lib.EB_OUT_BF16, out_dtype=_lib.EB_OUT_F16), _lib.EB_ERR_INVALID_ARG),
    (dict(dtype=_lib.EB_OUT_BF16, out_dtype=_lib.EB_OUT_F32), _lib.EB_ERR_INVALID_ARG),
    (dict(activation=3), _lib.EB_ERR_INVALID_ARG), (dict(activation=-1), _lib.EB_ERR_INVALID_ARG),
    (dict(n=0), _lib.EB_ERR_INVALID_ARG), (dict(k=0), _lib.EB_ERR_INVALID_ARG),
    (dict(num_groups=0), _lib.EB_ERR_INVALID_ARG), (dict(num_groups=_lib.EB_MAX_GROUPS + 1), _lib.EB_ERR_TOO_LARGE),
    (dict(k=_lib.EB_MAX_I8_COLS + 1), _lib.EB_ERR_TOO_LARGE), (dict(positions=1 << 31), _lib.EB_ERR_TOO_LARGE),
    (dict(n=(1 << 30) + 1), _lib.EB_ERR_TOO_LARGE), (dict(positions=(1 << 31) - 1024), _lib.EB_ERR_TOO_LARGE),
    (dict(dtype=_lib.EB_OUT_F16, out_dtype=_lib.EB_OUT_F16, k=(1 << 30) + 1), _lib.EB_ERR_TOO_LARGE),
    (dict(positions=-1), _lib.EB_ERR_INVALID_ARG), (dict(offsets=None), _lib.EB_ERR_INVALID_ARG),
    (dict(positions=9), _lib.EB_ERR_INVALID_ARG), (dict(out_rows_total=7), _lib.EB_ERR_INVALID_ARG),
    (dict(x=None), _lib.EB_ERR_INVALID_ARG), (dict(weight=None), _lib.EB_ERR_INVALID_ARG),
    (dict(out=None), _lib.EB_ERR_INVALID_ARG), (dict(status=None), _lib.EB_ERR_INVALID_ARG),
    (dict(x_scale=None), _lib.EB_ERR_INVALID_ARG), (dict(w_scale=None), _lib.EB_ERR_INVALID_ARG),
    (dict(x_ld=16), _lib.EB_ERR_INVALID_ARG), (dict(w_ld=16), _lib.EB_ERR_INVALID_ARG),
    (dict(w_group_ld=496), _lib.EB_ERR_INVALID_ARG), (dict(out_ld=15), _lib.EB_ERR_INVALID_ARG),
    (dict(out=P + 1), _lib.EB_ERR_INVALID_ARG), (dict(out=P + 2, out_dtype=_lib.EB_OUT_F32), _lib.EB_ERR_INVALID_ARG),
    (dict(offsets=P + 2), _lib.EB_ERR_INVALID_ARG), (dict(in_rows=P + 1), _lib.EB_ERR_INVALID_ARG),
    (dict(bias=P + 2), _lib.EB_ERR_INVALID_ARG), (dict(w_scale=P + 3), _lib.EB_ERR_INVALID_ARG),
    (dict(x=P + 8), _lib.EB_ERR_UNSUPPORTED), (dict(weight=P + 8), _lib.EB_ERR_UNSUPPORTED),
    (dict(x_ld=40), _lib.EB_ERR_UNSUPPORTED), (dict(w_ld=40, w_group_ld=1024), _lib.EB_ERR_UNSUPPORTED),
    (dict(w_group_ld=520), _lib.EB_ERR_UNSUPPORTED)])
def test_linear_refuses(lib, change, code):
    assert product(lib, **change) == code
    assert lib.eb_last_error()


def test_linear_no_positions_is_no_work(lib):
    assert product(lib, positions=0, x=None, weight=None, out=None) == _lib.EB_OK
    assert lib.eb_linear(None, 0, None) == _lib.EB_ERR_INVALID_ARG
    assert lib.eb_linear_check_status(None, 0, None) == _lib.EB_ERR_INVALID_ARG


def test_host_tensors_are_refused():
    x = torch.zeros(4, 16)
    with pytest.raises(ValueError):
        linear.quantize_rows(x)
    with pytest.raises(ValueError):
        linear.group_rows(torch.zeros(4, dtype=torch.int32), 2)
    with pytest.raises(ValueError):
        linear.int8_linear(x.to(torch.int8), torch.ones(4), torch.zeros(2, 16, dtype=torch.int8), torch.ones(2))
    with pytest.raises(ValueError):
        linear.grouped_linear(x.bfloat16(), torch.zeros(2, 8, 16).bfloat16(), torch.zeros(3, dtype=torch.int32))


def test_wide_rows_are_recognised():
    """`pack_rows` copies exactly the layouts that the products cannot read in place, and keeps their values."""
    wide = linear._wide_strides
    base = torch.arange(6 * 40, dtype=torch.int16).view(6, 40)
    assert linear.pack_rows(base[:, :37]).data_ptr() == base.data_ptr() and wide(base[:, :37]) == (40, 240)
    for t in (base[:, 1:33], base.flatten()[: 5 * 41].view(5, 41), base[:, ::2], base.t(), base[:1].expand(6, 40)):
        assert wide(t) is None
        packed = linear.pack_rows(t)
        assert wide(packed) is not None and torch.equal(packed, t)
    assert wide(torch.zeros(1, 13, dtype=torch.int8)) == (16, 16)
    cube = linear.pack_rows(torch.arange(3 * 5 * 7).view(3, 5, 7).to(torch.int8))
    assert wide(cube) == (16, 80) and wide(cube[:1]) == (16, 80) and wide(cube[:, :1]) == (16, 80)
    assert wide(cube.transpose(0, 1)) is None and wide(cube[1:, 1:]) == (16, 80)


def test_args_struct_matches_the_header(tmp_path):
    """Offsets of the ctypes mirror equal the C compiler's."""
    import os
    import subprocess

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [f[0] for f in _lib.EbLinearArgs._fields_]
    src = tmp_path / "o.c"
    src.write_text('#include <stdio.h>\n#include "recflex_b200.h"\nint main(void) {\n' + "".join(
        f'printf("%zu\\n", offsetof(eb_linear_args, {n}));\n' for n in names) + 'printf("%zu\\n", sizeof(eb_linear_args)); return 0; }\n')
    exe = tmp_path / "o"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [getattr(_lib.EbLinearArgs, n).offset for n in names] + [C.sizeof(_lib.EbLinearArgs)]
    assert np.all(np.diff(got) > 0)
    # the packed form holds the same bytes
    values = list(range(1, len(names) + 1))
    assert _lib.pack_linear_args(*values) == bytes(_lib.EbLinearArgs(*values))

"""Dense layers behind the pooled rows: rows in 8 bits, their matrix product, rows by expert, products by expert.

The reference's model runs `torch.nn.Linear` on the pooled rows (RecFlex/rec_modules.py:143-179) and has none of
these.  All of them call librecflex_b200.so (`eb_quantize_rows`, `eb_linear`, `eb_group_rows`) on the current stream,
never synchronise with the host, and may be captured into a CUDA graph once one of them has run on the device.

They are forward only, like the embedding layer in front of them: an argument that requires a gradient is refused
while gradients are being recorded, and so is one that carries a forward-mode tangent.  Row numbers and offsets live
on the GPU and are checked there: bad ones never fault, and `check_status` reports them.
"""
from __future__ import annotations

import ctypes as C
import functools
import threading
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as _forward_ad
import torch.nn as nn
from torch.autograd.graph import increment_version as _increment_version

from . import _lib

MAX_GROUPS = _lib.EB_MAX_GROUPS
_FLOATS = {torch.float32: _lib.EB_OUT_F32, torch.bfloat16: _lib.EB_OUT_BF16, torch.float16: _lib.EB_OUT_F16}
_ACTIVATIONS = {"none": _lib.EB_ACT_NONE, "relu": _lib.EB_ACT_RELU, "sigmoid": _lib.EB_ACT_SIGMOID}
_INDEX = {torch.int32: _lib.EB_I32, torch.int64: _lib.EB_I64}

_status_lock = threading.Lock()
_status = {}  # device index: (its status word, the word's address)


def _status_word(index: int) -> int:
    """Address of the device's status word, made at the first call.  Calls only set bits in it: all streams share it."""
    word = _status.get(index)
    if word is None:
        with _status_lock:
            word = _status.get(index)
            if word is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the first call on a device must come before any stream capture")
                t = torch.zeros(1, dtype=torch.int32, device=f"cuda:{index}")
                torch.cuda.current_stream(index).synchronize()
                word = _status[index] = (t, t.data_ptr())
    return word[1]


def check_status(device=None) -> None:
    """Raise if a product since the last check met offsets or row numbers outside their range.

    Waits for the device's current stream and answers for the products in front of it there; what products on other
    streams report is seen by this check or by the next one, whichever comes after it."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"check_status needs a CUDA device, got {device}")
    index = torch.cuda.current_device() if device.index is None else device.index
    word = _status.get(index)
    if word is not None:
        _lib.check(_lib.load().eb_linear_check_status(word[1], index, torch.cuda.current_stream(index).cuda_stream))


_Tensor = torch.Tensor
_I8, _I32 = (torch.int8,), (torch.int32,)
# the current stream's handle by device index, without the stream object around it (not there in a torch without CUDA)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _check(name: str, t: torch.Tensor, dims: int, dtypes, index: Optional[int] = None) -> int:
    """The index of the device of a tensor argument that is what it has to be.  (What a call checks first is what costs
    least to ask for; the rest words the refusal.)"""
    if type(t) is _Tensor and t.dtype in dtypes and t.dim() == dims and not t.requires_grad and _forward_ad._current_level < 0:
        at = t.get_device()
        if at == index or (index is None and at >= 0 and t.is_cuda):
            return at
    if not isinstance(t, _Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if index is not None and t.get_device() != index:
        raise ValueError(f"{name} must live on cuda:{index}, it lives on {t.device}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, it has {t.dim()}")
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: dtype {t.dtype} is not one of {', '.join(str(d) for d in dtypes)}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: these layers are forward only (detach it or use torch.no_grad())")
    if _forward_ad._current_level >= 0 and _forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a forward-mode tangent: these layers are forward only (take its primal)")
    return t.get_device()


def _vector(name: str, t: torch.Tensor, shape, dtype: torch.dtype, index: int) -> torch.Tensor:
    if type(t) is _Tensor and t.dtype is dtype and t.is_contiguous() and t.get_device() == index and not t.requires_grad \
            and _forward_ad._current_level < 0 and (t.numel() == shape[0] and t.dim() == 1 if len(shape) == 1 else t.shape == shape):
        return t
    _check(name, t, len(shape), (dtype,), index)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)}, it is {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _wide_strides(t: torch.Tensor) -> Optional[Tuple[int, int]]:
    """(elements between rows, elements between matrices) of `t` [..., rows, k] as the products read it: rows on 16-byte
    boundaries that do not overlap.  None for any other layout.  Where there is one row or matrix, its stride is free
    and reported as a packed tensor has it."""
    shape, stride = t.shape, t.stride()
    k, rows = shape[-1], shape[-2]
    per = 16 // t.element_size()
    if t.data_ptr() % 16 or (stride[-1] != 1 and k > 1):
        return None
    ld = stride[-2]
    if rows <= 1:
        ld = (k + per - 1) // per * per
    elif ld < k or ld % per:
        return None
    group_ld = ld * max(1, rows)
    if t.dim() == 3 and shape[0] > 1:
        group_ld = stride[0]
        if group_ld < ld * (rows - 1) + k or group_ld % per:
            return None
    return ld, group_ld


def _empty_wide(shape, dtype: torch.dtype, device) -> torch.Tensor:
    """Uninitialised [..., rows, k] whose rows start on 16-byte boundaries."""
    per = 16 // dtype.itemsize
    ld = (shape[-1] + per - 1) // per * per
    strides = (ld, 1) if len(shape) == 2 else (ld * shape[1], ld, 1)
    return torch.empty_strided(shape, strides, dtype=dtype, device=device)


def pack_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [rows, k] or [experts, n, k] as it is if its rows start on 16-byte boundaries, otherwise a copy whose rows do.
    The products take any layout and make this copy themselves; weights are better laid out once."""
    if _wide_strides(t) is not None:
        return t
    return _empty_wide(tuple(t.shape), t.dtype, t.device).copy_(t)


def _span(t: torch.Tensor) -> Tuple[int, int]:
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1 if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + last * t.element_size()


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits with one scale a row: `(q, scale)` with `q` int8 `[rows, k]`, `scale` float32 `[rows]`.

    `scale = max|x| / 127` of the row, and `q` the nearest integer (ties to even) to `x / scale`.  A row of zeros has
    scale 0; a row that holds an infinity or a NaN has codes 0 and a scale that is not finite, so that its products are
    NaN.  `x`: `[rows, k]` float32, bfloat16 or float16 with any strides.  The rows of `q` start on 16-byte boundaries.
    """
    index = _check("x", x, 2, _FLOATS)
    rows, k = x.shape
    ld, step = x.stride()
    if k > 1 and step != 1 or rows > 1 and ld < k:
        x = x.contiguous()
        ld = k
    device, q_ld = x.device, (k + 15) // 16 * 16
    q = torch.empty_strided((rows, k), (q_ld, 1), dtype=torch.int8, device=device)
    scale = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=device)
    code = _lib.load().eb_quantize_rows(x.data_ptr(), rows, k, ld if rows > 1 else k, _FLOATS[x.dtype], q.data_ptr(), q_ld,
                                        scale.data_ptr(), index, _current_stream(index))
    if code:
        _lib.check(code)
    return q, scale


@functools.lru_cache(maxsize=256)
def _group_workspace(rows: int, num_groups: int) -> int:
    """Bytes of scratch that eb_group_rows needs for these sizes."""
    if not -2 ** 31 <= num_groups < 2 ** 31:  # ctypes would keep its low half
        raise ValueError(f"num_groups must lie in [1, {MAX_GROUPS}], got {num_groups}")
    need = C.c_size_t()
    _lib.check(_lib.load().eb_group_rows_workspace_bytes(rows, num_groups, C.byref(need)))
    return need.value


def group_rows(groups: torch.Tensor, num_groups: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows by expert: `(order, offsets)`, both int32.

    `groups`: `[rows]` int32 or int64 expert numbers.  `order` lists the row numbers expert by expert, each expert's
    rows in increasing order, then the rows whose number lies outside `[0, num_groups)` (-1 for padding, say).  Expert
    g owns `order[offsets[g]:offsets[g + 1]]`: the `offsets` that `grouped_linear` takes.
    """
    index = _check("groups", groups, 1, _INDEX)
    if not groups.is_contiguous():
        groups = groups.contiguous()
    rows, device, num_groups = groups.shape[0], groups.device, int(num_groups)
    need = _group_workspace(rows, num_groups)
    order = torch.empty_strided((rows,), (1,), dtype=torch.int32, device=device)
    offsets = torch.empty_strided((num_groups + 1,), (1,), dtype=torch.int32, device=device)
    ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=device) if need else None
    code = _lib.load().eb_group_rows(groups.data_ptr(), rows, num_groups, _INDEX[groups.dtype], order.data_ptr(),
                                     offsets.data_ptr(), ws.data_ptr() if need else None, need, index,
                                     _current_stream(index))
    if code:
        _lib.check(code)
    return order, offsets


def _product(index, x, weight, bias, activation, x_scale, weight_scale, offsets, in_rows, out_rows, out_dtype, out):
    x_rows, k = x.shape
    if weight.dim() == 3:
        groups, n, w_k = weight.shape
        lead = (groups, n)
    else:
        n, w_k = weight.shape
        groups, lead = 1, (n,)
    act = _ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
    if k != w_k:
        raise ValueError(f"x has {k} columns, weight has {w_k}")
    if n < 1 or k < 1 or groups < 1:
        raise ValueError(f"weight must not be empty, it is {list(weight.shape)}")
    # tensors made here stay referenced until the launch is on the stream
    positions = x_rows
    in_ptr = out_ptr = offsets_ptr = bias_ptr = x_scale_ptr = w_scale_ptr = 0
    if in_rows is not None:
        _check("in_rows", in_rows, 1, _I32, index)
        in_rows = in_rows if in_rows.is_contiguous() else in_rows.contiguous()
        positions, in_ptr = in_rows.shape[0], in_rows.data_ptr()
    if out_rows is not None:
        _check("out_rows", out_rows, 1, _I32, index)
        if out_rows.shape[0] != positions:
            raise ValueError(f"out_rows has {out_rows.shape[0]} entries for {positions} rows")
        out_rows = out_rows if out_rows.is_contiguous() else out_rows.contiguous()
        out_ptr = out_rows.data_ptr()
    if offsets is not None:
        offsets = _vector("offsets", offsets, (groups + 1,), torch.int32, index)
        offsets_ptr = offsets.data_ptr()
    if bias is not None:
        bias = _vector("bias", bias, lead, torch.float32, index)
        bias_ptr = bias.data_ptr()
    if x.dtype is torch.int8:
        if x_scale is None or weight_scale is None:
            raise ValueError("8-bit products need x_scale and weight_scale")
        x_scale = _vector("x_scale", x_scale, (x_rows,), torch.float32, index)
        weight_scale = _vector("weight_scale", weight_scale, lead, torch.float32, index)
        x_scale_ptr, w_scale_ptr = x_scale.data_ptr(), weight_scale.data_ptr()
        dtype = _lib.EB_ROW_I8
        if out_dtype is None:
            out_dtype = torch.bfloat16 if out is None else out.dtype
    else:
        if x_scale is not None or weight_scale is not None:
            raise ValueError("scales belong to 8-bit products only")
        if out_dtype is not None and out_dtype is not x.dtype:
            raise TypeError(f"products of {x.dtype} give {x.dtype}, not {out_dtype}")
        out_dtype = x.dtype
        dtype = _FLOATS[out_dtype]
    out_code = _FLOATS.get(out_dtype)
    if out_code is None:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    zero_rest = 0
    given = out is not None
    if not given:
        # Rows on 16-byte boundaries, as the next product reads them and the tiles store them (int8 65536 x 256 x 431:
        # 21 us, packed 86); up to 16 units, where the gaps would be a good part of the result, they are packed.
        per_out = 16 // out_dtype.itemsize
        out_ld = n if n <= 16 else (n + per_out - 1) // per_out * per_out
        # without out_rows every position is a row of the result, and the kernel fills those of no group with zeros
        if out_rows is None:
            out = torch.empty_strided((positions, n), (out_ld, 1), dtype=out_dtype, device=x.device)
            zero_rest = int(offsets is not None)
        else:
            out = torch.zeros((positions, out_ld), dtype=out_dtype, device=x.device)
            if out_ld != n:
                out = out[:, :n]
        result_rows = positions
    else:
        _check("out", out, 2, (out_dtype,), index)
        if out.shape[1] != n or (n > 1 and out.stride(1) != 1) or (out.shape[0] > 1 and out.stride(0) < n):
            raise ValueError(f"out must be [rows, {n}] with unit column stride and rows that do not overlap")
        if out_rows is None and out.shape[0] < positions:
            raise ValueError(f"out has {out.shape[0]} rows for {positions}")
        lo, hi = _span(out)
        for t in (x, weight, bias, x_scale, weight_scale, offsets, in_rows, out_rows):
            if t is not None:
                first, last = _span(t)
                if first < hi and lo < last:
                    raise ValueError("out must not share memory with the arguments")
        result_rows = out.shape[0]
        out_ld = out.stride(0) if result_rows > 1 else n
    # layouts that are read in place; the usual ones are recognised without asking for everything (_wide_strides)
    x_ptr, weight_ptr, (x_ld, step) = x.data_ptr(), weight.data_ptr(), x.stride()
    per = 16 if dtype == _lib.EB_ROW_I8 else 8
    if step != 1 or x_ld % per or x_ld < k or x_ptr % 16:
        strides = _wide_strides(x)
        if strides is None:
            x = pack_rows(x)
            strides = _wide_strides(x)
        x_ld, x_ptr = strides[0], x.data_ptr()
    w_strides = weight.stride()
    if groups == 1 and w_strides[-1] == 1 and w_strides[-2] % per == 0 and w_strides[-2] >= k and weight_ptr % 16 == 0:
        w_ld, w_group_ld = w_strides[-2], w_strides[-2] * n
    else:
        strides = _wide_strides(weight)
        if strides is None:
            weight = pack_rows(weight)
            strides = _wide_strides(weight)
        (w_ld, w_group_ld), weight_ptr = strides, weight.data_ptr()
    args = _lib.pack_linear_args(x_ptr, weight_ptr, bias_ptr, x_scale_ptr, w_scale_ptr, offsets_ptr, in_ptr, out_ptr,
                                 out.data_ptr(), _status_word(index), x_rows, x_ld, w_ld, w_group_ld, positions,
                                 result_rows, out_ld, n, k, groups, dtype, out_code, act, zero_rest)
    code = _lib.load().eb_linear(args, index, _current_stream(index))
    if code:
        _lib.check(code)
    if given:  # what autograd has saved of it is no longer what it was
        _increment_version(out)
    return out


def int8_linear(q: torch.Tensor, q_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                bias: Optional[torch.Tensor] = None, activation: str = "none",
                out_dtype: Optional[torch.dtype] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """`activation((q @ weight.T) * q_scale[:, None] * weight_scale + bias)` of 8-bit rows and weights.

    `q` int8 `[rows, k]` and `q_scale` float32 `[rows]` as `quantize_rows` gives them; `weight` int8 `[n, k]`,
    `weight_scale` float32 `[n]`; `bias` float32 `[n]`.  The products are summed exactly in 32-bit integers (k up to
    131071), scaled in fp32 and rounded once to `out_dtype` (float32, bfloat16, the default, or float16).
    Above 16 units a result that is allocated here has its rows on 16-byte boundaries: for other widths it is not packed.
    """
    index = _check("q", q, 2, _I8)
    _check("weight", weight, 2, _I8, index)
    return _product(index, q, weight, bias, activation, q_scale, weight_scale, None, None, None, out_dtype, out)


def grouped_linear(x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   activation: str = "none", in_rows: Optional[torch.Tensor] = None,
                   out_rows: Optional[torch.Tensor] = None, x_scale: Optional[torch.Tensor] = None,
                   weight_scale: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
                   out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One matrix product per expert over ragged runs of rows:
    `out[out_rows[i]] = activation(x[in_rows[i]] @ weight[g].T + bias[g])` for `offsets[g] <= i < offsets[g + 1]`.

    `x` `[rows, k]` bfloat16 or float16 (summed in fp32, result of the same type), or int8 with `x_scale` float32
    `[rows]` (result bfloat16 unless `out_dtype` says otherwise); `weight` `[experts, n, k]` of the same type, with
    `weight_scale` float32 `[experts, n]` for int8; `bias` float32 `[experts, n]`; `offsets` int32 `[experts + 1]`,
    `in_rows` and `out_rows` int32 row numbers (i itself where a list is not given).  `group_rows` makes both.

    Positions of no expert (behind the last offset, or in front of the first) give rows of zeros when the result is
    allocated here, and leave the rows of a given `out` as they were.  No row number may stand twice in `out_rows`.
    Above 16 units a result that is allocated here has its rows on 16-byte boundaries: for other widths it is not packed.
    """
    index = _check("x", x, 2, (torch.bfloat16, torch.float16, torch.int8))
    _check("weight", weight, 3, (x.dtype,), index)
    if offsets is None:
        raise ValueError("offsets must be an int32 tensor")
    return _product(index, x, weight, bias, activation, x_scale, weight_scale, offsets, in_rows, out_rows, out_dtype, out)


class _Layer(nn.Module):
    """What the layers keep wherever they are moved: weights whose rows start on 16-byte boundaries (a copy to another
    device or type is packed, and every product would lay it out again), and biases and scales in 32 bits, as the
    products take them, also where `half()` or `to(dtype)` change the rest of a model."""

    def _apply(self, fn, recurse=True):
        kept = {name: self._buffers[name] for name in ("bias", "weight_scale") if self._buffers[name] is not None}
        super()._apply(fn, recurse)
        for name, before in kept.items():
            now = self._buffers[name]
            if now.dtype is not torch.float32:
                self._buffers[name] = before.to(now.device)
        self._buffers["weight"] = pack_rows(self._buffers["weight"])
        return self

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs):
        # 8-bit codes copied into 16-bit weights, or the other way round, would be no weights at all
        given, kind = state_dict.get(prefix + "weight"), self._buffers["weight"].dtype
        if given is not None and (given.dtype is torch.int8) != (kind is torch.int8):
            error_msgs.append(f"{prefix}weight is {given.dtype}, the layer's is {kind}: quantise the one that is not")
            return
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys, error_msgs)
        self._buffers["weight"] = pack_rows(self._buffers["weight"])  # assigned ones come in any layout and type
        for name in ("bias", "weight_scale"):
            if self._buffers[name] is not None:
                self._buffers[name] = self._buffers[name].float()


class Int8Linear(_Layer):
    """A linear layer in 8 bits: `weight` `[n, k]` is quantised once, one scale per output unit; every call quantises
    its rows, one scale per row, and multiplies 8-bit integers.  The result has the type of the argument."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none"):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
        q, scale = quantize_rows(weight.detach())
        self.activation = activation
        self.register_buffer("weight", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if bias is None else bias.detach().float())

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        q, scale = quantize_rows(x)
        return int8_linear(q, scale, self.weight, self.weight_scale, self.bias, self.activation, x.dtype)


class GroupedLinear(_Layer):
    """One linear layer per expert: `weight` `[experts, n, k]` in bfloat16 or float16, `bias` `[experts, n]`.

    `forward(x, offsets, in_rows, out_rows)` is `grouped_linear`.  `quantize()` turns the weights into 8 bits with one
    scale per expert and output unit; from then on every call quantises its rows."""

    def __init__(self, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none"):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}, got {activation!r}")
        _check("weight", weight.detach(), 3, (torch.bfloat16, torch.float16))
        self.activation = activation
        self.register_buffer("weight", pack_rows(weight.detach()))
        self.register_buffer("weight_scale", None)
        self.register_buffer("bias", None if bias is None else bias.detach().float())

    def quantize(self) -> "GroupedLinear":
        if self.weight.dtype != torch.int8:
            experts, n, k = self.weight.shape
            q, scale = quantize_rows(self.weight.reshape(experts * n, k))
            self.weight = q.unflatten(0, (experts, n))
            self.weight_scale = scale.view(experts, n)
        return self

    def forward(self, x: torch.Tensor, offsets: torch.Tensor, in_rows: Optional[torch.Tensor] = None,
                out_rows: Optional[torch.Tensor] = None) -> torch.Tensor:
        if self.weight.dtype != torch.int8:
            return grouped_linear(x, self.weight, offsets, self.bias, self.activation, in_rows, out_rows)
        q, scale = quantize_rows(x)
        return grouped_linear(q, self.weight, offsets, self.bias, self.activation, in_rows, out_rows, scale,
                              self.weight_scale, x.dtype)

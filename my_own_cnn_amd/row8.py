"""Layers of token networks on 8-bit rows over libmiq_qconv's C-ABI: the root-mean-square norm with the
residual's addition, activations as 8-bit rows, int8 products with a scale for each token and output
channel, and the same by experts.

No reference counterpart.  A tensor (..., C) is rows of C channels, as in the embedding and act8 calls,
whose rules for strides, streams, allocations and repeated results hold here too.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

from ._capi import check, lib
from .conv import _stream
from .train import (_IDS, _REAL, _act, _alike, _alloc, _dense, _halves, _here, _kind, _on_device, _output, _raw_stream,
                    _rows, _workspace, torch)

if torch is not None:
    _I8, _I32, _F32, _BF16 = torch.int8, torch.int32, torch.float32, torch.bfloat16


class Row8(NamedTuple):
    """8-bit rows: int8 `codes` (..., C) and float32 `scales` (...); a value stands for code * scale, a
    row whose scale is NaN for NaN.  Made by rms_row8 and act_row8, of weights (K, C) too."""

    codes: "torch.Tensor"
    scales: "torch.Tensor"


class ExpertsPlan(NamedTuple):
    """(token, slot) pairs sorted by expert, int32: `offsets` (experts + 1) of each expert's pairs, `rows`
    (tokens * slots) the token of each sorted pair, -1 behind the last, and `places`, of the ids'
    shape, where each pair went, -1 for an id without an expert."""

    offsets: "torch.Tensor"
    rows: "torch.Tensor"
    places: "torch.Tensor"


# The calls' checks are inline, like train.py's: on small tensors a call is bound by its time on the host.
_MAKE = tuple.__new__


def _new_row8(lead, c: int, like, kept: Optional[Row8], stream) -> Row8:
    """Storage for 8-bit rows (*lead, c): `kept`, or new."""
    if kept is not None:
        _dense(kept[0], torch.int8, "codes")
        _dense(kept[1], torch.float32, "scales")
        if kept[0].shape != lead + (c,) or kept[1].shape != lead:
            raise ValueError(f"kept must hold codes of shape {lead + (c,)} and scales of shape {lead}")
        return Row8(kept[0], kept[1])
    if stream is None:
        shape = lead + (c,)
        if like.shape == shape and like.is_contiguous():
            return _MAKE(Row8, (torch.empty_like(like, dtype=_I8), like.new_empty(lead, dtype=_F32)))
        return _MAKE(Row8, (like.new_empty(shape, dtype=_I8), like.new_empty(lead, dtype=_F32)))
    return Row8(_alloc(lead + (c,), _I8, like.device, stream), _alloc(lead, _F32, like.device, stream))


def _row8(x, what: str):
    """Shape of 8-bit rows (..., C)."""
    codes, scales = x
    at = codes.get_device()
    shape = codes.shape
    if (at < 0 or at != _here() or codes.dtype is not _I8 or scales.dtype is not _F32 or scales.get_device() != at or
            not codes.is_contiguous() or not scales.is_contiguous() or scales.shape != shape[:-1] or not shape):
        _dense(codes, _I8, f"{what} codes")
        _dense(scales, _F32, f"{what} scales")
        if not shape:
            raise ValueError(f"{what} codes must have a channel dimension")
        raise ValueError(f"{what} scales must be {tuple(shape[:-1])}, got {tuple(scales.shape)}")
    return shape


def _vector(v, size: int, what: str):
    """(address, kind) of a real vector of `size` values."""
    kind = _REAL.get(v.dtype)
    if kind is None or v.get_device() != _here() or v.shape != (size,) or not v.is_contiguous():
        _kind(v.dtype, what)
        _on_device(v, what)
        raise ValueError(f"{what} must be contiguous, of shape {(size,)}")
    return v.data_ptr(), kind


def _f32_of(v, shape, what: str):
    """Address of a contiguous float32 tensor of `shape`, NULL for None."""
    if v is None:
        return None
    if v.shape != shape:
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(v.shape)}")
    return _dense(v, torch.float32, what)


def _handle(like, stream):
    return _raw_stream(like.get_device()) if stream is None else _stream(stream)


# ---- norm ---------------------------------------------------------------------------------------

def _added(x, add, total, shape, stream):
    """(address and row distance of add, tensor, address and row distance of the sum)."""
    if add is None:
        if total is not None:
            raise ValueError("total needs add")
        return None, 0, None, None, 0
    if add.shape != shape or add.dtype != x.dtype:
        raise ValueError(f"add must be {x.dtype} of shape {shape}")
    ld_add = _rows(add, "add")[2]
    if total is None and stream is None and ld_add == shape[-1] and x.is_contiguous():
        total, ld = torch.empty_like(x), ld_add
    else:
        total, ld = _output(total, shape, x.dtype, x, stream)
    return add.data_ptr(), ld_add, total, total.data_ptr(), ld


def rms_fprop(x, gain, *, add=None, eps: float = 1e-6, out=None, total=None, stream=None):
    """x * gain / sqrt(mean(x^2) + eps) by rows of x (..., C), float32 or bfloat16; gain (C,), float32 or
    bfloat16.  With `add`, of x's shape and type, the norm is that of s = x + add rounded to the type,
    and the result is (y, s); `total` receives s and may be x or add.  eps in 1e-30 .. 1e30."""
    kind = _kind(x.dtype, "x")
    rows, c, ld = _rows(x, "x")
    shape = tuple(x.shape)
    gain_at, gain_kind = _vector(gain, c, "gain")
    add_at, ld_add, total, total_at, ld_total = _added(x, add, total, shape, stream)
    if x.is_contiguous():
        y, ld_y = _alike(out, x, shape, x.dtype, stream)
    else:
        y, ld_y = _output(out, shape, x.dtype, x, stream)
    status = lib().miq_rms_fprop(x.data_ptr(), add_at, gain_at, total_at, y.data_ptr(), rows, c, ld, ld_add, ld_total,
                                 ld_y, eps, kind, gain_kind, _handle(x, stream))
    if status:
        check(status, "rms_fprop")
    return y if add is None else (y, total)


def rms_row8(x, gain, *, add=None, eps: float = 1e-6, kept: Optional[Row8] = None, total=None, stream=None):
    """rms_fprop with the norm as 8-bit rows: a Row8, or with `add` (Row8, s).  `kept`: a Row8 to write
    into."""
    kind = _kind(x.dtype, "x")
    rows, c, ld = _rows(x, "x")
    shape = tuple(x.shape)
    gain_at, gain_kind = _vector(gain, c, "gain")
    add_at, ld_add, total, total_at, ld_total = _added(x, add, total, shape, stream)
    held = _new_row8(shape[:-1], c, x, kept, stream)
    status = lib().miq_rms_row8(x.data_ptr(), add_at, gain_at, total_at, held[0].data_ptr(), held[1].data_ptr(), rows, c,
                                ld, ld_add, ld_total, eps, kind, gain_kind, _handle(x, stream))
    if c == 0 and not status:  # rows of nothing: the entry point leaves their scales, this one writes the least
        status = lib().miq_act_row8(None, None, held[1].data_ptr(), held[1].numel(), 0, 0, _act("none"), 0, kind,
                                    _handle(x, stream))
    if status:
        check(status, "rms_row8")
    return held if add is None else (held, total)


def rms_bprop_workspace_size(rows: int, c: int) -> int:
    """Bytes of device workspace rms_bprop(..., workspace=...) needs (no GPU access)."""
    out = C.c_size_t()
    check(lib().miq_rms_bprop_workspace_size(rows, c, C.byref(out)), "rms_bprop_workspace_size")
    return out.value


def rms_bprop(dy, x, gain, *, dsum=None, eps: float = 1e-6, out=None, dgain=None, dtype=None, accumulate: bool = False,
              workspace=None, stream=None):
    """(dx, dgain): the backward pass of rms_fprop at x, which is the sum s where the norm had an addend;
    dx is then the gradient of both.  dy and `dsum`, a gradient that reaches s by another way and is
    added to dx, are of x's shape and type; `out` receives dx.  dgain (C,) is float32 or bfloat16
    (`dtype`, default float32) and summed in an order fixed by the sizes; `accumulate` adds it to
    `dgain`.  `workspace`: a device buffer of at least rms_bprop_workspace_size() bytes, not used by
    another call in flight; None allocates one from PyTorch for this call."""
    kind = _kind(x.dtype, "x")
    rows, c, ld = _rows(x, "x")
    shape = tuple(x.shape)
    if dy.shape != shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must be {x.dtype} of shape {shape}")
    ld_dy = _rows(dy, "dy")[2]
    gain_at, gain_kind = _vector(gain, c, "gain")
    dsum_at, ld_dsum = None, 0
    if dsum is not None:
        if dsum.shape != shape or dsum.dtype != x.dtype:
            raise ValueError(f"dsum must be {x.dtype} of shape {shape}")
        dsum_at, ld_dsum = dsum.data_ptr(), _rows(dsum, "dsum")[2]
    if accumulate and dgain is None:
        raise ValueError("accumulate needs dgain")
    if dgain is None:
        dtype = torch.float32 if dtype is None else dtype
        dgain_kind = _kind(dtype, "dtype")
        dgain = _output(None, (c,), dtype, x, stream)[0]
        dgain_at = dgain.data_ptr()
    else:
        if dtype is not None and dgain.dtype != dtype:
            raise ValueError(f"dgain must be {dtype}")
        dgain_at, dgain_kind = _vector(dgain, c, "dgain")
    if x.is_contiguous():
        dx, ld_dx = _alike(out, x, shape, x.dtype, stream)
    else:
        dx, ld_dx = _output(out, shape, x.dtype, x, stream)
    at, size, held = _workspace(workspace, "miq_rms_bprop_workspace_size", (rows, c), x.device, stream)
    status = lib().miq_rms_bprop(dy.data_ptr(), x.data_ptr(), gain_at, dsum_at, dx.data_ptr(), dgain_at, rows, c, ld_dy,
                                 ld, ld_dsum, ld_dx, eps, 1 if accumulate else 0, kind, gain_kind, dgain_kind, at, size,
                                 _handle(x, stream))
    if status:
        check(status, "rms_bprop")
    return dx, dgain


# ---- 8-bit rows -----------------------------------------------------------------------------------

def act_row8(x, act: str = "none", *, gated: bool = False, kept: Optional[Row8] = None, stream=None) -> Row8:
    """act(x) by rows of x (..., C), float32 or bfloat16, as 8-bit rows; with `gated`, x holds rows of a
    gate and of what it multiplies, (..., 2C), and the rows are act(gate) * up, (..., C).  `act`:
    'none' (8-bit rows of x itself, of a layer's weights for one), 'relu', 'silu' or 'gelu'."""
    kind, which = _kind(x.dtype, "x"), _act(act)
    rows, width, ld = _rows(x, "x")
    c = _halves(width, gated)
    lead = tuple(x.shape)[:-1]
    if width == 0:
        rows = x.shape[:-1].numel()
    held = _new_row8(lead, c, x, kept, stream)
    status = lib().miq_act_row8(x.data_ptr(), held[0].data_ptr(), held[1].data_ptr(), rows, c, ld, which,
                                1 if gated else 0, kind, _handle(x, stream))
    if status:
        check(status, "act_row8")
    return held


def row8_expand(x: Row8, *, dtype=None, out=None, stream=None):
    """What 8-bit rows stand for, code * scale, as float32 or bfloat16 (`dtype`, default float32)."""
    shape = _row8(x, "x")
    codes, scales = x
    if dtype is None:
        dtype = out.dtype if out is not None else _F32
    kind = _REAL.get(dtype)
    if kind is None:
        _kind(dtype, "dtype")
    c = shape[-1]
    if out is None and stream is None:
        y, ld_y, handle = torch.empty_like(codes, dtype=dtype), c, _raw_stream(codes.get_device())
    else:
        (y, ld_y), handle = _output(out, tuple(shape), dtype, codes, stream), _handle(codes, stream)
    status = lib().miq_row8_expand(codes.data_ptr(), scales.data_ptr(), y.data_ptr(), scales.numel(), c, ld_y, kind, handle)
    if status:
        check(status, "row8_expand")
    return y


# ---- products ---------------------------------------------------------------------------------------

def plan_row8_linear(rows: int, c: int, k: int, experts: int = 1):
    """(few, rows, channels, copied) of row8_linear and, with `experts`, row8_experts on as many rows:
    whether the weights go straight to the matrix instructions, a tile's rows and channels, and
    whether rows of codes are first copied to the workspace (no GPU access)."""
    out = (C.c_int32 * 4)()
    check(lib().miq_plan_row8_linear(rows, c, k, experts, out), "plan_row8_linear")
    return bool(out[0]), out[1], out[2], bool(out[3])


def row8_workspace_size(x_rows: int, rows: int, c: int, k: int, experts: int = 1) -> int:
    """Bytes of device workspace row8_linear(..., workspace=...) (x_rows == rows) and, with `experts`,
    row8_experts need: 0 wherever c is a multiple of 16, and for few rows (no GPU access)."""
    out = C.c_size_t()
    check(lib().miq_row8_workspace_size(x_rows, rows, c, k, experts, C.byref(out)), "row8_workspace_size")
    return out.value


def row8_linear(x: Row8, w: Row8, *, bias=None, add=None, dtype=None, out=None, workspace=None, stream=None):
    """A linear layer of 8-bit rows x (..., C) by 8-bit weights w (K, C): the exact int8 product times the
    row's and the channel's scale, plus `bias` (K,), float32, plus `add` (..., K), of the result's
    type; (..., K), float32 or bfloat16 (`dtype`, default bfloat16).  `out` may be `add`.
    `workspace`: a device buffer of at least row8_workspace_size() bytes, not used by another call in
    flight; None allocates one from PyTorch for this call where it needs one."""
    shape = _row8(x, "x")
    w_shape = _row8(w, "w")
    c = shape[-1]
    if len(w_shape) != 2 or w_shape[1] != c:
        raise ValueError(f"w must be (output channels, {c}), got {tuple(w_shape)}")
    k = w_shape[0]
    if dtype is None:
        dtype = out.dtype if out is not None else (add.dtype if add is not None else _BF16)
    kind = _REAL.get(dtype)
    if kind is None:
        _kind(dtype, "dtype")
    y_shape = (shape[0], k) if len(shape) == 2 else tuple(shape[:-1]) + (k,)
    add_at, ld_add = None, 0
    if add is not None:
        if add.shape != y_shape or add.dtype is not dtype:
            raise ValueError(f"add must be {dtype} of shape {y_shape}")
        add_at, ld_add = add.data_ptr(), _rows(add, "add")[2]
    codes, scales = x
    if out is None and stream is None:
        y, ld_y, handle = codes.new_empty(y_shape, dtype=dtype), k, _raw_stream(codes.get_device())
    else:
        (y, ld_y), handle = _output(out, y_shape, dtype, codes, stream), _handle(codes, stream)
    rows = scales.numel()
    at, size, held = None, 0, None
    if c % 16:
        at, size, held = _workspace(workspace, "miq_row8_workspace_size", (rows, rows, c, k, 1), codes.device, stream)
    status = lib().miq_row8_linear(codes.data_ptr(), scales.data_ptr(), w[0].data_ptr(), w[1].data_ptr(),
                                   None if bias is None else _f32_of(bias, (k,), "bias"), add_at, y.data_ptr(), rows, c,
                                   k, ld_add, ld_y, kind, at, size, handle)
    if status:
        check(status, "row8_linear")
    return y


# ---- experts ------------------------------------------------------------------------------------------

def experts_plan(ids, experts: int, *, stream=None) -> ExpertsPlan:
    """Sorts the (token, slot) pairs of `ids` (tokens, slots) or (tokens,), int32 or int64, by expert, in
    their order within an expert; ids outside [0, experts) are left out."""
    if ids.dtype not in _IDS:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    shape = tuple(ids.shape)
    if len(shape) not in (1, 2):
        raise ValueError("ids must be (tokens, slots) or (tokens,)")
    slots = shape[1] if len(shape) == 2 else 1
    if experts < 1:
        raise ValueError("experts must be at least 1")
    ids_at = _dense(ids, ids.dtype, "ids")
    if stream is None:
        offsets = ids.new_empty(experts + 1, dtype=_I32)
        rows = ids.new_empty(ids.numel(), dtype=_I32)
        places = torch.empty_like(ids, dtype=_I32)
    else:
        offsets, rows, places = (_alloc(s, torch.int32, ids.device, stream) for s in ((experts + 1,), (ids.numel(),), shape))
    status = lib().miq_experts_plan(ids_at, offsets.data_ptr(), rows.data_ptr(), places.data_ptr(), shape[0], slots,
                                    experts, _IDS[ids.dtype], _handle(ids, stream))
    if status:
        check(status, "experts_plan")
    return _MAKE(ExpertsPlan, (offsets, rows, places))


def row8_experts(x: Row8, w: Row8, offsets, *, rows=None, bias=None, dtype=None, out=None, workspace=None,
                 stream=None):
    """row8_linear by experts: rows offsets[e] .. offsets[e + 1] - 1 of the result by the weights w[e] of
    w (experts, K, C) and bias (experts, K).  Row i takes row rows[i] of x (N, C), or row i without
    `rows`; an entry of `rows` outside x stands for a row of zeros.  offsets (experts + 1,) and
    `rows` are int32 tensors on the device, as experts_plan gives them; offsets rise and end within
    the rows.  Rows of the result behind the last expert's are not written.  `workspace`: as of
    row8_linear."""
    shape = _row8(x, "x")
    w_shape = _row8(w, "w")
    if len(shape) != 2:
        raise ValueError("x must be (rows, channels)")
    n, c = shape
    if len(w_shape) != 3 or w_shape[2] != c:
        raise ValueError(f"w must be (experts, output channels, {c}), got {tuple(w_shape)}")
    experts, k, _ = w_shape
    if offsets.shape != (experts + 1,):
        raise ValueError(f"offsets must be {(experts + 1,)}, got {tuple(offsets.shape)}")
    offsets_at = _dense(offsets, _I32, "offsets")
    x_rows, rows_at = n, None
    if rows is not None:
        if rows.dim() != 1:
            raise ValueError("rows must have one dimension")
        n, rows_at = rows.numel(), _dense(rows, _I32, "rows")
    if dtype is None:
        dtype = out.dtype if out is not None else _BF16
    kind = _REAL.get(dtype)
    if kind is None:
        _kind(dtype, "dtype")
    codes, scales = x
    if out is None and stream is None:
        y, ld_y, handle = codes.new_empty((n, k), dtype=dtype), k, _raw_stream(codes.get_device())
    else:
        (y, ld_y), handle = _output(out, (n, k), dtype, codes, stream), _handle(codes, stream)
    at, size, held = None, 0, None
    if c % 16:
        at, size, held = _workspace(workspace, "miq_row8_workspace_size", (x_rows, n, c, k, experts), codes.device, stream)
    status = lib().miq_row8_experts(codes.data_ptr(), scales.data_ptr(), w[0].data_ptr(), w[1].data_ptr(),
                                    None if bias is None else _f32_of(bias, (experts, k), "bias"), offsets_at, rows_at,
                                    y.data_ptr(), x_rows, n, c, k, experts, ld_y, kind, at, size, handle)
    if status:
        check(status, "row8_experts")
    return y


def experts_join(y, places, share=None, *, add=None, out=None, stream=None):
    """The experts' rows back to their tokens: out[t] = add[t] + sum over s of share[t, s] * y[places[t, s]],
    summed in float32 in the order of s; places outside y add nothing.  y (N, C), float32 or bfloat16;
    places (tokens, slots) or (tokens,), int32, as experts_plan gives it; share of places' shape,
    float32 (default: ones); add (tokens, C) of y's type.  `out` may be `add`."""
    kind = _kind(y.dtype, "y")
    if y.dim() != 2:
        raise ValueError("y must be (rows, channels)")
    _, c, ld = _rows(y, "y")
    shape = tuple(places.shape)
    if len(shape) not in (1, 2):
        raise ValueError("places must be (tokens, slots) or (tokens,)")
    slots = shape[1] if len(shape) == 2 else 1
    places_at = _dense(places, _I32, "places")
    share_at = _f32_of(share, shape, "share")
    add_at, ld_add = None, 0
    if add is not None:
        if add.shape != (shape[0], c) or add.dtype != y.dtype:
            raise ValueError(f"add must be {y.dtype} of shape {(shape[0], c)}")
        add_at, ld_add = add.data_ptr(), _rows(add, "add")[2]
    to, ld_out = _output(out, (shape[0], c), y.dtype, y, stream)
    status = lib().miq_experts_join(y.data_ptr(), places_at, share_at, add_at, to.data_ptr(), y.shape[0], shape[0], slots, c,
                                    ld, ld_add, ld_out, kind, _handle(y, stream))
    if status:
        check(status, "experts_join")
    return to


__all__ = ["ExpertsPlan", "Row8", "act_row8", "experts_join", "experts_plan", "plan_row8_linear", "rms_bprop",
           "rms_bprop_workspace_size", "rms_fprop", "rms_row8", "row8_expand", "row8_experts", "row8_linear",
           "row8_workspace_size"]

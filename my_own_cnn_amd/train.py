"""Training operators of token networks over libmiq_qconv's C-ABI: the embedding table's lookup and
gradient, and activations kept in 8 bits between the forward and the backward pass.

No reference counterpart.  Rows are what the convolutions call NHWC pixels: a tensor of shape
(..., C) is rows of C channels.  Channels are dense; rows may lie apart (a slice of wider rows),
but leading dimensions must have one common row distance.  Every call is asynchronous on the given
(default: PyTorch's current) HIP stream, and gives the same bits for the same inputs.  What a call
allocates itself belongs to the stream it runs on.
"""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple, Optional

from ._capi import ACTS, MIQ_BF16, MIQ_F32, MIQ_I32, MIQ_I64, check, lib
from .conv import _current_device, _raw_stream, _stream

try:
    import torch
except ImportError:  # pragma: no cover
    torch = None

GROUP = 32  # channels that share an exponent byte

_REAL = {torch.float32: MIQ_F32, torch.bfloat16: MIQ_BF16} if torch is not None else {}
_IDS = {torch.int32: MIQ_I32, torch.int64: MIQ_I64} if torch is not None else {}


class Act8(NamedTuple):
    """A tensor kept in 8 bits: int8 `codes` of its shape and uint8 exponent bytes `scales`, one per
    32 channels of a row, (..., ceil(C / 32)); a value stands for code * 2^(scale - 127), the whole
    group for NaN where the byte is 255.  `gated` rows hold a gate and what it multiplies, C channels
    each, grouped apart.  `act` is the activation that was applied to the kept tensor."""

    codes: "torch.Tensor"
    scales: "torch.Tensor"
    act: str = "none"
    gated: bool = False


# A call below takes 7 to 9 us on the host, 3.4 of them in the entry point, 1 to 1.5 for each tensor it
# allocates: small layers are bound by it.  So its checks come inline, their messages from a function,
# shapes are plain tuples (torch's own take 0.3 us longer to join and to allocate from), and a tensor
# shaped like another comes from empty_like (1.1 us for 1.7).
_here = _current_device if _current_device is not None else (torch.cuda.current_device if torch is not None else None)
if _raw_stream is None:  # pragma: no cover - older torch
    def _raw_stream(device):
        return torch.cuda.current_stream(device).cuda_stream


def _kind(dtype, what: str) -> int:
    kind = _REAL.get(dtype)
    if kind is None:
        raise ValueError(f"{what} must be float32 or bfloat16, got {dtype}")
    return kind


def _act(act: str) -> int:
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}, got {act!r}")
    return ACTS[act]


def _on_device(t, what: str) -> None:
    at = t.get_device()
    if at < 0:
        raise ValueError(f"{what} must live in device memory")
    if at != _here():
        raise ValueError(f"{what} must live on the current device")


def _rows(t, what: str):
    """(rows, channels, row distance) of a tensor (..., C)."""
    at = t.get_device()
    if at < 0 or at != _here():
        _on_device(t, what)
    shape = t.shape
    if not shape:
        raise ValueError(f"{what} must have a channel dimension")
    c = shape[-1]
    if t.is_contiguous():
        return (t.numel() // c if c else 0), c, c
    stride = t.stride()
    if c > 1 and stride[-1] != 1:
        raise ValueError(f"{what}: channels must be dense")
    rows, ld = 1, c
    for size, step in zip(reversed(shape[:-1]), reversed(stride[:-1])):
        if size == 1:
            continue
        if rows == 1:
            ld = step
        elif step != rows * ld:
            raise ValueError(f"{what}: rows must have one common distance")
        rows *= size
    if rows > 1 and ld < c:
        raise ValueError(f"{what}: rows must not overlap")
    return rows, c, max(ld, c)


def _dense(t, dtype, what: str) -> int:
    if t.dtype != dtype or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {dtype}")
    at = t.get_device()
    if at < 0 or at != _here():
        _on_device(t, what)
    return t.data_ptr()


def _alloc(shape, dtype, device, stream):
    """A new tensor whose memory belongs to the stream of the call."""
    if stream is None:
        return torch.empty(shape, dtype=dtype, device=device)
    handle = _stream(stream)
    own = torch.cuda.ExternalStream(handle, device) if handle else torch.cuda.default_stream(device)
    with torch.cuda.stream(own):
        return torch.empty(shape, dtype=dtype, device=device)


def _output(out, shape, dtype, like, stream):
    """(tensor, row distance) of a call's result: `out`, or a new one on the device of `like`."""
    if out is None:
        if stream is None:
            return like.new_empty(shape, dtype=dtype), shape[-1]
        return _alloc(shape, dtype, like.device, stream), shape[-1]
    if out.shape != shape or out.dtype != dtype:
        raise ValueError(f"out must be {dtype} of shape {shape}")
    return out, _rows(out, "out")[2]


def _alike(out, like, shape, dtype, stream):
    """_output for a result of the shape of `like`, which is contiguous."""
    if out is None and stream is None:
        return torch.empty_like(like, dtype=dtype), shape[-1]
    return _output(out, shape, dtype, like, stream)


_sizes = {}  # workspace bytes by problem


def _workspace(workspace, size: str, problem, device, stream):
    """(address, bytes) of the caller's workspace, or of one allocated for this call and the tensor
    that holds it."""
    need = _sizes.get((size, problem))
    if need is None:
        got = C.c_size_t()
        check(getattr(lib(), size)(*problem, C.byref(got)), size)
        need = got.value
        if len(_sizes) < 4096:
            _sizes[size, problem] = need
    if workspace is not None:
        _on_device(workspace, "workspace")
        if not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous")
        return workspace.data_ptr(), workspace.numel() * workspace.element_size(), workspace
    if need == 0:
        return None, 0, None
    held = _alloc((need,), torch.uint8, device, stream)
    return held.data_ptr(), need, held


# ---- embedding ------------------------------------------------------------------------------

def embed_fprop(table, ids, *, scale: float = 1.0, dtype=None, out=None, stream=None):
    """scale * table[ids]: rows of `table` (vocab, C), float32 or bfloat16, by `ids` (any shape,
    int32 or int64), rounded once to `dtype` (default: the table's).  A position whose id lies
    outside [0, vocab) gets a row of zeros.  Returns (*ids.shape, C)."""
    kind = _kind(table.dtype, "table")
    if table.dim() != 2:
        raise ValueError("table must be (vocab, channels)")
    if ids.dtype not in _IDS:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    _, c, ld = _rows(table, "table")
    vocab = table.shape[0]
    ids_at = _dense(ids, ids.dtype, "ids")
    if dtype is None:
        dtype = out.dtype if out is not None else table.dtype
    y_kind = _kind(dtype, "dtype")
    y, ld_y = _output(out, tuple(ids.shape) + (c,), dtype, table, stream)
    status = lib().miq_embed_fprop(table.data_ptr(), ids_at, y.data_ptr(), vocab, c, ids.numel(), ld, ld_y, scale, kind,
                                   _IDS[ids.dtype], y_kind,
                                   _raw_stream(table.get_device()) if stream is None else _stream(stream))
    if status:
        check(status, "embed_fprop")
    return y


def embed_grad_workspace_size(vocab: int, c: int, tokens: int) -> int:
    """Bytes of device workspace embed_grad(..., workspace=...) needs (no GPU access)."""
    out = C.c_size_t()
    check(lib().miq_embed_grad_workspace_size(vocab, c, tokens, C.byref(out)), "embed_grad_workspace_size")
    return out.value


def plan_embed_grad(vocab: int, c: int, tokens: int):
    """(launches that sort the tokens, parts that the sorted tokens are cut into) of embed_grad, zeros
    where nothing is sorted: one launch without a workspace (no GPU access)."""
    out = (C.c_int32 * 2)()
    check(lib().miq_plan_embed_grad(vocab, c, tokens, out), "plan_embed_grad")
    return out[0], out[1]


def embed_grad(dy, ids, vocab: int, *, scale: float = 1.0, dtype=None, accumulate: bool = False, out=None,
               workspace=None, stream=None):
    """The gradient of embed_fprop with respect to the table: (vocab, C), float32 or bfloat16
    (`dtype`, default float32), row v the sum of scale * dy over the positions whose id is v, in an
    order fixed by the ids and the sizes.  `accumulate` adds it to `out` and touches only rows that have a token.
    `workspace`: a device buffer of at least embed_grad_workspace_size() bytes, not used by another
    call in flight; None allocates one from PyTorch for this call."""
    kind = _kind(dy.dtype, "dy")
    if ids.dtype not in _IDS:
        raise ValueError(f"ids must be int32 or int64, got {ids.dtype}")
    _, c, ld = _rows(dy, "dy")
    if dy.shape[:-1] != ids.shape:
        raise ValueError(f"dy must be (*ids.shape, channels), got {tuple(dy.shape)} and {tuple(ids.shape)}")
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    ids_at = _dense(ids, ids.dtype, "ids")
    if dtype is None:
        dtype = out.dtype if out is not None else torch.float32
    d_kind = _kind(dtype, "dtype")
    tokens = ids.numel()
    d, ld_d = _output(out, (vocab, c), dtype, dy, stream)
    at, size, held = _workspace(workspace, "miq_embed_grad_workspace_size", (vocab, c, tokens), dy.device, stream)
    status = lib().miq_embed_grad(dy.data_ptr(), ids_at, d.data_ptr(), vocab, c, tokens, ld, ld_d, scale,
                                  1 if accumulate else 0, kind, _IDS[ids.dtype], d_kind, at, size,
                                  _raw_stream(dy.get_device()) if stream is None else _stream(stream))
    if status:
        check(status, "embed_grad")
    return d


# ---- activations kept in 8 bits -----------------------------------------------------------------

def _halves(width: int, gated: bool) -> int:
    if not gated:
        return width
    if width % 2:
        raise ValueError("gated rows hold a gate and what it multiplies: an even number of channels")
    return width // 2


def _new_kept(x, shape, lead, groups: int, act: str, gated: bool, kept: Optional[Act8], stream) -> Act8:
    """Storage for x (of `shape`, rows `lead`) kept in 8 bits: `kept`, or new."""
    if kept is not None:
        _dense(kept.codes, torch.int8, "codes")
        _dense(kept.scales, torch.uint8, "scales")
        if kept.codes.shape != shape or kept.scales.shape != lead + (groups,):
            raise ValueError(f"kept must hold codes of shape {shape} and {groups} scales a row")
        return Act8(kept.codes, kept.scales, act, gated)
    if stream is None:
        codes = torch.empty_like(x, dtype=torch.int8) if x.is_contiguous() else x.new_empty(shape, dtype=torch.int8)
        return Act8(codes, x.new_empty(lead + (groups,), dtype=torch.uint8), act, gated)
    return Act8(_alloc(shape, torch.int8, x.device, stream), _alloc(lead + (groups,), torch.uint8, x.device, stream), act,
                gated)


def _kept(kept: Act8):
    """(rows, channels, shape of the codes, shape of their rows) of a kept tensor."""
    codes, scales, _, gated = kept
    at = codes.get_device()
    if (codes.dtype != torch.int8 or scales.dtype != torch.uint8 or at < 0 or at != _here() or
            scales.get_device() != at or not codes.is_contiguous() or not scales.is_contiguous()):
        _dense(codes, torch.int8, "codes")
        _dense(scales, torch.uint8, "scales")
    shape = tuple(codes.shape)
    if not shape:
        raise ValueError("codes must have a channel dimension")
    width = shape[-1]
    c = _halves(width, True) if gated else width
    groups = (c + 31) // GROUP * (2 if gated else 1)
    lead = shape[:-1]
    if scales.shape != lead + (groups,):
        raise ValueError(f"scales must be {lead + (groups,)}, got {tuple(scales.shape)}")
    return (codes.numel() // width if width else codes.shape[:-1].numel()), c, shape, lead


def act8_fprop(x, act: str = "silu", *, gated: bool = False, out=None, kept: Optional[Act8] = None, stream=None):
    """(act(x), x kept in 8 bits) in one pass over x (..., C); with `gated`, x holds rows of a gate and
    of what it multiplies, (..., 2C), and the result is act(gate) * up, (..., C).  `act`: 'none',
    'relu', 'silu' or 'gelu'.  The activation is that of x itself, not of the kept values.  `kept`:
    an Act8 to write into."""
    dtype = x.dtype
    kind, which = _kind(dtype, "x"), _act(act)
    rows, width, ld = _rows(x, "x")
    shape = tuple(x.shape)
    lead = shape[:-1]
    c = _halves(width, True) if gated else width
    if gated or not x.is_contiguous():
        y, ld_y = _output(out, lead + (c,), dtype, x, stream)
    else:
        y, ld_y = _alike(out, x, shape, dtype, stream)
    held = _new_kept(x, shape, lead, (c + 31) // GROUP * (2 if gated else 1), act, gated, kept, stream)
    status = lib().miq_act8_fprop(x.data_ptr(), y.data_ptr(), held[0].data_ptr(), held[1].data_ptr(), rows, c, ld, ld_y,
                                  which, 1 if gated else 0, kind,
                                  _raw_stream(x.get_device()) if stream is None else _stream(stream))
    if status:
        check(status, "act8_fprop")
    return y, held


def act8_keep(x, *, kept: Optional[Act8] = None, stream=None) -> Act8:
    """x (..., C) kept in 8 bits: the input of a layer whose weight gradient act8_grad computes, or
    that act8_expand gives back."""
    kind = _kind(x.dtype, "x")
    rows, c, ld = _rows(x, "x")
    shape = tuple(x.shape)
    held = _new_kept(x, shape, shape[:-1], (c + 31) // GROUP, "none", False, kept, stream)
    status = lib().miq_act8_fprop(x.data_ptr(), None, held[0].data_ptr(), held[1].data_ptr(), rows, c, ld, c, 0, 0, kind,
                                  _raw_stream(x.get_device()) if stream is None else _stream(stream))
    if status:
        check(status, "act8_keep")
    return held


def act8_expand(kept: Act8, *, apply: bool = False, dtype=None, out=None, stream=None):
    """The kept values as float32 or bfloat16 (`dtype`, default float32; exact in both), or with
    `apply` the activation of them recomputed: act(x') or act(gate') * up'."""
    rows, c, shape, lead = _kept(kept)
    codes, scales, act, gated = kept
    if dtype is None:
        dtype = out.dtype if out is not None else torch.float32
    kind = _kind(dtype, "dtype")
    halves = gated and not apply  # the halves of a gated row are rows of their own
    if gated and apply:
        y, ld_y = _output(out, lead + (c,), dtype, codes, stream)
    else:
        y, ld_y = _alike(out, codes, shape, dtype, stream)
    if halves:
        if not y.is_contiguous():
            raise ValueError("out must be contiguous for the values of gated rows")
        rows, ld_y = 2 * rows, c
    status = lib().miq_act8_expand(codes.data_ptr(), scales.data_ptr(), y.data_ptr(), rows, c, ld_y,
                                   _act(act) if apply else 0, 1 if gated and apply else 0, kind,
                                   _raw_stream(codes.get_device()) if stream is None else _stream(stream))
    if status:
        check(status, "act8_expand")
    return y


def act8_bprop(dy, kept: Act8, *, out=None, stream=None):
    """The backward pass of act8_fprop at the kept values: dy * act'(x'), or for gated rows
    [dy * up' * act'(gate'), dy * act(gate')]; dy (..., C), float32 or bfloat16."""
    kind = _kind(dy.dtype, "dy")
    rows, c, shape, lead = _kept(kept)
    codes, scales, act, gated = kept
    if dy.shape != lead + (c,):
        raise ValueError(f"dy must be {lead + (c,)}, got {tuple(dy.shape)}")
    _, _, ld = _rows(dy, "dy")
    dx, ld_dx = _alike(out, codes, shape, dy.dtype, stream)
    status = lib().miq_act8_bprop(dy.data_ptr(), codes.data_ptr(), scales.data_ptr(), dx.data_ptr(), rows, c, ld, ld_dx,
                                  _act(act), 1 if gated else 0, kind,
                                  _raw_stream(dy.get_device()) if stream is None else _stream(stream))
    if status:
        check(status, "act8_bprop")
    return dx


def act8_grad_workspace_size(rows: int, c: int, k: int, dtype=None) -> int:
    """Bytes of device workspace act8_grad(..., workspace=...) needs for a dy of `dtype` (default
    float32), rows x k, and kept rows of c channels (no GPU access)."""
    out = C.c_size_t()
    kind = _kind(dtype if dtype is not None else torch.float32, "dtype")
    check(lib().miq_act8_grad_workspace_size(rows, c, k, kind, C.byref(out)), "act8_grad_workspace_size")
    return out.value


def plan_act8_grad(rows: int, c: int, k: int, dtype=None):
    """(side of dw's tiles, parts that the rows are split into) of act8_grad for a dy of `dtype`
    (default float32), rows x k, and kept rows of c channels (no GPU access)."""
    out = (C.c_int32 * 2)()
    kind = _kind(dtype if dtype is not None else torch.float32, "dtype")
    check(lib().miq_plan_act8_grad(rows, c, k, kind, out), "plan_act8_grad")
    return out[0], out[1]


def act8_grad(dy, kept: Act8, *, dtype=None, accumulate: bool = False, out=None, workspace=None, stream=None):
    """The weight gradient of a linear (1x1) layer from its kept input: dw[k, c] = sum over the rows
    of dy[row, k] * x'[row, c], (K, C), float32 or, for a bfloat16 dy, bfloat16 (`dtype`, default
    float32).  dy (..., K).  `accumulate` adds it to `out`.  `workspace`: a device buffer of at least
    act8_grad_workspace_size() bytes, not used by another call in flight; None allocates one from
    PyTorch for this call."""
    kind = _kind(dy.dtype, "dy")
    if kept.gated:
        raise ValueError("act8_grad takes a layer's input, not gated rows")
    rows, c, _, lead = _kept(kept)
    _, k, ld = _rows(dy, "dy")
    if dy.shape[:-1] != lead:
        raise ValueError(f"dy and the kept rows differ: {tuple(dy.shape[:-1])} and {lead}")
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    if dtype is None:
        dtype = out.dtype if out is not None else torch.float32
    dw_kind = _kind(dtype, "dtype")
    dw, ld_dw = _output(out, (k, c), dtype, dy, stream)
    at, size, held = _workspace(workspace, "miq_act8_grad_workspace_size", (rows, c, k, kind), dy.device, stream)
    status = lib().miq_act8_grad(dy.data_ptr(), kept.codes.data_ptr(), kept.scales.data_ptr(), dw.data_ptr(), rows, c, k,
                                 ld, ld_dw, 1 if accumulate else 0, kind, dw_kind, at, size,
                                 _raw_stream(dy.get_device()) if stream is None else _stream(stream))
    if status:
        check(status, "act8_grad")
    return dw


__all__ = ["Act8", "act8_bprop", "act8_expand", "act8_fprop", "act8_grad", "act8_grad_workspace_size", "act8_keep",
           "embed_fprop", "embed_grad", "embed_grad_workspace_size", "plan_act8_grad", "plan_embed_grad"]

"""Head norms with the position rotation, for the operands of a gather:

    y = Rot(w o x / sqrt(mean(x^2) + eps))

on every head row x of Q, R and S in one pass, with the gradients of x and w.  (The reference's module neither norms
its heads nor takes positions: att3ntion/_autograd.py:327-329 refuses them.)
"""
from __future__ import annotations

import ctypes as C

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _cuda_kernels as _ck
from ._cabi import lib

_TYPE = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_HEAD_DIMS = (16, 32, 64, 128)
_BF16 = torch.bfloat16


def rotary_table(length: int, dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """FP32 [length, dim]: for every position the cosines of its dim / 2 angles position * base^(-2 i / dim), then their
    sines.  The angles are formed in 64 bits, where positions of any size keep their fraction of a turn."""
    if length < 1 or dim < 2 or dim % 2:
        raise ValueError(f"rotary_table: needs length >= 1 and an even dim >= 2, got {length}, {dim}")
    freq = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def _head_rows(t: torch.Tensor) -> torch.Tensor:
    """`t` [B,N,H,D] if the kernels can read its rows where they lie (16-byte aligned, contiguous), else a copy."""
    if t.data_ptr() % 16 == 0:
        if t.is_contiguous():                            # D is a multiple of 16: every row is aligned
            return t
        step = 16 // t.element_size()
        if t.stride(3) == 1 and all(s % step == 0 for n, s in zip(t.shape[:3], t.stride()) if n > 1) and max(_strides(t)[1:]) < 1 << 31:
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    # a dimension of one entry may carry any stride
    (B, N, H, _), (a, b, c, _) = t.shape, t.stride()
    return a if B > 1 else 0, b if N > 1 else 0, c if H > 1 else 0


def _read(t: torch.Tensor):
    """(tensor that the kernels read, its address, its three strides) for a checked [B,N,H,D] tensor."""
    at = t.data_ptr()
    if not at & 15 and t.is_contiguous():
        _, N, H, D = t.shape
        return t, at, N * H * D, H * D, D
    t = _head_rows(t)
    return (t, t.data_ptr(), *_strides(t))


def _scale(w, who: str, name: str, D: int, device):
    """(scale that the kernels read, its address, its type's number); address 0 without one."""
    if w is None:
        return None, 0, 0
    kind = _TYPE.get(w.dtype) if isinstance(w, torch.Tensor) else None
    if kind is None or w.dim() != 1 or w.shape[0] != D:
        raise RuntimeError(f"{who}: {name} must be a [{D}] tensor of bf16, fp16 or fp32")
    if w.device != device:
        raise RuntimeError(f"{who}: {name} must be on the inputs' device")
    at = w.data_ptr()
    if at & 15 or not w.is_contiguous():
        w = w.detach().clone(memory_format=torch.contiguous_format)
        at = w.data_ptr()
    return w, at, kind


def _check_heads(who: str, xs, names):
    """Common shape contract of [B,N,heads,D] tensors; returns (B, N, D)."""
    x0 = xs[0]
    if not isinstance(x0, torch.Tensor) or x0.dim() != 4:
        raise RuntimeError(f"{who}: {names[0]} must be a [B,N,heads,D] tensor")
    B, N, heads, D = x0.shape
    dtype, dev = x0.dtype, x0.get_device()
    if dtype not in _TYPE:
        raise RuntimeError(f"{who}: all inputs must share one type of bf16, fp16 and fp32")
    if D not in _HEAD_DIMS:
        raise RuntimeError(f"{who}: head dim must be 16, 32, 64 or 128, got {D}")
    for name, x in zip(names, xs):
        if x is not x0:
            if not isinstance(x, torch.Tensor) or x.dim() != 4:
                raise RuntimeError(f"{who}: {name} must be a [B,N,heads,D] tensor")
            b, n, heads, d = x.shape
            if x.dtype is not dtype:
                raise RuntimeError(f"{who}: all inputs must share one type of bf16, fp16 and fp32")
            if b != B or n != N or d != D:
                raise RuntimeError(f"{who}: {name} is {tuple(x.shape)}, expected batch, length and head dim of {names[0]} "
                                   f"{tuple(x0.shape)}")
            if x.get_device() != dev:
                raise RuntimeError(f"{who}: all inputs must be on one device")
        if heads < 1:
            raise RuntimeError(f"{who}: {name} has no heads")
    return B, N, D


def _check_table(who: str, table, D: int, device):
    """(table, rows, rot); no table rotates nothing."""
    if table is None:
        return None, 0, 0
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.float32 or table.shape[0] < 1:
        raise RuntimeError(f"{who}: table must be FP32 [positions, rotated columns] with at least one position")
    rot = table.shape[1]
    if not 8 <= rot <= D or rot % 8:
        raise RuntimeError(f"{who}: rotated columns must be a multiple of 8 up to the head dim {D}, got {rot}")
    if table.device != device:
        raise RuntimeError(f"{who}: table must be on the inputs' device")
    if not table.is_contiguous() or table.data_ptr() % 16:
        table = table.clone(memory_format=torch.contiguous_format)
    return table, table.shape[0], rot


def _check_positions(who: str, positions, B: int, N: int, device):
    """(positions or None, bytes, batch stride, position stride)."""
    if positions is None:
        return None, 0, 0, 0
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{who}: positions must be an int32 or int64 tensor")
    if tuple(positions.shape) not in {(N,), (B, N), (1, N)}:
        raise RuntimeError(f"{who}: positions must be [{N}] or [{B},{N}], got {tuple(positions.shape)}")
    if positions.device != device:
        raise RuntimeError(f"{who}: positions must be on the inputs' device")
    along = positions.stride(-1) if N > 1 else 0
    return positions, positions.element_size(), positions.stride(0) if positions.dim() == 2 and positions.shape[0] > 1 else 0, along


def _on_gpu(who: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{who}: inputs must be CUDA tensors")


_ZEROS = (0,) * 9
_NAMES = tuple(f"input {k}" for k in range(5))
_Rows = {n: C.c_int64 * (21 * n) for n in range(1, 6)}         # att3_head_rows arrays


def _forward(xs, ws, table, positions, eps, interleaved, heads_first):
    who = "norm_rotate"
    B, N, D = _check_heads(who, xs, _NAMES)
    dev, n = xs[0].device, len(xs)
    table, rows, rot = _check_table(who, table, D, dev)
    positions, pos_bytes, pos_b, pos_n = _check_positions(who, positions, B, N, dev)
    if positions is None and table is not None and N > rows:
        raise RuntimeError(f"{who}: {N} positions and a table of {rows}")
    if not eps >= 0:
        raise RuntimeError(f"{who}: eps must not be negative, got {eps}")
    words, ys, held = [], [], []
    scales = [_scale(w, who, f"weight {k}", D, dev) for k, w in enumerate(ws)]
    _on_gpu(who, xs[0])
    with _ck._on_device(dev):
        for x, (w, w_at, kind) in zip(xs, scales):
            H = x.shape[2]
            x, at, xb, xn, xh = _read(x)
            if heads_first:
                y = torch.empty((B, H, N, D), dtype=_BF16, device=dev)
                yb, yn, yh = H * N * D, D, N * D
            else:
                y = torch.empty((B, N, H, D), dtype=_BF16, device=dev)
                yb, yn, yh = N * H * D, H * D, D
            words += (at, xb, xn, xh, w_at, kind, 1, y.data_ptr(), yb, yn, yh, *_ZEROS, H)
            ys.append(y)
            held.append(x)                                   # copies live until the launch
        _ck._call(lib.att3_norm_rotate_forward, _Rows[n](*words), n, _TYPE[xs[0].dtype], _ck._ptr(table), rows, rot,
                  interleaved, _ck._ptr(positions), pos_bytes, pos_b, pos_n, B, N, D, eps, _ck._raw_stream(dev))
    return ys


class _NormRotateFn(Function):
    @staticmethod
    def forward(ctx, n, table, positions, eps, interleaved, heads_first, *tensors):
        xs, ws = tensors[:n], tensors[n:]
        ys = _forward(xs, ws, table, positions, eps, interleaved, heads_first)
        ctx.save_for_backward(table, positions, *tensors)        # checked by now: the backward takes them as they are
        ctx.n, ctx.eps, ctx.interleaved, ctx.heads_first = n, eps, interleaved, heads_first
        return tuple(ys)

    @staticmethod
    @once_differentiable
    def backward(ctx, *dys):
        table, positions, *tensors = ctx.saved_tensors
        xs, ws = tensors[:ctx.n], tensors[ctx.n:]
        who = "norm_rotate"
        B, N, _, D = xs[0].shape
        dev = xs[0].device
        table, rows, rot = _check_table(who, table, D, dev)
        positions, pos_bytes, pos_b, pos_n = _check_positions(who, positions, B, N, dev)
        with _ck._on_device(dev):
            # scratch of this call alone: a captured graph keeps it in its own pool
            nbytes = lib.att3_norm_rotate_workspace_bytes(ctx.n, D)
            scratch = torch.empty(nbytes, dtype=torch.uint8, device=dev)
            words, held, dxs, dws = [], [], [], []
            for x, w, dy in zip(xs, ws, dys):
                H, dtype = x.shape[2], x.dtype
                dx = torch.empty(x.shape, dtype=dtype, device=dev)
                dw = torch.empty(D, dtype=torch.float32, device=dev) if w is not None else None
                w, w_at, kind = _scale(w, who, "weight", D, dev)
                dy, dy_at, gb, gn, gh = _read(dy.transpose(1, 2) if ctx.heads_first else dy)
                x, at, xb, xn, xh = _read(x)
                words += (at, xb, xn, xh, w_at, kind, 1, 0, 0, 0, 0, dy_at, gb, gn, gh, dx.data_ptr(), N * H * D, H * D, D,
                          dw.data_ptr() if dw is not None else 0, H)
                held += (x, w, dy)
                dxs.append(dx)
                dws.append(dw)
            _ck._call(lib.att3_norm_rotate_backward, _Rows[ctx.n](*words), ctx.n, _TYPE[dtype], _ck._ptr(table), rows,
                      rot, ctx.interleaved, _ck._ptr(positions), pos_bytes, pos_b, pos_n, B, N, D, ctx.eps,
                      scratch.data_ptr(), nbytes, _ck._raw_stream(dev))
        dws = [dw if w is None or w.dtype == torch.float32 else dw.to(w.dtype) for w, dw in zip(ws, dws)]
        return (None,) * 6 + (*dxs, *dws)


def norm_rotate(xs, weights=None, table=None, positions=None, *, eps=1e-6, interleaved=False, heads_first=False):
    """Norms and rotates the head rows of one to five tensors in one pass.

    xs: [B,N,heads,D] tensors (heads may differ; any strides) of one type of bf16, fp16 and fp32, D in {16,32,64,128};
    a single tensor is taken too.  weights: a [D] scale or None for each, or None; a tensor without a scale is not
    normed.  table: FP32 [positions, rot], see `rotary_table`; the first `rot` columns (a multiple of 8) of every
    row are turned by its position's angles, pairing columns (d, d + rot/2), or (2d, 2d + 1) with interleaved=True; None:
    no rotation.  positions: int32 or int64 [N] or [B,N], None for 0 .. N-1.  A position outside the table is read as
    position 0 and reported by `device_status()`.

    Returns BF16 tensors, [B,N,heads,D] contiguous, or [B,heads,N,D] with heads_first=True.  Gradients of the inputs come
    back in their type, those of the scales are summed in FP32 in a fixed order; cotangents are taken as BF16."""
    single = isinstance(xs, torch.Tensor)
    xs = (xs,) if single else tuple(xs)
    if not 1 <= len(xs) <= 5:
        raise RuntimeError(f"norm_rotate: one to five tensors, got {len(xs)}")
    ws = (None,) * len(xs) if weights is None else (weights,) if isinstance(weights, torch.Tensor) else tuple(weights)
    if len(ws) != len(xs):
        raise RuntimeError(f"norm_rotate: {len(xs)} tensors and {len(ws)} weights")
    eps, interleaved, heads_first = float(eps), int(bool(interleaved)), bool(heads_first)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (*xs, *ws)):
        ys = _NormRotateFn.apply(len(xs), table, positions, eps, interleaved, heads_first, *xs, *ws)
    else:
        ys = tuple(_forward(xs, ws, table, positions, eps, interleaved, heads_first))
    return ys[0] if single else ys

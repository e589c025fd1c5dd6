"""Head norms with the position rotation, for the operands of a gather:

    y = Rot(w o x / sqrt(mean(x^2) + eps))

on every head row x of Q, R and S in one pass, with the gradients of x and w.  (The reference's module neither norms
its heads nor takes positions: att3ntion/_autograd.py:327-329 refuses them.)
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _cabi  # noqa: F401  (the library that the binding is linked against; says what to do if it is missing)

try:
    from . import _serve_native as _native
except ImportError as _error:
    class _Missing:
        """Stands for a binding that is not built, or built against another torch: what needs it says so when it is called,
        and the operators that go through the C ABI alone are not held up."""

        def __init__(self, why):
            self._why = why

        def __getattr__(self, name):
            raise ImportError(f"{name}: the torch binding att3ntion_b200/_serve_native.so cannot be loaded ({self._why}); build it with "
                              "`python -m att3ntion_b200.build`")

    _native = _Missing(str(_error))

_TYPES = (torch.bfloat16, torch.float16, torch.float32)
_HEAD_DIMS = (16, 32, 64, 128)


def rotary_table(length: int, dim: int, base: float = 10000.0, device=None) -> torch.Tensor:
    """FP32 [length, dim]: for every position the cosines of its dim / 2 angles position * base^(-2 i / dim), then their
    sines.  The angles are formed in 64 bits, where positions of any size keep their fraction of a turn."""
    if length < 1 or dim < 2 or dim % 2:
        raise ValueError(f"rotary_table: needs length >= 1 and an even dim >= 2, got {length}, {dim}")
    freq = float(base) ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=device) / dim)
    angle = torch.arange(length, dtype=torch.float64, device=device)[:, None] * freq
    return torch.cat((angle.cos(), angle.sin()), 1).float()


# The binding checks every call and declines one that is not in order; what follows says why.

def _check_scale(w, who: str, name: str, D: int, device):
    if w is None:
        return
    if not isinstance(w, torch.Tensor) or w.dim() != 1 or w.shape[0] != D or w.dtype not in _TYPES:
        raise RuntimeError(f"{who}: {name} must be a [{D}] tensor of bf16, fp16 or fp32")
    if w.device != device:
        raise RuntimeError(f"{who}: {name} must be on the inputs' device")


def _check_heads(who: str, xs, names):
    """Common shape contract of [B,N,heads,D] tensors; returns (B, N, D)."""
    x0 = xs[0]
    if not isinstance(x0, torch.Tensor) or x0.dim() != 4:
        raise RuntimeError(f"{who}: {names[0]} must be a [B,N,heads,D] tensor")
    B, N, heads, D = x0.shape
    dtype, dev = x0.dtype, x0.get_device()
    if dtype not in _TYPES:
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
    if table is None:
        return
    if not isinstance(table, torch.Tensor) or table.dim() != 2 or table.dtype != torch.float32 or table.shape[0] < 1:
        raise RuntimeError(f"{who}: table must be FP32 [positions, rotated columns] with at least one position")
    rot = table.shape[1]
    if not 8 <= rot <= D or rot % 8:
        raise RuntimeError(f"{who}: rotated columns must be a multiple of 8 up to the head dim {D}, got {rot}")
    if table.device != device:
        raise RuntimeError(f"{who}: table must be on the inputs' device")


def _check_positions(who: str, positions, B: int, N: int, device):
    if positions is None:
        return
    if not isinstance(positions, torch.Tensor) or positions.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{who}: positions must be an int32 or int64 tensor")
    if tuple(positions.shape) not in {(N,), (B, N), (1, N)}:
        raise RuntimeError(f"{who}: positions must be [{N}] or [{B},{N}], got {tuple(positions.shape)}")
    if positions.device != device:
        raise RuntimeError(f"{who}: positions must be on the inputs' device")


def _check_eps(who: str, eps):
    if not float(eps) >= 0:
        raise RuntimeError(f"{who}: eps must not be negative, got {eps}")


def _no_tangent(who: str, *tensors) -> None:
    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{who}: has no forward-mode derivative, and an argument carries a tangent")


def _on_gpu(who: str, t: torch.Tensor) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{who}: inputs must be CUDA tensors")


def _refuse_norm_rotate(xs, ws, table, positions, eps):
    who = "norm_rotate"
    if not 1 <= len(xs) <= 5:
        raise RuntimeError(f"{who}: one to five tensors, got {len(xs)}")
    if len(ws) != len(xs):
        raise RuntimeError(f"{who}: {len(xs)} tensors and {len(ws)} weights")
    B, N, D = _check_heads(who, xs, [f"input {k}" for k in range(len(xs))])
    dev = xs[0].device
    for k, w in enumerate(ws):
        _check_scale(w, who, f"weight {k}", D, dev)
    _check_table(who, table, D, dev)
    _check_positions(who, positions, B, N, dev)
    if positions is None and table is not None and N > table.shape[0]:
        raise RuntimeError(f"{who}: {N} positions and a table of {table.shape[0]}")
    _check_eps(who, eps)
    _no_tangent(who, *xs, *ws, table)
    if table is not None and table.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{who}: the table has no gradient; detach it")
    _on_gpu(who, xs[0])
    raise RuntimeError(f"{who}: arguments of a type or size that the kernels do not take")


def norm_rotate(xs, weights=None, table=None, positions=None, *, eps=1e-6, interleaved=False, heads_first=False):
    """Norms and rotates the head rows of one to five tensors in one pass.

    xs: [B,N,heads,D] tensors (heads may differ; any strides) of one type of bf16, fp16 and fp32, D in {16,32,64,128};
    a single tensor is taken too.  weights: a [D] scale or None for each, or None; a tensor without a scale is not
    normed.  table: FP32 [positions, rot], see `rotary_table`; the first `rot` columns (a multiple of 8) of every
    row are turned by its position's angles, pairing columns (d, d + rot/2), or (2d, 2d + 1) with interleaved=True; None:
    no rotation.  positions: int32 or int64 [N] or [B,N], None for 0 .. N-1.  A position outside the table is read as
    position 0 and reported by `device_status()`.

    Returns BF16 tensors, [B,N,heads,D] contiguous, or [B,heads,N,D] with heads_first=True.  Gradients of the inputs come
    back in their type, those of the scales are summed in FP32 in a fixed order; cotangents are taken as BF16.  The table has no
    gradient, and there is no forward-mode derivative: arguments that ask for either are refused."""
    single = isinstance(xs, torch.Tensor)
    xs = (xs,) if single else tuple(xs)
    if weights is None:
        weights = (None,) * len(xs)
    elif isinstance(weights, torch.Tensor):
        weights = (weights,)
    ys = _accepted(_native.norm_rotate, xs, weights, table, positions, eps, interleaved, heads_first)
    if ys is None:
        _refuse_norm_rotate(xs, weights, table, positions, eps)
    return ys[0] if single else ys


def _accepted(call, *args):
    """The binding's answer, or None if it declined the call or could not take the arguments' types."""
    try:
        return call(*args)
    except TypeError:
        return None

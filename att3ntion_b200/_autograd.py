"""``HypergraphAttention`` and its autograd bridge, API-compatible with the reference
module (att3ntion/_autograd.py:12-405): same constructor arguments, parameter names
and shapes (so state dicts load either way), same forward semantics

    y = Wo( gelu(Y_q) + gelu(Y_r) + gelu(Y_s) [+ the three scatter terms] )

with QuickGELU, heads split from ``d_model``, inputs cast to BF16 at the kernel
boundary and the sequence padded to a multiple of 16 with the padding invisible.
``gather_mode=1`` keeps only the Q-anchored gather and, for head sizes 64 and 128,
routes to ``single_gather_attention`` (optionally windowed).

Beyond the reference, keyword arguments add per-head RMS norms of Q, R and S (``qk_norm``), the position rotation of
the same rows (``rotary_base``), and first keys that stay visible outside the window (``sinks``); a windowed layer is
served from a ``GatherCache`` with ``prefill`` and ``decode``.
"""
from __future__ import annotations

import os

import torch
import torch.nn as nn
from torch.autograd import Function

from . import _custom_op  # noqa: F401  (registers torch.ops.att3ntion.hypergraph_{forward,backward})
from ._norm_rotate import norm_rotate, rotary_table
from ._single_gather import single_gather_attention, single_gather_heads_last, window_mask

TILE = 16
_CHECK_GRADS = os.getenv("ATT3NTION_CHECK_GRADS", "0").lower() in {"1", "true", "yes", "on"}


def _pad_to_multiple(t: torch.Tensor, multiple: int, dim: int = 2):
    """Right-pads `dim` of `t` with zeros to a multiple of `multiple`; returns (tensor, pad)."""
    extra = (-t.size(dim)) % multiple
    if extra == 0:
        return t, 0
    pad = [0, 0] * t.ndim
    pad[2 * (t.ndim - 1 - dim) + 1] = extra          # F.pad lists dims from the last one backwards
    return torch.nn.functional.pad(t, pad), extra


def _normalize_self_attn_mask(mask, batch: int, n: int, device):
    """None, or a contiguous bool [batch, n, n] on `device` from a [n,n] / [1,n,n] / [batch,n,n] mask."""
    if mask is None:
        return None
    if mask.ndim == 2:
        if tuple(mask.shape) != (n, n):
            raise ValueError(f"2D mask must have shape {(n, n)}, got {tuple(mask.shape)}")
        mask = mask.unsqueeze(0)
    elif mask.ndim != 3:
        raise ValueError(f"mask must have ndim 2 or 3, got ndim={mask.ndim}")
    if tuple(mask.shape[-2:]) != (n, n):
        raise ValueError(f"mask must have trailing shape {(n, n)}, got {tuple(mask.shape)}")
    if mask.shape[0] not in (1, batch):
        raise ValueError(f"mask batch dim must be 1 or {batch}, got {mask.shape[0]}")
    if mask.shape[0] == 1 and batch > 1:
        mask = mask.expand(batch, -1, -1)
    return mask.to(device=device, dtype=torch.bool).contiguous()


class _HypergraphAttentionAutograd(Function):
    """Casts and pads at the kernel boundary, calls the registered ops, crops and casts back."""

    @staticmethod
    def forward(ctx, Q, R, S, Vq_1, Vq_2, Vr_1, Vr_2, Vs_1, Vs_2, mask, dropout_rate=0.0, scatter=False,
                gather_mode=0):
        n = Q.size(2)
        if mask is not None and (R.size(2) != n or S.size(2) != n):
            raise ValueError("masked CUDA hypergraph attention requires equal sequence lengths")
        mask = _normalize_self_attn_mask(mask, Q.size(0), n, Q.device)
        xs = [_pad_to_multiple(t.contiguous().to(torch.bfloat16), TILE)[0]
              for t in (Q, R, S, Vq_1, Vq_2, Vr_1, Vr_2, Vs_1, Vs_2)]
        n_pad = xs[0].size(2) - n
        if mask is None:
            mask_t = torch.empty(0, device=Q.device, dtype=torch.bool)
        else:
            mask_t = torch.nn.functional.pad(mask, (0, n_pad, 0, n_pad), value=False).contiguous() if n_pad else mask
        out = torch.ops.att3ntion.hypergraph_forward(*xs, mask_t, float(dropout_rate), n, n, n, int(gather_mode))
        Ys, stats = out[:6], out[6:]
        ctx.save_for_backward(*xs, *stats, mask_t, *Ys[:3])
        ctx.n, ctx.dtype = n, Q.dtype
        return tuple(y[:, :, :n].to(Q.dtype) for y in Ys)

    @staticmethod
    def backward(ctx, *cot):
        saved = ctx.saved_tensors
        xs, stats, mask_t, Y3 = saved[:9], saved[9:15], saved[15], saved[16:19]
        n_full = xs[0].size(2)
        gs = []
        for g, y in zip(cot, (*Y3, *Y3)):
            if g is None:
                gs.append(torch.zeros_like(y))
            else:
                gs.append(_pad_to_multiple(g.contiguous().to(torch.bfloat16), TILE)[0])
        grads = torch.ops.att3ntion.hypergraph_backward(*gs, *xs, *stats, mask_t, *Y3)
        grads = [g[:, :, :ctx.n].to(ctx.dtype) if n_full != ctx.n else g.to(ctx.dtype) for g in grads]
        if _CHECK_GRADS:
            for name, g in zip(("Q", "R", "S", "Vq_1", "Vq_2", "Vr_1", "Vr_2", "Vs_1", "Vs_2"), grads):
                if not torch.isfinite(g).all():
                    raise RuntimeError(f"grad_{name} contains non-finite values")
        return (*grads, None, None, None, None)


class QuickGELU(nn.Module):
    def forward(self, x: torch.Tensor):
        return x * torch.sigmoid(1.702 * x)


def _captured(device) -> bool:
    """Whether the device's current stream is being captured into a graph."""
    if device.type != "cuda":
        return False
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


class HypergraphAttention(nn.Module):
    """Three-way hypergraph attention layer on the sm_100a kernels.

    qk_norm: RMS norms with learned scales over the heads of Q, R and S.  rotary_base: rotates those rows by their
    position's angles (see `rotary_table`; pairs of columns half a head apart).  sinks (with a window): the first `sinks`
    keys stay visible to every later query."""

    def __init__(self, d_model, n_heads, dropout_rate=0, scatter=False, gather_mode=0, window=0, *, qk_norm=False,
                 rotary_base=None, sinks=0, norm_eps=1e-6):
        super().__init__()
        if d_model % n_heads != 0:
            raise ValueError(f"d_model ({d_model}) must be divisible by n_heads ({n_heads})")
        if gather_mode not in (0, 1):
            raise ValueError(f"gather_mode must be 0 (Q, R and S anchored) or 1 (Q anchored only), got {gather_mode}")
        if scatter and gather_mode != 0:
            raise ValueError("scatter requires all three gathers (gather_mode=0)")
        if window and gather_mode != 1:
            raise ValueError("window requires the Q-anchored gather only (gather_mode=1)")
        if sinks < 0 or (sinks and not window):
            raise ValueError("sinks are first keys that stay visible outside a window: they need window > 0")
        self.d_model, self.n_heads, self.head_dim = d_model, n_heads, d_model // n_heads
        if (qk_norm or rotary_base) and self.head_dim not in (16, 32, 64, 128):
            raise ValueError(f"qk_norm and rotary_base need a head dim of 16, 32, 64 or 128, got {self.head_dim}")
        self.sinks, self.rotary_base, self.norm_eps = sinks, rotary_base, norm_eps
        self.scatter, self.gather_mode, self.window = scatter, gather_mode, window
        inner = n_heads * self.head_dim
        self.Wq = nn.Linear(d_model, inner, bias=False)
        self.Wr = nn.Linear(d_model, inner, bias=False)
        self.Ws = nn.Linear(d_model, inner, bias=False)
        vmul = 2 if scatter else 1
        # the Q-anchored gather never reads Vq, so the one-gather variant has no Wv_q
        self.Wv_q = None if gather_mode == 1 else nn.Linear(d_model, inner * vmul, bias=True)
        self.Wv_r = nn.Linear(d_model, inner * vmul, bias=True)
        self.Wv_s = nn.Linear(d_model, inner * vmul, bias=True)
        self.Wo = nn.Linear(inner, d_model, bias=True)
        self.dropout = nn.Dropout(dropout_rate)
        self.gelu = QuickGELU()
        self.q_norm, self.r_norm, self.s_norm = (nn.Parameter(torch.ones(self.head_dim)) if qk_norm else None
                                                 for _ in range(3))
        self._tables = []

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        # value projections saved with / without the scatter half load into either configuration
        for name in ("Wv_q", "Wv_r", "Wv_s"):
            module = getattr(self, name)
            if module is None:
                continue
            for suffix, target in (("weight", module.weight), ("bias", module.bias)):
                key = f"{prefix}{name}.{suffix}"
                loaded = state_dict.get(key)
                if loaded is None or loaded.shape == target.shape or loaded.ndim != target.ndim:
                    continue
                if loaded.shape[0] == 2 * target.shape[0] and loaded.shape[1:] == target.shape[1:]:
                    state_dict[key] = loaded[: target.shape[0]].contiguous()
                elif 2 * loaded.shape[0] == target.shape[0] and loaded.shape[1:] == target.shape[1:]:
                    grown = torch.zeros_like(target)
                    grown[: loaded.shape[0]] = loaded
                    state_dict[key] = grown
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)

    def _rotary(self, length, device):
        """The angle table, at least `length` positions long, or None.  It grows by doubling, and the shorter ones are kept:
        a captured graph may still read them.  Every later caller gets what this one makes, so it is an ordinary tensor
        whatever mode the caller is in, and finished when this returns, on whatever stream the next one works.  During a
        capture it would be filled by the graph's replays only: that one is the graph's own and not kept."""
        if not self.rotary_base:
            return None
        for t in reversed(self._tables):
            if t.device == device and t.shape[0] >= length:
                return t
        if _captured(device):
            return rotary_table(length, self.head_dim, self.rotary_base, device)
        most = max((t.shape[0] for t in self._tables if t.device == device), default=256)
        with torch.inference_mode(False), torch.no_grad():
            table = rotary_table(max(length, 2 * most), self.head_dim, self.rotary_base, device)
        if type(table) is torch.Tensor:                         # and not a stand-in of a tracer
            if device.type == "cuda":
                torch.cuda.current_stream(device).synchronize()
            self._tables.append(table)
        return table

    def __getstate__(self):
        return {**self.__dict__, "_tables": []}                 # copies make their own

    def __setstate__(self, state):
        super().__setstate__(state)
        # a layer that was pickled before it had these
        for name, value in (("sinks", 0), ("rotary_base", None), ("norm_eps", 1e-6), ("_tables", [])):
            self.__dict__.setdefault(name, value)
        for name in ("q_norm", "r_norm", "s_norm"):
            if name not in self._parameters:
                self.__dict__.setdefault(name, None)

    def _qrs(self, x, heads_first):
        """The score operands of every position, [B,N,H,D] or [B,H,N,D]: projected, and normed and rotated in one pass
        (then bf16) if the layer has either."""
        b, n, _ = x.shape
        qrs = [w(x).view(b, n, self.n_heads, self.head_dim) for w in (self.Wq, self.Wr, self.Ws)]
        if self.q_norm is None and not self.rotary_base:
            return [t.permute(0, 2, 1, 3) for t in qrs] if heads_first else qrs
        return norm_rotate(qrs, (self.q_norm, self.r_norm, self.s_norm), self._rotary(n, x.device), eps=self.norm_eps,
                           heads_first=heads_first)

    def _heads(self, t, width=None):
        b, n, _ = t.shape
        return t.reshape(b, n, self.n_heads, width or self.head_dim).permute(0, 2, 1, 3)

    def forward(self, x, rotary_emb=None, mask=None):
        if rotary_emb is not None:
            raise ValueError("CUDA HypergraphAttention does not support rotary embeddings")
        b, n, _ = x.shape
        if self.q_norm is not None or self.rotary_base or self.sinks:
            return self._extended(x, mask)
        Q, R, S = self.Wq(x), self.Wr(x), self.Ws(x)
        window_only = bool(self.window) and mask is None      # then the kernels derive the window from indices
        if self.window:
            win = window_mask(n, self.window, x.device)
            mask = win if mask is None else mask.to(device=x.device, dtype=torch.bool) & win

        if self.gather_mode == 1 and self.head_dim in (64, 128) and window_only and self.window <= 128 and n % TILE == 0:
            # window-only calls read the projections where they lie ([B,N,H,D] views, no permute-and-copy) and take
            # the activation from the kernel's epilogue
            split = lambda t: t.view(b, n, self.n_heads, self.head_dim)
            y = single_gather_heads_last(split(Q), split(R), split(S), split(self.Wv_r(x)), split(self.Wv_s(x)),
                                         min(self.window, n), act=True)
            return self.Wo(y.reshape(b, n, self.n_heads * self.head_dim))

        if self.gather_mode == 1 and self.head_dim in (64, 128):
            y = single_gather_attention(self._heads(Q), self._heads(R), self._heads(S), self._heads(self.Wv_r(x)),
                                        self._heads(self.Wv_s(x)), None if window_only else mask,
                                        min(self.window, n))
            y = self.gelu(y).permute(0, 2, 1, 3).contiguous().view(b, n, self.n_heads * self.head_dim)
            return self.Wo(y)

        return self._three_gather(x, self._heads(Q), self._heads(R), self._heads(S), mask)

    def _three_gather(self, x, Q, R, S, mask):
        b, n, _ = x.shape
        if self.scatter:
            Vq_1, Vq_2 = self._heads(self.Wv_q(x), 2 * self.head_dim).split(self.head_dim, dim=-1)
            Vr_1, Vr_2 = self._heads(self.Wv_r(x), 2 * self.head_dim).split(self.head_dim, dim=-1)
            Vs_1, Vs_2 = self._heads(self.Wv_s(x), 2 * self.head_dim).split(self.head_dim, dim=-1)
        else:
            Vr_1, Vs_1 = self._heads(self.Wv_r(x)), self._heads(self.Wv_s(x))
            Vq_1 = torch.zeros_like(Vr_1) if self.Wv_q is None else self._heads(self.Wv_q(x))
            Vq_2, Vr_2, Vs_2 = torch.zeros_like(Vq_1), torch.zeros_like(Vr_1), torch.zeros_like(Vs_1)

        Y_q, Y_r, Y_s, Y_q_, Y_r_, Y_s_ = _HypergraphAttentionAutograd.apply(
            Q, R, S, Vq_1, Vq_2, Vr_1, Vr_2, Vs_1, Vs_2, mask,
            self.dropout.p, self.scatter, self.gather_mode)
        y = self.gelu(Y_q)
        if self.gather_mode == 0:
            y = y + self.gelu(Y_r) + self.gelu(Y_s)
        if self.scatter:
            y = y + self.gelu(Y_q_) + self.gelu(Y_r_) + self.gelu(Y_s_)
        y = y.permute(0, 2, 1, 3).contiguous().view(b, n, self.n_heads * self.head_dim)
        return self.Wo(y)

    # ------------------------------------------------------------------ norms, rotation, sinks

    def _gather(self, x, Q, R, S, Vr, Vs, mask, last):
        """The Q-anchored gather and its output projection; operands [B,N,H,D] if `last`, else [B,H,N,D]."""
        b, n, _ = x.shape
        if last:
            y = single_gather_heads_last(Q, R, S, Vr, Vs, min(self.window, n), act=True)
        else:
            y = single_gather_attention(Q, R, S, Vr, Vs, mask, 0 if self.sinks else min(self.window, n))
            y = self.gelu(y.to(x.dtype)).permute(0, 2, 1, 3)
        return self.Wo(y.to(x.dtype).reshape(b, n, self.n_heads * self.head_dim))

    def _reads_in_place(self, n, mask):
        """Whether the windowed kernels take the projections where they lie, [B,N,H,D]."""
        return mask is None and not self.sinks and 0 < self.window <= 128 and n % TILE == 0

    def _extended(self, x, mask):
        b, n, _ = x.shape
        last = self.gather_mode == 1 and self.head_dim in (64, 128) and self._reads_in_place(n, mask)
        Q, R, S = self._qrs(x, heads_first=not last)
        if self.window and not last and (mask is not None or self.sinks):
            win = window_mask(n, self.window, x.device, self.sinks)
            mask = win if mask is None else mask.to(device=x.device, dtype=torch.bool) & win
        if self.gather_mode == 1 and self.head_dim in (64, 128):
            split = lambda t: t.view(b, n, self.n_heads, self.head_dim) if last else self._heads(t)
            return self._gather(x, Q, R, S, split(self.Wv_r(x)), split(self.Wv_s(x)), mask, last)
        if self.window and mask is None:
            mask = window_mask(n, self.window, x.device)
        # the gather's outputs come in the operands' type, which is the kernels' own here
        return self._three_gather(x, *(t.to(x.dtype) for t in (Q, R, S)), mask)

    # ------------------------------------------------------------------ serving

    def _check_serving(self, who, x, cache):
        if self.gather_mode != 1 or not self.window or self.head_dim not in (64, 128):
            raise ValueError(f"{who}: needs gather_mode=1, a window and a head dim of 64 or 128")
        if x.dim() != 3 or x.shape[0] != cache.sequences:
            raise ValueError(f"{who}: x must be [{cache.sequences},length,{self.d_model}], got {tuple(x.shape)}")

    @torch.no_grad()
    def prefill(self, x, cache, counts=None):
        """The layer over the prompts x [B,N,d_model] of empty sequences, storing their rows in `cache`.  counts (a list of
        ints): the prompts' lengths, right-padded to N; what comes back behind a prompt's end means nothing.  A sequence
        of count 0 is left as it is, so that one that was cleared can start anew beside the others."""
        self._check_serving("prefill", x, cache)
        b, n, _ = x.shape
        if any(have and new for have, new in zip(cache.host_lengths, cache._counts(counts, n))):
            raise ValueError("prefill: the sequences of its prompts must be empty")
        # a window of causal keys: the padding behind a prompt is never seen by its own positions
        last = self._reads_in_place(n, None)
        Q, R, S = self._qrs(x, heads_first=not last)
        vr, vs = self.Wv_r(x), self.Wv_s(x)
        split = lambda t: t.view(b, n, self.n_heads, self.head_dim)
        side = (lambda t: t) if last else (lambda t: t.transpose(1, 2))
        mask = window_mask(n, self.window, x.device, self.sinks) if self.sinks else None
        vr, vs = split(vr), split(vs)
        R_, S_ = side(R), side(S)
        cache.append(R_, S_, vr.to(R_.dtype), vs.to(R_.dtype), counts=counts)
        return self._gather(x, Q, R, S, side(vr), side(vs), mask, last)

    @torch.no_grad()
    def decode(self, x, cache, counts=None):
        """The layer over one new token of every sequence, x [B,1,d_model], after storing its rows in `cache`: the last
        `window` cached tokens and the first `sinks` are visible.  counts (a list of 0 and 1): a sequence of 0 sits out,
        nothing is stored for it and what comes back for it means nothing."""
        self._check_serving("decode", x, cache)
        if x.shape[1] != 1:
            raise ValueError(f"decode: one token a sequence, got {x.shape[1]}")
        b = x.shape[0]
        split = lambda t: t.view(b, 1, self.n_heads, self.head_dim)
        table = self._rotary(max(cache.host_positions, default=0) + 1, x.device)
        q = cache.append(split(self.Wr(x)), split(self.Ws(x)), split(self.Wv_r(x)), split(self.Wv_s(x)), counts=counts, Q=split(self.Wq(x)),
                         weights=(self.q_norm, self.r_norm, self.s_norm), table=table, eps=self.norm_eps)
        y = self.gelu(cache.decode(q[:, 0], window=self.window, sinks=self.sinks, counts=counts).to(x.dtype))
        return self.Wo(y.reshape(b, 1, self.n_heads * self.head_dim))

"""Serving the single gather: a paged cache of the rows that later queries need, the gather of one new token over it,
and eviction from it.  (The reference has no form for single tokens.)

A pool is BF16 [pages, page_size, Hkv, D] contiguous, one each for R, S, Vr and Vs.  `page_table` int32 [B, entries]
names the page of slots p * page_size .. of every sequence, `lengths` int32 [B] the slots in use.  Both are read on the
device, so captured graphs follow them; an entry outside its table is never followed, and `device_status()` reports it.
`GatherCache` keeps all of these for a batch of sequences.
"""
from __future__ import annotations

import torch

from ._norm_rotate import _accepted, _check_eps, _check_heads, _check_scale, _check_table, _native, _no_tangent, _on_gpu

_BF16 = torch.bfloat16
_POOLS = ("R", "S", "Vr", "Vs")


_NEW = ("R", "S", "Vr", "Vs", "Q")


def _check_pools(who, pools):
    if len(pools) != 4:
        raise RuntimeError(f"{who}: pools are the four tensors R, S, Vr, Vs, got {len(pools)}")
    first = pools[0]
    shape = dev = None
    for name, p in zip(_POOLS, pools):
        if not isinstance(p, torch.Tensor) or p.dtype is not _BF16 or p.dim() != 4 or not p.is_contiguous():
            raise RuntimeError(f"{who}: pool {name} must be a contiguous bf16 [pages,page_size,Hkv,D] tensor")
        if shape is None:
            shape, dev = p.shape, p.get_device()
        elif p.shape != shape or p.get_device() != dev:
            raise RuntimeError(f"{who}: the pools must share one shape and device")
        if p.data_ptr() & 15:
            raise RuntimeError(f"{who}: pool {name} must start on a 16-byte boundary")
    if 0 in shape:
        raise RuntimeError(f"{who}: the pools are empty")
    return first


def _check_table_of_pages(who, page_table, lengths, device, name="page_table", B=None):
    if not isinstance(page_table, torch.Tensor) or page_table.dim() != 2 or page_table.dtype != torch.int32:
        raise RuntimeError(f"{who}: {name} must be an int32 [B,entries] tensor")
    if page_table.shape[1] < 1 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise RuntimeError(f"{who}: {name} needs at least one entry a sequence, neighbours in memory")
    if B is not None and page_table.shape[0] != B:
        raise RuntimeError(f"{who}: {name} has {page_table.shape[0]} rows for {B} sequences")
    if page_table.device != device:
        raise RuntimeError(f"{who}: {name} must be on the pools' device")
    if lengths is not None:
        _check_ints(who, "lengths", lengths, page_table.shape[0], device)


def _check_ints(who, name, t, B, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.shape != (B,) or not t.is_contiguous():
        raise RuntimeError(f"{who}: {name} must be a contiguous int32 [{B}] tensor")
    if t.device != device:
        raise RuntimeError(f"{who}: {name} must be on the pools' device")


def _check_mass(who, mass, pool):
    if mass is not None and not (isinstance(mass, torch.Tensor) and mass.dtype == torch.float32 and mass.is_contiguous()
                                 and mass.shape == pool.shape[:3] and mass.device == pool.device):
        raise RuntimeError(f"{who}: mass must be a contiguous FP32 {tuple(pool.shape[:3])} tensor on the pools' device")


def _no_grad(who, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{who}: has no gradient; call it under torch.no_grad()")
    _no_tangent(who, *tensors)


def gather_cache_append(pools, page_table, lengths, R, S, Vr, Vs, *, counts=None, Q=None, weights=None, table=None,
                        positions=None, mass=None, eps=1e-6, interleaved=False):
    """Stores new rows R, S, Vr, Vs [B,T,Hkv,D] (any strides; bf16, fp16 or fp32) at slots lengths[b] .. of every
    sequence; `counts` (int32 [B]) stores only the first counts[b] of them.  `lengths` itself is left as it is.

    weights (a scale [D] or None each for Q, R, S) norms and `table` rotates R and S on the way, as `norm_rotate` does,
    at positions lengths[b] + t, or positions[b] + t if `positions` (int32 [B]) is given.  Q [B,T,Hq,D], if given, goes
    through the same pass and is returned as bf16, all T rows of it.  mass, if given, is zeroed at the slots written.
    No two sequences may write the same slot of a page.  A slot behind the page table's end, or on a page that the pool
    does not have, is left out and reported by `device_status()`."""
    weights = (None,) * 3 if weights is None else weights
    got = _accepted(_native.append, pools, page_table, lengths, R, S, Vr, Vs, counts, Q, weights, table, positions, mass, eps, interleaved)
    if got is None:
        _refuse_append(pools, page_table, lengths, (R, S, Vr, Vs) if Q is None else (R, S, Vr, Vs, Q), counts, weights, table, positions,
                       mass, eps)
    return got if Q is not None else None


def _refuse_append(pools, page_table, lengths, new, counts, weights, table, positions, mass, eps):
    who = "gather_cache_append"
    pool = _check_pools(who, pools)
    B, T, D = _check_heads(who, new, _NEW)
    dev, Hkv = pool.device, pool.shape[2]
    if new[0].device != dev or D != pool.shape[3] or any(x.shape[2] != Hkv for x in new[:4]):
        raise RuntimeError(f"{who}: new rows must be [B,T,{Hkv},{pool.shape[3]}] on the pools' device")
    _check_table_of_pages(who, page_table, lengths, dev, B=B)
    if counts is not None:
        _check_ints(who, "counts", counts, B, dev)
    if positions is not None:
        _check_ints(who, "positions", positions, B, dev)
    _check_mass(who, mass, pool)
    if len(weights) != 3:
        raise RuntimeError(f"{who}: weights are three scales, of Q, R and S")
    _no_grad(who, *new, *weights, *pools, table, mass)
    for k, w in enumerate(weights):
        _check_scale(w, who, f"weight {k}", D, dev)
    _check_table(who, table, D, dev)
    _check_eps(who, eps)
    _on_gpu(who, pool)
    raise RuntimeError(f"{who}: arguments of a type or size that the kernels do not take")


def single_gather_decode(Q, pools, page_table, lengths, *, window=0, sinks=0, mass=None):
    """The gather of one new token of every sequence over its cached rows (the token's own, appended before, among them):

        Y[b,h] = sum_{j,k} softmax_{(j,k)}(Q[b,h] . R_j . S_k / sqrt(D)) Vr_j o Vs_k

    Q [B,Hq,D] (cast to bf16), D in {64,128}, Hq a multiple of the pools' Hkv; returns [B,Hq,D] in Q's type.  window > 0
    makes the last `window` slots and the first `sinks` visible, window=0 all of them.  A sequence of length 0 gives
    zeros.  Scores are formed without rounding Q o R (what precise=True does in `single_gather_attention`).

    mass (FP32 [pages,page_size,Hkv]), if given, gains every visible slot's share of the attention: the mean over the
    key head's query heads of half the probability of the pairs that hold the slot as j plus half of those that hold it
    as k, 1 in all for every sequence and key head.  A slot that several sequences share gains each one's, in no fixed order.
    The call's scratch memory goes by what the page table could hold, not by the lengths: with masses about 12 bytes a query head and
    slot (of the window and sinks, if there is a window) and 8 bytes an SM and slot."""
    y = _accepted(_native.decode, Q, pools, page_table, lengths, window, sinks, mass)
    if y is None:
        _refuse_decode(Q, pools, page_table, lengths, window, sinks, mass)
    return y


def _refuse_decode(Q, pools, page_table, lengths, window, sinks, mass):
    who = "single_gather_decode"
    pool = _check_pools(who, pools)
    if not isinstance(Q, torch.Tensor) or Q.dim() != 3 or not Q.is_floating_point():
        raise RuntimeError(f"{who}: Q must be a [B,Hq,D] tensor")
    B, Hq, D = Q.shape
    Hkv = pool.shape[2]
    if D not in (64, 128):
        raise RuntimeError(f"{who}: D must be 64 or 128, got {D}")
    if D != pool.shape[3]:
        raise RuntimeError(f"{who}: Q has head dim {D}, the pools {pool.shape[3]}")
    if Hq < 1 or Hq % Hkv:
        raise RuntimeError(f"{who}: Hq={Hq} is not divisible by Hkv={Hkv}")
    if Q.device != pool.device:
        raise RuntimeError(f"{who}: Q must be on the pools' device")
    _check_table_of_pages(who, page_table, lengths, pool.device, B=B)
    if int(window) < 0 or int(sinks) < 0:
        raise RuntimeError(f"{who}: window and sinks must not be negative, got {window}, {sinks}")
    if sinks and not window:
        raise RuntimeError(f"{who}: sinks go with a window")
    _check_mass(who, mass, pool)
    _no_grad(who, Q, *pools, mass)
    _on_gpu(who, Q)
    raise RuntimeError(f"{who}: arguments of a type or size that the kernels do not take")


def gather_cache_evict(pools, mass, page_table, lengths, keep, *, sinks=0, recent=0, out_table=None):
    """Trims every sequence and key head to min(lengths[b], keep) slots: the first `sinks`, the last `recent` and, between
    them, those with the largest `mass` (equal ones: the lowest slots; NaN counts as largest).  The kept rows of all
    pools move with their mass, in order, to slots 0 .. , in place, or to the pages of `out_table`, which must then name
    none that a sequence of the call reads; in place, no two sequences may share a page.  Slots behind the last kept one
    are left as they are.  Key heads of a sequence may keep different slots.

    Returns (kept int32 [B,Hkv,keep], the slots that stayed, -1 behind the last; new lengths int32 [B])."""
    got = _accepted(_native.evict, pools, mass, page_table, lengths, keep, sinks, recent, out_table)
    if got is None:
        _refuse_evict(pools, mass, page_table, lengths, keep, sinks, recent, out_table)
    return got


def _refuse_evict(pools, mass, page_table, lengths, keep, sinks, recent, out_table):
    who = "gather_cache_evict"
    pool = _check_pools(who, pools)
    D = pool.shape[3]
    if D not in (16, 32, 64, 128):
        raise RuntimeError(f"{who}: head dim must be 16, 32, 64 or 128, got {D}")
    if mass is None:
        raise RuntimeError(f"{who}: needs the mass that it goes by")
    _check_mass(who, mass, pool)
    _check_table_of_pages(who, page_table, lengths, pool.device)
    _no_grad(who, *pools, mass)
    B = page_table.shape[0]
    if int(keep) < 1 or int(sinks) < 0 or int(recent) < 0 or int(sinks) + int(recent) > int(keep):
        raise RuntimeError(f"{who}: sinks + recent must fit in keep >= 1, got {sinks} + {recent} in {keep}")
    slots = page_table.shape[1] * pool.shape[1]
    if out_table is not None:
        _check_table_of_pages(who, out_table, None, pool.device, "out_table", B)
        if out_table.shape[1] * pool.shape[1] < min(int(keep), slots):
            raise RuntimeError(f"{who}: out_table has no room for {min(int(keep), slots)} slots")
    _on_gpu(who, pool)
    raise RuntimeError(f"{who}: arguments of a type or size that the kernels do not take")


class GatherCache:
    """A paged gather cache of a batch of sequences: pools, page table and lengths on the device, and the book-keeping of
    pages on the host.  A sequence that is done is left out by a count of 0 (`append`, `decode`), or emptied by `clear` and
    filled anew.

    sequences: rows of the page table.  pages: pages of `page_size` slots in each pool.  slots: the most that a sequence
    may hold.  track_mass: add up every token's share of the attention in `decode`, for `evict`.

    Pages are handed out in Python when a call needs them, so these methods are not for capture into a graph: a captured
    step calls the functions above on tensors of its own (or this cache's), which read lengths and tables as they are.
    `reserve` copies the table from pageable memory when a call needs a page, and counts are copied likewise: both wait for
    the stream."""

    def __init__(self, sequences, n_kv_heads, head_dim, *, pages, slots, page_size=64, track_mass=False, device="cuda"):
        if min(sequences, n_kv_heads, pages, slots, page_size) < 1:
            raise ValueError("GatherCache: sequences, heads, pages, slots and page_size must be positive")
        if head_dim not in (64, 128):
            raise ValueError(f"GatherCache: head_dim must be 64 or 128, got {head_dim}")
        self.sequences, self.page_size, self.slots = sequences, page_size, slots
        shape = (pages, page_size, n_kv_heads, head_dim)
        with torch.inference_mode(False):           # a cache made in inference mode may be used outside it
            self.pools = [torch.zeros(shape, dtype=_BF16, device=device) for _ in range(4)]
            self.mass = torch.zeros(shape[:3], dtype=torch.float32, device=device) if track_mass else None
            self._book = torch.full((sequences, -(-slots // page_size)), -1, dtype=torch.int32)      # the host's page table
            self.page_table = self._book.to(device, copy=True)
            # slots in use and tokens seen (which stay apart once tokens have been evicted), one tensor so that one add moves both
            self._counters = torch.zeros((2, sequences), dtype=torch.int32, device=device)
            self.lengths, self.positions = self._counters[0], self._counters[1]
        self.host_lengths, self.host_positions = [0] * sequences, [0] * sequences
        self._free = list(range(pages - 1, -1, -1))

    def _counts(self, counts, T):
        if counts is None:
            return [T] * self.sequences
        counts = [int(c) for c in counts]
        if len(counts) != self.sequences or any(not 0 <= c <= T for c in counts):
            raise ValueError(f"GatherCache: counts must be {self.sequences} numbers of 0 .. {T}")
        return counts

    def _on_device(self, counts):
        return torch.tensor(counts, dtype=torch.int32, device=self.page_table.device)

    def reserve(self, counts):
        """Hands out the pages that `counts[b]` more slots of every sequence need."""
        want = []
        for b, c in enumerate(counts):
            n = self.host_lengths[b] + c
            if n > self.slots:
                raise RuntimeError(f"GatherCache: sequence {b} would hold {n} slots, at most {self.slots}")
            have, need = -(-self.host_lengths[b] // self.page_size), -(-n // self.page_size)
            want += [(b, k) for k in range(have, need) if int(self._book[b, k]) < 0]
        if len(want) > len(self._free):
            raise RuntimeError(f"GatherCache: {len(want)} pages needed, {len(self._free)} free")
        for b, k in want:
            self._book[b, k] = self._free.pop()
        if want:
            self.page_table.copy_(self._book)

    def append(self, R, S, Vr, Vs, *, counts=None, Q=None, weights=None, table=None, eps=1e-6, interleaved=False):
        """`gather_cache_append` at the sequences' ends (R .. [B,T,Hkv,D]; counts: a list of ints, all T by default);
        rotations go by the number of tokens seen, evicted ones included.  Returns Q's rows, if given."""
        T = R.shape[1]
        host = self._counts(counts, T)
        self.reserve(host)
        on_device = None if counts is None else self._on_device(host)
        q = gather_cache_append(self.pools, self.page_table, self.lengths, R, S, Vr, Vs, counts=on_device, Q=Q, weights=weights,
                                table=table, positions=self.positions, mass=self.mass, eps=eps, interleaved=interleaved)
        self._counters.add_(T if on_device is None else on_device)
        for b, c in enumerate(host):
            self.host_lengths[b] += c
            self.host_positions[b] += c
        return q

    def decode(self, Q, *, window=0, sinks=0, counts=None):
        """`single_gather_decode` of Q [B,Hq,D] over the cached rows, adding to the masses if they are tracked.  counts (a
        list of 0 and 1): a sequence of 0 sits out, gives zeros and keeps its masses."""
        lengths = self.lengths if counts is None else self.lengths * self._on_device(self._counts(counts, 1))
        return single_gather_decode(Q, self.pools, self.page_table, lengths, window=window, sinks=sinks, mass=self.mass)

    def evict(self, keep, *, sinks=0, recent=0):
        """`gather_cache_evict` in place; the pages behind the kept slots become free.  Returns the slots that stayed,
        int32 [B,Hkv,keep].

        Masses come from `decode` alone: rows that were appended since have none yet, and slots that no query sees, behind
        a window, gain none.  keep = sinks + recent = sinks + window keeps what a windowed layer sees and frees the rest."""
        if self.mass is None:
            raise RuntimeError("GatherCache.evict: the cache does not track masses (track_mass=True)")
        kept, left = gather_cache_evict(self.pools, self.mass, self.page_table, self.lengths, keep, sinks=sinks, recent=recent)
        self.lengths.copy_(left)
        for b in range(self.sequences):
            self.host_lengths[b] = min(self.host_lengths[b], int(keep))
            self._release(b, -(-self.host_lengths[b] // self.page_size))
        self.page_table.copy_(self._book)
        return kept

    def _release(self, b, first):
        for k in range(first, self._book.shape[1]):
            page = int(self._book[b, k])
            if page >= 0:
                self._free.append(page)
                self._book[b, k] = -1

    def clear(self, sequence):
        """Empties one sequence and frees its pages."""
        self._release(sequence, 0)
        self.host_lengths[sequence] = self.host_positions[sequence] = 0
        self._counters[:, sequence] = 0
        self.page_table.copy_(self._book)

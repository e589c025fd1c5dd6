"""What the serving operators refuse, and their host-side logic: no GPU needed."""
import ctypes as C
import re

import pytest
import torch

from conftest import REPO
from att3ntion_b200 import (GatherCache, HypergraphAttention, _cabi, gather_cache_append, gather_cache_evict, norm_rotate,
                            rotary_table, single_gather_decode, window_mask)

lib = _cabi.lib
INT = torch.int32


def test_struct_sizes():
    """Every member of the two structs is 8 bytes wide, so that a binding may fill them as arrays of 64-bit integers: the
    header's declarations have as many as _cabi says."""
    header = (REPO / "include" / "att3_b200.h").read_text()

    def count(name):
        body = re.sub(r"/\*.*?\*/", "", re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, re.S).group(1), flags=re.S)
        assert all(t in ("const void*", "void*", "int64_t", "float*", "const int32_t*") for t in
                   re.findall(r"([\w ]+\*?) \w+(?:\[\d+\])?;", body.replace("\n", " ").strip()) for t in [t.strip()])
        return sum(int(m.group(1) or 1) for m in re.finditer(r"\w+(?:\[(\d+)\])?;", body))

    assert count("att3_head_rows") == _cabi.HEAD_ROWS_WORDS
    assert count("att3_gather_pages") == _cabi.GATHER_PAGES_WORDS


def test_rotary_table_keeps_far_angles():
    t = rotary_table(1 << 17, 16, 10000.0)
    p, i = 131071, 3
    a = torch.tensor(p * 10000.0 ** (-2 * i / 16), dtype=torch.float64)
    assert t.shape == (1 << 17, 16) and t.dtype == torch.float32
    assert abs(t[p, i] - a.cos()) < 1e-7 and abs(t[p, 8 + i] - a.sin()) < 1e-7
    for bad in ((0, 16), (4, 7), (4, 0)):
        with pytest.raises(ValueError, match="rotary_table"):
            rotary_table(*bad)


def test_window_mask_with_sinks():
    m = window_mask(9, 3, "cpu", 2)
    for q in range(9):
        for k in range(9):
            assert bool(m[q, k]) == (k <= q and (k > q - 3 or k < 2))
    assert torch.equal(window_mask(9, 3, "cpu"), window_mask(9, 3, "cpu", 0))


def bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("match,call", [
    ("B,N,heads,D", lambda: norm_rotate(bf(2, 3, 64))),
    ("head dim", lambda: norm_rotate(bf(1, 2, 3, 48))),
    ("one type", lambda: norm_rotate([bf(1, 2, 3, 64), torch.zeros(1, 2, 3, 64)])),
    ("one type", lambda: norm_rotate(torch.zeros(1, 2, 3, 64, dtype=torch.float64))),
    ("expected batch", lambda: norm_rotate([bf(1, 2, 3, 64), bf(1, 3, 3, 64)])),
    ("no heads", lambda: norm_rotate(bf(1, 2, 0, 64))),
    ("weights", lambda: norm_rotate([bf(1, 2, 3, 64)], [None, None])),
    ("one to five", lambda: norm_rotate([])),
    (r"weight 0 must be a \[64\]", lambda: norm_rotate(bf(1, 2, 3, 64), torch.ones(32))),
    ("table must be FP32", lambda: norm_rotate(bf(1, 2, 3, 64), None, bf(8, 64))),
    ("multiple of 8", lambda: norm_rotate(bf(1, 2, 3, 64), None, torch.zeros(8, 12))),
    ("multiple of 8", lambda: norm_rotate(bf(1, 2, 3, 64), None, torch.zeros(8, 128))),
    ("9 positions", lambda: norm_rotate(bf(1, 9, 3, 64), None, torch.zeros(8, 64))),
    ("positions must be", lambda: norm_rotate(bf(2, 9, 3, 64), None, torch.zeros(16, 64), torch.zeros(2, dtype=INT))),
    ("int32 or int64", lambda: norm_rotate(bf(2, 9, 3, 64), None, torch.zeros(16, 64), torch.zeros(9))),
    ("eps", lambda: norm_rotate(bf(1, 2, 3, 64), torch.ones(64), eps=-1.0)),
    ("eps", lambda: norm_rotate(bf(1, 2, 3, 64), torch.ones(64), eps=float("nan"))),
    ("CUDA", lambda: norm_rotate(bf(1, 2, 3, 64))),
])
def test_norm_rotate_refuses(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def cache_args(P=4, page=16, Hkv=2, D=64, B=2, entries=3, table=INT, lengths=INT):
    return [bf(P, page, Hkv, D) for _ in range(4)], torch.zeros(B, entries, dtype=table), torch.zeros(B, dtype=lengths)


def append(T=1, Hkv=2, D=64, B=2, new=None, cache=None, **kw):
    pools, table, lengths = cache or cache_args()
    new = new or [bf(B, T, Hkv, D) for _ in range(4)]
    return gather_cache_append(pools, table, lengths, *new, **kw)


@pytest.mark.parametrize("match,call", [
    ("four tensors", lambda: append(cache=(cache_args()[0][:3], *cache_args()[1:]))),
    ("pool S must be", lambda: append(cache=([bf(4, 16, 2, 64), torch.zeros(4, 16, 2, 64)] + [bf(4, 16, 2, 64)] * 2, *cache_args()[1:]))),
    ("pool Vr must be", lambda: append(cache=([bf(4, 16, 2, 64)] * 2 + [bf(4, 2, 16, 64).transpose(1, 2)] * 2, *cache_args()[1:]))),
    ("one shape", lambda: append(cache=([bf(4, 16, 2, 64)] * 3 + [bf(5, 16, 2, 64)], *cache_args()[1:]))),
    ("empty", lambda: append(cache=cache_args(P=0))),
    ("new rows must be", lambda: append(Hkv=3)),
    ("new rows must be", lambda: append(D=128)),
    ("int32", lambda: append(cache=cache_args(table=torch.int64))),
    ("lengths", lambda: append(cache=cache_args(lengths=torch.int64))),
    ("rows for", lambda: append(B=3)),
    ("counts", lambda: append(counts=torch.zeros(3, dtype=INT))),
    ("positions", lambda: append(positions=torch.zeros(2, dtype=torch.int64))),
    ("mass", lambda: append(mass=torch.zeros(4, 16, 1))),
    ("three scales", lambda: append(weights=[None, None])),
    ("gradient", lambda: append(new=[bf(2, 1, 2, 64).requires_grad_() for _ in range(4)])),
    ("CUDA", lambda: append()),
])
def test_append_refuses(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def decode(Q=None, cache=None, **kw):
    pools, table, lengths = cache or cache_args()
    return single_gather_decode(bf(2, 4, 64) if Q is None else Q, pools, table, lengths, **kw)


@pytest.mark.parametrize("match,call", [
    (r"\[B,Hq,D\]", lambda: decode(bf(2, 1, 4, 64))),
    ("64 or 128", lambda: decode(bf(2, 4, 32), cache_args(D=32))),
    ("head dim", lambda: decode(bf(2, 4, 128))),
    ("divisible", lambda: decode(bf(2, 3, 64))),
    ("divisible", lambda: decode(bf(2, 0, 64))),
    ("rows for", lambda: decode(bf(3, 4, 64))),
    ("negative", lambda: decode(window=-1)),
    ("negative", lambda: decode(window=4, sinks=-1)),
    ("go with a window", lambda: decode(sinks=2)),
    ("mass", lambda: decode(mass=torch.zeros(4, 16, 2, dtype=torch.float64))),
    ("gradient", lambda: decode(bf(2, 4, 64).requires_grad_())),
    ("neighbours", lambda: decode(cache=(cache_args()[0], torch.zeros(2, 6, dtype=INT)[:, ::2], cache_args()[2]))),
    ("at least one entry", lambda: decode(cache=cache_args(entries=0))),
    ("CUDA", lambda: decode()),
])
def test_decode_refuses(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def evict(keep=8, mass=torch.zeros(4, 16, 2), cache=None, **kw):
    pools, table, lengths = cache or cache_args()
    return gather_cache_evict(pools, mass, table, lengths, keep, **kw)


@pytest.mark.parametrize("match,call", [
    ("needs the mass", lambda: evict(mass=None)),
    ("mass must be", lambda: evict(mass=torch.zeros(4, 16, 1))),
    ("sinks \\+ recent", lambda: evict(keep=0)),
    ("sinks \\+ recent", lambda: evict(keep=8, sinks=5, recent=4)),
    ("sinks \\+ recent", lambda: evict(keep=8, sinks=-1)),
    ("no room", lambda: evict(keep=20, out_table=torch.zeros(2, 1, dtype=INT))),
    ("rows for", lambda: evict(out_table=torch.zeros(3, 3, dtype=INT))),
    ("head dim", lambda: evict(cache=cache_args(D=48))),
    ("CUDA", lambda: evict()),
])
def test_evict_refuses(match, call):
    with pytest.raises(RuntimeError, match=match):
        call()


def words(n):
    return (C.c_int64 * n)()


def test_c_entries_refuse_before_any_device_work():
    """Null and odd arguments of the C functions come back as status codes with a message."""
    one = C.c_void_p(256)
    rows = words(21 * 4)
    for k in range(4):
        rows[21 * k + 20] = 2                              # heads
    bad = _cabi.ERR_INVALID

    def forward(t=rows, n=1, x_type=0, table=None, table_rows=0, rot=0, pos=None, pos_bytes=0, B=1, N=1, D=64, eps=1e-6):
        return lib.att3_norm_rotate_forward(t, n, x_type, table, table_rows, rot, 0, pos, pos_bytes, 0, 0, B, N, D, eps, None)

    for kw, text in ((dict(t=None), "tensors"), (dict(n=0), "tensors"), (dict(n=6), "tensors"), (dict(D=40), "head dim"),
                     (dict(B=-1), "negative"), (dict(x_type=3), "element type"), (dict(eps=-1.0), "eps"),
                     (dict(rot=12), "multiple of 8"), (dict(rot=72), "multiple of 8"), (dict(rot=64), "table"),
                     (dict(rot=64, table=C.c_void_p(8), table_rows=4), "table"), (dict(pos=one, pos_bytes=2), "4 or 8 bytes"),
                     (dict(t=words(21)), "no heads"), (dict(), "null tensor"), (dict(B=1 << 20, N=1 << 20), "2^30 rows")):
        assert forward(**kw) == bad and text in _cabi.last_error(), (kw, _cabi.last_error())
    assert forward(B=0) == forward(N=0) == _cabi.OK        # nothing to do

    pages = words(5)
    pages[0], pages[1], pages[2], pages[3], pages[4] = 256, 4, 4, 8, 16

    def changed(k, v):
        p = words(5)
        p[:] = list(pages)
        p[k] = v
        return p

    def do_decode(q=one, pages=pages, B=2, Hq=4, Hkv=2, D=64, window=0, sinks=0, ws=None, nbytes=0, mass=None):
        return lib.att3_sg_decode(q, one, one, one, one, mass, one, pages, one, B, Hq, Hkv, D, window, sinks, ws, nbytes, None)

    for kw, text in ((dict(Hq=3), "divisible"), (dict(Hkv=0), "divisible"), (dict(D=32), "64 or 128"), (dict(window=-1), "negative"),
                     (dict(pages=None), "page table"), (dict(pages=changed(0, 0)), "page table"), (dict(pages=changed(4, 0)), "positive"),
                     (dict(pages=changed(3, 1 << 40)), "2^31"), (dict(pages=changed(2, 1 << 40)), "2^31"), (dict(q=None), "null"),
                     (dict(q=C.c_void_p(264)), "aligned"), (dict(B=1 << 23), "too many heads"),
                     (dict(B=1 << 17, mass=one), "65535"), (dict(window=1 << 30, sinks=1 << 30), "too wide")):
        assert do_decode(**kw) == bad and text in _cabi.last_error(), (kw, _cabi.last_error())
    assert do_decode() == _cabi.ERR_WORKSPACE and "workspace" in _cabi.last_error()
    n = lib.att3_sg_decode_workspace_bytes(2, 4, 2, 64, 0, 0, 64, 0)
    assert 0 < n <= lib.att3_sg_decode_workspace_bytes(2, 4, 2, 64, 0, 0, 64, 1)
    assert do_decode(ws=one, nbytes=n - 1) == _cabi.ERR_WORKSPACE
    assert do_decode(B=0) == _cabi.OK
    assert lib.att3_sg_decode_workspace_bytes(2, 3, 2, 64, 0, 0, 64, 0) == 0

    def do_evict(R=one, pages=pages, out=pages, Hkv=2, D=64, keep=8, sinks=0, recent=0):
        return lib.att3_gather_cache_evict(R, one, one, one, one, pages, out, one, one, one, 2, Hkv, D, keep, sinks, recent, None)

    for kw, text in ((dict(Hkv=0), "head dimension"), (dict(D=8), "head dim"), (dict(keep=0), "sinks + recent"),
                     (dict(sinks=5, recent=4), "sinks + recent"), (dict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), "sinks + recent"),
                     (dict(out=None), "page table"), (dict(keep=60, out=changed(2, 1)), "no room"),
                     (dict(out=changed(3, 9)), "same pools"), (dict(R=None), "null"), (dict(R=C.c_void_p(8)), "aligned")):
        assert do_evict(**kw) == bad and text in _cabi.last_error(), (kw, _cabi.last_error())

    def do_append(n=4, t=rows, pages=pages, lengths=one):
        return lib.att3_gather_cache_append(t, n, 0, None, 0, 0, 0, None, pages, lengths, None, None, 1, 1, 64, 1e-6, None)

    for kw, text in ((dict(n=3), "R, S, Vr, Vs"), (dict(pages=None), "page table"), (dict(lengths=None), "null lengths"), (dict(), "null tensor")):
        assert do_append(**kw) == bad and text in _cabi.last_error(), (kw, _cabi.last_error())

    assert lib.att3_norm_rotate_backward(rows, 1, 0, None, 0, 0, 0, None, 0, 0, 0, 0, 1, 64, 1e-6, None, 0, None) == _cabi.ERR_WORKSPACE
    assert lib.att3_norm_rotate_workspace_bytes(0, 64) == 0 < lib.att3_norm_rotate_workspace_bytes(1, 64)


def test_cache_hands_out_pages_and_takes_them_back():
    c = GatherCache(3, 1, 64, pages=6, slots=40, page_size=16, device="cpu")
    c.reserve([16, 1, 0])
    assert (c.page_table >= 0).sum(1).tolist() == [1, 1, 0] and len(c._free) == 4
    c.host_lengths = [16, 1, 0]
    c.reserve([1, 15, 33])
    assert (c.page_table >= 0).sum(1).tolist() == [2, 1, 3] and len(c._free) == 0
    used = c.page_table[c.page_table >= 0].tolist()
    assert sorted(used) == list(range(6))
    c.host_lengths = [17, 16, 33]
    with pytest.raises(RuntimeError, match="1 pages needed, 0 free"):
        c.reserve([0, 1, 0])
    with pytest.raises(RuntimeError, match="at most 40"):
        c.reserve([24, 0, 0])
    c.clear(2)
    assert len(c._free) == 3 and c.page_table[2].tolist() == [-1, -1, -1] and c.host_lengths == [17, 16, 0]
    c.reserve([0, 1, 0])
    assert len(c._free) == 2
    with pytest.raises(ValueError, match="counts"):
        c._counts([1, 2], 4)
    with pytest.raises(ValueError, match="counts"):
        c._counts([1, 5, 0], 4)
    with pytest.raises(RuntimeError, match="track_mass"):
        c.evict(4)
    for kw in (dict(pages=0, slots=4), dict(pages=4, slots=0)):
        with pytest.raises(ValueError):
            GatherCache(1, 1, 64, device="cpu", **kw)
    with pytest.raises(ValueError, match="head_dim"):
        GatherCache(1, 1, 32, pages=1, slots=1, device="cpu")


def test_layer_arguments():
    with pytest.raises(ValueError, match="sinks"):
        HypergraphAttention(64, 1, gather_mode=1, sinks=2)
    with pytest.raises(ValueError, match="head dim"):
        HypergraphAttention(96, 2, qk_norm=True)
    plain = HypergraphAttention(128, 2, gather_mode=1, window=16)
    assert not any("norm" in k for k in plain.state_dict())          # what was saved before loads as before
    layer = HypergraphAttention(128, 2, gather_mode=1, window=16, qk_norm=True, rotary_base=1e4)
    assert {k for k in layer.state_dict()} - {k for k in plain.state_dict()} == {"q_norm", "r_norm", "s_norm"}
    a = layer._rotary(10, torch.device("cpu"))
    assert a.shape == (512, 64) and layer._rotary(512, torch.device("cpu")) is a
    b = layer._rotary(513, torch.device("cpu"))
    assert b.shape == (1024, 64) and torch.equal(b[:512], a) and layer._tables[0] is a
    cache = GatherCache(2, 2, 64, pages=4, slots=32, page_size=16, device="cpu")
    for x, match in ((torch.zeros(1, 4, 128), "x must be"), (torch.zeros(2, 128), "x must be")):
        with pytest.raises(ValueError, match=match):
            layer.prefill(x, cache)
    with pytest.raises(ValueError, match="one token"):
        layer.decode(torch.zeros(2, 2, 128), cache)
    with pytest.raises(ValueError, match="needs gather_mode=1"):
        HypergraphAttention(128, 2, gather_mode=1).decode(torch.zeros(2, 1, 128), cache)
    cache.host_lengths[0] = 3
    with pytest.raises(ValueError, match="empty"):
        layer.prefill(torch.zeros(2, 4, 128), cache)


# --------------------------------------------------------------------------- the decode's ring of stages

class Phases:
    """An mbarrier as its waiters see it: only the parity of the running phase."""

    def __init__(self, arrivals):
        self.need, self.left, self.done = arrivals, arrivals, 0

    def arrive(self):
        self.left -= 1
        if self.left == 0:
            self.done, self.left = self.done + 1, self.need

    def passes(self, parity):
        return self.done % 2 != parity


def ring_ends(arrivals, busy, fills, stages, last):
    """Copy warps of the ring (busy[w]: it has bytes to bring) and its reader, one step at a time, warp `last` only when no
    other can go on: whether all of them end."""
    full, empty = [Phases(arrivals) for _ in range(stages)], [Phases(1) for _ in range(stages)]
    landed, at, read = [0] * fills, [0] * len(busy), 0

    def copy_step(w):
        f = at[w]
        if f == fills or (f >= stages and not empty[f % stages].passes((f // stages - 1) % 2)):
            return False
        if w == 0 or arrivals > 1:
            full[f % stages].arrive()
        landed[f] += busy[w]
        at[w] += 1
        return True

    while True:
        if read < fills and full[read % stages].passes((read // stages) % 2) and landed[read] == sum(busy):
            empty[read % stages].arrive()
            read += 1
        elif not any(copy_step(w) for w in range(len(busy)) if w != last) and not copy_step(last):
            return read == fills and all(a == fills for a in at)


@pytest.mark.parametrize("stages", [3, 8])
@pytest.mark.parametrize("busy", [(1, 0, 0), (1, 1, 0), (1, 1, 1)])
def test_no_copy_warp_misses_a_phase_of_the_ring(stages, busy):
    """Boxes of 128 rows leave two of the three copy warps without work, boxes of 64 one.  Whichever of them is late, the
    ring's barriers must not go round twice meanwhile; with one arrival a stage they could."""
    source = (REPO / "att3ntion_b200" / "csrc" / "serve_decode.cuh").read_text()
    warps = re.search(r"DEC_COPY_WARPS = (\d+);", source).group(1)
    count = re.search(r"mbar_init\(&bars\[DB_KV_FULL0 \+ x\], (\w+)\)", source).group(1)
    arrivals = int(warps if count == "DEC_COPY_WARPS" else count)
    for fills in range(1, 8 * stages):
        for last in range(3):
            assert ring_ends(arrivals, busy, fills, stages, last), (fills, last)
    assert not all(ring_ends(1, (1, 0, 0), fills, stages, 1) for fills in range(1, 8 * stages))


def test_kernels_set_up_early_use_no_read_only_loads():
    """The serving kernels start while the kernel before them, which may write their inputs, still runs: loads that want
    memory constant for the kernel's whole life are not theirs to use."""
    sources = list((REPO / "att3ntion_b200" / "csrc").glob("serve_*.cu*"))
    assert len(sources) >= 5
    for path in sources:
        code = re.sub(r"//.*", "", path.read_text())
        assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", code), path.name


def test_decode_refuses_heads_whose_rows_pass_32_bits():
    """2^24 key heads of 128 make a slot of 2^32 bytes, which the copies' 32-bit pitch cannot hold."""
    assert lib.att3_sg_decode_workspace_bytes(1, 1 << 24, 1 << 24, 128, 0, 0, 16, 0) == 0
    assert "too many heads" in _cabi.last_error()
    assert lib.att3_sg_decode_workspace_bytes(1, (1 << 24) - 1, (1 << 24) - 1, 128, 0, 0, 16, 0) > 0


# --------------------------------------------------------------------------- what autograd would miss

def dual(t):
    return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("call", [
    lambda: norm_rotate(dual(bf(1, 2, 3, 64))),
    lambda: norm_rotate([bf(1, 2, 3, 64)] * 2, [None, dual(torch.ones(64))]),
    lambda: norm_rotate(bf(1, 2, 3, 64), None, dual(torch.zeros(8, 64))),
    lambda: append(new=[bf(2, 1, 2, 64)] * 3 + [dual(bf(2, 1, 2, 64))]),
    lambda: append(weights=[None, dual(torch.ones(64)), None]),
    lambda: append(Q=dual(bf(2, 1, 4, 64))),
    lambda: append(cache=([bf(4, 16, 2, 64)] * 3 + [dual(bf(4, 16, 2, 64))], *cache_args()[1:])),
    lambda: decode(dual(bf(2, 4, 64))),
    lambda: decode(cache=([dual(bf(4, 16, 2, 64))] + [bf(4, 16, 2, 64)] * 3, *cache_args()[1:])),
    lambda: decode(mass=dual(torch.zeros(4, 16, 2))),
    lambda: evict(mass=dual(torch.zeros(4, 16, 2))),
    lambda: evict(cache=([bf(4, 16, 2, 64)] * 3 + [dual(bf(4, 16, 2, 64))], *cache_args()[1:])),
])
@pytest.mark.parametrize("grad", [True, False])
def test_tangents_are_refused(call, grad):
    """A dual tensor requires no gradient, and forward differentiation goes on under no_grad."""
    with torch.set_grad_enabled(grad), torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            call()


@pytest.mark.parametrize("call", [
    lambda: norm_rotate(bf(1, 2, 3, 64), None, torch.zeros(8, 64, requires_grad=True)),
    lambda: append(cache=([bf(4, 16, 2, 64).requires_grad_()] + [bf(4, 16, 2, 64)] * 3, *cache_args()[1:])),
    lambda: append(table=torch.zeros(8, 64, requires_grad=True)),
    lambda: decode(mass=torch.zeros(4, 16, 2, requires_grad=True)),
    lambda: evict(mass=torch.zeros(4, 16, 2, requires_grad=True)),
    lambda: evict(cache=([bf(4, 16, 2, 64).requires_grad_()] + [bf(4, 16, 2, 64)] * 3, *cache_args()[1:])),
])
def test_gradients_that_there_are_none_of_are_refused(call):
    with pytest.raises(RuntimeError, match="gradient"):
        call()


# --------------------------------------------------------------------------- the layer's angle table

def test_angle_table_is_an_ordinary_tensor_whoever_asks_first():
    import copy
    from torch._subclasses.fake_tensor import FakeTensorMode
    cpu = torch.device("cpu")
    layer = HypergraphAttention(64, 1, gather_mode=1, window=16, rotary_base=1e4)
    with FakeTensorMode():
        layer._rotary(8, cpu)
    assert layer._tables == []
    with torch.inference_mode():
        t = layer._rotary(8, cpu)
    assert not t.is_inference() and layer._rotary(512, cpu) is t
    (t * torch.ones(1, requires_grad=True)).sum().backward()                      # saved for the backward pass
    twin = copy.deepcopy(layer)
    assert twin._tables == [] and layer._tables[0] is t and torch.equal(twin._rotary(8, cpu), t)


def test_layers_pickled_before_they_had_norms_and_tables_load():
    import pickle
    old = HypergraphAttention(64, 1, gather_mode=1, window=16)
    for name in ("sinks", "rotary_base", "norm_eps", "_tables", "q_norm", "r_norm", "s_norm"):
        old.__dict__.pop(name)
    new = pickle.loads(pickle.dumps(old))
    assert new.sinks == 0 and not new.rotary_base and new.q_norm is None and new._rotary(4, torch.device("cpu")) is None
    normed = pickle.loads(pickle.dumps(HypergraphAttention(64, 1, gather_mode=1, window=16, qk_norm=True, rotary_base=10.0)))
    assert isinstance(normed.q_norm, torch.nn.Parameter) and normed.rotary_base == 10.0 and normed._tables == []


def test_cache_made_in_inference_mode_is_used_outside_it():
    with torch.inference_mode():
        c = GatherCache(2, 1, 64, pages=4, slots=32, page_size=16, track_mass=True, device="cpu")
    assert not any(t.is_inference() for t in (*c.pools, c.mass, c.page_table, c.lengths, c.positions))
    c._counters.add_(1)
    assert c.lengths.tolist() == c.positions.tolist() == [1, 1]
    c.reserve([17, 0])
    with torch.inference_mode():
        c._counters.add_(1)
        c.clear(0)
    assert c.lengths.tolist() == [0, 2] and len(c._free) == 4


def test_scratch_for_masses_goes_by_the_slots():
    """Linear in the page table's width and in the heads: 12 bytes a query head and slot, 8 an SM and slot, and what the call
    without masses takes."""
    sms = 148
    for B, Hq, Hkv, D in ((1, 8, 1, 128), (16, 8, 8, 64), (8, 32, 4, 128)):
        for slots in (1 << 12, 1 << 15, 1 << 16, 131072, 1 << 20):
            plain = lib.att3_sg_decode_workspace_bytes(B, Hq, Hkv, D, 0, 0, slots, 0)
            extra = lib.att3_sg_decode_workspace_bytes(B, Hq, Hkv, D, 0, 0, slots, 1) - plain
            tail = 256 * (B * Hq + sms) * 16 + 65536            # references, partial tiles, rounding of the parts
            assert 0 < extra <= 13 * B * Hq * slots + 9 * sms * slots + tail, (B, Hq, slots, extra)


def test_training_does_without_the_serving_binding():
    """Without the torch binding the layers and operators of the C ABI import and construct; what needs it says so."""
    import subprocess
    import sys
    code = """
import sys
sys.modules["att3ntion_b200._serve_native"] = None
import torch, att3ntion
from att3ntion_b200 import GatherCache, HypergraphAttention, norm_rotate, single_gather_attention
HypergraphAttention(64, 1)
cache = GatherCache(1, 1, 64, pages=1, slots=16, page_size=16, track_mass=True, device="cpu")
x = torch.zeros(1, 1, 1, 64)
for call in (lambda: norm_rotate(x), lambda: cache.append(x, x, x, x), lambda: cache.decode(x[0]), lambda: cache.evict(1)):
    try:
        call()
    except ImportError as e:
        assert "att3ntion_b200.build" in str(e), e
    else:
        raise SystemExit("no ImportError")
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=REPO)
    assert r.returncode == 0 and r.stdout.strip() == "fine", r.stderr


def test_counts_of_sequences_that_sit_out():
    layer = HypergraphAttention(64, 1, gather_mode=1, window=16)
    cache = GatherCache(2, 1, 64, pages=4, slots=32, page_size=16, device="cpu")
    for bad in ([1], [2, 0], [-1, 1]):
        with pytest.raises(ValueError, match="counts"):
            cache.decode(bf(2, 1, 64), counts=bad)
        with pytest.raises(ValueError, match="counts"):
            layer.decode(torch.zeros(2, 1, 64), cache, counts=bad)
    cache.host_lengths = [3, 0]
    for counts in (None, [1, 0], [4, 4]):
        with pytest.raises(ValueError, match="must be empty"):
            layer.prefill(torch.zeros(2, 4, 64), cache, counts=counts)
    with pytest.raises(ValueError, match="counts"):
        layer.prefill(torch.zeros(2, 4, 64), cache, counts=[0, 5])


def test_import_brings_no_tracer():
    """The package's layers import in milliseconds; torch's tracer takes seconds."""
    import subprocess
    import sys
    code = "import sys, torch; before = 'torch._dynamo' in sys.modules; import att3ntion; print(before, 'torch._dynamo' in sys.modules)"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=REPO)
    assert r.returncode == 0 and len(set(r.stdout.split())) == 1, (r.stdout, r.stderr)


def test_library_builds_without_torch():
    import subprocess
    import sys
    code = "import sys; sys.modules['torch'] = None; from att3ntion_b200 import build; print(build.build())"
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=REPO)
    assert r.returncode == 0 and r.stdout.strip().endswith("libatt3_b200.so") and "not built" in r.stderr, r.stderr

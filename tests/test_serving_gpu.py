"""Head norms with rotation, gather-cache append, single-token gather and eviction on the GPU against their definitions
in 64 bits.

Tolerances.  A rounding to BF16 is off by at most 2^-8 of the value.  The gather's result has one, and one of every
probability before the second product: |Y - Y64| <= 2^-8 |Y| + 2^-8 A with A = sum P |Vr o Vs|, both times 1 + 2^-8
for the order of the two.  What remains is FP32: a score is a sum of 2 D products of magnitude |q r s| / sqrt(D), a
relative error of the probabilities of at most 2 D 2^-24 sum|q r s| / sqrt(D) (1e-4 for the largest used here, and a
tensor core may cut where it would round, so twice that)."""
import pytest
import torch

from helpers import serving_ref as ref

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8                        # BF16


def rand(g, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=g).to(dtype)


def close(got, want, tol, what=""):
    d = (got.double().cpu() - want).abs()
    bad = d > tol
    assert not bad.any() and torch.isfinite(got).all(), f"{what}: off by {d.max():.3g}, {int(bad.sum())} of {bad.numel()} over, worst excess {(d - tol).max():.3g}"


# --------------------------------------------------------------------------- head norms with rotation

NORM_CASES = [
    # B, N, heads, D, rot, type, interleaved, heads_first
    (1, 1, (1,), 16, 8, torch.float32, False, False),
    (2, 5, (3, 1), 16, 16, torch.bfloat16, False, True),
    (2, 7, (4, 2, 2), 32, 16, torch.float16, True, False),
    (3, 33, (8, 1, 1), 64, 32, torch.bfloat16, False, False),
    (1, 129, (5, 5, 5), 64, 64, torch.float32, True, True),
    (2, 65, (8, 2, 2), 128, 128, torch.bfloat16, False, False),
    (1, 31, (6, 3, 1), 128, 48, torch.float32, False, True),
    (2, 40, (2, 2, 2, 2, 2), 128, 0, torch.bfloat16, False, False),
    (1, 1000, (9, 1, 1), 128, 64, torch.float16, True, True),
]


@pytest.mark.parametrize("B,N,heads,D,rot,dtype,interleaved,heads_first", NORM_CASES)
@pytest.mark.parametrize("scaled", ["all", "some"])
def test_norm_rotate_and_gradients(B, N, heads, D, rot, dtype, interleaved, heads_first, scaled):
    from att3ntion_b200 import norm_rotate, rotary_table
    g = torch.Generator().manual_seed(B * 1000 + N)
    eps = 1e-5
    table = rotary_table(N + 500, rot) if rot else None
    pos = torch.randint(0, N + 500, (B, N), generator=g)
    xs = [rand(g, B, N, h, D, dtype=dtype) * 2 for h in heads]
    ws = [None if scaled == "some" and k % 2 else 1 + 0.3 * torch.randn(D, generator=g) for k in range(len(heads))]
    dys = [rand(g, B, h, N, D) if heads_first else rand(g, B, N, h, D) for h in heads]
    leaves = [x.cuda().requires_grad_() for x in xs]
    scales = [None if w is None else w.cuda().requires_grad_() for w in ws]
    ys = norm_rotate(leaves, scales, table.cuda() if rot else None, pos.cuda(), eps=eps, interleaved=interleaved, heads_first=heads_first)
    torch.autograd.backward(ys, [d.cuda() for d in dys])
    for x, w, dy, y, leaf, scale in zip(xs, ws, dys, ys, leaves, scales):
        x64 = x.double().requires_grad_()
        w64 = None if w is None else w.double().requires_grad_()
        y64 = ref.norm_rotate(x64, w64, table.double() if rot else None, pos, eps, interleaved)
        shaped = y64.transpose(1, 2) if heads_first else y64
        # one rounding, and a dozen FP32 operations on values of the row's size
        slack = 2e-6 * y64.detach().abs().amax(-1, keepdim=True)
        close(y, shaped.detach(), HALF * shaped.detach().abs() + (slack.transpose(1, 2) if heads_first else slack), "y")
        shaped.backward(dy.double())
        half = torch.finfo(dtype).eps / 2
        close(leaf.grad, x64.grad, half * x64.grad.abs() + 4e-6 * x64.grad.abs().amax(-1, keepdim=True) + 1e-6 * (0 if w is None else 1), "dx")
        assert leaf.grad.dtype == dtype
        if w is not None:
            # B N heads terms, each with a few FP32 roundings, summed in two levels
            u = (x64 * (x64.pow(2).mean(-1, keepdim=True) + eps).rsqrt()).detach()
            terms = (dy.double().transpose(1, 2) if heads_first else dy.double()).abs().amax(-1, keepdim=True) * u.abs()
            close(scale.grad, w64.grad, 3e-6 * terms.sum((0, 1, 2)) + 1e-7, "dw")


@pytest.mark.parametrize("make", ["sliced", "transposed", "expanded", "odd offset", "columns apart"])
def test_norm_rotate_takes_any_strides(make):
    from att3ntion_b200 import norm_rotate, rotary_table
    g = torch.Generator().manual_seed(5)
    B, N, H, D = 2, 19, 3, 64
    if make == "sliced":                                 # the heads of a joint projection
        x = rand(g, B, N, H + 4, D).cuda()[:, :, 2:2 + H]
    elif make == "transposed":
        x = rand(g, B, H, N, D).cuda().transpose(1, 2)
    elif make == "expanded":
        x = rand(g, B, 1, H, D).cuda().expand(B, N, H, D)
    elif make == "odd offset":
        x = rand(g, B * N * H * D + 1).cuda()[1:].view(B, N, H, D)
    else:
        x = rand(g, B, N, H, D * 2).cuda()[..., ::2]
    w, table = (1 + torch.rand(D + 1, generator=g)).cuda()[1:], rotary_table(N, 32).cuda()
    x = x.detach().requires_grad_()
    y = norm_rotate(x, w, table)
    want = norm_rotate(x.detach().contiguous().clone(), w.clone(), table)
    assert torch.equal(y, want)
    dy = rand(g, B, H, N, D).cuda().transpose(1, 2)
    (dx,) = torch.autograd.grad(y, x, dy)
    x2 = x.detach().contiguous().clone().requires_grad_()
    (dx2,) = torch.autograd.grad(norm_rotate(x2, w.clone(), table), x2, dy.contiguous())
    assert torch.equal(dx, dx2)


def test_norm_rotate_empty_and_repeatable():
    from att3ntion_b200 import norm_rotate
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.empty(2, 0, 3, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    y = norm_rotate(x, w)
    assert y.shape == x.shape
    gx, gw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
    assert gx.shape == x.shape and not gw.any()
    x = torch.randn(3, 700, 5, 64, device="cuda", requires_grad=True)
    dy = torch.randn(3, 700, 5, 64, device="cuda").bfloat16()
    first = torch.autograd.grad(norm_rotate(x, w), [x, w], dy)
    for _ in range(3):
        for a, b in zip(first, torch.autograd.grad(norm_rotate(x, w), [x, w], dy)):
            assert torch.equal(a, b)


def test_norm_rotate_reports_a_position_outside_its_table():
    from att3ntion_b200 import _cuda_kernels as ck, norm_rotate, rotary_table
    x = torch.randn(1, 4, 2, 64, device="cuda")
    table = rotary_table(8, 64).cuda()
    pos = torch.tensor([0, 7, 3, 1], device="cuda")
    norm_rotate(x, None, table, pos)
    ck.device_status()
    for bad in (8, -1, 1 << 40):
        got = norm_rotate(x, None, table, torch.tensor([0, bad, 3, 1], device="cuda"))
        with pytest.raises(RuntimeError, match="position"):
            ck.device_status()
        assert torch.isfinite(got).all()
        ck.device_status()                               # reported once


# --------------------------------------------------------------------------- a cache to work on

class Made:
    """Pools with random rows, pages handed out in random order, -1 in the entries behind each sequence's last page."""

    def __init__(self, seed, lengths, Hkv, D, page, room=0, scale=1.0):
        g = self.g = torch.Generator().manual_seed(seed)
        self.B, self.page = len(lengths), page
        need = [-(-(n + room) // page) for n in lengths]
        total = sum(need) + 2
        order = torch.randperm(total, generator=g).int()
        self.table = torch.full((self.B, max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = order[at: at + k]
            at += k
        self.free = order[at:]
        self.pools = [rand(g, total, page, Hkv, D) * scale for _ in range(4)]
        self.mass = torch.rand(total, page, Hkv, generator=g)
        self.lengths = torch.tensor(lengths, dtype=torch.int32)

    def gpu(self):
        return [p.cuda() for p in self.pools], self.table.cuda(), self.lengths.cuda()


# --------------------------------------------------------------------------- append

@pytest.mark.parametrize("B,T,Hq,Hkv,D,page,dtype,interleaved", [
    (1, 1, 1, 1, 16, 1, torch.float32, False),
    (3, 1, 8, 1, 128, 16, torch.bfloat16, False),
    (4, 37, 6, 2, 64, 7, torch.float16, True),
    (2, 130, 4, 4, 128, 64, torch.float32, False),
])
@pytest.mark.parametrize("normed", [True, False])
def test_append(B, T, Hq, Hkv, D, page, dtype, interleaved, normed):
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_append, rotary_table
    g = torch.Generator().manual_seed(T + page)
    have = [int(torch.randint(0, 3 * page, (1,), generator=g)) for _ in range(B)]
    c = Made(1, have, Hkv, D, page, room=T)
    pools, table, lengths = c.gpu()
    mass = c.mass.cuda()
    new = [rand(g, B, T, Hkv, D, dtype=dtype) for _ in range(4)]
    Q = rand(g, B, T, Hq, D, dtype=dtype)
    counts = torch.randint(0, T + 1, (B,), generator=g).int()
    counts[0] = T
    start = torch.randint(0, 300, (B,), generator=g).int()
    ws = [1 + 0.3 * torch.randn(D, generator=g) for _ in range(3)] if normed else None
    rot = rotary_table(300 + T, D // 2) if normed else None
    out = gather_cache_append(pools, table, lengths, *[x.cuda() for x in new], counts=counts.cuda(), Q=Q.cuda(),
                              weights=None if ws is None else [w.cuda() for w in ws], table=None if rot is None else rot.cuda(),
                              positions=start.cuda(), mass=mass, interleaved=interleaved)
    ck.device_status()
    pos = start.long()[:, None] + torch.arange(T)
    want = [p.double() for p in c.pools]
    rows = [x.double() for x in new]
    q64 = Q.double()
    if normed:
        t64 = rot.double()
        q64 = ref.norm_rotate(q64, ws[0].double(), t64, pos, 1e-6, interleaved)
        rows[0] = ref.norm_rotate(rows[0], ws[1].double(), t64, pos, 1e-6, interleaved)
        rows[1] = ref.norm_rotate(rows[1], ws[2].double(), t64, pos, 1e-6, interleaved)
    wmass = c.mass.clone()
    for b in range(B):
        for t in range(int(counts[b])):
            e = have[b] + t
            at = (int(c.table[b, e // page]), e % page)
            for w, r in zip(want, rows):
                w[at] = r[b, t]
            wmass[at] = 0
    close(out, q64, HALF * q64.abs() + 1e-5, "Q")
    for k, (p, w) in enumerate(zip(pools, want)):
        close(p, w, HALF * w.abs() + (1e-5 if normed and k < 2 else 0), f"pool {k}")
    assert torch.equal(mass.cpu(), wmass) and torch.equal(lengths.cpu(), c.lengths)


def test_append_leaves_out_what_has_no_page():
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_append
    c = Made(2, [3, 30], 1, 64, 16, room=2)
    c.table[0, 0] = 999                                  # a page that the pool does not have
    c.lengths[1] = 47                                    # the second of two new slots lies behind the table's end
    pools, table, lengths = c.gpu()
    new = [torch.randn(2, 2, 1, 64, device="cuda") for _ in range(4)]
    gather_cache_append(pools, table, lengths, *new)
    with pytest.raises(RuntimeError, match="page"):
        ck.device_status()
    for p, old, x in zip(pools, c.pools, new):
        want = old.cuda()
        if table.shape[1] > 2:
            want[int(c.table[1, 2]), 15] = x[1, 0].bfloat16()
        assert torch.equal(p, want)


# --------------------------------------------------------------------------- the gather of one new token

DECODE_CASES = [
    # lengths, Hq, Hkv, D, page, window, sinks
    ([1], 1, 1, 128, 16, 0, 0),
    ([0, 1, 2, 0], 4, 2, 64, 16, 0, 0),
    ([128], 8, 1, 128, 16, 128, 0),
    ([5, 200, 127, 128, 129], 8, 1, 128, 16, 128, 0),
    ([300, 17, 132, 131, 133], 8, 2, 128, 32, 128, 4),
    ([31, 32, 33, 64, 65, 96, 97], 3, 1, 128, 7, 0, 0),
    ([700, 1, 259], 2, 2, 128, 64, 0, 0),
    ([1000], 1, 1, 64, 128, 0, 0),
    ([513, 40], 6, 3, 64, 1, 0, 0),
    ([77, 900, 16], 16, 1, 128, 16, 16, 0),
    ([77, 900, 16], 8, 8, 64, 16, 1, 3),
    ([600, 256], 4, 1, 128, 256, 300, 37),
    ([50] * 40, 8, 4, 128, 16, 33, 1),
    # at most 128 visible slots, heads in blocks of 8, 4, 2 and 1
    ([40, 3, 128, 97, 0, 31], 15, 1, 64, 16, 100, 7),
    ([20, 1, 16], 22, 2, 128, 32, 0, 0),
    # at most 192 visible slots: one step of keys a tile
    ([192, 191, 129, 160, 161, 5, 0], 8, 2, 128, 32, 0, 0),
    ([1000, 193, 192, 150, 40], 3, 1, 128, 16, 150, 42),
    ([500, 133, 700], 8, 8, 64, 16, 128, 5),
    ([140] * 30, 16, 1, 64, 64, 130, 2),
]


@pytest.mark.parametrize("lengths,Hq,Hkv,D,page,window,sinks", DECODE_CASES)
@pytest.mark.parametrize("with_mass", [False, True])
def test_decode(lengths, Hq, Hkv, D, page, window, sinks, with_mass):
    from att3ntion_b200 import _cuda_kernels as ck, single_gather_decode
    c = Made(3, lengths, Hkv, D, page)
    Q = rand(c.g, c.B, Hq, D)
    Y64, A, share = ref.decode(Q, c.pools, c.table, lengths, window, sinks)
    pools, table, dev_lengths = c.gpu()
    mass = c.mass.cuda() if with_mass else None
    Y = single_gather_decode(Q.cuda(), pools, table, dev_lengths, window=window, sinks=sinks, mass=mass)
    ck.device_status()
    close(Y, Y64, (1 + HALF) * HALF * (Y64.abs() + A) + 2e-4 * A, "Y")
    if with_mass:
        want = c.mass.double()
        for at, v in share.items():
            want[at] += v
        # FP32 sums and exponentials, and the old value's rounding
        close(mass, want, 2.0 ** -24 * want + 2e-5 * (want - c.mass.double()), "mass")
        untouched = want == c.mass.double()
        assert torch.equal(mass.cpu()[untouched], c.mass[untouched])


@pytest.mark.parametrize("scale", [1e-3, 4.0])
def test_decode_small_and_large_scores(scale):
    """Scores from 1e-9 to hundreds: the softmax is flat, or one pair takes everything."""
    from att3ntion_b200 import single_gather_decode
    lengths = [300, 70]
    c = Made(4, lengths, 1, 128, 16, scale=scale)
    Q = rand(c.g, 2, 4, 128) * scale
    Y64, A, _ = ref.decode(Q, c.pools, c.table, lengths)
    pools, table, n = c.gpu()
    Y = single_gather_decode(Q.cuda(), pools, table, n)
    # sum |q r s| / sqrt(D) is 64 times larger at scale 4
    close(Y, Y64, (1 + HALF) * HALF * (Y64.abs() + A) + 2e-4 * max(1.0, scale ** 3) * A, "Y")


def test_decode_never_reads_behind_the_lengths():
    """NaN and infinity in every slot that is not visible, in spare pages too."""
    from att3ntion_b200 import single_gather_decode
    lengths, page, window, sinks = [150, 20, 77], 16, 60, 5
    c = Made(6, lengths, 2, 64, page)
    Q = rand(c.g, 3, 4, 64)
    pools, table, n = c.gpu()
    want = single_gather_decode(Q.cuda(), pools, table, n, window=window, sinks=sinks)
    seen = torch.zeros(c.pools[0].shape[:2], dtype=torch.bool)
    for b, length in enumerate(lengths):
        for e in ref.visible(length, window, sinks):
            seen[int(c.table[b, e // page]), e % page] = True
    for k, p in enumerate(pools):
        p[~seen.cuda()] = float("nan") if k % 2 else float("inf")
    got = single_gather_decode(Q.cuda(), pools, table, n, window=window, sinks=sinks)
    assert torch.isfinite(want).all() and torch.equal(got, want)


def test_decode_does_not_depend_on_the_batch_around_it():
    """A sequence's result alone and in a batch differs by the order of FP32 sums at most."""
    from att3ntion_b200 import single_gather_decode
    lengths = [400, 1, 260, 33, 900, 0, 128]
    c = Made(7, lengths, 2, 128, 16)
    Q = rand(c.g, c.B, 8, 128).cuda()
    pools, table, n = c.gpu()
    Y = single_gather_decode(Q, pools, table, n)
    for b in range(c.B):
        one = single_gather_decode(Q[b: b + 1], pools, table[b: b + 1], n[b: b + 1])
        # both round an FP32 sum to BF16 once; P's rounding moves with the strip's reference: compare as two estimates
        _, A, _ = ref.decode(Q[b: b + 1].cpu(), c.pools, c.table[b: b + 1], lengths[b: b + 1])
        close(one, Y[b: b + 1].double().cpu(), 2 * ((1 + HALF) * HALF * (Y[b: b + 1].double().cpu().abs() + A) + 2e-4 * A))
    again = single_gather_decode(Q, pools, table, n)
    assert torch.equal(Y, again)


def test_decode_reports_bad_tables():
    from att3ntion_b200 import _cuda_kernels as ck, single_gather_decode
    c = Made(8, [100, 40], 1, 128, 16)
    Q = rand(c.g, 2, 4, 128).cuda()
    pools, table, n = c.gpu()
    want = single_gather_decode(Q, pools, table, n)
    ck.device_status()
    bad = table.clone()
    bad[0, 3] = 10 ** 6
    got = single_gather_decode(Q, pools, bad, n)
    with pytest.raises(RuntimeError, match="page"):
        ck.device_status()
    assert torch.equal(got[1], want[1])
    for length in (-5, 10 ** 6):
        m = n.clone()
        m[0] = length
        got = single_gather_decode(Q, pools, torch.where(table < 0, torch.zeros_like(table), table), m)
        with pytest.raises(RuntimeError, match="length"):
            ck.device_status()
        assert torch.equal(got[1], want[1])
    assert not single_gather_decode(Q, pools, table, torch.zeros_like(n)).any()
    ck.device_status()


# --------------------------------------------------------------------------- eviction

@pytest.mark.parametrize("lengths,Hkv,D,page,keep,sinks,recent", [
    ([1], 1, 64, 16, 1, 0, 0),
    ([0, 5, 100], 2, 128, 16, 40, 4, 10),
    ([333, 334, 332], 3, 64, 7, 333, 0, 333),
    ([700, 2, 699], 1, 16, 64, 100, 50, 50),
    ([1500], 2, 128, 128, 1499, 1, 1),
    ([3000, 2100, 1025], 1, 32, 32, 1024, 4, 500),
])
@pytest.mark.parametrize("masses", ["random", "ties", "odd values"])
@pytest.mark.parametrize("where", ["in place", "fresh pages", "copy of the table"])
def test_evict(lengths, Hkv, D, page, keep, sinks, recent, masses, where):
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_evict
    c = Made(9, lengths, Hkv, D, page)
    if masses == "ties":
        c.mass = (c.mass * 4).floor()
    elif masses == "odd values":
        odd = torch.tensor([0.0, -0.0, -1.0, float("inf"), -float("inf"), float("nan"), 1e-42, 3.0])
        c.mass = odd[(c.mass * 8).long()]
    slots = ref.evict(c.mass, c.table, lengths, keep, sinks, recent)
    out = c.table
    if where == "fresh pages":
        per = -(-min(keep, c.table.shape[1] * page) // page)
        base = c.pools[0].shape[0]
        out = (base + torch.randperm(c.B * per, generator=c.g)).int().view(c.B, per)
        c.pools = [torch.cat([p, rand(c.g, c.B * per, *p.shape[1:])]) for p in c.pools]
        c.mass = torch.cat([c.mass, torch.rand(c.B * per, page, Hkv, generator=c.g)])
    want, wmass = [p.clone() for p in c.pools], c.mass.clone()
    for b in range(c.B):
        for h in range(Hkv):
            for r, e in enumerate(slots[b][h]):
                to, frm = (int(out[b, r // page]), r % page, h), (int(c.table[b, e // page]), e % page, h)
                for w, p in zip(want, c.pools):
                    w[to] = p[frm]
                wmass[to] = c.mass[frm]
    pools, table, n = c.gpu()
    mass = c.mass.cuda()
    to = None if where == "in place" else out.cuda() if where == "fresh pages" else table.clone()
    kept, left = gather_cache_evict(pools, mass, table, n, keep, sinks=sinks, recent=recent, out_table=to)
    ck.device_status()
    assert left.tolist() == [min(k, keep) for k in lengths]
    for b in range(c.B):
        for h in range(Hkv):
            assert kept[b, h].tolist() == slots[b][h] + [-1] * (keep - len(slots[b][h]))
    for p, w in zip(pools, want):
        assert torch.equal(p.cpu(), w)
    assert torch.equal(mass.cpu().view(torch.int32), wmass.view(torch.int32))


def test_evict_long_sequence_reads_the_mass_again():
    """More slots than the keys' shared memory holds."""
    from att3ntion_b200 import gather_cache_evict
    n, keep, page = 60001, 777, 128
    c = Made(10, [n], 1, 16, page)
    c.mass = (c.mass * 1000).floor()
    pools, table, length = c.gpu()
    kept, left = gather_cache_evict(pools, c.mass.cuda(), table, length, keep, sinks=3, recent=7)
    m = ref.rows_of(c.mass, c.table, 0, list(range(n)))[:, 0].double()
    m[:3] = m[n - 7:] = float("inf")
    want = m.sort(descending=True, stable=True).indices[:keep].sort().values
    assert torch.equal(kept[0, 0].long().cpu(), want) and left.item() == keep


# --------------------------------------------------------------------------- streams, graphs, together

def test_other_stream_and_device_guard():
    from att3ntion_b200 import norm_rotate, single_gather_decode
    c = Made(11, [500, 300], 1, 128, 16)
    Q = rand(c.g, 2, 8, 128).cuda()
    pools, table, n = c.gpu()
    x = torch.randn(2, 300, 4, 64, device="cuda")
    want = single_gather_decode(Q, pools, table, n), norm_rotate(x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append((single_gather_decode(Q, pools, table, n), norm_rotate(x)))
    torch.cuda.synchronize()
    for y, z in got:
        assert torch.equal(y, want[0]) and torch.equal(z, want[1])


def test_captured_step_follows_the_lengths():
    """Append and decode captured once, replayed while the sequences grow, two graphs in turn."""
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_append, rotary_table, single_gather_decode
    B, Hq, Hkv, D, page = 2, 4, 1, 64, 16
    c = Made(12, [10, 120], Hkv, D, page, room=40)
    pools, table, n = c.gpu()
    twin = [p.clone() for p in pools]
    rot = rotary_table(200, D).cuda()
    w = [torch.ones(D, device="cuda")] * 3
    new = [torch.randn(B, 1, Hkv, D, device="cuda") for _ in range(4)]
    Q = torch.randn(B, 1, Hq, D, device="cuda")
    one = torch.ones(B, dtype=torch.int32, device="cuda")

    def step(ps, lengths):
        q = gather_cache_append(ps, table, lengths, *new, Q=Q, weights=w, table=rot)
        lengths.add_(one)
        return single_gather_decode(q[:, 0], ps, table, lengths, window=64, sinks=2)

    m = n.clone()
    step([p.clone() for p in pools], n.clone())                        # warm-up outside the capture
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = step(pools, n)
        graphs.append((gr, y))
    for k in range(24):
        for x in (*new, Q):
            x.normal_()
        gr, y = graphs[k % 2]
        gr.replay()
        want = step(twin, m)
        assert torch.equal(y, want) and torch.equal(n, m)
    for p, t in zip(pools, twin):
        assert torch.equal(p, t)
    ck.device_status()


def test_captured_on_two_streams_that_fork_and_join():
    """Each kernel follows the ones that it reads from, whichever stream and kind of work they came from."""
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_append, norm_rotate, rotary_table, single_gather_decode
    B, Hq, Hkv, D, page = 3, 4, 2, 64, 16
    c = Made(21, [10, 120, 63], Hkv, D, page, room=40)
    pools, table, n = c.gpu()
    rot = rotary_table(200, D).cuda()
    w = torch.rand(D, device="cuda")
    new = [torch.randn(B, 1, Hkv, D, device="cuda") for _ in range(4)]
    Q = torch.randn(B, 1, Hq, D, device="cuda")
    big = torch.randn(1 << 22, device="cuda")
    side = torch.cuda.Stream()

    def step(ps, lengths):
        here = torch.cuda.current_stream()
        side.wait_stream(here)
        with torch.cuda.stream(side):
            q = norm_rotate(Q * (1 + big.sum().tanh()), weights=w, table=rot, positions=lengths[:, None])
        gather_cache_append(ps, table, lengths, *new, weights=[None, w, w], table=rot)
        seen = lengths + 1
        here.wait_stream(side)
        y = single_gather_decode(q[:, 0], ps, table, seen, window=64)
        return y, norm_rotate(y[:, None], weights=w)

    twin = [p.clone() for p in pools]
    want = step([p.clone() for p in pools], n)                         # warm-up outside the capture
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        got = step(pools, n)
    for _ in range(5):
        for x in (*new, Q, big):
            x.normal_()
        n.add_(1)
        want = step(twin, n)
        torch.cuda.synchronize()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(pools, twin))
    ck.device_status()


def test_pages_past_32_bits_of_a_pool():
    """The same rows on pages that begin 2^31 elements (2^32 bytes) into the pools give the same bits."""
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_append, gather_cache_evict, rotary_table, single_gather_decode
    Hkv, D, page = 8, 128, 64
    c = Made(23, [300, 45], Hkv, D, page, room=1)
    near, table, n = c.gpu()
    count, skip = near[0].shape[0], (1 << 31) // (page * Hkv * D)
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 18 GB")
    far = [torch.empty(skip + count, page, Hkv, D, dtype=torch.bfloat16, device="cuda") for _ in near]
    for f, x in zip(far, near):
        f[skip:] = x
    moved = torch.where(table < 0, table, table + skip)
    masses = [c.mass.cuda(), torch.zeros(skip + count, page, Hkv, device="cuda")]
    masses[1][skip:] = masses[0]
    new = [torch.randn(2, 1, Hkv, D, device="cuda") for _ in range(4)]
    Q = torch.randn(2, 8, D, device="cuda", dtype=torch.bfloat16)
    rot = rotary_table(400, D).cuda()
    got = []
    for pools, pages, mass in ((near, table, masses[0]), (far, moved, masses[1])):
        gather_cache_append(pools, pages, n, *new, table=rot, mass=mass)
        seen = n + 1
        out = [single_gather_decode(Q, pools, pages, seen, mass=mass), single_gather_decode(Q, pools, pages, seen, window=100, sinks=2)]
        out += [single_gather_decode(Q, pools, pages, seen)]
        out += gather_cache_evict(pools, mass, pages, seen, 90, sinks=2, recent=10)
        got.append(out + [p[-count:] for p in pools] + [mass[-count:]])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    ck.device_status()


def test_tables_that_are_part_of_a_larger_one():
    """Page tables and lengths as slices of a server's own."""
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_append, gather_cache_evict, single_gather_decode
    c = Made(13, [100, 37, 64], 1, 64, 16, room=8)
    pools, table, n = c.gpu()
    wide = torch.full((5, table.shape[1] + 9), -7, dtype=torch.int32, device="cuda")
    wide[1:4, 4: 4 + table.shape[1]] = table
    part = wide[1:4, 4: 4 + table.shape[1]]
    twin = [p.clone() for p in pools]
    mass, twin_mass = c.mass.cuda(), c.mass.cuda()
    new = [rand(c.g, 3, 2, 1, 64).cuda() for _ in range(4)]
    Q = rand(c.g, 3, 3, 64).cuda()
    results = []
    for ps, m, t in ((pools, mass, part), (twin, twin_mass, table)):
        gather_cache_append(ps, t, n, *new, mass=m)
        y = single_gather_decode(Q, ps, t, n + 2, window=50, sinks=1, mass=m)
        kept, left = gather_cache_evict(ps, m, t, n + 2, 40, sinks=1, recent=3)
        results.append((y, kept, left, m, *ps))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    ck.device_status()


def test_queries_behind_a_count_need_no_angles():
    """A padded batch at the end of the angle table: the padding's positions lie behind it."""
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_append, rotary_table
    for Hkv, Hq in ((1, 1), (2, 4)):
        c = Made(14, [60, 10], Hkv, 64, 16, room=8)
        pools, table, n = c.gpu()
        rot = rotary_table(64, 64).cuda()
        new = [torch.randn(2, 8, Hkv, 64, device="cuda") for _ in range(4)]
        Q = torch.randn(2, 8, Hq, 64, device="cuda")
        counts = torch.tensor([4, 8], dtype=torch.int32, device="cuda")
        q = gather_cache_append(pools, table, n, *new, counts=counts, Q=Q, table=rot)
        ck.device_status()
        assert torch.isfinite(q).all()
        gather_cache_append(pools, table, n, *new, counts=counts + torch.tensor([1, 0], dtype=torch.int32, device="cuda"), Q=Q, table=rot)
        with pytest.raises(RuntimeError, match="position"):
            ck.device_status()


def test_empty_batches():
    from att3ntion_b200 import gather_cache_append, gather_cache_evict, single_gather_decode
    pools = [torch.zeros(2, 16, 1, 64, device="cuda", dtype=torch.bfloat16) for _ in range(4)]
    table, n = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    new = [torch.zeros(0, 4, 1, 64, device="cuda") for _ in range(4)]
    assert gather_cache_append(pools, table, n, *new) is None
    assert gather_cache_append(pools, table, n, *new, Q=torch.zeros(0, 4, 2, 64, device="cuda")).shape == (0, 4, 2, 64)
    assert single_gather_decode(torch.zeros(0, 2, 64, device="cuda"), pools, table, n).shape == (0, 2, 64)
    kept, left = gather_cache_evict(pools, torch.zeros(2, 16, 1, device="cuda"), table, n, 5)
    assert kept.shape == (0, 1, 5) and left.shape == (0,)
    table, n = torch.zeros(3, 1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda")
    new = [torch.zeros(3, 0, 1, 64, device="cuda") for _ in range(4)]
    assert gather_cache_append(pools, table, n, *new, Q=torch.zeros(3, 0, 2, 64, device="cuda")).shape == (3, 0, 2, 64)


def test_norm_rotate_captured_with_its_backward():
    """Forward and backward captured, replayed on new inputs; a capture beside a live eager graph of the same leaves is
    refused where it can still be refused."""
    from att3ntion_b200 import norm_rotate, rotary_table
    x = torch.randn(2, 33, 3, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda", requires_grad=True)
    dy = torch.randn(2, 33, 3, 64, device="cuda").bfloat16()
    table = rotary_table(40, 32).cuda()

    def step():
        y = norm_rotate(x, w, table)
        return (y, *torch.autograd.grad(y, [x, w], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            x.normal_()
            dy.normal_()
        graph.replay()
        got_now = [t.detach().clone() for t in got]
        want = step()
        for a, b in zip(got_now, want):
            assert torch.equal(a, b)
        del want
    del got                                # it kept the leaves' accumulators of the capture's stream
    alive = norm_rotate(x, w, table)
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside the capture"):
        with torch.cuda.graph(other):
            step()
    assert torch.isfinite(alive).all()
    torch.cuda.synchronize()


def test_norm_rotate_gradients_have_no_gradients():
    from att3ntion_b200 import norm_rotate
    x = torch.randn(1, 2, 1, 64, device="cuda", requires_grad=True)
    y = norm_rotate(x, torch.ones(64, device="cuda"))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.float().sum(), x, create_graph=True)


# --------------------------------------------------------------------------- the layer

@pytest.mark.parametrize("kw", [dict(window=128, qk_norm=True, rotary_base=10000.0), dict(window=16, qk_norm=True),
                                dict(window=33, rotary_base=500.0, sinks=3), dict(window=200, qk_norm=True, rotary_base=1e4),
                                dict(window=64)])
@pytest.mark.parametrize("head_dim,dtype", [(64, torch.float32), (128, torch.bfloat16)])
def test_layer_prefill_and_decode_follow_its_forward(kw, head_dim, dtype):
    """Prompts of different lengths, then tokens one by one, against the forward pass over the whole sequences.  The two
    round at different places, so they are held to the gate that the forward itself is held to (relative 0.03 in the
    2-norm; the forward rounds Q o R, the decode does not)."""
    from att3ntion_b200 import GatherCache, HypergraphAttention
    torch.manual_seed(3)
    B, N, H = 3, 150, 2
    layer = HypergraphAttention(H * head_dim, H, gather_mode=1, **kw).cuda().to(dtype)
    x = torch.randn(B, N, H * head_dim, device="cuda", dtype=dtype)
    with torch.no_grad():
        want = layer(x)
    prompts = [140, 1, 97]
    cache = GatherCache(B, H, head_dim, pages=40, slots=N, page_size=16)
    y = layer.prefill(x[:, :140], cache, counts=prompts)
    base = layer.Wo.bias.detach().double()
    # The layer's results hold the output bias too and are rounded with it: each by half a step of its type, relative to
    # the whole value.  With the bias an order of magnitude above the rest (0.06 against 0.002 here) that is no part of
    # the 0.03 above but comes on top, once for either side.
    half_step = torch.finfo(dtype).eps / 2

    def near(a, b):
        a, b = a.detach().double(), b.detach().double()
        tol = 0.03 * (b - base).norm() + half_step * (a.norm() + b.norm())
        assert torch.isfinite(a).all() and (a - b).norm() <= tol, (float((a - b).norm()), float(tol))
    for b, n in enumerate(prompts):
        near(y[b, :n], want[b, :n])
    for _ in range(10):
        at = cache.host_lengths
        step = torch.stack([x[b, at[b]] for b in range(B)])[:, None]
        where = list(at)
        y = layer.decode(step, cache)
        for b in range(B):
            near(y[b, 0], want[b, where[b]])
    assert cache.lengths.tolist() == cache.host_lengths == [n + 10 for n in prompts]


def test_layer_trains_with_norms_and_rotation():
    """Gradients of the extended layer against central differences of its own loss in the direction of the gradient."""
    from att3ntion_b200 import HypergraphAttention
    torch.manual_seed(4)
    for mode, window in ((1, 16), (1, 0), (0, 0)):
        layer = HypergraphAttention(64, 1, gather_mode=mode, window=window, qk_norm=True, rotary_base=100.0).cuda()
        x = torch.randn(1, 32, 64, device="cuda")
        dy = torch.randn(1, 32, 64, device="cuda")
        layer(x).backward(dy)
        for name in ("q_norm", "r_norm", "s_norm", "Wq.weight", "Ws.weight"):
            p = dict(layer.named_parameters())[name]
            assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.norm() > 0, name
            # The loss is a sum of N D terms of BF16 results: 2^-9 rms each, so 2^-9 |dy o y| in all; a step that moves the
            # loss by 30 times that leaves the difference quotient good to a tenth.
            with torch.no_grad():
                direction = p.grad / p.grad.norm()
                noise = float((dy * layer(x)).norm()) * 2.0 ** -9
                h = max(0.05, 30 * noise / float(p.grad.norm()))
                if h > 0.3 * float(p.norm()):
                    continue                                    # a gradient too small to be seen through the rounding
                p.add_(direction, alpha=h)
                up = float((layer(x).double() * dy.double()).sum())
                p.add_(direction, alpha=-2 * h)
                down = float((layer(x).double() * dy.double()).sum())
                p.add_(direction, alpha=h)
            assert abs((up - down) / (2 * h) - float(p.grad.norm())) <= 0.25 * float(p.grad.norm()), (mode, name)


def test_cache_run_append_decode_evict_decode():
    """A cache that tracks masses through steps, an eviction and further steps, against the definitions in 64 bits."""
    from att3ntion_b200 import GatherCache, rotary_table
    g = torch.Generator().manual_seed(21)
    B, Hq, Hkv, D, page = 2, 4, 2, 64, 8
    cache = GatherCache(B, Hkv, D, pages=24, slots=80, page_size=page, track_mass=True)
    table = rotary_table(200, D)
    ws = [1 + 0.2 * torch.randn(D, generator=g) for _ in range(3)]
    kept_rows = [[[[] for _ in range(4)] for _ in range(Hkv)] for _ in range(B)]     # what each head's slots must hold
    share = [[[] for _ in range(Hkv)] for _ in range(B)]
    seen = [0, 0]

    def step(T, counts):
        new = [rand(g, B, T, Hkv, D) for _ in range(4)]
        q = rand(g, B, T, Hq, D)
        got = cache.append(*[t.cuda() for t in new], counts=counts, Q=q.cuda(), weights=[w.cuda() for w in ws], table=table.cuda())
        for b in range(B):
            for t in range(T if counts is None else counts[b]):
                pos = torch.tensor([[seen[b]]])
                rows = [x[b: b + 1, t: t + 1].double() for x in new]
                for k in (0, 1):
                    rows[k] = ref.norm_rotate(rows[k], ws[k + 1].double(), table.double(), pos, 1e-6, False)
                for h in range(Hkv):
                    for k in range(4):
                        kept_rows[b][h][k].append(rows[k][0, 0, h])
                    share[b][h].append(0.0)
                seen[b] += 1
        return got

    def check(q):
        y = cache.decode(q)
        for b in range(B):
            for h in range(Hq):
                k = h // (Hq // Hkv)
                R, S, Vr, Vs = (torch.stack(t) for t in kept_rows[b][k])
                x = (q[b, h].double().cpu() * R) @ S.T / 8.0
                p = torch.softmax(x.flatten(), 0).view_as(x)
                Y, A = ((p @ Vs) * Vr).sum(0), ((p @ Vs.abs()) * Vr.abs()).sum(0)
                # R and S were rounded to BF16 on the way in: each factor of a score by 2^-8 at most, so a score by 2^-7 of
                # its sum of magnitudes, and the probabilities by twice that
                slack = 2.0 ** -7 * float(((q[b, h].double().cpu().abs() * R.abs()) @ S.abs().T / 8.0).max()) * 2
                assert ((y[b, h].double().cpu() - Y).abs() <= 3 * HALF * (Y.abs() + A) + slack * A).all()
                part = (p.sum(0) + p.sum(1)) / (2 * (Hq // Hkv))
                share[b][k] = [a + float(v) for a, v in zip(share[b][k], part)]

    step(30, [30, 17])
    for _ in range(4):
        check(step(1, None)[:, 0])
    kept = cache.evict(20, sinks=2, recent=5)
    assert cache.lengths.tolist() == cache.host_lengths == [20, 20] and cache.positions.tolist() == seen == [34, 21]
    for b in range(B):
        for h in range(Hkv):
            slots = kept[b, h].tolist()
            assert slots == sorted(set(slots)) and slots[:2] == [0, 1] and slots[-5:] == list(range(seen[b] - 5, seen[b]))
            # what left had no more mass than what stayed (up to the rounding of R and S)
            out = [share[b][h][e] for e in range(seen[b]) if e not in slots]
            mid = [share[b][h][e] for e in slots[2:-5]]
            assert max(out) <= min(mid) * 1.2
            kept_rows[b][h] = [[t[e] for e in slots] for t in kept_rows[b][h]]
            share[b][h] = [share[b][h][e] for e in slots]
    assert len(cache._free) == 24 - 2 * 3
    for _ in range(6):
        check(step(1, None)[:, 0])
    cache.clear(0)
    assert cache.lengths.tolist() == [0, 26] and len(cache._free) == 24 - 4


# --------------------------------------------------------------------------- what the calls above left out

@pytest.mark.parametrize("page", [64, 128, 384])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_whole_boxes_many_times_round_the_ring(page, D):
    """Pages whose boxes leave copy warps without work, stretches of many key steps, repeated: same bits, no wait given up."""
    from att3ntion_b200 import _cuda_kernels as ck, single_gather_decode
    lengths = [4000, 129, 2560]
    c = Made(31, lengths, 2, D, page)
    Q = rand(c.g, 3, 4, D)
    pools, table, n = c.gpu()
    q = Q.cuda()
    first = single_gather_decode(q, pools, table, n)
    for _ in range(50):
        assert torch.equal(single_gather_decode(q, pools, table, n), first)
    ck.device_status()
    Y64, A, _ = ref.decode(Q[1:2], c.pools, c.table[1:2], lengths[1:2])
    close(first[1:2], Y64, (1 + HALF) * HALF * (Y64.abs() + A) + 2e-4 * A, "Y")


def test_evict_that_keeps_everything():
    """keep = 2^31 - 1, "all of them": the places behind the last slot are -1 up to the end."""
    from att3ntion_b200 import _cuda_kernels as ck, gather_cache_evict
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 12 GB")
    c = Made(32, [100], 1, 16, 16)
    pools, table, n = c.gpu()
    kept, left = gather_cache_evict(pools, c.mass.cuda(), table, n, 2 ** 31 - 1, sinks=1, recent=2)
    ck.device_status()
    assert kept.shape == (1, 1, 2 ** 31 - 1) and left.tolist() == [100]
    assert kept[0, 0, :100].tolist() == list(range(100))
    assert all(bool((kept[0, 0, a: a + (1 << 28)] == -1).all()) for a in range(100, 2 ** 31 - 1, 1 << 28))
    for p, old in zip(pools, c.pools):
        assert torch.equal(p.cpu(), old)


@pytest.mark.parametrize("eps", [0.0, 1e-60])
@pytest.mark.parametrize("N,heads,D,dtype", [(5, (3, 1), 64, torch.float32), (17, (1,), 128, torch.bfloat16), (1, (5, 8), 16, torch.float16)])
def test_norm_rotate_gradients_without_eps(N, heads, D, dtype, eps):
    """eps = 0, or one that is 0 in FP32, on rows that are nowhere zero; numbers of rows that leave groups of rows part empty."""
    from att3ntion_b200 import norm_rotate
    g = torch.Generator().manual_seed(N)
    xs = [rand(g, 2, N, h, D, dtype=dtype).double().sign().to(dtype) * (1 + torch.rand(2, N, h, D, generator=g)).to(dtype) for h in heads]
    ws = [1 + 0.3 * torch.randn(D, generator=g) for _ in heads]
    leaves, scales = [x.cuda().requires_grad_() for x in xs], [w.cuda().requires_grad_() for w in ws]
    dys = [rand(g, 2, N, h, D) for h in heads]
    ys = norm_rotate(leaves, scales, eps=eps)
    torch.autograd.backward(ys, [d.cuda() for d in dys])
    half = torch.finfo(dtype).eps / 2
    for x, w, dy, y, leaf, scale in zip(xs, ws, dys, ys, leaves, scales):
        x64, w64 = x.double().requires_grad_(), w.double().requires_grad_()
        y64 = ref.norm_rotate(x64, w64, None, None, 0.0, False)
        close(y, y64.detach(), HALF * y64.detach().abs() + 2e-6 * y64.detach().abs().amax(-1, keepdim=True), "y")
        y64.backward(dy.double())
        close(leaf.grad, x64.grad, half * x64.grad.abs() + 4e-6 * x64.grad.abs().amax(-1, keepdim=True) + 1e-6, "dx")
        u = (x64 * x64.pow(2).mean(-1, keepdim=True).rsqrt()).detach()
        close(scale.grad, w64.grad, 3e-6 * (dy.double().abs().amax(-1, keepdim=True) * u.abs()).sum((0, 1, 2)) + 1e-7, "dw")


def test_derivatives_are_refused_on_the_gpu():
    """Tangents, and arguments without a gradient that want one: none is dropped in silence."""
    from torch.autograd import forward_ad
    from att3ntion_b200 import gather_cache_append, gather_cache_evict, norm_rotate, rotary_table, single_gather_decode
    c = Made(33, [20, 9], 1, 64, 16, room=1)
    pools, table, n = c.gpu()
    mass, rot = c.mass.cuda(), rotary_table(64, 64).cuda()
    new = [torch.randn(2, 1, 1, 64, device="cuda") for _ in range(4)]
    Q = torch.randn(2, 4, 64, device="cuda")
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
    calls = [lambda d: norm_rotate(d(new[0])), lambda d: norm_rotate(new[0], d(rot[0])), lambda d: norm_rotate(new[0], None, d(rot)),
             lambda d: gather_cache_append(pools, table, n, *new[:3], d(new[3])), lambda d: gather_cache_append(pools, table, n, *new, mass=d(mass)),
             lambda d: gather_cache_append([d(pools[0]), *pools[1:]], table, n, *new), lambda d: gather_cache_append(pools, table, n, *new, table=d(rot)),
             lambda d: single_gather_decode(d(Q), pools, table, n), lambda d: single_gather_decode(Q, [*pools[:3], d(pools[3])], table, n),
             lambda d: single_gather_decode(Q, pools, table, n, mass=d(mass)), lambda d: gather_cache_evict(pools, d(mass), table, n, 4)]
    before = [p.clone() for p in (*pools, mass)]
    for k, call in enumerate(calls):
        for grad in (True, False):
            with torch.set_grad_enabled(grad), forward_ad.dual_level(), pytest.raises(RuntimeError, match="tangent"):
                call(dual)
        if k > 1:
            with pytest.raises(RuntimeError, match="gradient"):
                call(lambda t: t.detach().requires_grad_())
    for call in (lambda: torch.func.jvp(norm_rotate, (new[0],), (new[1],)), lambda: torch.func.vmap(norm_rotate)(torch.stack(new))):
        with pytest.raises(RuntimeError):
            call()
    leaf = new[0].clone().requires_grad_()
    with forward_ad.dual_level(), pytest.raises(RuntimeError):
        norm_rotate(dual(leaf))
    assert all(torch.equal(a, b) for a, b in zip(before, (*pools, mass)))


@pytest.mark.parametrize("first", ["inference mode", "capture", "side stream"])
def test_angle_table_first_made_elsewhere(first):
    """A layer whose first call ran in inference mode, was captured, or ran behind other work of a side stream, then trains."""
    import copy
    from att3ntion_b200 import HypergraphAttention
    torch.manual_seed(6)
    layer = HypergraphAttention(128, 2, gather_mode=1, window=16, rotary_base=1e4, qk_norm=True).cuda()
    x = torch.randn(2, 48, 128, device="cuda")
    twin = copy.deepcopy(layer)
    want = twin(x)
    want.sum().backward()
    if first == "inference mode":
        with torch.inference_mode():
            assert torch.equal(layer(x), want)
    elif first == "capture":
        graph = torch.cuda.CUDAGraph()
        with torch.no_grad(), torch.cuda.graph(graph):
            y = layer(x)
    else:
        torch.full((1 << 20,), float("nan"), device="cuda")       # what the table's memory may hold before it is filled
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            torch.cuda._sleep(1 << 28)
            layer._rotary(48, x.device)
    got = layer(x)
    got.sum().backward()
    assert torch.equal(got, want)
    for a, b in zip(layer.parameters(), twin.parameters()):
        assert torch.equal(a.grad, b.grad)
    if first == "capture":
        for _ in range(2):
            graph.replay()
            assert torch.equal(y, want)


def test_cache_in_and_out_of_inference_mode():
    from att3ntion_b200 import GatherCache
    new = [torch.randn(2, 3, 1, 64, device="cuda") for _ in range(4)]
    q = torch.randn(2, 4, 64, device="cuda")
    out = []
    for made, used in ((True, False), (False, True), (False, False)):
        with torch.inference_mode(made):
            c = GatherCache(2, 1, 64, pages=4, slots=32, page_size=16, track_mass=True)
        with torch.inference_mode(used):
            c.append(*new)
            c.append(*new, counts=[1, 0])
            y = c.decode(q)
            kept = c.evict(2)
        assert c.lengths.tolist() == [2, 2] and c.positions.tolist() == [4, 3]
        out.append((y, kept))
    assert all(torch.equal(a, b) for o in out[:2] for a, b in zip(o, out[2]))


@pytest.mark.parametrize("through", ["view", "projection", "scale"])
def test_norm_rotate_captured_on_what_the_capture_makes_of_leaves(through):
    """The leaves behind a view, a projection or a cast count as the inputs do; inputs computed before the capture do not
    stand in its way."""
    from att3ntion_b200 import norm_rotate
    x = torch.randn(2, 33, 192, device="cuda", requires_grad=True)
    weight = torch.randn(192, 192, device="cuda", requires_grad=True)
    w = torch.rand(64, device="cuda", dtype=torch.float64, requires_grad=True)
    dy = torch.randn(2, 33, 3, 64, device="cuda").bfloat16()

    def forward():
        if through == "view":
            return norm_rotate(x.view(2, 33, 3, 64)), [x]
        if through == "projection":
            return norm_rotate((x.detach() @ weight).view(2, 33, 3, 64)), [weight]
        return norm_rotate(x.detach().view(2, 33, 3, 64), w.float()), [w]

    def step():
        y, leaves = forward()
        return (y, *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.detach().clone() for t in step()]
    torch.cuda.current_stream().wait_stream(side)
    alive = forward()
    other = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="outside the capture"):
        with torch.cuda.graph(other):
            forward()
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    h = (x @ weight).view(2, 33, 3, 64)                   # its graph stays alive
    part = torch.cuda.CUDAGraph()
    with torch.cuda.graph(part):
        norm_rotate(h)
    torch.cuda.synchronize()


@pytest.mark.parametrize("lengths,Hq,Hkv,D,page,window,sinks", [
    # many tiles of a head on one CTA, begun and ended inside a tile's keys; last tiles of one half
    ([2000], 24, 3, 64, 64, 0, 0),
    ([1924, 300, 129, 257], 16, 2, 128, 16, 0, 0),
    ([1500, 40, 900, 385], 32, 4, 64, 32, 700, 30),
    ([700] * 12, 16, 16, 128, 64, 0, 0),
])
def test_masses_over_many_tiles(lengths, Hq, Hkv, D, page, window, sinks):
    from att3ntion_b200 import _cuda_kernels as ck, single_gather_decode
    c = Made(34, lengths, Hkv, D, page)
    # scores that grow along the sequence, so that what was added up before has to follow a new maximum
    for b, n in enumerate(lengths):
        for p in range(-(-n // page)):
            c.pools[0][int(c.table[b, p])] *= 0.2 + 2.0 * p * page / n
    Q = rand(c.g, c.B, Hq, D)
    Y64, A, share = ref.decode(Q, c.pools, c.table, lengths, window, sinks)
    pools, table, n = c.gpu()
    mass = c.mass.cuda()
    Y = single_gather_decode(Q.cuda(), pools, table, n, window=window, sinks=sinks, mass=mass)
    ck.device_status()
    close(Y, Y64, (1 + HALF) * HALF * (Y64.abs() + A) + 4e-4 * A, "Y")
    want = c.mass.double()
    for at, v in share.items():
        want[at] += v
    # as in test_decode, at scores up to 2.2 times as large
    close(mass, want, 2.0 ** -24 * want + 5e-5 * (want - c.mass.double()), "mass")
    again = c.mass.cuda()
    assert torch.equal(single_gather_decode(Q.cuda(), pools, table, n, window=window, sinks=sinks, mass=again), Y) and torch.equal(again, mass)


@pytest.mark.parametrize("D,with_mass", [(64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("where", ["rows", "columns"])
def test_decode_scores_below_the_range_count_nothing(D, with_mass, where):
    """Scores that are -inf in FP32 for whole groups of rows, or for the first steps of keys, beside ordinary ones.  All
    factors are powers of two, so the products are exact."""
    from att3ntion_b200 import single_gather_decode
    n, page = 420, 64
    c = Made(36, [n], 1, D, page)
    Q = torch.zeros(1, 2, D, dtype=torch.bfloat16)
    Q[..., 0] = 2.0 ** 40
    for k in (0, 1):
        c.pools[k].zero_()
        c.pools[k][..., 0] = 2.0 ** -20
    for e in range(288):
        at = (int(c.table[0, e // page]), e % page)
        c.pools[0 if where == "rows" else 1][at + (0, 0)] = -2.0 ** 120       # a score of -2^140 / sqrt(D)
    Y64, A, share = ref.decode(Q, c.pools, c.table, [n])
    pools, table, length = c.gpu()
    mass = c.mass.cuda() if with_mass else None
    Y = single_gather_decode(Q.cuda(), pools, table, length, mass=mass)
    close(Y, Y64, (1 + HALF) * HALF * (Y64.abs() + A) + 2e-4 * A, "Y")
    if with_mass:
        want = c.mass.double()
        for at, v in share.items():
            want[at] += v
        close(mass, want, 2.0 ** -24 * want + 2e-5 * (want - c.mass.double()), "mass")


def test_masses_with_a_wide_table():
    """Tables for 131072 slots of 16 sequences, most of it empty: the scratch is by the slot and fits."""
    from att3ntion_b200 import _cuda_kernels as ck, single_gather_decode
    lengths = [100] * 15 + [700]
    c = Made(35, lengths, 1, 128, 16)
    pools, table, n = c.gpu()
    wide = torch.full((16, 131072 // 16), -1, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    Q = rand(c.g, 16, 8, 128).cuda()
    out = []
    for t in (table, wide):
        mass = c.mass.cuda()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        out.append((single_gather_decode(Q, pools, t, n, mass=mass), mass))
        assert torch.cuda.max_memory_allocated() - before < 1 << 30
    ck.device_status()
    assert all(torch.equal(a, b) for a, b in zip(*out))


@pytest.mark.parametrize("kw", [dict(window=16, qk_norm=True, rotary_base=1e4), dict(window=48, sinks=3)])
def test_sequences_that_end_and_start_at_their_own_time(kw):
    """One sequence ends, is cleared and starts anew while the others go on or sit out: each gives what it gives alone."""
    from att3ntion_b200 import GatherCache, HypergraphAttention
    torch.manual_seed(8)
    layer = HypergraphAttention(128, 2, gather_mode=1, **kw).cuda()
    x = torch.randn(3, 80, 128, device="cuda")
    new = torch.randn(1, 80, 128, device="cuda")
    make = lambda n: GatherCache(n, 2, 64, pages=10 * n, slots=80, page_size=8, track_mass=True)
    cache, alone = make(3), [make(3) for _ in range(2)]

    def near(a, b):                                     # projections of another batch may be summed in another order
        assert (a - b).norm() <= 0.01 * b.norm()

    layer.prefill(x[:, :30], cache, counts=[30, 12, 25])
    for _ in range(3):
        layer.decode(x[:, 40:41], cache)
    assert cache.host_lengths == [33, 15, 28]
    cache.clear(1)
    layer.decode(x[:, 41:42], cache, counts=[1, 0, 1])
    assert cache.host_lengths == cache.lengths.tolist() == [34, 0, 29] and cache.host_positions == [34, 0, 29]
    assert len(cache._free) == 30 - 5 - 4 and cache.page_table[1].tolist() == [-1] * 10
    y = layer.prefill(torch.cat([x[:1, :20], new[:, :20], x[:1, :20]]), cache, counts=[0, 17, 0])
    assert cache.host_lengths == [34, 17, 29]
    before = cache.mass.clone()
    y2 = layer.decode(torch.cat([x[:1, 42:43], new[:, 17:18], x[2:, 42:43]]), cache, counts=[1, 1, 0])
    assert cache.host_lengths == cache.lengths.tolist() == [35, 18, 29]
    pages = cache.page_table[2][:4].long()
    assert torch.equal(cache.mass[pages], before[pages])           # what sat out gained nothing
    # the same three sequences, each with a batch of copies of its own
    for b, (rows, steps) in enumerate((((x[0:1, :30], 30), (40, 40, 40, 41, 42)), ((new[:, :20], 17), (17,)))):
        c = alone[b]
        z = layer.prefill(rows[0].expand(3, -1, -1).contiguous(), c, counts=[rows[1]] * 3)
        if b == 1:
            near(y[1, :17], z[1, :17])
        source = x[0:1] if b == 0 else new
        for s in steps:
            z = layer.decode(source[:, s: s + 1].expand(3, -1, -1).contiguous(), c)
        near(y2[b], z[b])


@pytest.mark.parametrize("N,head_dim,kw", [
    (48, 64, dict(gather_mode=1, window=16, qk_norm=True, rotary_base=100.0, sinks=3)),
    (48, 64, dict(gather_mode=1, window=16, qk_norm=True, rotary_base=100.0)),
    (45, 128, dict(gather_mode=1, window=20, qk_norm=True, rotary_base=1e4, sinks=1)),
    (40, 64, dict(gather_mode=1, window=200, rotary_base=1e4, sinks=5)),
    (33, 128, dict(gather_mode=1, qk_norm=True)),
    (48, 32, dict(gather_mode=1, window=9, qk_norm=True, rotary_base=100.0, sinks=4)),
    (32, 64, dict(gather_mode=0, qk_norm=True, rotary_base=100.0)),
    (27, 16, dict(gather_mode=0, qk_norm=True, rotary_base=100.0)),
])
def test_layer_gradients_against_64_bits(N, head_dim, kw):
    """Every parameter's gradient, and the input's, of the layer with norms, rotation and sinks against a restatement in 64
    bits whose gather operands are rounded to BF16 as the layer's are.

    Tolerances, in the 2-norm.  A gather's gradient dO of an operand O is held to |error| <= g |dO|, g = 0.06 for Q, R, S and
    0.04 for the values, the result to 0.03 |Y| (the gates of the operators' own tests).  The result's error moves its
    cotangent too, by 0.03 |Y| max |dY gelu''| / |dY|, and BF16 rounds it by 2^-8: both are added to g.  From there on all is
    linear: |error dW| <= g |dO| s |X|_2 with s the largest factor of the norm's backward pass, |w| / rms.  A scale's gradient
    sums error times u = x / rms over the rows, whose errors are roundings of their own: taken as independent, their sum has
    the 2-norm sum error^2 u^2, at most (g |dO| max |u|)^2.  The output projection: 0.03 |Y| max |gelu'| |dy|_2
    + 2^-8 |gelu(Y)| |dy|_2; a projection's bias: g |dO| sqrt(rows)."""
    from oracle import triplet_oracle as O
    from att3ntion_b200 import HypergraphAttention, rotary_table, window_mask
    torch.manual_seed(N + head_dim)
    B, H = 2, 2
    layer = HypergraphAttention(H * head_dim, H, **kw).cuda()
    with torch.no_grad():
        for p in (layer.q_norm, layer.r_norm, layer.s_norm):
            if p is not None:
                p.uniform_(0.5, 1.5)
    x, dy = torch.randn(B, N, H * head_dim, device="cuda", requires_grad=True), torch.randn(B, N, H * head_dim, device="cuda")
    layer(x).backward(dy)

    P = {n: p.detach().double().cpu().requires_grad_() for n, p in layer.named_parameters()}
    X = x.detach().double().cpu().requires_grad_()
    round_bf16 = lambda t: t + (t.detach().to(torch.bfloat16).double() - t.detach())
    heads = lambda t: t.view(B, N, H, head_dim).transpose(1, 2)
    table = rotary_table(N, head_dim, kw["rotary_base"]).double() if kw.get("rotary_base") else None
    pos = torch.arange(N).expand(B, N)
    ops, factor, spread = {}, {}, {}
    for name, w, scale in (("Q", "Wq", "q_norm"), ("R", "Wr", "r_norm"), ("S", "Ws", "s_norm")):
        raw = (X @ P[w + ".weight"].T).view(B, N, H, head_dim)
        t = ref.norm_rotate(raw, P.get(scale), table, pos, 1e-6, False)
        inverse = (raw.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt().detach() if scale in P else None
        factor[name] = 1.0 if inverse is None else float(P[scale].detach().abs().max() * inverse.max())
        spread[name] = None if inverse is None else float((raw.detach() * inverse).abs().max())
        ops[name] = round_bf16(t.transpose(1, 2))
    for name, w in (("Vr", "Wv_r"), ("Vs", "Wv_s"), ("Vq", "Wv_q")):
        if w + ".weight" in P:
            ops[name], factor[name] = round_bf16(heads(X @ P[w + ".weight"].T + P.get(w + ".bias", 0.0))), 1.0
    for t in ops.values():
        t.retain_grad()
    mask = window_mask(N, kw["window"], "cpu", kw.get("sinks", 0)).expand(B, N, N) if kw.get("window") else None
    zero = torch.zeros_like(ops["Vr"])
    out, _ = O.hypergraph_dense(ops["Q"], ops["R"], ops["S"], ops.get("Vq", zero), zero, ops["Vr"], zero, ops["Vs"], zero, mask=mask,
                                gather_mode=kw["gather_mode"], scatter=False)
    out = [t for t in out[: 3 if kw["gather_mode"] == 0 else 1]]
    for t in out:
        t.retain_grad()
    acts = [t * torch.sigmoid(1.702 * t) for t in out]
    y = sum(acts).transpose(1, 2).reshape(B, N, H * head_dim)
    (y @ P["Wo.weight"].T + P["Wo.bias"]).backward(dy.double().cpu())

    more = 2.0 ** -8
    for t, a in zip(out, acts):
        s = torch.sigmoid(1.702 * t.detach())
        first, second = s + 1.702 * t.detach() * s * (1 - s), 1.702 * s * (1 - s) * (2 + 1.702 * t.detach() * (1 - 2 * s))
        cotangent = t.grad / first                                     # before the activation
        more = max(more, 2.0 ** -8 + 0.03 * float(t.detach().norm() * (cotangent * second).abs().max() / t.grad.norm()))
    assert more < 0.2
    share = {n: ((0.04 if n[0] == "V" else 0.06) + more) * float(t.grad.norm()) * factor[n] for n, t in ops.items()}
    flat = X.detach().flatten(0, 1)
    size = float(torch.linalg.matrix_norm(flat, 2))
    of = {"Wq": "Q", "Wr": "R", "Ws": "S", "Wv_r": "Vr", "Wv_s": "Vs", "Wv_q": "Vq"}
    tol = {"Wo.bias": 1e-5 * float(dy.norm()) * N}
    edge = float(torch.linalg.matrix_norm(dy.double().cpu().flatten(0, 1), 2))
    tol["Wo.weight"] = edge * sum(0.03 * float(t.detach().norm()) * 1.1 + 2.0 ** -8 * float(a.detach().norm()) for t, a in zip(out, acts))
    total = 0.0
    for w, o in of.items():
        if w + ".weight" in P:
            tol[w + ".weight"] = share[o] * size
            if w + ".bias" in P:
                tol[w + ".bias"] = share[o] * (B * N) ** 0.5
            total += share[o] * float(torch.linalg.matrix_norm(P[w + ".weight"].detach(), 2))
    for scale, o in (("q_norm", "Q"), ("r_norm", "R"), ("s_norm", "S")):
        if scale in P:
            tol[scale] = share[o] / factor[o] * spread[o]
    assert set(tol) == set(P)
    for name, p in layer.named_parameters():
        off = float((p.grad.double().cpu() - P[name].grad).norm())
        assert off <= tol[name], (name, off, tol[name], float(P[name].grad.norm()))
        if not name.endswith("bias"):                              # a tolerance that a wrong gradient would meet says nothing
            assert tol[name] < 0.9 * float(P[name].grad.norm()), (name, tol[name], float(P[name].grad.norm()))
    off = float((x.grad.double().cpu() - X.grad).norm())
    assert off <= total, (off, total)


def test_masses_of_shared_pages_gain_every_share():
    """Sequences with a common prefix, or a table that names a page twice: no share is lost."""
    from att3ntion_b200 import _cuda_kernels as ck, single_gather_decode
    B, page = 24, 32
    c = Made(37, [300] + [40] * (B - 1), 2, 64, page)
    c.table[1:, :7] = c.table[0, :7]
    c.table[3, 5] = c.table[3, 2]
    lengths = [300, 224] + [200 + b for b in range(B - 2)]
    Q = rand(c.g, B, 4, 64)
    _, _, share = ref.decode(Q, c.pools, c.table, lengths)
    pools, table, _ = c.gpu()
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    want = c.mass.double()
    for at, v in share.items():
        want[at] += v
    for _ in range(5):
        mass = c.mass.cuda()
        single_gather_decode(Q.cuda(), pools, table, n, mass=mass)
        # FP32 sums and exponentials of each share, and a rounding of the running value an addition (25 of them)
        close(mass, want, 25 * 2.0 ** -24 * want + 2e-5 * (want - c.mass.double()), "mass")
    ck.device_status()

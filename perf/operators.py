"""Measured calls of the operators that serve a windowed gather: head norms with the position rotation, appending to a
paged gather cache, the gather of one new token over that cache, and eviction from it.

A gather cache holds, for every cached token and key head, the four rows R, S, Vr, Vs that a later query needs.  Its
pools are [pages, page_size, Hkv, D]; `table[b, p]` names the page that holds slots p*page_size .. of sequence b, and
`lengths[b]` says how many slots are in use.

`run` computes each operator in its plain form (elementary torch operations in 32 bits, rounded once at the end) unless
`own` is set, in which case it makes the framework's calls.  `exact` states the definitions again in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-6
DEVICE = "cuda"


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # One decoding step of 64 sequences: queries and keys of one token each.  Launch latency is everything.
        dict(name="norm step", op="norm", B=64, N=1, Hq=8, Hkv=1, D=128, rot=128, dtype="bfloat16", far=100000,
             interleaved=False, heads_first=False, train=False),
        # A training step at the headline shape (batch 4, 8 query heads over one key head, 8192 tokens): both directions.
        dict(name="norm train", op="norm", B=4, N=8192, Hq=8, Hkv=1, D=128, rot=128, dtype="bfloat16", far=0,
             interleaved=False, heads_first=False, train=True),
        # The 64-wide configuration (batch 4, 8 heads, 2048 tokens) of an FP32 model, padded length, half the head
        # rotated in neighbouring pairs, results laid out heads first for the dense gather.
        dict(name="norm train fp32", op="norm", B=4, N=2047, Hq=8, Hkv=8, D=64, rot=32, dtype="float32", far=0,
             interleaved=True, heads_first=True, train=True),
        # A decoding step's append: one new token of each of 64 sequences, normed, rotated and stored.
        dict(name="append step", op="append", B=64, T=1, Hq=8, Hkv=1, D=128, rot=128, page=16, have=8000,
             dtype="bfloat16", normed=True, ragged=False),
        # Prompts of up to 2000 tokens of 16 sequences stored as they are (the prompt's own pass has normed them).
        dict(name="append prompts", op="append", B=16, T=2000, Hq=0, Hkv=4, D=128, rot=0, page=64, have=0,
             dtype="bfloat16", normed=False, ragged=True),
        # One user's next token, window 128: the smallest serving call.
        dict(name="decode one", op="decode", B=1, Hq=8, Hkv=1, D=128, length=8192, window=128, sinks=0, page=16,
             ragged=False, mass=False),
        # A serving batch at window 128 with four sinks, lengths all different.
        dict(name="decode batch", op="decode", B=128, Hq=8, Hkv=1, D=128, length=4000, window=128, sinks=4, page=32,
             ragged=True, mass=False),
        # No window, 64-wide heads each with keys of its own, ragged lengths from one token up.
        dict(name="decode ragged", op="decode", B=16, Hq=8, Hkv=8, D=64, length=2000, window=0, sinks=0, page=16,
             ragged=True, mass=False),
        # Long sequences, every pair visible: the largest call, all tensor-core work.
        dict(name="decode long", op="decode", B=2, Hq=8, Hkv=1, D=128, length=8191, window=0, sinks=0, page=128,
             ragged=False, mass=False),
        # The same call with every token's share of the attention added up for a later eviction.
        dict(name="decode mass", op="decode", B=4, Hq=8, Hkv=2, D=128, length=2500, window=0, sinks=0, page=64,
             ragged=True, mass=True),
        # A small cache trimmed to half.
        dict(name="evict small", op="evict", B=2, Hkv=1, D=128, length=700, keep=333, sinks=4, recent=64, page=16),
        # A serving batch trimmed together.
        dict(name="evict batch", op="evict", B=32, Hkv=4, D=128, length=8000, keep=4000, sinks=4, recent=256, page=64),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["norm", "append", "decode", "decode", "evict"])
    Hkv = rng.choice([1, 1, 2, 4, 8])
    D = rng.choice([64, 128, 128])
    page = rng.choice([16, 32, 64, 128])
    if op == "norm":
        D = rng.choice([16, 32, 64, 128])
        B, Hq = _spread(rng, 1, 64), Hkv * rng.choice([1, 2, 4, 8])
        most = max(1, min(8192, (4 * 8192 * 10 * 128) // (2 * B * (Hq + 2 * Hkv) * D)))
        N = _spread(rng, min(most, rng.choice([1, 1, 200])), most)
        return dict(op=op, B=B, N=N, Hq=Hq, Hkv=Hkv, D=D, rot=rng.choice([D, D, D // 2, 0]),
                    dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), far=rng.choice([0, 100000]),
                    interleaved=rng.random() < 0.5, heads_first=rng.random() < 0.5, train=rng.random() < 0.6)
    if op == "append":
        B, normed = _spread(rng, 1, 64), rng.random() < 0.6
        T = _spread(rng, 1, max(1, min(4000, (16 * 2000 * 4 * 128) // (2 * B * Hkv * D))))
        return dict(op=op, B=B, T=T, Hq=Hkv * rng.choice([1, 4, 8]) if normed else 0, Hkv=Hkv, D=D,
                    rot=rng.choice([D, D // 2]) if normed else 0, page=page, have=rng.choice([0, _spread(rng, 1, 4000)]),
                    dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), normed=normed, ragged=rng.random() < 0.5)
    if op == "decode":
        Hq = Hkv * rng.choice([1, 2, 4, 8])
        window = rng.choice([0, 0, 0, 16, 64, 128, 128, _spread(rng, 1, 500)])
        sinks = rng.choice([0, 4, _spread(rng, 1, 40)]) if window else 0
        length = _spread(rng, rng.choice([1, 100, 100]), 8000)
        seen = min(length, window + sinks) if window else length
        B = _spread(rng, 1, max(1, min(128, (2 * 8 * 8191 * 8191) // (Hq * seen * seen))))
        while B * Hq * seen * seen > 2 * 8 * 8191 * 8191:
            length = seen = seen // 2
        return dict(op=op, B=B, Hq=Hq, Hkv=Hkv, D=D, length=length, window=window, sinks=sinks, page=page,
                    ragged=rng.random() < 0.6, mass=rng.random() < 0.3)
    length = _spread(rng, rng.choice([2, 200]), 8000)
    B = _spread(rng, 1, max(1, (32 * 8000 * 4 * 128) // (length * Hkv * D * 2)))
    B = min(B, 64)
    keep = rng.randint(1, length)
    sinks = min(keep, rng.choice([0, 4]))
    return dict(op=op, B=B, Hkv=Hkv, D=D, length=length, keep=keep, sinks=sinks,
                recent=rng.randint(0, keep - sinks), page=page)


# --------------------------------------------------------------------------- inputs

def _table(far, rot):
    """[far, rot] FP32: the cosines of every position, then the sines, from angles in 64 bits."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=DEVICE)
    a = torch.arange(far, dtype=torch.float64, device=DEVICE)[:, None] * 10000.0 ** (-2.0 * i / rot)[None]
    return torch.cat([a.cos(), a.sin()], 1).float()


def _lengths(case, key, seed):
    """int32 [B]: all alike, or spread from one token to the longest, the longest among them."""
    B, most = case["B"], case[key]
    if not case.get("ragged"):
        return torch.full((B,), most, dtype=torch.int32, device=DEVICE)
    g = torch.Generator().manual_seed(seed)
    n = 1 + (torch.rand(B, generator=g) * most).long().clamp(max=most - 1)
    n[int(torch.randint(0, B, (1,), generator=g))] = most
    return n.int().to(DEVICE)


def _paged(g, B, slots, page, spare=0):
    """Page table [B, pages] of a pool whose pages lie in random order, and the number of pages in the pool."""
    per = -(-slots // page)
    total = B * per + spare
    order = torch.randperm(total, device=DEVICE, generator=g)
    return order[: B * per].view(B, per).int().contiguous(), total


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    randn = lambda *s, dtype=torch.bfloat16: torch.randn(*s, generator=g, device=DEVICE).to(dtype)  # noqa: E731
    s = dict(case=case)
    op, D = case["op"], case["D"]
    if op == "norm":
        B, N, Hq, Hkv = case["B"], case["N"], case["Hq"], case["Hkv"]
        dt = getattr(torch, case["dtype"])
        s["xs"] = [randn(B, N, h, D, dtype=dt).mul_(1.7).requires_grad_(case["train"]) for h in (Hq, Hkv, Hkv)]
        s["weights"] = [(1 + 0.2 * randn(D, dtype=torch.float32)).requires_grad_(case["train"]) for _ in range(3)]
        s["table"] = _table(max(N, case["far"]), case["rot"]) if case["rot"] else None
        s["positions"] = (torch.randint(0, case["far"] - N + 1, (B, 1), generator=g, device=DEVICE)
                          + torch.arange(N, device=DEVICE)) if case["far"] and case["rot"] else None
        if case["train"]:
            s["dys"] = [randn(*((B, h, N, D) if case["heads_first"] else (B, N, h, D))) for h in (Hq, Hkv, Hkv)]
    elif op == "append":
        B, T, Hq, Hkv, page = case["B"], case["T"], case["Hq"], case["Hkv"], case["page"]
        dt = getattr(torch, case["dtype"])
        s["counts"] = _lengths(case, "T", seed) if case["ragged"] else None
        # the sequences' earlier pages lie elsewhere in a user's pool: the table's entries for them are not looked at
        first, last = case["have"] // page, (case["have"] + T - 1) // page
        part, total = _paged(g, B, (last - first + 1) * page, page, 1)
        s["page_table"] = torch.zeros(B, last + 1, dtype=torch.int32, device=DEVICE)
        s["page_table"][:, first:] = part
        s["lengths"] = torch.full((B,), case["have"], dtype=torch.int32, device=DEVICE)
        s["pools"] = [torch.zeros(total, page, Hkv, D, dtype=torch.bfloat16, device=DEVICE) for _ in range(4)]
        s["new"] = [randn(B, T, Hkv, D, dtype=dt) for _ in range(4)]
        s["Q"] = randn(B, T, Hq, D, dtype=dt) if case["normed"] else None
        s["weights"] = [1 + 0.2 * randn(D, dtype=torch.float32) for _ in range(3)] if case["normed"] else None
        s["table"] = _table(case["have"] + T, case["rot"]) if case["normed"] else None
    elif op == "decode":
        B, Hq, Hkv, page = case["B"], case["Hq"], case["Hkv"], case["page"]
        s["lengths"] = _lengths(case, "length", seed)
        s["page_table"], total = _paged(g, B, case["length"], page)
        s["pools"] = [randn(total, page, Hkv, D) for _ in range(4)]
        s["Q"] = randn(B, Hq, D)
        s["mass"] = torch.rand(total, page, Hkv, generator=g, device=DEVICE) * 1e-3 if case["mass"] else None
    else:
        B, Hkv, page = case["B"], case["Hkv"], case["page"]
        gl = torch.Generator().manual_seed(seed)
        n = case["length"] - (torch.rand(B, generator=gl) * 0.3 * case["length"]).long()
        s["lengths"] = n.clamp(min=1).int().to(DEVICE)
        per, out = -(-case["length"] // page), -(-case["keep"] // page)
        tables, total = _paged(g, B, (per + out) * page, page)
        # the kept tokens go to fresh pages: the old ones may still serve a sequence that was forked from this one
        s["page_table"], s["out_table"] = tables[:, :per].contiguous(), tables[:, per:].contiguous()
        s["pools"] = [randn(total, page, Hkv, D) for _ in range(4)]
        # attention that tokens have gathered: a few carry much, the newest none yet
        m = torch.rand(total, page, Hkv, generator=g, device=DEVICE)
        s["mass"] = torch.where(m < 0.02, torch.zeros_like(m), -m.log())
    return s


# --------------------------------------------------------------------------- plain forms

def _norm_plain(x, w, table, pos, interleaved):
    """x [B,N,H,D]: divided by its root mean square, times w, the first `rot` columns rotated by the position's angles."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    if table is None:
        return y
    rot = table.shape[1]
    cs = table[pos].unsqueeze(-2)                       # [B,N,1,rot] or [N,1,rot]
    c, s = cs[..., : rot // 2], cs[..., rot // 2:]
    if interleaved:
        a, b = y[..., 0:rot:2], y[..., 1:rot:2]
        r = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
    else:
        a, b = y[..., : rot // 2], y[..., rot // 2: rot]
        r = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([r, y[..., rot:]], -1)


def _run_norm(s):
    case, xs, ws = s["case"], s["xs"], s["weights"]
    pos = s["positions"]
    if own:
        from att3ntion_b200 import norm_rotate
        ys = norm_rotate(xs, ws, s["table"], pos, eps=EPS, interleaved=case["interleaved"],
                         heads_first=case["heads_first"])
    else:
        if pos is None:
            pos = torch.arange(case["N"], device=DEVICE)
        ys = [_norm_plain(xs[0], ws[0], s["table"], pos, case["interleaved"]),
              _norm_plain(xs[1], ws[1], s["table"], pos, case["interleaved"]),
              _norm_plain(xs[2], ws[2], s["table"], pos, case["interleaved"])]
        ys = [(y.transpose(1, 2).contiguous() if case["heads_first"] else y).to(torch.bfloat16) for y in ys]
    if not case["train"]:
        return list(ys)
    grads = torch.autograd.grad(ys, [*xs, *ws], s["dys"])
    return [y.detach() for y in ys] + list(grads)


def _run_append(s):
    case, pools, new = s["case"], s["pools"], s["new"]
    if own:
        from att3ntion_b200 import gather_cache_append
        q = gather_cache_append(pools, s["page_table"], s["lengths"], *new, counts=s["counts"], Q=s["Q"],
                                weights=s["weights"], table=s["table"], eps=EPS)
        return dict(pools=list(pools), Q=q)
    t = torch.arange(case["T"], device=DEVICE)
    pos = s["lengths"].long()[:, None] + t              # [B,T]: slot, and here the position too
    R, S, Vr, Vs = new
    q = None
    if case["normed"]:
        wq, wr, ws = s["weights"]
        q = _norm_plain(s["Q"], wq, s["table"], pos, False).to(torch.bfloat16)
        R, S = _norm_plain(R, wr, s["table"], pos, False), _norm_plain(S, ws, s["table"], pos, False)
    pages = s["page_table"].long().gather(1, pos // case["page"])
    rows = pages * case["page"] + pos % case["page"]
    if s["counts"] is not None:
        live = t[None] < s["counts"][:, None]
        rows, R, S, Vr, Vs = rows[live], R[live], S[live], Vr[live], Vs[live]
    Hkv, D = case["Hkv"], case["D"]
    at = rows.reshape(-1)
    pools[0].view(-1, Hkv, D)[at] = R.reshape(-1, Hkv, D).to(torch.bfloat16)
    pools[1].view(-1, Hkv, D)[at] = S.reshape(-1, Hkv, D).to(torch.bfloat16)
    pools[2].view(-1, Hkv, D)[at] = Vr.reshape(-1, Hkv, D).to(torch.bfloat16)
    pools[3].view(-1, Hkv, D)[at] = Vs.reshape(-1, Hkv, D).to(torch.bfloat16)
    return dict(pools=list(pools), Q=q)


def _run_decode(s):
    case, Q, pools, table, lengths = s["case"], s["Q"], s["pools"], s["page_table"], s["lengths"]
    mass = s["mass"].clone() if s["mass"] is not None else None      # a pass adds to it: each starts from the same
    if own:
        from att3ntion_b200 import single_gather_decode
        y = single_gather_decode(Q, pools, table, lengths, window=case["window"], sinks=case["sinks"], mass=mass)
        return dict(Y=y, mass=mass)
    B, Hq, Hkv, D, page = case["B"], case["Hq"], case["Hkv"], case["D"], case["page"]
    # the visible slots of each sequence, in order: the first `sinks`, then the last `window`
    n = lengths.long()
    most = min(case["length"], case["window"] + case["sinks"]) if case["window"] else case["length"]
    e = torch.arange(most, device=DEVICE)[None]
    seen = n.clamp(max=case["window"] + case["sinks"]) if case["window"] else n
    skip = (n - seen)[:, None]
    slot = torch.where(e < case["sinks"], e, e + skip) if case["window"] else e.expand(B, most)
    live = e < seen[:, None]
    slot = torch.where(live, slot, torch.zeros_like(slot))
    rows = table.long().gather(1, slot // page) * page + slot % page
    R, S, Vr, Vs = (p.view(-1, Hkv, D)[rows].float().transpose(1, 2).unsqueeze(2) for p in pools)   # [B,Hkv,1,E,D]
    q = Q.float().view(B, Hkv, Hq // Hkv, 1, D)
    X = (q * R) @ S.transpose(-1, -2) * (D ** -0.5)                                          # [B,Hkv,G,E,E]
    both = live[:, None, None, :, None] & live[:, None, None, None, :]
    X = X.masked_fill_(~both, -math.inf)
    X = X.sub_(X.amax((-1, -2), keepdim=True)).exp_()
    X = X.div_(X.sum((-1, -2), keepdim=True))
    y = ((X @ Vs) * Vr).sum(-2).reshape(B, Hq, D).to(torch.bfloat16)
    if mass is not None:
        share = (X.sum(-1) + X.sum(-2)).sum(2) / (2 * (Hq // Hkv))                           # [B,Hkv,E]
        mass.view(-1, Hkv).index_put_((rows[live],), share.transpose(1, 2)[live], accumulate=True)
    return dict(Y=y, mass=mass)


def _run_evict(s):
    case, pools, mass = s["case"], s["pools"], s["mass"]
    if own:
        from att3ntion_b200 import gather_cache_evict
        kept, n = gather_cache_evict(pools, mass, s["page_table"], s["lengths"], case["keep"], sinks=case["sinks"],
                                     recent=case["recent"], out_table=s["out_table"])
        return dict(pools=list(pools), mass=mass, kept=kept, lengths=n)
    B, Hkv, page, keep, most = case["B"], case["Hkv"], case["page"], case["keep"], case["length"]
    n = s["lengths"].long()[:, None]
    slot = torch.arange(most, device=DEVICE)[None]                                           # [1,L]
    rows = s["page_table"].long().gather(1, (slot // page).expand(B, most)) * page + slot % page
    m = mass.view(-1, Hkv)[rows].transpose(1, 2)                                             # [B,Hkv,L]
    held = ((slot < case["sinks"]) | (slot >= n - case["recent"])) & (slot < n)
    # first the held ones, then by mass, ties by slot, the unused slots last
    key = torch.where(held[:, None], math.inf, m).masked_fill((slot >= n)[:, None], -math.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices[..., :keep].sort(-1).values  # [B,Hkv,keep]
    r = torch.arange(keep, device=DEVICE)
    left = n.clamp(max=keep)                                                                 # [B,1]
    live = (r[None] < left)[:, None].expand(B, Hkv, keep)
    kept = torch.where(live, order, -1)
    to = s["out_table"].long().gather(1, (r[None] // page).expand(B, keep)) * page + r[None] % page
    b, h, _ = live.nonzero(as_tuple=True)
    src, dst = rows[b, kept[live]], to[:, None].expand(B, Hkv, keep)[live]
    pools[0].view(-1, Hkv, case["D"])[dst, h] = pools[0].view(-1, Hkv, case["D"])[src, h]
    pools[1].view(-1, Hkv, case["D"])[dst, h] = pools[1].view(-1, Hkv, case["D"])[src, h]
    pools[2].view(-1, Hkv, case["D"])[dst, h] = pools[2].view(-1, Hkv, case["D"])[src, h]
    pools[3].view(-1, Hkv, case["D"])[dst, h] = pools[3].view(-1, Hkv, case["D"])[src, h]
    mass.view(-1, Hkv)[dst, h] = mass.view(-1, Hkv)[src, h]
    return dict(pools=list(pools), mass=mass, kept=kept.int(), lengths=left[:, 0].int())


def run(state):
    return dict(norm=_run_norm, append=_run_append, decode=_run_decode, evict=_run_evict)[state["case"]["op"]](state)


# --------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    op, B, Hkv, D = case["op"], case["B"], case["Hkv"], case["D"]
    size = {"float32": 4}.get(case.get("dtype"), 2)
    if op == "norm":
        rows = B * case["N"] * (case["Hq"] + 2 * Hkv)
        places = case["N"] * (B if case["far"] else 1)
        moved = rows * D * (size + 2) + places * case["rot"] * 4
        flops = rows * D * 6
        if case["train"]:
            moved += rows * D * (2 * size + 2) + places * case["rot"] * 4       # x and dy read, dx written
            flops += rows * D * 14
        return {"bytes": moved, "flops": flops}
    if op == "append":
        mean = (1 + case["T"]) / 2 if case["ragged"] else case["T"]
        rows = B * mean * (case["Hq"] + 4 * Hkv)
        return {"bytes": rows * D * (size + 2) + B * mean * case["rot"] * 4, "flops": rows * D * 3}
    if op == "decode":
        # the sum over sequences of what a query sees, and of its square, for lengths spread evenly over 1 .. longest
        n, cap = case["length"], case["window"] + case["sinks"] if case["window"] else case["length"]
        each = range(1, n + 1) if case["ragged"] else [n]
        one = sum(min(i, cap) for i in each) / len(each)
        two = sum(min(i, cap) ** 2 for i in each) / len(each)
        return {"bytes": B * (Hkv * one * D * 8 + case["Hq"] * D * 4 + (Hkv * one * 8 if case["mass"] else 0)),
                "flops": B * case["Hq"] * two * D * 4}
    n = 0.85 * case["length"]
    left = min(n, case["keep"])
    return {"bytes": B * Hkv * (n * 4 + left * (D * 16 + 8 + 4)), "flops": 0}


# --------------------------------------------------------------------------- the definitions, in 64 bits

def _rotation(positions, table, D, interleaved):
    """[..., D, D] matrices that rotate a head's columns, one a position, in 64 bits."""
    rot = table.shape[1]
    half = rot // 2
    i = torch.arange(half, device=DEVICE)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    t = table.double()[positions]
    M = torch.eye(D, dtype=torch.float64, device=DEVICE).repeat(*positions.shape, 1, 1)
    M[..., a, a], M[..., b, b] = t[..., :half], t[..., :half]
    M[..., a, b], M[..., b, a] = -t[..., half:], t[..., half:]
    return M


def _normed64(x, w, M, dy=None):
    """M (w o x / rms(x)) of x [B,N,H,D] and, for a cotangent, the gradients of x and w from the quotient rule."""
    x, w = x.detach().double(), w.detach().double()
    D = x.shape[-1]
    rms = ((x ** 2).sum(-1, keepdim=True) / D + EPS).sqrt()
    u = x / rms
    y = u * w if M is None else torch.einsum("...nij,...nhj->...nhi", M, u * w)
    if dy is None:
        return y, None, None
    g = dy.double() if M is None else torch.einsum("...nij,...nhi->...nhj", M, dy.double())
    dw = torch.einsum("bnhd,bnhd->d", g, u)
    gw = g * w
    return y, gw / rms - x * (gw * x).sum(-1, keepdim=True) / (D * rms ** 3), dw


def _exact_norm(s):
    case = s["case"]
    ys, dxs, dws = [], [], []
    for k in range(3):
        y, dx, dw = [], [], 0
        for b in range(case["B"]):
            M = None
            if s["table"] is not None:
                p = torch.arange(case["N"], device=DEVICE) if s["positions"] is None else s["positions"][b]
                M = _rotation(p, s["table"], case["D"], case["interleaved"])[None]
            dy = None
            if case["train"]:
                dy = s["dys"][k][b: b + 1]
                dy = dy.permute(0, 2, 1, 3) if case["heads_first"] else dy
            yb, dxb, dwb = _normed64(s["xs"][k][b: b + 1], s["weights"][k], M, dy)
            y.append(yb.permute(0, 2, 1, 3) if case["heads_first"] else yb)
            dx.append(dxb)
            dw = dw if dwb is None else dw + dwb
        ys.append(torch.cat(y).contiguous())
        if case["train"]:
            dxs.append(torch.cat(dx))
            dws.append(dw)
    return ys + dxs + dws


def _exact_append(s):
    case, page = s["case"], s["case"]["page"]
    pools, q = [p.double() for p in s["pools"]], []
    for b in range(case["B"]):
        n0, T = int(s["lengths"][b]), case["T"]
        M = None if not case["normed"] else _rotation(torch.arange(n0, n0 + T, device=DEVICE), s["table"], case["D"], False)
        rows = [t[b].double() for t in s["new"]]
        if case["normed"]:
            q.append(_normed64(s["Q"][b], s["weights"][0], M)[0])
            rows[0] = _normed64(rows[0], s["weights"][1], M)[0]
            rows[1] = _normed64(rows[1], s["weights"][2], M)[0]
        n = T if s["counts"] is None else int(s["counts"][b])
        slots = torch.arange(n0, n0 + n, device=DEVICE)
        pages, within = s["page_table"][b].long()[slots // page], slots % page
        for p, r in zip(pools, rows):
            p[pages, within] = r[:n]
    return dict(pools=pools, Q=torch.stack(q) if q else None)


def _exact_decode(s):
    case, page = s["case"], s["case"]["page"]
    G = case["Hq"] // case["Hkv"]
    Y = torch.zeros(case["B"], case["Hq"], case["D"], dtype=torch.float64, device=DEVICE)
    mass = None if s["mass"] is None else s["mass"].double()
    for b, n in enumerate(s["lengths"].tolist()):
        slots = torch.arange(n, device=DEVICE)
        if case["window"]:
            slots = slots[(slots < case["sinks"]) | (slots >= n - case["window"])]
        pages, within = s["page_table"][b].long()[slots // page], slots % page
        for h in range(case["Hq"]):
            R, S, Vr, Vs = (p[pages, within, h // G].double() for p in s["pools"])
            x = torch.einsum("d,jd,kd->jk", s["Q"][b, h].double(), R, S) / math.sqrt(case["D"])
            p = torch.exp(x - torch.logsumexp(x.flatten(), 0))
            Y[b, h] = torch.einsum("jk,jd,kd->d", p, Vr, Vs)
            if mass is not None:
                mass[pages, within, h // G] += (p.sum(0) + p.sum(1)) / (2 * G)
    return dict(Y=Y, mass=mass)


def _exact_evict(s):
    case, page = s["case"], s["case"]["page"]
    pools, mass = [p.double() for p in s["pools"]], s["mass"].double()
    kept = torch.full((case["B"], case["Hkv"], case["keep"]), -1, dtype=torch.int32, device=DEVICE)
    left = []
    for b, n in enumerate(s["lengths"].tolist()):
        k = min(n, case["keep"])
        left.append(k)
        slots = torch.arange(n, device=DEVICE)
        at = s["page_table"][b].long()[slots // page], slots % page
        r = torch.arange(k, device=DEVICE)
        to = s["out_table"][b].long()[r // page], r % page
        for h in range(case["Hkv"]):
            m = [(-1 if i < case["sinks"] or i >= n - case["recent"] else 0, -v, i)
                 for i, v in enumerate(s["mass"][at[0], at[1], h].tolist())]
            chosen = torch.tensor(sorted(i for _, _, i in sorted(m)[:k]), device=DEVICE)
            kept[b, h, :k] = chosen.int()
            for p, source in zip([*pools, mass], [*s["pools"], s["mass"]]):
                p[to[0], to[1], h] = source[at[0][chosen], at[1][chosen], h].double()
    return dict(pools=pools, mass=mass, kept=kept, lengths=torch.tensor(left, dtype=torch.int32, device=DEVICE))


def exact(case, seed):
    s = prepare(case, seed)
    return dict(norm=_exact_norm, append=_exact_append, decode=_exact_decode, evict=_exact_evict)[case["op"]](s)

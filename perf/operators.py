"""The operators of a speculative decoding step, as a user's program calls them and in plain torch.

A step of the hybrid verifier over cached sequences runs three operators:

* ``cache``: new K/V rows are written into pages (bf16, or e4m3 with one power-of-two
  scale per token and head) and a range of positions is read back as bf16;
* ``attention``: T drafted nodes per sequence (T = 1: plain decoding) attend to the cached
  prefix and to their ancestors among the drafted nodes;
* ``advance`` / ``verify`` / ``accept``: the gated delta rule from a carried state: tokens
  that move the state on, a tree of drafted tokens that leaves it alone, and the
  state after the accepted path of such a tree.

Head layouts are those of the verifier (24 query / 4 key heads of 256 channels, 16 key /
48 value heads of 128 channels), the draft (40 / 8 heads of 128) and narrower ones.
"""

import math
import random

import torch

own = False

F8 = torch.float8_e4m3fn
EXP_BIAS, EXP_MIN, EXP_MAX = 127, -117, 118
CHUNK = 64


# ------------------------------------------------------------------------------ cases
def listed():
    return [
        # the accepted tokens of one step of a small batch, kept in bf16: launch latency
        dict(name="cache_append", op="cache", b=8, new=4, lo=120, hi=1500, hk=4, d=256, page=64, e4m3=False,
             whole=False),
        # a batch of prompts quantised into the cache and read back for the next prompt chunk
        dict(name="cache_prompt", op="cache", b=6, new=2048, lo=2048, hi=9001, hk=8, d=128, page=16, e4m3=True,
             whole=True),
        # one user, one token, a short conversation: the smallest decoding call
        dict(name="decode_one", op="attention", b=1, t=1, lo=700, hi=700, hq=24, hk=4, d=256, page=64, e4m3=False,
             gate=True),
        # plain decoding of a large ragged batch over a quantised cache
        dict(name="decode_batch", op="attention", b=64, t=1, lo=1, hi=8191, hq=24, hk=4, d=256, page=64, e4m3=True,
             gate=True),
        # a tree of drafted tokens in the draft's own head layout, small pages, no output gate
        dict(name="tree_draft", op="attention", b=8, t=29, lo=100, hi=4001, hq=40, hk=8, d=128, page=16, e4m3=False,
             gate=False),
        # a tree that fills one tile of stacked rows over long bf16 caches
        dict(name="tree_long", op="attention", b=32, t=21, lo=4000, hi=24001, hq=24, hk=4, d=256, page=64,
             e4m3=False, gate=True),
        # a wide tree over long quantised caches: the most arithmetic for each byte of cache
        dict(name="tree_wide", op="attention", b=8, t=61, lo=6000, hi=32003, hq=24, hk=4, d=256, page=128, e4m3=True,
             gate=True),
        # one user, one token: the recurrent form's smallest call
        dict(name="delta_step", op="advance", b=1, t=1, nk=16, nv=48, d=128),
        # a chunk of two prompts carried on from their states, an odd length
        dict(name="delta_prompt", op="advance", b=2, t=333, nk=16, nv=48, d=128),
        # a tree of a mid-sized batch
        dict(name="delta_tree", op="verify", b=16, t=16, nk=16, nv=48, d=128),
        # a wide tree of a large batch
        dict(name="delta_tree_wide", op="verify", b=32, t=61, nk=16, nv=48, d=128),
        # the accepted paths of a large batch
        dict(name="delta_accept", op="accept", b=64, t=16, nk=16, nv=48, d=128),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["cache", "attention", "attention", "attention", "advance", "verify", "accept"])
    if op == "cache":
        hk, d = rng.choice([(4, 256), (8, 128), (2, 64), (1, 128)])
        b, new = _spread(rng, 1, 48), _spread(rng, 1, 2048)
        new = max(1, min(new, 12288 // b))
        hi = max(new, min(_spread(rng, new, 12000), 48000 // b))
        return dict(op=op, b=b, new=new, lo=rng.randint(new, hi), hi=hi, hk=hk, d=d, page=rng.choice([16, 32, 64, 128]),
                    e4m3=rng.random() < 0.7, whole=rng.random() < 0.5)
    if op == "attention":
        hq, hk, d = rng.choice([(24, 4, 256), (24, 4, 256), (40, 8, 128), (8, 2, 64), (4, 4, 128), (8, 1, 128)])
        t = rng.choice([1, _spread(rng, 2, 64), _spread(rng, 2, 64)])
        b = _spread(rng, 1, 64)
        hi = _spread(rng, 1, 32768)
        hi = max(1, min(hi, 440000 // b, int(9.2e6 / (b * t)) if t > 1 else hi))
        return dict(op=op, b=b, t=t, lo=rng.choice([0, rng.randint(0, hi), hi]), hi=hi, hq=hq, hk=hk, d=d,
                    page=rng.choice([16, 32, 64, 128]), e4m3=rng.random() < 0.5, gate=rng.random() < 0.6)
    nk, nv, d = rng.choice([(16, 48, 128), (16, 48, 128), (2, 4, 64), (4, 4, 128)])
    if op == "advance":
        t = rng.choice([1, _spread(rng, 2, 400)])
        b = _spread(rng, 1, max(1, min(64, 700 // t)))
    else:
        t, b = _spread(rng, 1, 64), _spread(rng, 1, 48)
        if b * t > 1950:
            b = 1950 // t
    return dict(op=op, b=b, t=t, nk=nk, nv=nv, d=d)


def _lens(c):
    """The sequences' lengths: evenly spread between lo and hi (prepare shuffles them)."""
    b, lo, hi = c["b"], c["lo"], c["hi"]
    return [hi if b == 1 else lo + (hi - lo) * i // (b - 1) for i in range(b)]


def work(c):
    b = c["b"]
    if c["op"] == "cache":
        row = 2 * c["hk"] * (c["d"] + 1 if c["e4m3"] else 2 * c["d"])  # one token's K and V in the cache
        back = sum(_lens(c)) if c["whole"] else b * c["new"]
        flat = 2 * c["hk"] * c["d"] * 2
        # what is written and read back in one pass comes from the cache once
        return {"bytes": b * c["new"] * (flat + row) + back * (row + flat), "flops": 0}
    if c["op"] == "attention":
        t, hq, hk, d = c["t"], c["hq"], c["hk"], c["d"]
        n = sum(_lens(c))
        row = 2 * hk * (d + 1 if c["e4m3"] else 2 * d)
        nodes = b * t * (2 * d * (hq * (3 if c["gate"] else 2) + 2 * hk) + 4 * hq)
        return {"bytes": n * row + nodes, "flops": 4 * hq * d * t * n + 2 * b * hq * d * t * (t + 1)}
    t, nk, nv, d = c["t"], c["nk"], c["nv"], c["d"]
    state = 4 * b * nv * d * d
    if c["op"] == "accept":
        return {"bytes": 2 * state + b * (2 * nk * d + 4 * nv * d), "flops": 3 * b * nv * d * d}
    tokens = b * t * (4 * nk * d + 4 * nv * d + 6 * nv)
    pairs = 4 * b * nv * t * min(t, CHUNK) * d
    if c["op"] == "verify":
        return {"bytes": state + tokens + 4 * b * t * nv * d, "flops": 4 * b * nv * t * d * d + pairs}
    return {"bytes": 2 * state + tokens, "flops": 6 * b * nv * t * d * d + pairs}


# ------------------------------------------------------------------------------ inputs
def _tree(rng, t):
    """Parents of t nodes in topological order: -1 is the last cached token, chains and branches."""
    return [-1 if i == 0 else max(-1, i - 1 - int(rng.expovariate(0.7))) for i in range(t)]


def _path(rng, parents):
    """A node drawn from the tree, and the way to it from the root."""
    at, way = rng.randrange(len(parents)), []
    while at >= 0:
        way.append(at)
        at = parents[at]
    return way[::-1]


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device="cuda")


def _encode(x):
    """Plain quantisation of rows [..., D]: (e4m3 codes, exponent bytes [...])."""
    x = x.float()
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(a)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(EXP_MIN, EXP_MAX)
    e = torch.where(a == 0, 0, e)
    y = torch.ldexp(x, -e[..., None].float())
    return torch.where(torch.isnan(y), y, y.clamp(-448, 448)).to(F8), (e + EXP_BIAS).to(torch.uint8)


def _scale(exps):
    """fp32 2^e of exponent bytes."""
    return torch.ldexp(torch.ones((), device=exps.device), exps.float() - EXP_BIAS)


def _pages(c, g, total):
    """One pool of K or V rows [pages, heads, page, d]: (rows, exponent bytes or None)."""
    shape = (total, c["hk"], c["page"], c["d"])
    pool = torch.empty(shape, device="cuda", dtype=F8 if c["e4m3"] else torch.bfloat16)
    exps = torch.empty(shape[:3], device="cuda", dtype=torch.uint8) if c["e4m3"] else None
    spread = torch.rand(c["hk"], 1, c["d"], device="cuda", generator=g) + 0.5  # channels differ in size
    step = max(1, (64 << 20) // (c["hk"] * c["page"] * c["d"]))
    for p in range(0, total, step):
        x = (torch.randn((min(step, total - p), *shape[1:]), device="cuda", generator=g) * spread).bfloat16()
        if c["e4m3"]:
            pool[p:p + step], exps[p:p + step] = _encode(x)
        else:
            pool[p:p + step] = x
    return pool, exps


def _cache(c, g, rng):
    """Pools, page table and lengths of ragged sequences whose pages are scattered over the pools."""
    page = c["page"]
    lens = _lens(c)
    rng.shuffle(lens)
    need = [-(-n // page) for n in lens]
    total = sum(need) + 1  # the last page belongs to nobody
    order = list(range(total - 1))
    rng.shuffle(order)
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (max(1, max(need)) - n))
        at += n
    k, ke = _pages(c, g, total)
    v, ve = _pages(c, g, total)
    return dict(k_pool=k, v_pool=v, k_exp=ke, v_exp=ve, table=_int(table), lens=_int(lens)), lens, table


def prepare(case, seed):
    c = case
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    b = c["b"]
    s = dict(case=c)
    if c["op"] == "cache":
        pools, lens, table = _cache(c, g, rng)
        s.update(pools)
        new, page = c["new"], c["page"]
        # rows of the sequences' last positions; a sequence keeps fewer of a step's tokens now and then
        keep = [new if c["whole"] else rng.randint(1, new) for _ in range(b)]
        slots = [[table[i][p // page] * page + p % page if p - (n - new) < keep[i] else -1 for p in range(n - new, n)]
                 for i, n in enumerate(lens)]
        s["slots"] = _int(slots, torch.int64).view(-1)
        s["rows_k"] = (randn(b * new, c["hk"], c["d"]) * 1.5).bfloat16()
        s["rows_v"] = randn(b * new, c["hk"], c["d"]).bfloat16()
        s["starts"] = _int([0 if c["whole"] else n - new for n in lens])
        s["length"] = max(lens) if c["whole"] else new
        return s
    t = c["t"]
    trees = [_tree(rng, t) for _ in range(b)]
    s["parents"] = _int(trees)
    counts = [t if t < 3 or rng.random() < 0.5 else rng.randint(max(1, t - 3), t) for _ in range(b)]
    s["counts"] = _int(counts)
    if c["op"] == "attention":
        s.update(_cache(c, g, rng)[0])
        hq, hk, d = c["hq"], c["hk"], c["d"]
        s["q"] = (randn(b, t, hq, d) * 2).bfloat16()
        s["k"], s["v"] = randn(b, t, hk, d).bfloat16(), randn(b, t, hk, d).bfloat16()
        s["gate"] = randn(b, t, hq, d).bfloat16() if c["gate"] else None
        return s
    nk, nv, d = c["nk"], c["nv"], c["d"]
    # a head's decay by its own rate, as the gates give it: slow heads and fast ones
    rate = torch.exp(torch.rand(nv, device="cuda", generator=g) * math.log(1600.0)) * 0.01
    s["g"] = -rate * torch.nn.functional.softplus(randn(b, t, nv))
    s["q"], s["k"] = randn(b, t, nk, d).bfloat16(), randn(b, t, nk, d).bfloat16()
    s["v"] = randn(b, t, nv, d).bfloat16()
    s["beta"] = torch.sigmoid(randn(b, t, nv)).bfloat16()
    s["state"] = randn(b, nv, d, d) * 0.2
    s["next"] = torch.empty_like(s["state"])
    if c["op"] == "accept":
        s["u"] = randn(b, t, nv, d) * 0.5
        paths = [_path(rng, p) for p in trees]
        s["path"] = _int([p + [-1] * (max(map(len, paths)) - len(p)) for p in paths])
    return s


# ------------------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    if c["op"] == "cache":
        return _plain_cache(s, c)
    if c["op"] == "attention":
        return _plain_attention(s, c)
    if c["op"] == "accept":
        return _plain_accept(s, c)
    return _plain_delta(s, c)


def _own(s, c):
    from nanospec_b200.ops import decode_ops as dops

    if c["op"] in ("cache", "attention"):
        cache = dops.PagedCache(s["k_pool"], s["v_pool"], s["k_exp"], s["v_exp"])
    if c["op"] == "cache":
        dops.cache_write(cache, s["rows_k"], s["rows_v"], s["slots"])
        return dops.cache_read(cache, s["table"], s["lens"], s["length"], starts=s["starts"])
    if c["op"] == "attention":
        return dops.tree_attention(s["q"], s["k"], s["v"], cache, s["table"], s["lens"], s["parents"],
                                   counts=s["counts"], gate=s["gate"])
    groups = c["nv"] // c["nk"]
    if c["op"] == "advance":
        return dops.gated_delta_advance(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], groups,
                                        counts=s["counts"], out_state=s["next"])
    if c["op"] == "verify":
        return dops.gated_delta_verify(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], s["parents"], groups,
                                       counts=s["counts"])
    return dops.gated_delta_accept(s["k"], s["g"], s["u"], s["path"], s["state"], groups, out_state=s["next"])


# ------------------------------------------------------------------------------ plain forms
def _decode(pool, exps):
    x = pool.float()
    return x if exps is None else x * _scale(exps)[..., None]


def _plain_cache(s, c):
    page, pages = c["page"], s["k_pool"].shape[0]
    # rows that are not kept go to the page that belongs to nobody
    slots = torch.where(s["slots"] < 0, (pages - 1) * page, s["slots"])
    at = (slots // page, slice(None), slots % page)
    pos = s["starts"][:, None].long() + torch.arange(s["length"], device="cuda")
    seen = (pos < s["lens"][:, None])[..., None, None]
    pos = torch.minimum(pos, (s["lens"][:, None].long() - 1).clamp_min(0))
    pg = torch.gather(s["table"].long(), 1, pos // page)
    out = []
    for x, pool, exps in ((s["rows_k"], s["k_pool"], s["k_exp"]), (s["rows_v"], s["v_pool"], s["v_exp"])):
        if c["e4m3"]:
            codes, e = _encode(x)
            pool.view(torch.uint8)[at] = codes.view(torch.uint8)
            exps[at] = e
            got = pool.view(torch.uint8)[pg, :, pos % page].view(F8).float() * _scale(exps[pg, :, pos % page])[..., None]
        else:
            pool[at] = x
            got = pool[pg, :, pos % page].float()
        out.append(torch.where(seen, got, 0.0).bfloat16())
    return tuple(out)


def _ancestors(parents, counts):
    """[b, t, t]: node a is node t or one of its ancestors; no rows or columns beyond the counts."""
    b, t = parents.shape
    i = torch.arange(t, device=parents.device)
    up = (parents[:, :, None] == i).float() + torch.eye(t, device=parents.device)
    for _ in range(max(1, (t - 1).bit_length())):
        up = (up @ up > 0).float()
    live = i < counts[:, None]
    return (up > 0) & live[:, :, None] & live[:, None, :]


def _dense(pool, exps, table, lens):
    """[b, heads, L, d] fp32 rows of the sequences, zeros beyond their lengths."""
    t = table.long().clamp_min(0)
    x = _decode(pool[t] if exps is None else pool.view(torch.uint8)[t].view(F8), None if exps is None else exps[t])
    x = x.transpose(1, 2).flatten(2, 3)
    live = torch.arange(x.shape[2], device=x.device) < lens[:, None]
    return torch.where(live[:, None, :, None], x, 0.0), live


def _plain_attention(s, c):
    b, t, hq, d = s["q"].shape
    hk = c["hk"]
    gr = hq // hk
    anc = _ancestors(s["parents"], s["counts"])
    kc, live = _dense(s["k_pool"], s["k_exp"], s["table"], s["lens"])
    q = s["q"].float().view(b, t, hk, gr, d).permute(0, 2, 3, 1, 4).reshape(b, hk, gr * t, d) * d ** -0.5
    row = (torch.arange(t, device="cuda") < s["counts"][:, None])[:, None, None, :]
    see = row.expand(b, 1, gr, t).reshape(b, 1, gr * t, 1) & live[:, None, None, :]
    far = torch.where(see, q @ kc.transpose(2, 3), -math.inf)
    del kc
    near = q @ s["k"].float().permute(0, 2, 3, 1)
    near = torch.where(anc[:, None, None].expand(b, 1, gr, t, t).reshape(b, 1, gr * t, t), near, -math.inf)
    top = torch.maximum(far.amax(-1), near.amax(-1))[..., None]
    at = torch.where(torch.isfinite(top), top, 0.0)
    far, near = torch.exp(far - at), torch.exp(near - at)
    total = far.sum(-1, keepdim=True) + near.sum(-1, keepdim=True)
    vc, _ = _dense(s["v_pool"], s["v_exp"], s["table"], s["lens"])
    o = far @ vc + near @ s["v"].float().transpose(1, 2)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (at + torch.log(total))[..., 0].view(b, hk, gr, t).reshape(b, hq, t)
    o = o.view(b, hk, gr, t, d).permute(0, 3, 1, 2, 4).reshape(b, t, hq, d)
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.bfloat16(), lse


def _unit(x):
    x = x.float()
    return x * torch.rsqrt((x * x).sum(-1, keepdim=True) + 1e-6)


def _heads(x, groups):
    """[b, t, heads, ...] -> [b, heads * groups, t, ...]"""
    return x.transpose(1, 2).repeat_interleave(groups, 1)


def _delta_nodes(q, k, v, g, beta, state, anc):
    """The delta rule over nodes whose ancestors are given: outputs, updates and total decays."""
    d = q.shape[-1]
    a = anc[:, None]
    total = (a.float() @ g[..., None])[..., 0]
    decay = torch.exp(torch.where(a, total[..., :, None] - total[..., None, :], -math.inf))
    strict = a & ~torch.eye(q.shape[2], dtype=torch.bool, device=q.device)
    grow = torch.exp(total)[..., None]
    m = -torch.where(strict, beta[..., None] * decay * (k @ k.transpose(2, 3)), 0.0)
    u = beta[..., None] * (v - grow * (k @ state))
    for _ in range(max(1, (q.shape[2] - 1).bit_length())):  # (I - m)^-1 = (I + m)(I + m^2)(I + m^4)...
        u, m = u + m @ u, m @ m
    o = (grow * (q @ state) + (decay * (q @ k.transpose(2, 3))) @ u) * d ** -0.5
    return o, u, total


def _plain_delta(s, c):
    groups, t = c["nv"] // c["nk"], c["t"]
    q, k = _heads(_unit(s["q"]), groups), _heads(_unit(s["k"]), groups)
    v, g, beta = _heads(s["v"].float(), 1), _heads(s["g"], 1), _heads(s["beta"].float(), 1)
    live = torch.arange(t, device="cuda") < s["counts"][:, None]
    if c["op"] == "verify":
        o, u, _ = _delta_nodes(q, k, v, g, beta, s["state"], _ancestors(s["parents"], s["counts"]))
        keep = live[:, :, None, None]
        return (torch.where(keep, o.transpose(1, 2), 0.0).bfloat16(),
                torch.where(keep, u.transpose(1, 2), 0.0).contiguous())
    state, outs = s["state"], []
    g = torch.where(live[:, None], g, 0.0)
    beta = torch.where(live[:, None], beta, 0.0)
    for i in range(0, t, CHUNK):
        part = [x[:, :, i:i + CHUNK] for x in (q, k, v, g, beta)]
        n = part[0].shape[2]
        chain = torch.ones(n, n, dtype=torch.bool, device="cuda").tril().expand(c["b"], n, n)
        o, u, total = _delta_nodes(*part, state, chain)
        left = total[..., -1:, None]
        state = torch.exp(left) * state + (torch.exp(left - total[..., None]) * part[1]).transpose(2, 3) @ u
        outs.append(o)
    o = torch.cat(outs, 2).transpose(1, 2)
    return torch.where(live[:, :, None, None], o, 0.0).bfloat16(), state


def _plain_accept(s, c):
    groups = c["nv"] // c["nk"]
    path = s["path"].long()
    on = path >= 0
    at = path.clamp_min(0)
    take = lambda x: torch.gather(x, 1, at.view(*at.shape, *[1] * (x.dim() - 2)).expand(*at.shape, *x.shape[2:]))  # noqa: E731
    g = torch.where(on[..., None], take(s["g"]), 0.0)
    total = g.cumsum(1)
    w = torch.where(on[..., None], torch.exp(total[:, -1:] - total), 0.0)
    k = (_unit(take(s["k"])).repeat_interleave(groups, 2) * w[..., None]).permute(0, 2, 3, 1)
    return torch.exp(total[:, -1])[..., None, None] * s["state"] + k @ take(s["u"]).transpose(1, 2)


# ------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s, c = prepare(case, seed), case
    return {"cache": _exact_cache, "attention": _exact_attention, "accept": _exact_accept}.get(
        c["op"], _exact_delta)(s, c)


def _exact_row(x, e4m3):
    """What a written row reads back as, from the definition of its scale and of e4m3."""
    x = x.double()
    if not e4m3:
        return x
    a = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(a / 448)
    e = torch.where(m == 0.5, e - 1, e).clamp(EXP_MIN, EXP_MAX)
    y = x * torch.exp2(-e.double())
    grid = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
    y = (torch.round(y / grid) * grid).clamp(-448, 448)
    return torch.where(a == 0, 0.0, y * torch.exp2(e.double()))


def _exact_cache(s, c):
    page, out = c["page"], []
    for name in "kv":
        pool = s[name + "_pool"]
        ex = s[name + "_exp"]
        rows = _exact_row(s["rows_" + name], c["e4m3"])
        res = torch.zeros(c["b"], s["length"], c["hk"], c["d"], device="cuda", dtype=torch.float64)
        for i, (n, st) in enumerate(zip(s["lens"].tolist(), s["starts"].tolist())):
            pg = s["table"][i, : -(-n // page)].long()
            x = pool[pg].double()
            if ex is not None:
                x = x * torch.exp2(ex[pg].double() - EXP_BIAS)[..., None]
            x = x.transpose(1, 2).flatten(0, 1)[:n]
            part = slice(i * c["new"], (i + 1) * c["new"])
            kept = (s["slots"][part] >= 0).view(-1, 1, 1)
            x[n - c["new"]:] = torch.where(kept, rows[part], x[n - c["new"]:])
            x = x[st:st + s["length"]]
            res[i, : len(x)] = x
        out.append(res)
    return tuple(out)


def _exact_attention(s, c):
    b, t, hq, d = s["q"].shape
    gr, page = hq // c["hk"], c["page"]
    out = torch.zeros(b, t, hq, d, device="cuda", dtype=torch.float64)
    lse = torch.full((b, hq, t), -math.inf, device="cuda", dtype=torch.float64)
    for i in range(b):
        n, live = int(s["lens"][i]), int(s["counts"][i])
        pg = s["table"][i, : -(-n // page)].long()
        keys = []
        for name in "kv":
            x = s[name + "_pool"][pg].double()
            if s[name + "_exp"] is not None:
                x = x * torch.exp2(s[name + "_exp"][pg].double() - EXP_BIAS)[..., None]
            keys.append(torch.cat((x.transpose(1, 2).flatten(0, 1)[:n], s[name][i].double()), 0))
        see = torch.zeros(t, n + t, dtype=torch.bool)
        parents = s["parents"][i].tolist()
        for a in range(live):
            see[a, :n] = True
            at = a
            while at >= 0:
                see[a, n + at] = True
                at = parents[at]
        see = see.cuda()
        for h in range(hq):
            sc = s["q"][i, :, h].double() @ keys[0][:, h // gr].T / math.sqrt(d)
            sc = sc.masked_fill(~see, -math.inf)[:live]
            lse[i, h, :live] = torch.logsumexp(sc, -1)
            out[i, :live, h] = torch.softmax(sc, -1) @ keys[1][:, h // gr]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].double())
    return out, lse


def _exact_delta(s, c):
    b, t, nv, d = s["v"].shape
    gr, tree = nv // c["nk"], c["op"] == "verify"
    out = torch.zeros(b, t, nv, d, device="cuda", dtype=torch.float64)
    upd = torch.zeros_like(out)
    last = torch.empty(b, nv, d, d, device="cuda", dtype=torch.float64)
    unit = lambda x: x.double() / torch.sqrt(x.double().square().sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    q = (unit(s["q"]) / math.sqrt(d)).repeat_interleave(gr, 2)
    k = unit(s["k"]).repeat_interleave(gr, 2)
    for i in range(b):
        start = s["state"][i].double()
        parents = s["parents"][i].tolist()
        states = {-1: start}
        for a in range(int(s["counts"][i])):
            st = states[parents[a] if tree else a - 1]
            st = st * torch.exp(s["g"][i, a].double())[:, None, None]
            u = s["beta"][i, a].double()[:, None] * (s["v"][i, a].double() - torch.einsum("hkv,hk->hv", st, k[i, a]))
            st = st + k[i, a][:, :, None] * u[:, None, :]
            if not tree:
                states.clear()
            states[a] = st
            out[i, a], upd[i, a] = torch.einsum("hkv,hk->hv", st, q[i, a]), u
        last[i] = states[max(states)]
    return (out, upd) if tree else (out, last)


def _exact_accept(s, c):
    gr = c["nv"] // c["nk"]
    state = s["state"].double()
    k = s["k"].double()
    k = (k / torch.sqrt(k.square().sum(-1, keepdim=True) + 1e-6)).repeat_interleave(gr, 2)
    for i, path in enumerate(s["path"].tolist()):
        for a in path:
            if a >= 0:
                state[i] = state[i] * torch.exp(s["g"][i, a].double())[:, None, None]
                state[i] += k[i, a][:, :, None] * s["u"][i, a].double()[:, None, :]
    return state

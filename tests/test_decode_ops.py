"""Decoding ops (paged cache, tree attention, gated delta rule from a state) against plain
64-bit statements, on the CPU path and on the GPU kernels.

Tolerances. Cache: none, every scaling is exact. Attention output (bf16): one rounding of
the result and one of each probability, 2^-9 relative each, so
|err| <= 2^-9 (|o| + 1.25 sum_j p_j |v_j|), times the gate; lse: fp32 sums of D products
and one exp2 / log2, 2e-5 + 2^-20 |lse|. Delta rule: fp32 with T dependent steps of D
products, (T + D) 2^-24 ~ 2e-5 of the norm for u and states; outputs add one bf16 rounding.
"""

import math
import random

import pytest
import torch

from nanospec_b200.ops import decode_ops as dops

F8 = torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
devices = pytest.mark.parametrize("dev", DEVICES)


@pytest.fixture(autouse=True)
def _device_error(request):
    dev = request.node.callspec.params.get("dev") if hasattr(request.node, "callspec") else None
    if dev == "cuda" and not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    torch.manual_seed(0)
    yield
    if dev == "cuda":
        assert dops.cuda_ops().device_error() == 0


def i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------------------ cache
def encode64(x):
    """What rows read back as: smallest e with amax <= 448 * 2^e, then e4m3 on that grid."""
    x = x.double()
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1, keepdim=True)
    m, e = torch.frexp(a / 448)
    e = torch.where(m == 0.5, e - 1, e).clamp(-117, 118)
    e = torch.where(a == 0, 0, e)
    y = x * torch.exp2(-e.double())
    mag = y.abs().clamp(2.0 ** -6, 448.0)
    grid = torch.exp2(torch.frexp(mag)[1].double() - 1 - 3)
    r = (torch.round(y / grid) * grid).clamp(-448, 448)
    return torch.where(torch.isnan(x), x, r * torch.exp2(e.double()))


def special_rows(x):
    """Rows that a cache meets at the edges, written over the first rows of x [n, Hk, D]."""
    x[0] = 0
    x[1] = x[1] * 1e-38
    x[2] = x[2] * 3e37
    x[3, :, 0], x[3, :, 1], x[3, :, 2] = math.nan, math.inf, -math.inf
    x[4] = 0
    x[4, :, 3] = 448.0 * 2.0 ** -5       # the largest magnitude exactly at the top code
    x[5] = 0
    x[5, :, 2] = 450.0                   # just beyond it
    x[6] = -x[6].abs()
    return x


@devices
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads,d,page", [(4, 256, 64), (2, 16, 16), (1, 80, 32), (8, 128, 128), (3, 64, 16)])
def test_cache_round_trip(dev, e4m3, heads, d, page):
    n = 37
    cache = dops.PagedCache.allocate(5, heads, page, d, dtype=F8 if e4m3 else torch.bfloat16, device=dev)
    qkv = torch.randn(n, 3, heads, d).bfloat16()
    special_rows(qkv[:, 1])
    slots = torch.randperm(5 * page)[:n]
    slots[10] = slots[20] = -1
    fused = qkv.to(dev)
    dops.cache_write(cache, fused[:, 1], fused[:, 2], slots.to(dev))  # strided rows
    keep = slots >= 0
    want = [encode64(qkv[keep, i]) if e4m3 else qkv[keep, i].double() for i in (1, 2)]
    table = torch.arange(5, dtype=torch.int32).flip(0)[None]
    got = dops.cache_read(cache, table.to(dev), i32([5 * page], dev), 5 * page)
    s = slots[keep]
    at = (4 - s // page) * page + s % page  # the table lists the pages backwards
    for g, w in zip(got, want):
        assert g.dtype == torch.bfloat16
        assert torch.equal(g[0].cpu()[at].double().nan_to_num(7e30), w.nan_to_num(7e30))


@devices
@pytest.mark.parametrize("e4m3", [False, True])
def test_cache_read_ranges(dev, e4m3):
    """Odd lengths, empty sequences, ranges that begin inside a page and end beyond the
    sequence; pages that nobody wrote are never read."""
    heads, d, page, lens = 2, 64, 16, [0, 1, 37, 16]
    cache = dops.PagedCache.allocate(9, heads, page, d, dtype=F8 if e4m3 else torch.bfloat16, device=dev)
    for x in (cache.k, cache.v):
        x.view(torch.uint8).fill_(0x7f if e4m3 else 0xff)  # NaN
    table = torch.tensor([[-1, -1, -1], [7, -1, -1], [3, 8, 0], [5, -1, -1]], dtype=torch.int32)
    rows = [torch.randn(n, heads, d).bfloat16() for n in lens]
    for i, n in enumerate(lens):
        pos = torch.arange(n)
        sl = table[i, pos // page].long() * page + pos % page
        dops.cache_write(cache, rows[i].to(dev), -rows[i].to(dev), sl.to(dev))
    starts = [0, 0, 5, 20]
    for st in (None, i32(starts, dev)):
        k, v = dops.cache_read(cache, table.to(dev), i32(lens, dev), 33, starts=st)
        for i, n in enumerate(lens):
            a = 0 if st is None else starts[i]
            want = torch.zeros(33, heads, d).double()
            part = (encode64(rows[i]) if e4m3 else rows[i].double())[a:a + 33]
            want[:len(part)] = part
            assert torch.equal(k[i].cpu().double(), want) and torch.equal(v[i].cpu().double(), -want)
    k, _ = dops.cache_read(cache, table.to(dev), i32(lens, dev), 0)
    assert k.shape == (4, 0, heads, d)


@devices
def test_cache_empty_write(dev):
    cache = dops.PagedCache.allocate(1, 2, 16, 32, device=dev)
    z = torch.empty(0, 2, 32, dtype=torch.bfloat16, device=dev)
    dops.cache_write(cache, z, z, torch.empty(0, dtype=torch.int64, device=dev))


# ------------------------------------------------------------------------------ attention
def random_tree(rng, t):
    return [-1 if i == 0 else rng.randint(max(-1, i - 4), i - 1) for i in range(t)]


class Problem:
    """Ragged cached sequences with scattered pages; NaN everywhere that nobody may look."""

    def __init__(self, dev, lens, t, hq, hk, d, page, e4m3, counts=None, gate=True, spread=2.0, seed=0, pages=None):
        rng = random.Random(seed)
        b = len(lens)
        self.args = dev, lens, t, hq, hk, d
        need = [-(-n // page) for n in lens]
        total = pages or sum(need) + 2
        self.cache = dops.PagedCache.allocate(total, hk, page, d, dtype=F8 if e4m3 else torch.bfloat16, device=dev)
        if pages is None:
            for x in (self.cache.k, self.cache.v):
                x.view(torch.uint8).fill_(0x7f if e4m3 else 0xff)
        order = list(range(total)) if pages is None else list(range(total - sum(need), total))
        rng.shuffle(order)
        width = max(1, max(need)) + 1
        table, at = [], 0
        for n in need:
            table.append(order[at:at + n] + [-1] * (width - n))
            at += n
        self.table, self.lens = i32(table, dev), i32(lens, dev)
        self.prefix = []
        for i, n in enumerate(lens):
            rows = torch.randn(n, 2, hk, d).bfloat16()
            rows[:, :, :, 0] *= 4
            pos = torch.arange(n)
            sl = torch.tensor(table[i])[pos // page] * page + pos % page
            dops.cache_write(self.cache, rows[:, 0].to(dev), rows[:, 1].to(dev), sl.to(dev))
            self.prefix.append(encode64(rows) if e4m3 else rows.double())
        self.parents = torch.tensor([random_tree(rng, t) for _ in range(b)], dtype=torch.int32)
        self.counts = counts
        # q, k, v and the gate as views into one fused projection
        width = 2 * hq * d + 2 * hk * d
        fused = torch.randn(b, t, width).bfloat16()
        fused[..., :2 * hq * d] *= spread
        for i, c in enumerate(counts or []):
            fused[i, c:] = math.nan
            self.parents[i, c:] = 12345
        self.cpu = self.split(fused)
        self.dev = self.split(fused.to(dev))
        if not gate:
            self.cpu[3] = self.dev[3] = None

    def split(self, fused):
        _, _, _, hq, hk, d = self.args
        qg = fused[..., :2 * hq * d].unflatten(-1, (hq, 2 * d))
        kv = fused[..., 2 * hq * d:].unflatten(-1, (2 * hk, d))
        return [qg[..., :d], kv[:, :, :hk], kv[:, :, hk:], qg[..., d:]]

    def run(self, **kw):
        dev = self.args[0]
        q, k, v, g = self.dev
        c = None if self.counts is None else i32(self.counts, dev)
        return dops.tree_attention(q, k, v, self.cache, self.table, self.lens, self.parents.to(dev), counts=c,
                                   gate=g, **kw)

    def check(self, out, lse, scale=None):
        _, lens, t, hq, hk, d = self.args
        out, lse = out.cpu().double(), lse.cpu().double()
        q, k, v, g = self.cpu
        scale = d ** -0.5 if scale is None else scale
        for i, n in enumerate(lens):
            live = t if self.counts is None else self.counts[i]
            for a in range(t):
                if a >= live:
                    assert (out[i, a] == 0).all() and (lse[i, :, a] == -math.inf).all()
                    continue
                way, at = [], a
                while at >= 0:
                    way.append(at)
                    at = int(self.parents[i, at])
                kk = torch.cat((self.prefix[i][:, 0], k[i, way].double())).repeat_interleave(hq // hk, 1)
                vv = torch.cat((self.prefix[i][:, 1], v[i, way].double())).repeat_interleave(hq // hk, 1)
                s = torch.einsum("hd,jhd->hj", q[i, a].double(), kk) * scale
                want_lse = torch.logsumexp(s, -1)
                p = torch.softmax(s, -1)
                o, mag = torch.einsum("hj,jhd->hd", p, vv), torch.einsum("hj,jhd->hd", p, vv.abs())
                f = 1.0 if g is None else torch.sigmoid(g[i, a].double())
                err = (out[i, a] - o * f).abs()
                assert (err <= 2.0 ** -9 * (o.abs() + 1.25 * mag) * f + 1e-6).all(), (i, a, err.max())
                err = (lse[i, :, a] - want_lse).abs()
                assert (err <= 2e-5 + 2.0 ** -20 * want_lse.abs()).all(), (i, a, err.max())


ATTENTION = [
    # lens, T, Hq, Hk, D, page, counts
    ([0], 1, 4, 4, 64, 16, None),                           # nothing but itself
    ([1, 64, 65, 63], 1, 24, 4, 256, 64, None),             # decoding, lengths about a tile
    ([0, 130, 17], 5, 8, 2, 64, 16, [5, 3, 0]),             # ragged trees, one with no node
    ([100, 333], 64, 6, 1, 128, 128, [64, 61]),             # the widest tree, several row tiles
    ([513, 5], 21, 24, 4, 256, 32, None),                   # one full tile of stacked rows
    ([70, 200], 7, 40, 8, 128, 16, [7, 2]),                 # the draft's heads
    ([90], 9, 4, 2, 16, 16, None),                          # narrow heads
    ([33, 128], 3, 10, 2, 80, 32, None),                    # a head_dim that no tile divides
    ([75], 4, 6, 6, 192, 64, None),
    ([40], 2, 130, 1, 64, 16, None),                        # more heads to a group than a tile has rows
    ([129], 64, 7, 7, 240, 16, None),
]


@devices
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("case", range(len(ATTENTION)))
def test_tree_attention(dev, e4m3, case):
    lens, t, hq, hk, d, page, counts = ATTENTION[case]
    p = Problem(dev, lens, t, hq, hk, d, page, e4m3, counts, gate=case % 2 == 0, seed=case)
    p.check(*p.run())


@devices
@pytest.mark.parametrize("e4m3", [False, True])
def test_tree_attention_scale_and_spread(dev, e4m3):
    """Scores far apart (one key takes all) and nearly equal ones."""
    for scale, spread in ((3.0, 4.0), (1e-3, 0.1)):
        p = Problem(dev, [150, 40], 6, 8, 2, 64, 16, e4m3, spread=spread)
        p.check(*p.run(scale=scale), scale=scale)


@devices
def test_tree_attention_shared_parents(dev):
    p = Problem(dev, [20, 90], 6, 4, 2, 64, 16, False)
    p.parents = p.parents[:1].expand(2, 6)
    a = p.run()
    p.check(*a)
    p.parents = p.parents[0]
    assert all(torch.equal(x, y) for x, y in zip(a, p.run()))


@devices
def test_tree_attention_value_scales(dev):
    """Rows of one quantised cache whose magnitudes differ by many powers of two."""
    p = Problem(dev, [128], 2, 4, 2, 64, 16, True, gate=False)
    rows = torch.randn(128, 2, 2, 64).bfloat16()
    rows[:, 1] *= torch.exp2(torch.randint(-40, 20, (128, 2, 1)).float()).bfloat16()
    pos = torch.arange(128)
    sl = p.table[0].cpu()[pos // 16].long() * 16 + pos % 16
    dops.cache_write(p.cache, rows[:, 0].to(dev), rows[:, 1].to(dev), sl.to(dev))
    p.prefix = [encode64(rows)]
    p.check(*p.run())


@pytest.mark.gpu
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("dev", ["cuda"])
def test_tree_attention_many_parts(dev, e4m3):
    """Few long sequences (every one split over many CTAs) next to short ones."""
    p = Problem(dev, [9001, 3, 0, 700], 3, 12, 2, 128, 64, e4m3, seed=3)
    p.check(*p.run())


@pytest.mark.gpu
@pytest.mark.parametrize("dev", ["cuda"])
def test_large_offsets(dev):
    """Pages whose element offsets pass 2^31 (and byte offsets 2^32)."""
    p = Problem(dev, [70, 33], 4, 8, 8, 256, 128, False, pages=(1 << 31) // (8 * 128 * 256) + 40)
    assert p.cache.k.numel() > 1 << 31
    p.check(*p.run())
    k, _ = dops.cache_read(p.cache, p.table, p.lens, 70)
    assert torch.equal(k[0].cpu().double(), p.prefix[0][:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("dev", ["cuda"])
def test_repeats_and_streams(dev):
    """The same bits every time, and on another stream."""
    p = Problem(dev, [4000, 900, 77], 9, 24, 4, 128, 64, True, seed=5)
    first = p.run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(4):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            again = p.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, again))
    s = Delta(dev, 3, 33, 2, 3, 128)
    a = s.verify()
    with torch.cuda.stream(side):
        b = s.verify()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@devices
def test_attention_no_sequences(dev):
    cache = dops.PagedCache.allocate(1, 2, 16, 64, device=dev)
    z = lambda h: torch.empty(0, 3, h, 64, dtype=torch.bfloat16, device=dev)  # noqa: E731
    out, lse = dops.tree_attention(z(4), z(2), z(2), cache, i32([], dev).view(0, 1), i32([], dev), i32([-1, 0, 1], dev))
    assert out.shape == (0, 3, 4, 64) and lse.shape == (0, 4, 3)


# ------------------------------------------------------------------------------ gated delta rule
class Delta:
    def __init__(self, dev, b, t, nk, groups, d, counts=None, seed=0, slow=False):
        rng = random.Random(seed)
        self.dev, self.shape, self.groups, self.counts = dev, (b, t, nk, d), groups, counts
        nv = nk * groups
        r = lambda *s: torch.randn(*s)  # noqa: E731
        self.q, self.k, self.v = r(b, t, nk, d).bfloat16(), r(b, t, nk, d).bfloat16(), r(b, t, nv, d).bfloat16()
        rate = torch.exp(torch.rand(nv) * 7) * (0.001 if slow else 0.02)
        self.g = -rate * torch.rand(b, t, nv)
        self.beta = torch.rand(b, t, nv).bfloat16()
        self.state = r(b, nv, d, d) * 0.3
        self.parents = torch.tensor([random_tree(rng, t) for _ in range(b)], dtype=torch.int32)
        for i, c in enumerate(counts or []):
            for x in (self.q, self.k, self.v, self.g, self.beta):
                x[i, c:] = math.nan
            self.parents[i, c:] = 777

    def to(self, *names):
        return [getattr(self, n).clone().to(self.dev) for n in names]

    def c(self):
        return None if self.counts is None else i32(self.counts, self.dev)

    def verify(self, **kw):
        return dops.gated_delta_verify(*self.to("q", "k", "v", "g", "beta", "state", "parents"), self.groups,
                                       counts=self.c(), **kw)

    def nodes64(self, chain):
        """(out, u, {sequence: states of its nodes}) node by node in 64 bits."""
        b, t, nk, d = self.shape
        unit = lambda x: x.double() / (x.double().square().sum(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
        q = (unit(self.q) / d ** 0.5).repeat_interleave(self.groups, 2)
        k = unit(self.k).repeat_interleave(self.groups, 2)
        out, u, states = torch.zeros_like(self.v).double(), torch.zeros_like(self.v).double(), {}
        for i in range(b):
            states[i] = {-1: self.state[i].double()}
            for n in range(t if self.counts is None else self.counts[i]):
                p = n - 1 if chain else int(self.parents[i, n])
                s = states[i][p] * self.g[i, n].double().exp()[:, None, None]
                u[i, n] = self.beta[i, n].double()[:, None] * (
                    self.v[i, n].double() - torch.einsum("hkv,hk->hv", s, k[i, n]))
                s = s + k[i, n][:, :, None] * u[i, n][:, None, :]
                states[i][n] = s
                out[i, n] = torch.einsum("hkv,hk->hv", s, q[i, n])
        return out, u, states


def near(got, want, rounding=0.0):
    got, want = got.cpu().double(), want.double()
    assert torch.isfinite(got).all()
    off, norm = (got - want).norm().item(), want.norm().item()
    assert off <= (2e-5 + rounding) * norm + 1e-30, (off, norm)


BF = 2.0 ** -9
DELTA = [(1, 1, 1, 1, 128, None), (2, 1, 2, 3, 128, None), (2, 5, 2, 1, 16, [5, 0]), (3, 16, 1, 3, 128, [16, 15, 1]),
         (2, 17, 2, 2, 64, [17, 9]), (1, 64, 1, 2, 128, None), (2, 61, 1, 1, 32, [61, 33]), (1, 48, 3, 1, 128, None)]


@devices
@pytest.mark.parametrize("case", range(len(DELTA)))
def test_delta_verify_and_accept(dev, case):
    b, t, nk, gr, d, counts = DELTA[case]
    s = Delta(dev, b, t, nk, gr, d, counts, seed=case, slow=case % 2 == 1)
    before = s.state.clone()
    out, u = s.verify()
    w_out, w_u, states = s.nodes64(False)
    near(out, w_out, BF)
    near(u, w_u)
    for i, c in enumerate(counts or []):
        assert (out[i, c:] == 0).all() and (u[i, c:] == 0).all()
    assert torch.equal(s.state, before)
    rng = random.Random(case)
    paths, want = [], []
    for i in range(b):
        n = t if counts is None else counts[i]
        at, way = (rng.randrange(n) if n else -1), []
        want.append(states[i][at])
        while at >= 0:
            way.append(at)
            at = int(s.parents[i, at])
        paths.append(way[::-1])
    m = max(map(len, paths)) + 1
    path = i32([p + [-1] * (m - len(p)) for p in paths], dev)
    k, g, state = s.to("k", "g", "state")
    new = torch.full_like(state, math.nan)
    ret = dops.gated_delta_accept(k, g, u, path, state, gr, out_state=new)
    assert ret is new and torch.equal(state.cpu(), before)
    near(new, torch.stack(want))
    dops.gated_delta_accept(k, g, u, path, state, gr)  # in place
    assert torch.equal(state, new)


ADVANCE = [(1, 1, 1, 1, 128, None), (3, 1, 2, 3, 128, [1, 0, 1]), (2, 7, 1, 2, 16, None), (2, 64, 1, 1, 64, None),
           (1, 65, 1, 2, 128, None), (2, 200, 1, 1, 128, [200, 131]), (2, 130, 2, 1, 32, [64, 128]),
           (1, 257, 1, 1, 128, None)]


@devices
@pytest.mark.parametrize("case", range(len(ADVANCE)))
def test_delta_advance(dev, case):
    b, t, nk, gr, d, counts = ADVANCE[case]
    s = Delta(dev, b, t, nk, gr, d, counts, seed=case, slow=case % 2 == 1)
    w_out, _, states = s.nodes64(True)
    want = torch.stack([states[i][max(states[i])] for i in range(b)])
    args = s.to("q", "k", "v", "g", "beta")
    state = s.state.clone().to(dev)
    new = torch.full_like(state, math.nan)
    out, ret = dops.gated_delta_advance(*args, state, gr, counts=s.c(), out_state=new)
    assert ret is new and torch.equal(state.cpu(), s.state)
    near(out, w_out, BF)
    near(new, want)
    for i, c in enumerate(counts or []):
        assert (out[i, c:] == 0).all()
    out2, ret = dops.gated_delta_advance(*args, state, gr, counts=s.c())
    assert ret is state and torch.equal(out2, out) and torch.equal(state, new)


@devices
def test_delta_steps_compose(dev):
    """Tokens one by one, in two chunks, and as one tree path give the same state."""
    s = Delta(dev, 2, 80, 1, 2, 64)
    a = s.to("q", "k", "v", "g", "beta")
    one = s.state.clone().to(dev)
    for t in range(80):
        dops.gated_delta_advance(*[x[:, t:t + 1] for x in a], one, 2)
    two = s.state.clone().to(dev)
    dops.gated_delta_advance(*[x[:, :33] for x in a], two, 2)
    dops.gated_delta_advance(*[x[:, 33:] for x in a], two, 2)
    near(two, one.cpu())
    three = s.state.clone().to(dev)
    for lo, hi in ((0, 40), (40, 80)):
        part = [x[:, lo:hi] for x in a]
        chain = torch.arange(-1, hi - lo - 1, dtype=torch.int32, device=dev)
        _, u = dops.gated_delta_verify(*part, three, chain, 2)
        path = torch.arange(hi - lo, dtype=torch.int32, device=dev).expand(2, -1).contiguous()
        dops.gated_delta_accept(part[1], part[3], u, path, three, 2)
    near(three, one.cpu())


@devices
def test_delta_rows_and_resets(dev):
    """A pool of states with idle rows; a decay of -inf forgets; strided inputs."""
    b, t, nk, gr, d = 3, 4, 1, 2, 32
    s = Delta(dev, b, t, nk, gr, d)
    s.g[0, 2] = -math.inf
    pool = torch.randn(6, nk * gr, d, d)
    rows = [4, -1, 0]
    s.state = torch.stack([pool[max(r, 0)] for r in rows])
    w_out, _, states = s.nodes64(True)
    fused = torch.cat((s.q, s.k, s.v), 2).to(dev)
    q, k, v = fused.split((nk, nk, nk * gr), 2)
    g, beta = s.to("g", "beta")
    got = pool.clone().to(dev)
    out, _ = dops.gated_delta_advance(q, k, v, g, beta, got, gr, rows=i32(rows, dev))
    want = pool.clone().double()
    want[4], want[0] = states[0][t - 1], states[2][t - 1]
    near(out[::2], w_out[::2], BF)
    assert (out[1] == 0).all()
    near(got, want)
    for r in (1, 2, 3, 5):
        assert torch.equal(got[r].cpu(), pool[r])
    out, u = dops.gated_delta_verify(q, k, v, g, beta, pool.clone().to(dev), s.parents.to(dev), gr, rows=i32(rows, dev))
    w_out, w_u, _ = s.nodes64(False)
    near(out[::2], w_out[::2], BF)
    near(u[::2], w_u[::2])
    assert (out[1] == 0).all() and (u[1] == 0).all()
    path = i32([[0], [0], [-1]], dev)
    got = pool.clone().to(dev)
    dops.gated_delta_accept(k, g, u, path, got, gr, rows=i32(rows, dev))
    assert torch.equal(got[1:4].cpu(), pool[1:4]) and torch.equal(got[0].cpu(), pool[0])
    assert not torch.equal(got[4].cpu(), pool[4])


# ------------------------------------------------------------------------------ refusals
@devices
def test_refusals(dev):
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)  # noqa: E731
    cache = dops.PagedCache.allocate(4, 2, 16, 64, device=dev)
    table, lens, parents = i32([[0, 1]], dev), i32([20], dev), i32([-1, 0, 1], dev)
    slots = torch.zeros(3, dtype=torch.int64, device=dev)
    q, k = bf(1, 3, 4, 64), bf(1, 3, 2, 64)
    ok = dict(q=q, k=k, v=k, cache=cache, table=table, lens=lens, parents=parents)

    def attention(**kw):
        dops.tree_attention(**{**ok, **kw})

    attention()
    bad = [
        lambda: dops.PagedCache.allocate(4, 2, 24, 64, device=dev),
        lambda: dops.PagedCache.allocate(4, 2, 16, 72, device=dev),
        lambda: dops.PagedCache.allocate(4, 2, 16, 272, device=dev),
        lambda: dops.cache_write(cache, bf(3, 2, 32), bf(3, 2, 32), slots),
        lambda: dops.cache_write(cache, bf(3, 2, 64), bf(2, 2, 64), slots),
        lambda: dops.cache_write(cache, bf(3, 2, 64), bf(3, 2, 64), slots.int()),
        lambda: dops.cache_read(cache, table, lens, -1),
        lambda: dops.cache_read(cache, table.long(), lens, 4),
        lambda: dops.cache_read(cache, table, lens, 4, starts=i32([0, 0], dev)),
        lambda: dops.cache_read(dops.PagedCache(cache.k, cache.v.bfloat16()[:3]), table, lens, 4),
        lambda: dops.cache_read(dops.PagedCache(cache.k.to(F8), cache.v.to(F8)), table, lens, 4),
        lambda: attention(q=bf(1, 3, 5, 64)),
        lambda: attention(k=bf(1, 3, 2, 32)),
        lambda: attention(q=bf(1, 3, 4, 32)),
        lambda: attention(parents=i32([-1, 0], dev)),
        lambda: attention(parents=parents.long()),
        lambda: attention(lens=i32([20, 20], dev)),
        lambda: attention(counts=i32([3, 3], dev)),
        lambda: attention(gate=bf(1, 3, 4, 32)),
        lambda: attention(scale=0.0),
        lambda: attention(scale=-1.0),
        lambda: attention(table=i32([0, 1], dev)),
        lambda: dops.tree_attention(bf(1, 65, 4, 64), bf(1, 65, 2, 64), bf(1, 65, 2, 64), cache, table, lens,
                                    torch.arange(-1, 64, dtype=torch.int32, device=dev)),
    ]
    f = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    d = dict(q=bf(1, 3, 2, 32), k=bf(1, 3, 2, 32), v=bf(1, 3, 4, 32), g=f(1, 3, 4), beta=bf(1, 3, 4),
             state=f(1, 4, 32, 32), groups=2)
    acc = dict(k=d["k"], g=d["g"], u=f(1, 3, 4, 32), path=i32([[0, 1]], dev), state=d["state"], groups=2)
    for call in (dops.gated_delta_advance, lambda **kw: dops.gated_delta_verify(**{"parents": parents, **kw})):
        call(**d)
        for change in (dict(groups=1), dict(k=bf(1, 3, 2, 16)), dict(v=bf(1, 2, 4, 32)), dict(g=d["g"].bfloat16()),
                       dict(state=f(1, 4, 32, 16)), dict(state=f(2, 4, 32, 32)), dict(state=d["state"].double()),
                       dict(rows=i32([0, 0], dev)), dict(counts=i32([0, 0], dev)),
                       dict(q=bf(1, 3, 2, 48), k=bf(1, 3, 2, 48), v=bf(1, 3, 4, 48), state=f(1, 4, 48, 48))):
            bad.append(lambda call=call, change=change: call(**{**d, **change}))
    bad.append(lambda: dops.gated_delta_advance(**d, out_state=f(2, 4, 32, 32)))
    bad.append(lambda: dops.gated_delta_verify(**d, parents=i32([-1], dev)))
    dops.gated_delta_accept(**acc)
    for change in (dict(u=f(1, 3, 4, 16)), dict(u=f(1, 3, 4, 32).bfloat16()), dict(path=i32([0], dev)),
                   dict(path=acc["path"].long()), dict(g=f(1, 3, 2)), dict(state=f(1, 4, 16, 16))):
        bad.append(lambda change=change: dops.gated_delta_accept(**{**acc, **change}))
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {i} was accepted")


def test_bad_indices_cpu():
    cache = dops.PagedCache.allocate(4, 2, 16, 64, device="cpu")
    z = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for slot in (-2, 64):
        with pytest.raises(IndexError):
            dops.cache_write(cache, z, z, torch.tensor([slot]))
    for table, lens in (([[9]], [5]), ([[0]], [17]), ([[0]], [-1])):
        with pytest.raises(IndexError):
            dops.cache_read(cache, i32(table, "cpu"), i32(lens, "cpu"), 8)
    s = Delta("cpu", 1, 3, 1, 1, 16)
    s.parents[0] = torch.tensor([-1, 2, 0])
    with pytest.raises(IndexError):
        s.verify()
    with pytest.raises(IndexError):
        s.verify(rows=i32([3], "cpu"))
    with pytest.raises(IndexError):
        dops.gated_delta_accept(s.k, s.g, torch.zeros(1, 3, 1, 16), i32([[3]], "cpu"), s.state)


@pytest.mark.gpu
@pytest.mark.parametrize("dev", ["cuda"])
def test_bad_indices_are_skipped(dev):
    """Every kernel skips accesses that its index tensors put out of range and sets code 4."""
    c = dops.cuda_ops()

    def flagged(call):
        assert c.device_error() == 0
        r = call()
        assert c.device_error() == 4
        c.clear_device_error()
        return r

    cache = dops.PagedCache.allocate(4, 2, 16, 64, dtype=F8, device=dev)
    z = torch.ones(3, 2, 64, dtype=torch.bfloat16, device=dev)
    cache.k.view(torch.uint8).zero_()
    cache.v.view(torch.uint8).zero_()
    cache.k_exp.fill_(127)
    cache.v_exp.fill_(127)
    flagged(lambda: dops.cache_write(cache, z, z, torch.tensor([0, 64, 1 << 40], device=dev)))
    assert int((cache.k.float() != 0).sum()) == 128
    for table, lens in (([[9, 0]], [20]), ([[0, 1]], [33]), ([[0, 1]], [-4])):
        flagged(lambda: dops.cache_read(cache, i32(table, dev), i32(lens, dev), 40))
        q, k = torch.ones(1, 2, 4, 64, dtype=torch.bfloat16, device=dev), z[None, :2]
        out, _ = flagged(lambda: dops.tree_attention(q, k, k, cache, i32(table, dev), i32(lens, dev),
                                                     i32([-1, 0], dev)))
        assert torch.isfinite(out).all()
    for parents, counts in (([-1, 1], [2]), ([-2, 0], [2]), ([-1, 0], [3]), ([-1, 0], [-1])):
        flagged(lambda: dops.tree_attention(q, k, k, cache, i32([[0, 1]], dev), i32([20], dev), i32(parents, dev),
                                            counts=i32(counts, dev)))
        s = Delta(dev, 1, 2, 1, 1, 64)
        s.parents, s.counts = torch.tensor(parents, dtype=torch.int32), counts
        flagged(s.verify)
    s = Delta(dev, 1, 2, 1, 1, 64)
    flagged(lambda: s.verify(rows=i32([1], dev)))
    k, g, state = s.to("k", "g", "state")
    u = torch.ones(1, 2, 1, 64, device=dev)
    for path in ([[2]], [[-2]]):
        flagged(lambda: dops.gated_delta_accept(k, g, u, i32(path, dev), state))
    assert torch.equal(state.cpu(), s.state)

"""Decoding ops where a size, an address, a scale or a value lies at an edge. Tolerances are those
of test_decode_ops.py."""

import math

import pytest
import torch

from nanospec_b200 import decode
from nanospec_b200.models import verifier as V
from nanospec_b200.ops import decode_ops as dops

from test_decode_ops import BF, Delta, Problem, _device_error, devices, encode64, i32, near  # noqa: F401

NARROW = [(2, 33, 1, 2, 16, None), (1, 64, 2, 1, 16, None), (2, 70, 2, 2, 16, [70, 41]), (2, 131, 1, 1, 16, [97, 131]),
          (1, 70, 1, 1, 32, None), (1, 70, 1, 1, 64, None)]


@devices
@pytest.mark.parametrize("case", range(len(NARROW)))
def test_delta_advance_narrow_heads(dev, case):
    """More tokens to a chunk than a narrow head's CTA has threads."""
    b, t, nk, gr, d, counts = NARROW[case]
    s = Delta(dev, b, t, nk, gr, d, counts, seed=case)
    w_out, _, states = s.nodes64(True)
    state = s.state.clone().to(dev)
    out, _ = dops.gated_delta_advance(*s.to("q", "k", "v", "g", "beta"), state, gr, counts=s.c())
    near(out, w_out, BF)
    near(state, torch.stack([states[i][max(states[i])] for i in range(b)]))


def shifted(x, by):
    """x, dense, at ``by`` elements into its storage."""
    return x.new_empty(x.numel() + by)[by:].view(x.shape).copy_(x)


@devices
@pytest.mark.parametrize("by", [1, 4])
@pytest.mark.parametrize("e4m3", [False, True])
def test_dense_operands_at_odd_addresses(dev, by, e4m3):
    """Dense views that begin off a 16-byte boundary give what aligned ones give."""
    p = Problem(dev, [90, 33], 5, 8, 2, 64, 16, e4m3)
    p.dev = [x.contiguous() for x in p.dev]
    want = p.run()
    p.dev = [shifted(x, by) for x in p.dev]
    assert all(x.is_contiguous() and (dev == "cpu" or x.data_ptr() % 16) for x in p.dev)
    assert all(torch.equal(a, b) for a, b in zip(p.run(), want))
    k, v = (torch.randn(7, 2, 64, device=dev).bfloat16() for _ in range(2))
    slots = torch.arange(7, device=dev) + p.table[1, 0] * 16
    got = []
    for a, b in ((k, v), (shifted(k, by), shifted(v, by))):
        dops.cache_write(p.cache, a, b, slots)
        got += [dops.cache_read(p.cache, p.table, p.lens, 7)]
    assert all(torch.equal(a, b) for a, b in zip(*got))


@devices
@pytest.mark.parametrize("by", [1, 2])
@pytest.mark.parametrize("t,d", [(1, 128), (20, 128), (40, 32)])
def test_dense_delta_operands_at_odd_addresses(dev, by, t, d):
    s = Delta(dev, 2, t, 1, 2, d)
    q, k, v, g, beta, state, parents = s.to("q", "k", "v", "g", "beta", "state", "parents")
    odd = [shifted(x, by) for x in (q, k, v, g, beta)]
    want, got = state.clone(), state.clone()
    a, b = dops.gated_delta_advance(q, k, v, g, beta, want, 2)[0], dops.gated_delta_advance(*odd, got, 2)[0]
    assert torch.equal(a, b) and torch.equal(want, got)
    a, b = (dops.gated_delta_verify(*x, state, parents, 2) for x in ((q, k, v, g, beta), odd))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    path = torch.arange(t, dtype=torch.int32, device=dev).expand(2, -1).contiguous()
    for m in {1, t}:
        want, got = torch.empty_like(state), torch.empty_like(state)
        dops.gated_delta_accept(k, g, a[1], path[:, :m].contiguous(), state, 2, out_state=want)
        dops.gated_delta_accept(odd[1], odd[3], shifted(a[1], by), path[:, :m].contiguous(), state, 2, out_state=got)
        assert torch.equal(want, got)


@devices
def test_out_states_that_overlap(dev):
    """States move on in place or to memory of their own: a row being read is nobody's to write."""
    s = Delta(dev, 3, 2, 1, 2, 16)
    q, k, v, g, beta, state = s.to("q", "k", "v", "g", "beta", "state")
    pool = torch.zeros(8, 2, 2, 16, 16, device=dev)
    flat = pool[:, 0].contiguous()
    u, path = torch.zeros(3, 2, 2, 16, device=dev), i32([[0, 1]] * 3, dev)
    want = state.clone()
    out = dops.gated_delta_advance(q, k, v, g, beta, want, 2)[0]
    for a, b in ((flat[:3], flat[3:6]), (flat[5:], flat[2:5]), (pool[:3, 0], pool[:3, 1]), (pool[:3, 1], pool[:3, 0]),
                 (pool[2:5, 1], pool[3:6, 0]), (flat[:3], flat[:3]), (pool[1:4, 1], pool[1:4, 1])):
        a.copy_(state)
        got, ret = dops.gated_delta_advance(q, k, v, g, beta, a, 2, out_state=b)
        assert ret is b and torch.equal(got, out) and torch.equal(b, want)
    for a, b in ((flat[:3], flat[1:4]), (flat[2:5], flat[:3]), (flat[:3], flat[:6:2]), (state, flat[:1].expand(3, -1, -1, -1)),
                 (pool[:3, 0], flat.as_strided((3, 2, 16, 16), (256, 256, 16, 1)))):
        with pytest.raises(ValueError):
            dops.gated_delta_advance(q, k, v, g, beta, a, 2, out_state=b)
        with pytest.raises(ValueError):
            dops.gated_delta_accept(k, g, u, path, a, 2, out_state=b)


def rewrite(p, rows):
    """Sequence 0's prefix of an e4m3 problem becomes rows [n, 2, Hk, D]."""
    dev, page = p.args[0], p.cache.page_size
    pos = torch.arange(len(rows))
    slots = p.table[0].cpu()[pos // page].long() * page + pos % page
    dops.cache_write(p.cache, rows[:, 0].to(dev), rows[:, 1].to(dev), slots.to(dev))
    p.prefix[0] = encode64(rows)


def aim(p, x):
    """Channel 0 of every query is x."""
    for q in (p.cpu[0], p.dev[0]):
        q[..., 0] = x


def scale_nodes(p, f):
    """The nodes' V times f [T] (powers of two)."""
    p.cpu[2] = (p.cpu[2].float() * f[None, :, None, None]).bfloat16()
    p.dev[2] = p.cpu[2].to(p.args[0])


@devices
@pytest.mark.parametrize("far", [16, 22, 26, 30, 100])
@pytest.mark.parametrize("n,b", [(128, 1), (400, 1), (400, 80)])
def test_value_scale_of_a_key_without_weight(dev, far, n, b):
    """One cached row of V is 2^far times the others', but its key has no probability."""
    if b > 1 and dev == "cpu":
        pytest.skip("the same statement as one sequence")
    p = Problem(dev, [n] + [300] * (b - 1), 2, 4, 2, 64, 16, True, gate=False)
    rows = torch.randn(n, 2, 2, 64).bfloat16()
    rows[:, 0, :, 0] = 0
    rows[5, 0, :, 0] = -160.0  # score -160 and e^-160 of the probability
    rows[5, 1] *= 2.0 ** far
    aim(p, 8.0)
    rewrite(p, rows)
    p.check(*p.run())


@devices
def test_value_scale_of_a_hidden_node(dev):
    """A drafted node that others do not see has V of 2^30 times theirs."""
    p = Problem(dev, [100], 4, 4, 2, 64, 16, True, gate=False)
    p.parents = i32([[-1, 0, 0, 2]], "cpu")
    scale_nodes(p, torch.tensor([1.0, 2.0 ** 30, 1.0, 1.0]))
    p.check(*p.run())


@devices
@pytest.mark.parametrize("n", [500, 6000])
def test_sink_without_value(dev, n):
    """One key takes nearly all the probability and has V = 0: the others are the output."""
    p = Problem(dev, [n], 1, 4, 2, 64, 16, True, gate=False)
    rows = torch.randn(n, 2, 2, 64).bfloat16()
    rows[:, 0] *= 0.25
    rows[:, 0, :, 0] = 0
    rows[3, 0, :, 0] = 17.0  # e^17 = 2^24.5 times the others' probability
    rows[3, 1] = 0
    aim(p, 8.0)
    rewrite(p, rows)
    p.check(*p.run())


@devices
def test_values_near_the_top_and_bottom(dev):
    """V rows at the ends of the exponents' range."""
    for e in (-110, 110):
        p = Problem(dev, [300], 2, 4, 2, 64, 16, True, gate=False)
        rows = torch.randn(300, 2, 2, 64).bfloat16()
        rows[:, 1] *= 2.0 ** e
        scale_nodes(p, torch.full((2,), 2.0 ** e))
        rewrite(p, rows)
        out, lse = p.run()
        p.prefix[0][:, 1] *= 2.0 ** -e
        p.cpu[2] = (p.cpu[2].float() * 2.0 ** -e).bfloat16()
        p.check(out.float() * 2.0 ** -e, lse)


@devices
@pytest.mark.parametrize("far", [2, 3, 70, 110])
@pytest.mark.parametrize("b", [1, 80])
def test_value_scale_of_a_key_with_weight(dev, far, b):
    """One cached row of V is 2^far times the others' and its key counts like any other; a
    sequence per CTA, and several."""
    if b > 1 and dev == "cpu":
        pytest.skip("the same statement as one sequence")
    p = Problem(dev, [400] + [300] * (b - 1), 2, 4, 2, 64, 16, True, gate=False)
    rows = torch.randn(400, 2, 2, 64).bfloat16()
    rows[:, 1].clamp_(-3, 3)
    rows[:, 1, :, 1] = 3.0  # the same scale in every row
    rows[5, 1] *= 2.0 ** far
    rewrite(p, rows)
    p.check(*p.run())


@devices
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n", [0, 700])
def test_scores_that_overflow_downwards(dev, e4m3, n):
    """Every score is -inf: zeros, lse -inf, however the keys are split."""
    p = Problem(dev, [n], 1, 4, 2, 64, 64, e4m3, gate=False)
    p.dev[0].fill_(3e38)
    p.dev[1].fill_(-3e38)
    if n:
        rows = torch.randn(n, 2, 2, 64).bfloat16()
        rows[:, 0] = -1e38
        rewrite(p, rows)
    out, lse = p.run()
    assert (out == 0).all() and (lse == -math.inf).all()


@devices
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("scale", [1e-30, 1e-60])
def test_vanishing_scale(dev, e4m3, scale):
    """Scores that vanish: the mean of what is seen."""
    p = Problem(dev, [200], 3, 4, 2, 64, 64, e4m3, gate=False)
    for q in (p.cpu[0], p.dev[0]):
        q[:, 1] = 0
    p.check(*p.run(scale=scale), scale=scale)


@devices
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_queries_that_are_not_finite(dev, e4m3, bad):
    """A query row that is not finite has no finite output, and leaves other rows alone."""
    p = Problem(dev, [200], 3, 4, 2, 64, 64, e4m3, gate=False)
    want = p.run()
    p.dev[0][0, 1, 2, 7] = bad
    out, lse = p.run()
    assert not torch.isfinite(out[0, 1, 2]).any() and not torch.isfinite(lse[0, 2, 1])
    out[0, 1, 2], lse[0, 2, 1] = want[0][0, 1, 2], want[1][0, 2, 1]
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dev", ["cuda"])
def test_refuses_tables_beyond_32_bits(dev):
    """Positions are counted in 32 bits, a tile beyond the last one included."""
    cache = dops.PagedCache.allocate(2, 1, 128, 16, device=dev)
    q = torch.zeros(1, 1, 1, 16, dtype=torch.bfloat16, device=dev)
    table = torch.zeros(1, (1 << 24) - 1, dtype=torch.int32, device=dev)
    with pytest.raises(ValueError):
        dops.tree_attention(q, q, q, cache, table, i32([100], dev), i32([-1], dev))


@devices
def test_refuses_no_key_heads(dev):
    z = lambda h: torch.zeros(1, 1, h, 64, dtype=torch.bfloat16, device=dev)  # noqa: E731
    cache = dops.PagedCache.allocate(2, 0, 16, 64, device=dev)
    with pytest.raises(ValueError):
        dops.tree_attention(z(4), z(0), z(0), cache, i32([[0]], dev), i32([3], dev), i32([-1], dev))


@devices
@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("n", [0, 1, 129])
def test_less_work_than_processors(dev, e4m3, n):
    """Fewer units of work than SMs: some blocks get no tile, every tile has a block of its own."""
    p = Problem(dev, [n], 1, 1, 1, 128, 16, e4m3)
    p.check(*p.run())


STAGE = {}


def stage_of(dev, kernel=4):
    if dev == "cuda" and not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    if (dev, kernel) not in STAGE:
        dtype = torch.bfloat16 if dev == "cuda" else torch.float32
        tc = V.tiny_hybrid_text_config(head_dim=32)
        tc["linear_conv_kernel_dim"] = kernel
        w = V.random_verifier_weights(tc, 0, 4, device="cpu", first=True, last=True, seed=1, std=0.15, dtype=dtype)
        STAGE[dev, kernel] = V.QwenStage(None, 0, 4, device=dev, first=True, last=True,
                                         weights={k: v.to(dev) for k, v in w.items()}, config=V.synthetic_hf_config(tc))
    return STAGE[dev, kernel]


def snapshot(s):
    return ([x.clone() for c in s.caches.values() for x in (c.k.view(torch.uint8), c.v.view(torch.uint8))]
            + [x.clone() for x in s.states.values()] + [x.clone() for x in s.convs.values()] + [s.lens.clone()])


@devices
def test_accept_refuses_what_is_no_path(dev):
    """Siblings, skipped or repeated ancestors, entries below -1: nothing changes, in particular
    not the next sequence's pages."""
    s = decode.DecodeSession(stage_of(dev), 2, 16, page_size=16)
    s.prompt(torch.zeros(2, 8, dtype=torch.int64))
    parents = i32([-1, 0, 0, 1], "cpu")
    s.verify(torch.zeros(2, 4, dtype=torch.int64), parents)
    before = snapshot(s)
    good = [0, 1, 3]
    for bad in ([1], [0, 3], [0, 0], [0, 1, 2], [0, -2], [4], [1, 0], [0] * 9, [0, 2, 3]):
        n = max(len(bad), 3)
        rows = [good + [-1] * (n - 3), bad + [-1] * (n - len(bad))]
        with pytest.raises(ValueError):
            s.accept(i32(rows, "cpu"))
        assert all(torch.equal(a, b) for a, b in zip(before, snapshot(s)))
    parents.fill_(-1)  # the session has its own
    s.accept(torch.tensor([[0, 0], [1, 2], [3, -1]]).T)  # the tree is still there; any integer type and strides will do
    assert s.lens.tolist() == [11, 10]


def test_prompt_drops_the_last_tree():
    s = decode.DecodeSession(stage_of("cpu"), 1, 32)
    s.verify(torch.zeros(1, 2, dtype=torch.int64), i32([-1, 0], "cpu"))
    s.prompt(torch.zeros(1, 8, dtype=torch.int64))
    with pytest.raises(ValueError):
        s.accept(i32([[0, 1]], "cpu"))


@devices
def test_session_without_convolution_history(dev):
    """A convolution of width 1 keeps no inputs."""
    stage = stage_of(dev, kernel=1)
    gen = torch.Generator().manual_seed(2)
    ids = torch.randint(0, stage.config["vocab_size"], (1, 12), generator=gen)
    s = decode.DecodeSession(stage, 1, 64, quantize=False)
    s.prompt(ids[:, :8])
    for i in range(8, 12):
        logits = s.verify(ids[:, i:i + 1], i32([-1], "cpu"))
        s.accept(i32([[0]], "cpu"))
    assert all(c.shape[1] == 0 for c in s.convs.values())
    x, _ = V.stage_forward(stage, ids.to(dev))
    want = (x.float() @ stage.lm_head.weight.float().T).cpu()[0, -1]
    got = logits[0, 0].float().cpu()
    assert torch.nn.functional.cosine_similarity(got, want, dim=0) > (0.99 if dev == "cuda" else 0.99999)

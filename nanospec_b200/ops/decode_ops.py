"""Decoding ops of the hybrid verifier: a paged K/V cache that quantises, attention of a
tree of drafted tokens over it, and the gated delta rule from a carried state.

One step of speculative decoding runs, per layer, ``tree_attention`` or
``gated_delta_verify`` over T drafted nodes (T = 1 is plain decoding); once the accepted
path is known, ``cache_write`` keeps its K/V rows and ``gated_delta_accept`` moves the
state on. Prompts go through ``gated_delta_advance``. The reference runs its verifier over
whole sequences from an empty state only (nanospec/train.py:53-157).

CUDA tensors run the sm_100a kernels of ``nanospec_b200._C`` on the current stream (bf16
activations, fp32 decays and states); CPU tensors run the statements in
``ops.reference``. Bad shapes, types and layouts raise ``ValueError``. Bad *values* of
index tensors (slots, page tables, lengths, parents, counts, paths) cannot be seen without
waiting for the GPU: there the kernels skip the access (a page that does not exist is
replaced by page 0 in ``tree_attention``) and set the device error word (code 4, see
``utils.health``); on the CPU they raise ``IndexError``.

Index tensors are int32 (``slots`` int64). Nodes at or beyond ``counts`` are padding: their
inputs are not used, their outputs are zeros (lse -inf).
"""

from __future__ import annotations

import torch

from . import reference as ref
from ._ext import cuda_ops

MAX_NODES = 64  # nodes of one tree: one attention key tile, one block of the delta rule


def _c():
    return cuda_ops()


def _need(ok, message):
    if not ok:
        raise ValueError("nanospec_b200: " + message)


class PagedCache:
    """K/V rows of one attention layer in pages: ``k``, ``v`` [pages, heads, page_size, D].

    bf16 pages hold the rows as they are. e4m3 pages (``torch.float8_e4m3fn``) hold codes
    and, per (row, head), one power-of-two scale as an exponent byte in ``k_exp`` /
    ``v_exp`` [pages, heads, page_size] (uint8, bias 127). Slot ``s`` is row
    ``s % page_size`` of page ``s // page_size``. Which pages a sequence owns is the
    caller's page table; pages need no initial values.
    """

    __slots__ = ("k", "v", "k_exp", "v_exp")

    def __init__(self, k, v, k_exp=None, v_exp=None):
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        if not k.is_cuda:  # CUDA pages are checked by every kernel call
            self.check()

    @classmethod
    def allocate(cls, pages, heads, page_size, head_dim, *, dtype=torch.bfloat16, device="cuda"):
        """Uninitialised pages; ``dtype`` torch.float8_e4m3fn makes the cache quantise."""
        shape = (pages, heads, page_size, head_dim)
        new = lambda s, t: torch.empty(s, dtype=t, device=device)  # noqa: E731
        exps = [new(shape[:3], torch.uint8) if dtype == torch.float8_e4m3fn else None for _ in range(2)]
        cache = cls(new(shape, dtype), new(shape, dtype), *exps)
        cache.check()
        return cache

    def check(self):
        k, v = self.k, self.v
        _need(k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype, "cache: k and v pages differ")
        _need(k.is_contiguous() and v.is_contiguous(), "cache: pages must be contiguous")
        _need(k.shape[2] in (16, 32, 64, 128), "cache: page_size must be 16, 32, 64 or 128")
        _need(k.shape[3] % 16 == 0 and 16 <= k.shape[3] <= 256, "cache: head_dim must be a multiple of 16 up to 256")
        if k.dtype == torch.float8_e4m3fn:
            for e in (self.k_exp, self.v_exp):
                _need(e is not None and e.dtype == torch.uint8 and e.shape == k.shape[:3] and e.is_contiguous(),
                      "cache: e4m3 pages need uint8 exponents [pages, heads, page_size]")
        else:
            _need(k.dtype.is_floating_point and k.dtype.itemsize > 1, "cache: pages must be bfloat16 or float8_e4m3fn")
            _need(self.k_exp is None and self.v_exp is None, "cache: only e4m3 pages have exponents")

    @property
    def page_size(self):
        return self.k.shape[2]


def cache_write(cache, k, v, slots):
    """Write token rows k, v [n, Hk, D] into ``slots`` [n] int64, quantising on the way into
    e4m3 pages. A slot of -1 drops its row; slots must not repeat within a call."""
    if k.is_cuda:
        _c().cache_write(cache.k, cache.v, cache.k_exp, cache.v_exp, k, v, slots)
        return
    pages, heads, page, d = cache.k.shape
    _need(k.shape == v.shape and k.dim() == 3 and k.shape[1:] == (heads, d), "cache_write: k and v must be [n, heads, D]")
    _need(slots.shape == k.shape[:1] and slots.dtype == torch.int64, "cache_write: slots must be int64 [n]")
    _check_range(slots, -1, pages * page, "slots")
    keep = slots >= 0
    s = slots[keep]
    for x, pool, exps in ((k, cache.k, cache.k_exp), (v, cache.v, cache.v_exp)):
        rows = x[keep]
        if exps is not None:
            rows, e = ref.cache_encode(rows)
            exps[s // page, :, s % page] = e
            pool, rows = pool.view(torch.uint8), rows.view(torch.uint8)
        pool[s // page, :, s % page] = rows.to(pool.dtype)


def cache_read(cache, table, lens, length, starts=None):
    """Read positions ``[starts[i], starts[i] + length)`` of every sequence back: bf16 k, v
    [b, length, Hk, D], zeros at and beyond ``lens[i]``. table [b, max_pages], lens and
    starts [b] (None: 0)."""
    if cache.k.is_cuda:
        return _c().cache_read(cache.k, cache.v, cache.k_exp, cache.v_exp, table, lens, starts, int(length))
    b = _check_table(cache, table, lens)
    _need(length >= 0, "cache_read: length must not be negative")
    _need(starts is None or (starts.shape == (b,) and starts.dtype == torch.int32), "cache_read: starts must be int32 [b]")
    page = cache.page_size
    first = torch.zeros_like(lens) if starts is None else starts
    _check_range(first, 0, 1 << 31, "starts")
    pos = first[:, None].long() + torch.arange(length)
    seen = pos < lens[:, None]
    pg = torch.gather(table.long(), 1, torch.where(seen, pos // page, 0)) if table.shape[1] else torch.zeros_like(pos)
    _check_range(pg[seen], 0, cache.k.shape[0], "page table")
    pg = torch.where(seen, pg, 0)
    out = []
    for pool, exps in ((cache.k, cache.k_exp), (cache.v, cache.v_exp)):
        if not seen.any():
            x = torch.zeros(*pos.shape, pool.shape[1], pool.shape[3])
        elif exps is not None:
            x = ref.cache_decode(pool.view(torch.uint8)[pg, :, pos % page].view(pool.dtype), exps[pg, :, pos % page])
        else:
            x = pool[pg, :, pos % page].float()
        x = torch.where(seen[..., None, None], x, torch.zeros(()))
        out.append(x.to(torch.bfloat16 if exps is not None else pool.dtype))
    return tuple(out)


def tree_attention(q, k, v, cache, table, lens, parents, counts=None, gate=None, scale=None):
    """Attention of T drafted nodes per sequence over the cached prefix and their ancestors.

    q [b, T, Hq, D] and the nodes' own k, v [b, T, Hk, D] (normalised and rotated, not yet
    in the cache); ``cache`` with table [b, max_pages] and lens [b]; parents [b, T] or [T]:
    the node before each node, -1 for children of the last cached token, parents[t] < t.
    Node t sees positions [0, lens) and itself and its ancestors. ``gate`` [b, T, Hq, D],
    when given, multiplies the output by sigmoid(gate); ``scale`` defaults to D^-1/2.
    Strided views are taken as they are when D is contiguous and rows are 16-byte aligned.
    Live nodes' k and v must be finite: a product with a masked one's zero probability is
    still formed. (Whatever lies in pages beyond ``lens`` or in padding nodes is not used.)
    In a quantised cache, on the GPU, terms p_j v_j whose probability times V scale is below
    2^-28 of the row's largest are dropped.

    Returns (out [b, T, Hq, D], lse [b, Hq, T] fp32, natural log, before the gate).
    """
    if q.is_cuda:
        return _c().tree_attention(q, k, v, cache.k, cache.v, cache.k_exp, cache.v_exp, table, lens, parents, counts,
                                   gate, scale)
    b, t, hq, d = q.shape
    _need(k.shape == v.shape == (b, t, cache.k.shape[1], cache.k.shape[3]) and d == cache.k.shape[3],
          "tree_attention: k and v must be [b, T, Hk, D] like the cache")
    _need(hq >= 1 and k.shape[2] >= 1 and hq % k.shape[2] == 0, "tree_attention: query heads must be a multiple of key heads")
    _need(gate is None or gate.shape == q.shape, "tree_attention: gate must have q's shape")
    _need(scale is None or scale > 0, "tree_attention: scale must be positive")
    _check_table(cache, table, lens)
    _need(len(lens) == b, "tree_attention: one length per sequence")
    parents, counts = _check_tree(parents, counts, b, t)
    pk, pv = cache_read(cache, table, lens, int(lens.max()) if b else 0)
    return ref.tree_attention(q, k, v, pk, pv, lens, ref.tree_ancestors(parents, counts), gate,
                              d ** -0.5 if scale is None else scale)


def gated_delta_advance(q, k, v, g, beta, state, groups=1, counts=None, rows=None, out_state=None):
    """The gated delta rule over T tokens from a carried state (any T >= 1; T = 1 decodes).

    Like ``verifier_ops.gated_delta_rule`` (q, k [b, T, nk, D] raw, v [b, T, nv, D], g fp32
    and beta [b, T, nv], value head h using key head h // groups), but in fp32 throughout,
    starting from ``state`` fp32 [n, nv, D, D] (key channel, value channel). Sequence i
    uses row ``rows[i]`` (None: i; -1: an idle sequence, zero outputs; rows must not repeat)
    and its first ``counts[i]`` tokens. The new states go to the same rows of ``out_state``
    (None: to ``state``, in place; otherwise memory apart from it). Returns
    (out [b, T, nv, D], out_state).
    """
    out_state = state if out_state is None else out_state
    if q.is_cuda:
        return _c().gdn_advance(q, k, v, g, beta, state, int(groups), counts, rows, out_state), out_state
    b, t = _check_delta(q, k, v, g, beta, state, groups)
    _check_out_state(state, out_state)
    chain = torch.arange(-1, t - 1, dtype=torch.int32)
    chain, counts = _check_tree(chain, counts, b, t, limit=False)
    live, rows = _check_rows(rows, b, state)
    r = lambda x: x.repeat_interleave(groups, 2)  # noqa: E731
    out, _, last = ref.gated_delta_nodes(r(q), r(k), v, g, beta, state[rows], chain, torch.where(live, counts, 0))
    out_state[rows[live]] = last[live]
    return out, out_state


def gated_delta_verify(q, k, v, g, beta, state, parents, groups=1, counts=None, rows=None):
    """The gated delta rule over a tree of T <= 64 drafted nodes; ``state`` stays as it is.

    Arguments as in ``gated_delta_advance`` and ``tree_attention``: node t continues from
    the state of node parents[t] (-1: ``state``). Returns (out [b, T, nv, D], u fp32
    [b, T, nv, D]); u holds the rows that the nodes would add, for ``gated_delta_accept``.
    Live nodes' inputs must be finite (g may be -inf): on the GPU a node that is not an
    ancestor is multiplied by zero. Padding nodes are not used.
    """
    if q.is_cuda:
        return _c().gdn_verify(q, k, v, g, beta, state, parents, int(groups), counts, rows)
    b, t = _check_delta(q, k, v, g, beta, state, groups)
    parents, counts = _check_tree(parents, counts, b, t)
    live, rows = _check_rows(rows, b, state)
    r = lambda x: x.repeat_interleave(groups, 2)  # noqa: E731
    out, u, _ = ref.gated_delta_nodes(r(q), r(k), v, g, beta, state[rows], parents, torch.where(live, counts, 0))
    return out, u


def gated_delta_accept(k, g, u, path, state, groups=1, rows=None, out_state=None):
    """Move ``state`` on along the accepted nodes ``path`` [b, m <= 64] of a verified tree
    (root first, -1 entries skipped): S <- e^{g_a} S + k_a u_a^T. k and g as given to
    ``gated_delta_verify``, u as it returned it. In place unless ``out_state`` (memory apart
    from ``state``) is given; ``rows`` must not repeat. Returns the new states."""
    out_state = state if out_state is None else out_state
    if k.is_cuda:
        _c().gdn_accept(k, g, u, path, state, int(groups), rows, out_state)
        return out_state
    b, t, nk, d = k.shape
    nv = nk * groups
    _need(u.shape == (b, t, nv, d) and u.dtype == torch.float32, "gated_delta_accept: u must be fp32 [b, T, nv, D]")
    _need(g.shape == (b, t, nv), "gated_delta_accept: g must be [b, T, nv]")
    _need(path.dim() == 2 and path.shape[0] == b and path.dtype == torch.int32,
          "gated_delta_accept: path must be int32 [b, m]")
    _need(t <= MAX_NODES and path.shape[1] <= MAX_NODES, "gated_delta_accept: at most 64 nodes, and path entries")
    _need(state.dim() == 4 and state.shape[1:] == (nv, d, d) and state.dtype == torch.float32,
          "gated delta rule: state must be fp32 [n, nv, D, D]")
    _check_out_state(state, out_state)
    _check_range(path, -1, t, "path")
    live, rows = _check_rows(rows, b, state)
    new = ref.gated_delta_accept(k.repeat_interleave(groups, 2), g, u, path, state[rows])
    out_state[rows[live]] = new[live]
    return out_state


# ------------------------------------------------------------------ checks of the CPU statements
def _check_range(t, lo, hi, name):
    if t.numel() and (int(t.min()) < lo or int(t.max()) >= hi):
        raise IndexError(f"nanospec_b200: {name} out of range")


def _check_table(cache, table, lens):
    cache.check()
    b = lens.shape[0]
    _need(lens.dim() == 1 and lens.dtype == torch.int32, "lens must be int32 [b]")
    _need(table.dim() == 2 and table.shape[0] == b and table.dtype == torch.int32,
          "table must be int32 [b, max_pages]")
    _check_range(lens, 0, table.shape[1] * cache.page_size + 1, "lens")
    return b


def _check_tree(parents, counts, b, t, limit=True):
    _need(parents.dtype == torch.int32 and parents.shape in ((t,), (b, t)), "parents must be int32 [T] or [b, T]")
    _need(counts is None or (counts.shape == (b,) and counts.dtype == torch.int32), "counts must be int32 [b]")
    _need(t >= 1 and (t <= MAX_NODES or not limit), f"a tree has 1 to {MAX_NODES} nodes")
    parents = parents.expand(b, t)
    if counts is None:
        counts = torch.full((b,), t, dtype=torch.int32)
    _check_range(counts, 0, t + 1, "counts")
    used = torch.arange(t) < counts[:, None]
    if bool((used & ((parents < -1) | (parents >= torch.arange(t)))).any()):
        raise IndexError("nanospec_b200: parents must come before their children")
    return torch.where(used, parents, -1), counts


def _check_delta(q, k, v, g, beta, state, groups):
    _need(q.dim() == 4 and v.dim() == 4, "gated delta rule: q, k, v must be [b, T, heads, D]")
    b, t, nk, d = q.shape
    nv = nk * groups
    _need(k.shape == q.shape and v.shape == (b, t, nv, d), "gated delta rule: k must have q's shape, v groups * nk heads")
    _need(g.shape == beta.shape == (b, t, nv) and g.dtype == torch.float32,
          "gated delta rule: g (fp32) and beta must be [b, T, nv]")
    _need(d in (16, 32, 64, 128), "gated delta rule: head_dim must be 16, 32, 64 or 128")
    _need(state.dim() == 4 and state.shape[1:] == (nv, d, d) and state.dtype == torch.float32,
          "gated delta rule: state must be fp32 [n, nv, D, D]")
    return b, t


def _check_out_state(state, out_state):
    _need(out_state.shape == state.shape and out_state.dtype == state.dtype,
          "gated delta rule: out_state must be like state")
    n, row, sx, sy = state.shape[0], state.shape[1:].numel(), state.stride(0), out_state.stride(0)
    _need(n <= 1 or sy >= row, "gated delta rule: rows of out_state overlap")
    off = (out_state.data_ptr() - state.data_ptr()) // 4
    same = off == 0 and (n <= 1 or sx == sy)
    apart = n == 0 or off >= (n - 1) * sx + row or -off >= (n - 1) * sy + row  # or rows interleave
    apart = apart or (n > 1 and sx == sy >= 2 * row and row <= off % sx <= sx - row)
    _need(same or apart, "gated delta rule: out_state must be state or lie apart from it")


def _check_rows(rows, b, state):
    if rows is None:
        _need(state.shape[0] == b, "gated delta rule: one state per sequence, or rows")
        return torch.ones(b, dtype=torch.bool), torch.arange(b)
    _need(rows.shape == (b,) and rows.dtype == torch.int32, "gated delta rule: rows must be int32 [b]")
    _check_range(rows, -1, state.shape[0], "rows")
    return rows >= 0, rows.long().clamp_min(0)

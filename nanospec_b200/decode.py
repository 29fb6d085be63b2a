"""Speculative decoding with the hybrid verifier: a session that keeps sequences' caches and states.

``DecodeSession`` holds, for a batch of sequences, one paged K/V cache per attention layer
(bf16, or e4m3 quantised as it is written), and per gated-delta layer the fp32 state and the
last inputs of the causal convolution. A step is

    logits = session.verify(tokens, parents)     # a tree of drafted tokens; nothing is kept
    path, token = greedy_path(tokens, parents, logits)
    session.accept(path)                         # keep the accepted nodes

Node 0 of a tree is the last token already sampled (its K/V is not cached yet), so plain
decoding is a tree of one node. ``prompt`` fills an empty session. The same statements run
on CPU tensors (plain torch) and on CUDA tensors (this repository's kernels); see
``ops.decode_ops`` for the operators. The reference verifies whole sequences only
(nanospec/train.py:53-157).

Example: ``python -m nanospec_b200.decode`` decodes with a small random verifier.
"""

from __future__ import annotations

import torch

from .models.verifier import QwenStage
from .ops import decode_ops as dops
from .ops import verifier_ops as vops


def tree_depths(parents):
    """Depth of every node (0: children of the last cached token) of parents [T] or [b, T] on the CPU."""
    p = parents.reshape(-1, parents.shape[-1])
    depth = torch.zeros_like(p)
    rows = torch.arange(p.shape[0])
    for t in range(p.shape[1]):
        up = p[:, t].long()
        if bool(((up < -1) | (up >= t)).any()):
            raise ValueError("nanospec_b200: parents must come before their children")
        depth[:, t] = torch.where(up < 0, 0, depth[rows, up.clamp_min(0)] + 1)
    return depth.view_as(parents)


def path_end(parents, path):
    """Last node (-1: none) of every row of path [b, m], which must be a way down the tree
    parents [b, T]: root first, each node the child of the one before, -1 skipped. On the CPU."""
    b, t = parents.shape
    if path.dim() != 2 or path.shape[0] != b or path.is_floating_point():
        raise ValueError("nanospec_b200: path must be integers [b, m], a row per sequence")
    if path.shape[1] > dops.MAX_NODES or bool(((path < -1) | (path >= t)).any()):
        raise ValueError("nanospec_b200: path must name nodes of the last tree, or -1")
    last = torch.full((b,), -1, dtype=torch.int64)
    for node in path.long().unbind(1):
        up = parents.gather(1, node.clamp_min(0)[:, None])[:, 0]
        if bool(((node >= 0) & (up != last)).any()):
            raise ValueError("nanospec_b200: path must lead from the last cached token down the tree")
        last = torch.where(node >= 0, node, last)
    return last


def greedy_path(tokens, parents, logits):
    """The nodes that greedy decoding keeps, and its next token.

    tokens [b, T] and parents [T] or [b, T] on the CPU, logits [b, T, V]. From node 0 on, a
    child is kept when its token is the argmax of its parent's logits. Returns (paths [b, m]
    int32 padded with -1, next tokens [b]) on the CPU.
    """
    best = logits.argmax(-1).cpu()
    b, t = tokens.shape
    parents = parents.expand(b, t)
    paths, nxt = [], []
    for i in range(b):
        at, path = 0, [0]
        while True:
            want = int(best[i, at])
            kids = [n for n in range(at + 1, t) if int(parents[i, n]) == at and int(tokens[i, n]) == want]
            if not kids:
                break
            at = kids[0]
            path.append(at)
        paths.append(path)
        nxt.append(int(best[i, at]))
    m = max(map(len, paths))
    return (torch.tensor([p + [-1] * (m - len(p)) for p in paths], dtype=torch.int32),
            torch.tensor(nxt, dtype=torch.int64))


class DecodeSession:
    """Caches and states of ``batch`` sequences of up to ``max_tokens`` tokens each.

    ``stage``: a whole verifier (embedding, all layers, norm and LM head). ``quantize``
    keeps K/V as e4m3. Sequence i owns pages [i * n, (i + 1) * n) of every layer's cache.
    """

    def __init__(self, stage: QwenStage, batch: int, max_tokens: int, *, page_size=64, quantize=True):
        if stage.embed_tokens is None or stage.norm is None or stage.lm_head is None:
            raise ValueError("nanospec_b200: decoding needs the whole verifier in one stage")
        tc = stage.config
        w = stage.embed_tokens.weight
        self.stage, self.batch, self.max_tokens = stage, batch, max_tokens
        self.device, self.dtype = w.device, w.dtype
        pages = -(-max_tokens // page_size)
        self.page_size = page_size
        self.table = torch.arange(batch * pages, dtype=torch.int32, device=self.device).view(batch, pages)
        self.lens = torch.zeros(batch, dtype=torch.int32)  # on the host; a device copy goes with each step
        kv_type = torch.float8_e4m3fn if quantize else self.dtype
        self.caches, self.states, self.convs = {}, {}, {}
        for i, layer in enumerate(stage.layers):
            if layer.linear_attn is not None:
                a = layer.linear_attn
                d = a.key_head_dim
                if d != a.value_head_dim:
                    raise ValueError("nanospec_b200: decoding needs equal key and value head sizes")
                self.states[i] = torch.zeros(batch, a.num_value_heads, d, d, device=self.device)
                conv = 2 * a.num_key_heads * d + a.num_value_heads * d
                self.convs[i] = torch.zeros(batch, a.conv1d.weight.shape[-1] - 1, conv, device=self.device,
                                            dtype=self.dtype)
            else:
                a = layer.self_attn
                self.caches[i] = dops.PagedCache.allocate(batch * pages, a.num_key_value_heads, page_size, a.head_dim,
                                                          dtype=kv_type, device=self.device)
        self.pending = None

    # ------------------------------------------------------------------ steps
    @torch.no_grad()
    def prompt(self, ids):
        """Run prompts ids [b, s] through an empty session; returns the last token's logits [b, V]."""
        if int(self.lens.max()) or ids.shape[0] != self.batch:
            raise ValueError("nanospec_b200: prompt() fills an empty session, one row per sequence")
        b, s = ids.shape
        self._fit(s)
        self.pending = None  # a tree over the empty session is none of this prompt's
        pos = torch.arange(s).expand(b, s)
        x = self._run(ids, pos, lambda i, attn, n: self._prompt_gdn(i, attn, n),
                      lambda i, attn, qg, k, v, cos, sin: self._prompt_attention(i, attn, qg, k, v, cos, sin))
        self.lens += s
        return self._logits(x[:, -1:])[:, 0]

    @torch.no_grad()
    def verify(self, tokens, parents):
        """Logits [b, T, V] of a tree of drafted tokens [b, T]; parents [T] or [b, T] (on the CPU,
        int32, -1: child of the last cached token). Kept until ``accept``."""
        b, t = tokens.shape
        if b != self.batch:
            raise ValueError("nanospec_b200: one tree per sequence")
        depth = tree_depths(parents).expand(b, t)
        self._fit(int(depth.max()) + 1)
        dev = self.device
        par = parents.to(torch.int32).expand(b, t).clone(memory_format=torch.contiguous_format)  # kept until accept()
        step = dict(tree=par, parents=par.to(dev), lens=self.lens.to(dev), windows=self._windows(par), layers={})
        x = self._run(tokens, self.lens[:, None] + depth, lambda i, attn, n: self._tree_gdn(step, i, attn, n),
                      lambda i, attn, qg, k, v, cos, sin: self._tree_attention(step, i, attn, qg, k, v, cos, sin))
        self.pending = step
        return self._logits(x)

    @torch.no_grad()
    def accept(self, path):
        """Keep the nodes ``path`` [b, m] (on the CPU, root first, -1 padding) of the last tree.

        Every row's nodes must be a way down from the last cached token (each the child of the
        one before); anything else raises ``ValueError`` and changes nothing.
        """
        step = self.pending
        if step is None:
            raise ValueError("nanospec_b200: accept() follows verify()")
        last = path_end(step["tree"], path)
        path = path.to(torch.int32).contiguous()
        self.pending = None
        b = path.shape[0]
        on = path >= 0
        # slots of the kept nodes: positions after the cached ones, in the order of the path
        at = self.lens[:, None].long() + on.long().cumsum(1) - 1
        slots = self._slots(torch.where(on, at, -1))
        node = path.clamp_min(0).long().to(self.device)
        dpath = path.to(self.device)
        rows = torch.arange(b, device=self.device)[:, None]
        # the convolution's inputs end with the last kept node (its window is the new tail)
        tail = self._tail(step["windows"], last).to(self.device)
        for i, keep in step["layers"].items():
            if i in self.caches:
                k, v = keep
                dops.cache_write(self.caches[i], k[rows, node].flatten(0, 1), v[rows, node].flatten(0, 1), slots)
            else:
                k, g, u, groups, raw = keep
                dops.gated_delta_accept(k, g, u, dpath, self.states[i], groups)
                self.convs[i] = raw[rows, tail].contiguous()
        self.lens += on.sum(1).to(torch.int32)

    # ------------------------------------------------------------------ the verifier's layers
    def _run(self, ids, pos, gdn, attention):
        x = vops.embedding(ids.to(self.device), self.stage.embed_tokens.weight)
        tables = {}
        for i, layer in enumerate(self.stage.layers):
            n = vops.qwen_norm(x, layer.input_layernorm.weight, layer.input_layernorm.eps)
            if layer.linear_attn is not None:
                out = gdn(i, layer.linear_attn, n)
            else:
                attn = layer.self_attn
                key = (attn.rotary_dim, attn.rope_theta)
                if key not in tables:
                    tables[key] = vops.rotary_factors(pos.to(self.device), *key, n.dtype)
                b, s, _ = n.shape
                d, hq, hk = attn.head_dim, attn.num_heads, attn.num_key_value_heads
                qg = _linear(n, attn.q_proj).view(b, s, hq, 2 * d)
                k, v = _linear(n, attn.k_proj).view(b, s, hk, d), _linear(n, attn.v_proj).view(b, s, hk, d)
                o = attention(i, attn, qg, k, v, *tables[key])
                out = _linear(o.reshape(b, s, hq * d), attn.o_proj)
            x = vops.add(x, out)
            n = vops.qwen_norm(x, layer.post_attention_layernorm.weight, layer.post_attention_layernorm.eps)
            mlp = layer.mlp
            x = vops.add(x, _linear(vops.silu_mul(_linear(n, mlp.gate_proj), _linear(n, mlp.up_proj)), mlp.down_proj))
        return x

    def _logits(self, x):
        x = vops.qwen_norm(x, self.stage.norm.weight, self.stage.norm.eps)
        return vops.fp8_linear(x, self.stage.lm_head.weight, None)

    def _project(self, attn, n):
        mixed = _linear(n, attn.in_proj_qkv)
        z, bp, ap = _linear(n, attn.in_proj_z), _linear(n, attn.in_proj_b), _linear(n, attn.in_proj_a)
        g, beta = vops.gdn_gates(ap, bp, attn.A_log, attn.dt_bias)
        return mixed, z, g, beta

    def _heads(self, attn, mixed):
        nk, nv, d = attn.num_key_heads, attn.num_value_heads, attn.key_head_dim
        q, k, v = mixed.split((nk * d, nk * d, nv * d), -1)
        return q.unflatten(-1, (nk, d)), k.unflatten(-1, (nk, d)), v.unflatten(-1, (nv, d)), nv // nk

    def _output(self, attn, out, z):
        b, s, nv, d = out.shape
        out = vops.qwen_gated_norm(out.reshape(-1, d), z.reshape(-1, d), attn.norm.weight, attn.norm.eps)
        return _linear(out.reshape(b, s, nv * d), attn.out_proj)

    def _prompt_gdn(self, i, attn, n):
        mixed, z, g, beta = self._project(attn, n)
        q, k, v, groups = self._heads(attn, vops.causal_conv_silu(mixed, attn.conv1d.weight))
        out, _ = dops.gated_delta_advance(q, k, v, g, beta, self.states[i], groups)
        self.convs[i] = torch.cat((self.convs[i], mixed), 1)[:, mixed.shape[1]:].contiguous()
        return self._output(attn, out, z)

    def _tree_gdn(self, step, i, attn, n):
        b, t, _ = n.shape
        mixed, z, g, beta = self._project(attn, n)
        raw = torch.cat((self.convs[i], mixed), 1)
        # the convolution's window of node t: itself and the inputs before it on its own path
        win = step["windows"].to(self.device)
        rows = torch.arange(b, device=self.device)[:, None, None]
        w = raw[rows, win].flatten(0, 1)  # [b * T, K, C]: one short sequence per node
        conv = vops.causal_conv_silu(w, attn.conv1d.weight)[:, -1].view(b, t, -1)
        q, k, v, groups = self._heads(attn, conv)
        out, u = dops.gated_delta_verify(q, k, v, g, beta, self.states[i], step["parents"], groups)
        step["layers"][i] = (k, g, u, groups, raw)
        return self._output(attn, out, z)

    def _rotated(self, attn, qg, k, cos, sin):
        d, rd = attn.head_dim, attn.rotary_dim
        return (vops.head_norm_partial_rope(qg[..., :d], attn.q_norm.weight, attn.q_norm.eps, cos, sin, rd),
                vops.head_norm_partial_rope(k, attn.k_norm.weight, attn.k_norm.eps, cos, sin, rd))

    def _prompt_attention(self, i, attn, qg, k, v, cos, sin):
        b, s = qg.shape[:2]
        _, kr = self._rotated(attn, qg, k, cos, sin)
        slots = self._slots(torch.arange(s).expand(b, s))
        dops.cache_write(self.caches[i], kr.flatten(0, 1), v.flatten(0, 1), slots)
        return vops.gated_attention(qg, k, v, attn.q_norm.weight, attn.k_norm.weight, attn.q_norm.eps, cos, sin,
                                    attn.rotary_dim)

    def _tree_attention(self, step, i, attn, qg, k, v, cos, sin):
        q, kr = self._rotated(attn, qg, k, cos, sin)
        out, _ = dops.tree_attention(q, kr, v, self.caches[i], self.table, step["lens"], step["parents"],
                                     gate=qg[..., attn.head_dim:])
        step["layers"][i] = (kr, v)
        return out

    # ------------------------------------------------------------------ positions
    def _fit(self, more):
        if int(self.lens.max()) + more > self.max_tokens:
            raise ValueError("nanospec_b200: the session's max_tokens are used up")

    def _slots(self, pos):
        """int64 slots (flattened, on the device) of positions [b, n] on the CPU; -1 stays -1."""
        first = torch.arange(self.batch)[:, None] * self.table.shape[1] * self.page_size
        return torch.where(pos < 0, -1, first + pos).reshape(-1).to(self.device)

    def _kernel(self):
        sizes = {c.shape[1] + 1 for c in self.convs.values()}
        if len(sizes) > 1:
            raise ValueError("nanospec_b200: convolutions of different widths")
        return sizes.pop() if sizes else 1

    def _windows(self, parents):
        """[b, T, K] rows of (kept inputs, nodes) that each node's convolution reads, oldest first."""
        b, t = parents.shape
        kk = self._kernel()
        up = torch.cat((torch.arange(-1, kk - 2).expand(b, kk - 1), parents.long() + kk - 1), 1)
        at = torch.arange(kk - 1, kk - 1 + t).expand(b, t)
        win = [at]
        for _ in range(kk - 1):
            win.append(up.gather(1, win[-1]))
        return torch.stack(win[::-1], -1)

    def _tail(self, windows, last):
        """[b, K - 1] rows of (kept inputs, nodes) that stay after node ``last`` (-1: none accepted)."""
        kk = windows.shape[-1]
        rows = torch.arange(len(last))
        return torch.where((last < 0)[:, None], torch.arange(kk - 1)[None], windows[rows, last.clamp_min(0)][:, 1:])


def _linear(x, lin):
    return vops.fp8_linear(x, lin.weight, lin.weight_scale_inv)


def main(argv=None):
    """Greedy decoding with random drafted trees against a small random verifier."""
    import argparse

    from .models.verifier import random_verifier_weights, synthetic_hf_config, tiny_hybrid_text_config

    p = argparse.ArgumentParser(description=main.__doc__)
    p.add_argument("--device", default="cuda" if torch.cuda.is_available() else "cpu")
    p.add_argument("--steps", type=int, default=16)
    p.add_argument("--nodes", type=int, default=12)
    a = p.parse_args(argv)
    tc = tiny_hybrid_text_config(head_dim=32)
    dtype = torch.bfloat16 if a.device.startswith("cuda") else torch.float32
    w = random_verifier_weights(tc, 0, tc["num_hidden_layers"], device=a.device, first=True, last=True, dtype=dtype,
                                std=0.3)
    stage = QwenStage(None, 0, tc["num_hidden_layers"], device=a.device, first=True, last=True, weights=w,
                      config=synthetic_hf_config(tc))
    gen = torch.Generator().manual_seed(0)
    batch, vocab = 4, tc["vocab_size"]
    ids = torch.randint(0, vocab, (batch, 40), generator=gen)
    session = DecodeSession(stage, batch, 40 + a.steps * a.nodes)
    token = session.prompt(ids).argmax(-1).cpu()
    kept = 0
    for _ in range(a.steps):
        # a drafted tree: the last token, then random continuations below random nodes
        parents = torch.tensor([-1] + [int(torch.randint(0, n, (), generator=gen)) for n in range(1, a.nodes)],
                               dtype=torch.int32)
        tokens = torch.randint(0, vocab, (batch, a.nodes), generator=gen)
        tokens[:, 0] = token
        logits = session.verify(tokens, parents)
        path, token = greedy_path(tokens, parents, logits)
        session.accept(path)
        kept += int((path >= 0).sum())
    print(f"{a.steps} steps, {kept / a.steps / batch:.2f} tokens kept per step, lengths {session.lens.tolist()}")


if __name__ == "__main__":
    main()

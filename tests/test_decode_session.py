"""DecodeSession: verifying trees over cached sequences equals running the verifier over
every root-to-node path from the start."""

import pytest
import torch

from nanospec_b200 import decode
from nanospec_b200.models import verifier as V

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
LAYERS = 4


@pytest.fixture(params=DEVICES)
def stage(request):
    if request.param == "cuda" and not torch.cuda.is_available():
        pytest.skip("needs a CUDA GPU")
    dtype = torch.bfloat16 if request.param == "cuda" else torch.float32
    tc = V.tiny_hybrid_text_config(head_dim=32)
    w = V.random_verifier_weights(tc, 0, LAYERS, device="cpu", first=True, last=True, seed=1, std=0.15, dtype=dtype)
    w = {k: v.to(request.param) for k, v in w.items()}
    yield V.QwenStage(None, 0, LAYERS, device=request.param, first=True, last=True, weights=w,
                      config=V.synthetic_hf_config(tc))
    if request.param == "cuda":
        from nanospec_b200.ops._ext import cuda_ops
        torch.cuda.synchronize()
        assert cuda_ops().device_error() == 0


def full_logits(stage, ids):
    x, _ = V.stage_forward(stage, ids.to(stage.embed_tokens.weight.device))
    return (x.float() @ stage.lm_head.weight.float().T).cpu()


def same(got, want, exact):
    got, want = got.float().cpu(), want.float()
    if exact:  # fp32 on the CPU
        assert torch.allclose(got, want, rtol=1e-3, atol=1e-3 * want.abs().max().item())
    else:  # bf16 activations (and 4-bit significands in a quantised cache) through four layers
        cos = torch.nn.functional.cosine_similarity(got.flatten(), want.flatten(), dim=0).item()
        assert cos > 0.99, cos


@pytest.mark.parametrize("quantize", [False, True])
def test_trees_equal_full_runs(stage, quantize):
    gen = torch.Generator().manual_seed(3)
    vocab, b = stage.config["vocab_size"], 2
    exact = stage.embed_tokens.weight.dtype == torch.float32 and not quantize
    seqs = [row for row in torch.randint(0, vocab, (b, 37), generator=gen)]
    session = decode.DecodeSession(stage, b, 128, page_size=16, quantize=quantize)
    same(session.prompt(torch.stack(seqs)), full_logits(stage, torch.stack(seqs))[:, -1], exact)
    trees = [torch.tensor([-1, 0, 0, 1, 1, 3, 2, 6, 6], dtype=torch.int32), torch.tensor([-1, 0, 1, 2], dtype=torch.int32),
             torch.tensor([-1], dtype=torch.int32)]
    paths = [[[0, 1, 3, 5], [0, 2]], [[0, 1, 2, 3], [0]], [[0], [0]]]
    for parents, kept in zip(trees, paths):
        t = len(parents)
        tokens = torch.randint(0, vocab, (b, t), generator=gen)
        logits = session.verify(tokens, parents)
        assert logits.shape == (b, t, vocab)
        for i in range(b):
            for n in range(t):
                way, at = [], n
                while at >= 0:
                    way.append(at)
                    at = int(parents[at])
                ids = torch.cat((seqs[i], tokens[i, way[::-1]]))[None]
                same(logits[i, n], full_logits(stage, ids)[0, -1], exact)
        m = max(map(len, kept))
        session.accept(torch.tensor([k + [-1] * (m - len(k)) for k in kept], dtype=torch.int32))
        seqs = [torch.cat((s, tokens[i, k])) for i, (s, k) in enumerate(zip(seqs, kept))]
        assert session.lens.tolist() == [len(s) for s in seqs]


def test_greedy_decoding_matches_drafts(stage):
    """A tree that holds the greedy continuation is kept whole; random drafts are not."""
    gen = torch.Generator().manual_seed(5)
    vocab = stage.config["vocab_size"]
    ids = torch.randint(0, vocab, (1, 20), generator=gen)

    def plain(steps):
        s = decode.DecodeSession(stage, 1, 64, quantize=False)
        tok, out = s.prompt(ids).argmax(-1).cpu(), []
        for _ in range(steps):
            out.append(int(tok))
            logits = s.verify(tok.view(1, 1), torch.tensor([-1], dtype=torch.int32))
            path, tok = decode.greedy_path(tok.view(1, 1), torch.tensor([-1]), logits)
            s.accept(path)
        return out

    want = plain(6)
    s = decode.DecodeSession(stage, 1, 64, quantize=False)
    assert int(s.prompt(ids).argmax(-1)) == want[0]
    # want[0] -> (want[1], a wrong token) -> want[2] below the right one
    tokens = torch.tensor([[want[0], (want[1] + 1) % vocab, want[1], want[2]]])
    parents = torch.tensor([-1, 0, 0, 2], dtype=torch.int32)
    path, nxt = decode.greedy_path(tokens, parents, s.verify(tokens, parents))
    if stage.embed_tokens.weight.dtype == torch.float32:  # bf16 logits may tie
        assert path.tolist() == [[0, 2, 3]] and int(nxt) == want[3]
    s.accept(path)


def test_refusals(stage):
    s = decode.DecodeSession(stage, 1, 32)
    with pytest.raises(ValueError):
        s.accept(torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError):
        s.verify(torch.zeros(2, 1, dtype=torch.int64), torch.tensor([-1], dtype=torch.int32))
    with pytest.raises(ValueError):
        s.verify(torch.zeros(1, 2, dtype=torch.int64), torch.tensor([-1, 1], dtype=torch.int32))
    with pytest.raises(ValueError):
        s.prompt(torch.zeros(1, 33, dtype=torch.int64))
    s.verify(torch.zeros(1, 1, dtype=torch.int64), torch.tensor([-1], dtype=torch.int32))
    with pytest.raises(ValueError):
        s.accept(torch.tensor([[1]], dtype=torch.int32))

"""Decoding ops where a size, an address, a scale or a value lies at an edge. Tolerances are those
of test_decode_ops.py."""

import pytest
import torch

from nanospec_b200.ops import decode_ops as dops

from test_decode_ops import BF, Delta, _device_error, devices, near  # noqa: F401

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

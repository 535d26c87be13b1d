"""The expert layer's accuracy as a whole: bounds on single values allow for
terms that all err to one side, a bound on the output's distance does not."""
import math

import pytest

from test_decode_gpu import _gen, _moe64, _randn
from test_decode_limits_cpu import EXPERTS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H,I,E", [(1, 4096, 448, 16), (9, 4096, 448, 16), (61, 4096, 448, 16), (17, 512, 448, 2),
                                     (3, 1001, 333, 7), (128, 1001, 333, 7), (128, 264, 40, 2), (40, 2501, 37, 32)])
@pytest.mark.parametrize("weights", ["float32", "bfloat16"])
@pytest.mark.parametrize("gates", ["equal", "softmax"])
def test_experts_distance_from_64_bits(cuda, T, H, I, E, weights, gates):
    import torch

    from aps2026_b200 import decode

    g, wt = _gen(T + H + I), getattr(torch, weights)
    x, logits = _randn(g, T, H), _randn(g, T, E)
    gate_up = (_randn(g, E, 2 * I, H) / math.sqrt(H)).to(wt)
    down = (_randn(g, E, H, I) / math.sqrt(I)).to(wt)
    out = torch.empty_like(x)
    decode.moe_decode_gpu(x, logits, gate_up, down, out, gates=gates)
    want, _ = _moe64(x, logits, gate_up, down, 1e-3, 2e-2, gates)
    off = (out.double() - want).norm(dim=1) / want.norm(dim=1)
    assert float(off.max()) < EXPERTS

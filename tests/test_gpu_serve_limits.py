"""The serving operators where their numbers end: weights that are none."""

import pytest
import torch

from test_gpu_serve import Drafts, _verify_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [37, 300, 50001])
@pytest.mark.parametrize("shape", ["chain", "tree"])
def test_negative_and_nan_draft_weights_are_zero(device, vocab, shape):
    """A token without any weight of the target's is not accepted because the draft's
    is negative, and gains none from it when others are refused."""
    for seed in range(6):
        d = Drafts([6, 9, 1, 12], vocab, shape, seed, noise=2.0)
        g = torch.Generator()
        g.manual_seed(seed)
        t = len(d.tokens)
        d.p[torch.rand(t, vocab, generator=g) < 0.5] = 0
        kind = torch.rand(t, vocab, generator=g)
        d.q[kind < 0.3] *= -1
        d.q[(kind > 0.3) & (kind < 0.4)] = float("nan")
        d.q[(kind > 0.4) & (kind < 0.45)] = -float("inf")
        # drafted tokens of each kind behind their parents
        d.tokens = torch.randint(0, vocab, (t,), generator=g).tolist()
        want = _verify_oracle(d.p, d.q.nan_to_num(0, neginf=0).clamp(min=0), d.tokens, d.parents, d.au, d.su, d.cu, d.n_max)
        assert d.run(device) == want

"""Log probabilities of tokens: results that do not belong to the call."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402


def test_results_of_another_call():
    """What the backward reads of a result has the size and kind that the forward gave it."""
    x, t = torch.randn(6, 40, device="cuda"), torch.arange(6, device="cuda")
    r = engine.token_logprobs(x, t, top=3)
    g = torch.ones(6, device="cuda")
    engine.token_logprobs_backward(x, t, r, g, g, torch.ones(6, 3, device="cuda"))
    less = engine.token_logprobs(x[:2], t[:2], top=3)
    for bad in (dict(norm=less.norm), dict(entropy=less.entropy), dict(top_indices=less.top_indices),
                dict(norm=r.norm[:, :1]), dict(norm=r.norm.double()), dict(norm=r.norm.half()),
                dict(entropy=r.entropy.half()), dict(top_indices=r.top_indices.int()),
                dict(top_indices=r.top_indices.cpu()), dict(norm=r.norm.cpu()), dict(entropy=r.entropy.cpu()),
                dict(top_indices=r.top_indices[..., :1]), dict(top_indices=r.top_indices.repeat(1, 20)),
                dict(logprob=less.logprob)):
        with pytest.raises(ValueError):
            engine.token_logprobs_backward(x, t, r._replace(**bad), g, g, torch.ones(6, 3, device="cuda"))

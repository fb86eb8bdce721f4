"""Log probabilities of tokens: results that do not belong to the call, ignored rows of anything, second
derivatives."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine, nn  # noqa: E402


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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [70, 5003, 50257])
def test_ignored_rows_may_hold_anything(dtype, vocab):
    """A padded row has no gradient, whatever its logits are; one that an entropy or an alternative counts in has."""
    x = torch.randn(6, vocab, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    t = torch.tensor([3, -100, 5, -100, -100, -100], device="cuda")
    clean = engine.token_logprobs(x, t, top=2)
    g = torch.randn(6, device="cuda")
    weight = (t >= 0).float()
    uses = ((g, None, None), (g, g * weight, None), (g, g * weight, torch.ones(6, 2, device="cuda") * weight[:, None]))
    want = [engine.token_logprobs_backward(x, t, clean, *use) for use in uses]
    x[1] = float("nan")
    x[3, vocab // 2], x[4] = float("inf"), -float("inf")
    got = engine.token_logprobs(x, t, top=2)
    assert not got.logprob[[1, 3, 4]].any()
    for use, ref in zip(uses, want):
        d = engine.token_logprobs_backward(x, t, got, *use)
        assert not d[[1, 3, 4, 5]].any() and torch.equal(d[[0, 2]], ref[[0, 2]])
    ones = torch.ones(6, device="cuda")
    d = engine.token_logprobs_backward(x, t, got, g, ones)
    assert d[1].isnan().all() and d[3].isnan().any() and not d[4].any() and d[5].any()
    d = engine.token_logprobs_backward(x, t, got, g, None, torch.ones(6, 2, device="cuda"))
    assert d[1].isnan().all() and d[5].any()


def test_no_second_derivative():
    """Of a gradient that the kernels made there is none: asked for one, torch raises instead of leaving a term out."""
    x = torch.randn(4, 30, device="cuda", requires_grad=True)
    result = nn.token_logprobs(x, torch.arange(4, device="cuda"))
    (g,) = torch.autograd.grad(result.logprob.sum() + result.entropy.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        (g.square().sum() + x.sum()).backward()

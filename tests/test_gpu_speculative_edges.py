"""Drafted trees through the models: entries of ``parents`` beyond 32 bits, steps that are refused."""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import nn, no_grad  # noqa: E402
from test_gpu_speculative import model  # noqa: E402


@pytest.mark.parametrize("entry", [2**32, 2**32 - 1, -(2**32) - 1, 2**31, 2**63 - 1])
def test_parents_beyond_32_bits_mark_padding(entry):
    lm = model()
    with no_grad(), torch.no_grad():
        lm.eval()
        logits = []
        for odd in (-2, entry):
            caches = lm.new_cache(1)
            lm(torch.tensor([[1, 2, 3, 4, 5]]), caches=caches)
            logits.append(lm(torch.tensor([[6, 7, 8, 9]]), caches=caches, parents=[[-1, 0, odd, 2]]))
    assert torch.equal(*logits)


@pytest.mark.parametrize("parents", [[[-1, 0.5, 1]], [[True, False, True]], [[-1, 0]], [-1, 0, 1]])
def test_parents_that_are_not_integers_a_token(parents):
    lm = model()
    with no_grad(), torch.no_grad():
        caches = lm.eval().new_cache(1)
        lm(torch.tensor([[1, 2]]), caches=caches)
        with pytest.raises(ValueError, match="parents"):
            lm(torch.tensor([[3, 4, 5]]), caches=caches, parents=parents)
        assert caches[0].length == 2


@pytest.mark.parametrize("dtype", [torch.int32, torch.int16, torch.int8])
def test_parents_of_any_integer_type(dtype):
    lm = model()
    parents = torch.tensor([[-1, 0, 0, 100]])
    with no_grad(), torch.no_grad():
        lm.eval()
        logits = []
        for given in (parents, parents.to(dtype)):
            caches = lm.new_cache(1)
            lm(torch.tensor([[1, 2, 3]]), caches=caches)
            logits.append(lm(torch.tensor([[4, 5, 6, 7]]), caches=caches, parents=given))
    assert torch.equal(*logits)


@pytest.mark.parametrize("rotary", [True, False])
def test_a_refused_tree_leaves_the_module_s_cache(rotary):
    np.random.seed(1)
    attention = nn.MultiHeadAttention(64, 4, rotary=rotary, device="cuda").eval()
    cache = nn.KVCache(1, 4, 16, 200)
    x = torch.randn(1, 70, 64, device="cuda")
    int32 = lambda *shape: torch.full(shape, -1, dtype=torch.int32, device="cuda")  # noqa: E731
    with no_grad(), torch.no_grad():
        attention(x[:, :5], cache=cache)
        for steps, parents in ((70, int32(1, 70)), (3, int32(1, 4)), (3, int32(1, 3).long()), (3, int32(2, 3)),
                               (3, int32(1, 3).cpu()), (3, int32(3))):
            with pytest.raises(ValueError):
                attention(x[:, :steps], cache=cache, parents=parents)
            assert cache.length == 5
        attention(x[:, :64], cache=cache, parents=int32(1, 64))
        assert cache.length == 69


def test_windowed_attention_has_no_second_derivative():
    """Asked for one, torch raises; a first derivative under create_graph is what it is without."""
    np.random.seed(2)
    attention = nn.MultiHeadAttention(64, 4, window=5, sinks=1, device="cuda").train()
    x = torch.randn(2, 20, 64, device="cuda", requires_grad=True)
    (plain,) = torch.autograd.grad(attention(x).square().sum(), x)
    (g,) = torch.autograd.grad(attention(x).square().sum(), x, create_graph=True)
    assert torch.equal(plain, g)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.square().sum().backward()

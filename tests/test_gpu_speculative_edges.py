"""Drafted trees through the models: entries of ``parents`` beyond 32 bits."""

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import no_grad  # noqa: E402
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

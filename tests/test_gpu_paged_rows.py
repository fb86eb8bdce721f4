"""Rows of different lengths in a ``PagedKVCache``: failed steps, truncation, refused calls."""

import numpy as np
import pytest

import oracle
from helpers import to_np
from test_gpu_paged_cache import Mirror, model, tensor

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import tensorsmith_b200 as ts  # noqa: E402
from tensorsmith_b200 import engine, nn  # noqa: E402


class Failure(Exception):
    pass


def fail(*_, **__):
    raise Failure


@pytest.mark.parametrize("where", ["before the first append", "between two layers", "after the last append"])
def test_a_failed_step_restores_every_row(where):
    lm = model()
    part = {"before the first append": lm.blocks[0].attention.q_proj, "between two layers": lm.blocks[1].attention_norm,
            "after the last append": lm.final_norm}[where]
    gen = torch.Generator().manual_seed(4)
    prompt, chunk, step, wrong = (torch.randint(0, 97, (2, n), generator=gen) for n in (70, 5, 1, 3))
    with ts.no_grad(), torch.no_grad():
        both = [lm.new_cache(2, 160, quantized="int4") for _ in range(2)]
        for caches in both:
            lm(prompt, caches=caches)
            caches[0].cache.fork([0, -1])
            lm(chunk, caches=caches)
        caches, twin = both
        good, part.forward = part.forward, fail
        with pytest.raises(Failure):
            lm(wrong, caches=caches)
        part.forward = good
        cache = caches[0].cache
        assert cache.lengths.tolist() == cache.seq_lens.tolist() == [75, 5]
        assert [layer.length for layer in caches] == [75, 75] and cache.free_pages() == twin[0].cache.free_pages()
        for _ in range(2):
            assert torch.equal(lm(step, caches=caches), lm(step, caches=twin))


def test_truncation_of_ragged_rows():
    m = Mirror(2, page_size=16)
    m.append(20)
    m.fork([0, -1, 1])
    m.append(7)
    m.cache.truncate([25, 3, 27])
    m.tokens = [[layer[:n] for layer in row] for row, n in zip(m.tokens, (25, 3, 27))]
    m.check()
    m.append(2)
    m.check()
    # a step that one layer has appended goes whole, whatever it is truncated to
    with ts.no_grad():
        m.cache.layers[0].append(*(tensor(torch.ones(3, 2, 4, 64, device="cuda")),) * 2)
    assert m.cache.lengths.tolist() == [31, 9, 33]
    m.cache.layers[1].truncate(29)
    assert m.cache.lengths.tolist() == [27, 5, 29] and [c.length for c in m.cache.layers] == [29, 29]
    m.check()
    m.truncate(6)
    m.check()
    for bad in ([6, 6, 6], [1, 2], [-1, 0, 0], [0.5, 0, 0], -1, 7):
        with pytest.raises(ValueError):
            m.cache.truncate(bad)
    m.check()


def test_quantized_takes_any_truth_value():
    lm = model()
    for value in (1, True, np.True_):
        assert all(cache.quantized for cache in lm.new_cache(1, 32, quantized=value))
    for value in (0, None, False, np.False_):
        assert not any(cache.quantized for cache in lm.new_cache(1, 32, quantized=value))
    prompt = torch.zeros(1, 4, dtype=torch.int64)
    for value, same in ((1, True), (None, False)):
        assert torch.equal(lm.generate(prompt, 3, temperature=0, quantized_cache=value),
                           lm.generate(prompt, 3, temperature=0, quantized_cache=same))


@pytest.mark.parametrize("is_causal", [True, False])
def test_the_attention_module_passes_the_mask_on(is_causal):
    """A chunk of five tokens over pages that hold them and seven before, against fp64 attention over the pages."""
    attention = model(layers=1).blocks[0].attention
    cache = nn.PagedKVCache(2, 1, 2, 32, 64, device="cuda:0", page_size=16)
    layer = cache.layers[0]
    gen = torch.Generator("cuda").manual_seed(0)
    first, x = (torch.randn(2, n, 128, generator=gen, device="cuda") for n in (7, 5))
    with ts.no_grad(), torch.no_grad():
        attention(first, cache=layer)
        got = attention(x, cache=layer, is_causal=is_causal)
        q = engine.rope(attention.q_proj(x).reshape(2, 5, 4, 32).permute(0, 2, 1, 3), offset=7)
        keys, values = (to_np(t._data).astype(np.float64) for t in layer.get())
        ref, _, _ = oracle.attention_int4(to_np(q).astype(np.float64), list(keys), list(values), [12, 12],
                                          is_causal=is_causal)
        want = attention.out_proj(torch.from_numpy(ref).float().cuda().permute(0, 2, 1, 3).reshape(2, 5, 128))
    # fp32 attention and one projection of 128 terms, at tf32 at worst
    assert (got - want).abs().max() <= 1e-3 * want.abs().max()


def test_attend_refuses_a_query_that_wants_gradients():
    m = Mirror(2, layers=1)
    m.append(3)
    layer = m.cache.layers[0]
    query = ts.tensor(np.ones((2, 2, 1, 64), np.float32), device="cuda:0", requires_grad=True)
    with pytest.raises(RuntimeError, match="inference-only"):
        layer.attend(query)
    with ts.no_grad():
        assert layer.attend(query).shape == (2, 2, 1, 64)


def test_a_refused_append_changes_nothing():
    m = Mirror(2, page_size=16)
    m.append(16)
    free = m.cache.free_pages()
    whole = tensor(torch.ones(2, 2, 1, 64, dtype=torch.int64, device="cuda"))
    with ts.no_grad(), pytest.raises(TypeError):
        m.cache.layers[0].append_rotary(whole, whole)
    assert m.cache.length == 16 and m.cache.free_pages() == free
    m.append(1)
    m.check()

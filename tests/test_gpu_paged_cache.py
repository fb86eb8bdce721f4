"""``PagedKVCache`` and the transformer that generates with it.

A layer's ``attend`` is held to fp64 attention over the values its pages stand for; forks, frees, truncation
and compaction must leave every row's tokens as they were written.  The transformer is compared with itself
attending over an ordinary cache that holds the dequantised pages.
"""

import numpy as np
import pytest

import oracle
from helpers import to_np

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
import tensorsmith_b200 as ts  # noqa: E402
from tensorsmith_b200 import engine, nn  # noqa: E402


def tensor(x):
    return ts.Tensor(x, device="cuda:0")


class Mirror:
    """A cache and, row by row, the tokens it should hold."""

    def __init__(self, rows, *, layers=2, heads=2, dim=64, capacity=300, seed=0, **kw):
        self.cache = nn.PagedKVCache(rows, layers, heads, dim, capacity, device="cuda:0", **kw)
        self.gen = torch.Generator("cuda").manual_seed(seed)
        self.tokens = [[[] for _ in range(layers)] for _ in range(rows)]  # [row][layer] of (k, v) [H, D]
        self.heads, self.dim = heads, dim

    def append(self, steps):
        rows = self.cache.batch_size
        for i, layer in enumerate(self.cache.layers):
            k, v = (torch.randn(rows, self.heads, steps, self.dim, generator=self.gen, device="cuda") for _ in range(2))
            with ts.no_grad():
                layer.append(tensor(k), tensor(v))
            for r in range(rows):
                for s in range(steps):
                    self.tokens[r][i].append(tuple(
                        oracle.dequantize_int4(*oracle.quantize_int4(to_np(x[r, :, s]))) for x in (k, v)))

    def fork(self, index):
        self.cache.fork(index)
        self.tokens = [[list(layer) for layer in self.tokens[s]] if s >= 0 else
                       [[] for _ in self.cache.layers] for s in index]

    def truncate(self, n):
        self.cache.truncate(n)
        self.tokens = [[layer[:n] for layer in row] for row in self.tokens]

    def check(self):
        assert self.cache.lengths.tolist() == [len(row[0]) for row in self.tokens]
        assert self.cache.seq_lens.tolist() == self.cache.lengths.tolist()
        for i, layer in enumerate(self.cache.layers):
            k, v = (to_np(t._data) for t in layer.get())
            for r, row in enumerate(self.tokens):
                for got, which in ((k, 0), (v, 1)):
                    want = np.stack([t[which] for t in row[i]], axis=1) if row[i] else np.zeros((self.heads, 0, self.dim))
                    np.testing.assert_array_equal(got[r, :, : want.shape[1]], want)
        engine.check_device_status()
        assert self.cache._counters[2] == 0
        held = self.cache.page_table[self.cache.page_table >= 0]
        refs = torch.bincount(held.long(), minlength=self.cache.num_pages)
        assert torch.equal(refs.int(), self.cache._refs) and int((refs == 0).sum()) == self.cache.free_pages()


@pytest.mark.parametrize("page", [16, 64])
def test_rows_keep_their_tokens(page):
    m = Mirror(3, page_size=page, num_pages=80)
    m.append(21)
    m.append(1)
    m.check()
    m.fork([0, 0, 2, 2, 2])
    m.append(1)
    m.check()
    m.fork([4, -1, 1])
    m.append(page)
    m.check()
    m.cache.compact()
    m.check()
    m.truncate(17)  # into pages that were shared
    m.append(3)
    m.check()
    m.cache.reorder([2, 0, 1])
    m.tokens = [m.tokens[i] for i in (2, 0, 1)]
    m.check()
    m.cache.free([0, 2])
    m.tokens[0] = [[] for _ in m.tokens[0]]
    m.tokens[2] = [[] for _ in m.tokens[2]]
    m.check()
    m.cache.reset()
    assert m.cache.free_pages() == 80 and m.cache.length == 0


def test_truncated_rows_do_not_write_to_shared_pages():
    m = Mirror(1, page_size=16, num_pages=30)
    m.append(64)
    m.fork([0, 0, 0])
    m.truncate(20)
    m.append(30)
    m.check()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_attend_over_ragged_rows(dtype):
    m = Mirror(2, layers=1, capacity=200, dtype=dtype)
    m.append(70)
    m.fork([0, 1, -1])
    m.append(5)
    q = torch.randn(3, 6, 5, 64, generator=m.gen, device="cuda").to(getattr(torch, dtype))
    with ts.no_grad():
        out = m.cache.layers[0].attend(tensor(q))
    lens = [75, 75, 5]
    # the appended rows are rounded to the cache's type before they are quantised
    keys, values = ([to_np(t._data)[r, :, :n].astype(np.float64) for r, n in enumerate(lens)]
                    for t in m.cache.layers[0].get())
    ref, _, spread = oracle.attention_int4(to_np(q).astype(np.float64), keys, values, lens)
    unit = {"float32": 2.0**-18, "bfloat16": 2.0**-8, "float16": 2.0**-11}[dtype]
    assert (np.abs(to_np(out._data) - ref) <= unit * np.abs(ref) + (unit / 4 + 2.0**-16) * spread).all()


def test_refusals():
    for bad in (dict(head_dim=48), dict(page_size=24), dict(num_pages=0)):
        with pytest.raises(ValueError):
            nn.PagedKVCache(**{**dict(batch_size=1, num_layers=1, num_heads=1, head_dim=64, max_seq_len=64,
                                      device="cuda:0"), **bad})
    with pytest.raises(TypeError):
        nn.PagedKVCache(1, 1, 1, 64, 64, device="cuda:0", dtype="float64")
    m = Mirror(2, num_pages=3, page_size=16, capacity=64)
    m.append(16)
    before = m.cache.page_table.clone()
    with pytest.raises(ValueError, match="free pages"):
        m.append(1)  # two pages are due, one is free
    assert torch.equal(before, m.cache.page_table) and m.cache.length == 16
    m.check()
    x = tensor(torch.zeros(2, 2, 1, 64, device="cuda"))
    layer = m.cache.layers[0]
    with ts.no_grad():
        for key, value in ((tensor(x._data[:1]), x), (x, tensor(x._data[..., :32])), (tensor(x._data[:, :, :0]),) * 2):
            with pytest.raises(ValueError):
                layer.append(key, value)
        with pytest.raises(ValueError, match="capacity"):
            layer.append(*(tensor(torch.zeros(2, 2, 49, 64, device="cuda")),) * 2)
        with pytest.raises(TypeError):
            layer.attend(tensor(x._data.half()))
    grad = ts.tensor(np.zeros((2, 2, 1, 64), np.float32), device="cuda:0", requires_grad=True)
    with pytest.raises(RuntimeError, match="inference-only"):
        layer.append(grad, grad)
    for rows in ([2], [-2], [[0]], [0.5], []):
        with pytest.raises(ValueError):
            m.cache.fork(rows)
    with pytest.raises(ValueError):
        m.cache.truncate(17)


def test_copies_that_writers_leave_one_another_fit_exactly():
    """Three rows share a partly filled page and two pages are free: the third writer keeps the page."""
    m = Mirror(1, num_pages=3, page_size=16, capacity=32)
    m.append(5)
    m.fork([0, 0, 0])
    m.append(1)
    m.check()
    assert m.cache.free_pages() == 0


def model(kv_heads=2, layers=2, context=160):
    np.random.seed(0)
    config = nn.TransformerConfig(vocab_size=97, dim=128, num_heads=4, num_layers=layers, num_kv_heads=kv_heads,
                                  max_seq_len=context)
    return nn.TransformerLM(config, device="cuda:0").eval()


def test_transformer_over_pages_matches_its_dequantised_cache():
    """Chunks and single tokens; the reference attends over the values that the pages stand for."""
    lm = model()
    tokens = torch.randint(0, 97, (2, 40), generator=torch.Generator().manual_seed(1))
    with ts.no_grad(), torch.no_grad():
        caches = lm.new_cache(2, 64, quantized="int4")
        plain = lm.new_cache(2, 64)
        paged_append = nn.PagedKVCache
        assert isinstance(caches[0].cache, paged_append)
        at = 0
        for n in (33, 1, 1, 5):
            got = lm(tokens[:, at:at + n], caches=caches)
            # the plain caches take the dequantised tokens in the place of what they would have appended
            class Taken:
                def __init__(self, cache, source):
                    self.inner, self.source = cache, source

                def __getattr__(self, name):
                    return getattr(self.inner, name)

                def append_rotary(self, key, value):
                    k, v = (tensor(t._data[:, :, at:at + n].contiguous()) for t in self.source.get())
                    return self.inner.append(k, v)

            want = lm(tokens[:, at:at + n], caches=[Taken(p, c) for p, c in zip(plain, caches)])
            assert (got - want).abs().max() <= 1e-4 * want.abs().max()  # fp32 attention on both sides
            at += n
        assert [c.length for c in caches] == [40, 40]


def test_a_failed_step_rolls_back():
    lm = model()
    tokens = torch.zeros(1, 8, dtype=torch.int64)
    with ts.no_grad(), torch.no_grad():
        caches = lm.new_cache(1, 32, quantized="int4")
        lm(tokens, caches=caches)
        with pytest.raises(ValueError, match="mask"):
            lm(tokens, caches=caches, attn_mask=torch.ones(1, 1, 8, 16, dtype=torch.bool, device="cuda"))
        caches[0].append(*(tensor(torch.zeros(1, 2, 3, 32, device="cuda")),) * 2)  # as if a later layer had failed
        for cache in caches:
            cache.truncate(8)
        assert [c.length for c in caches] == [8, 8] and caches[0].cache.length == 8
        assert lm(tokens[:, :1], caches=caches).shape == (1, 1, 97)


def test_generate_shares_prompts_between_samples():
    lm = model()
    prompt = torch.randint(0, 97, (2, 70), generator=torch.Generator().manual_seed(2))
    greedy = lm.generate(prompt, 12, temperature=0, quantized_cache="int4")
    both = lm.generate(prompt, 12, temperature=0, quantized_cache="int4", num_samples=3)
    assert both.shape == (6, 82)
    for r in range(6):  # a sample's rows share pages with the others and still see only their own tokens
        assert torch.equal(both[r], greedy[r // 3])
    sampled = lm.generate(prompt, 12, quantized_cache="int4", num_samples=3,
                          generator=torch.Generator("cuda").manual_seed(3))
    assert len({tuple(row.tolist()) for row in sampled}) > 2
    plain = lm.generate(prompt, 12, temperature=0, num_samples=2)
    assert torch.equal(plain[0], plain[1]) and plain.shape == (4, 82)
    with pytest.raises(ValueError):
        lm.generate(prompt, 2, num_samples=0)
    with pytest.raises(ValueError):
        lm.new_cache(1, 32, quantized="int2")
    with pytest.raises(ValueError):
        lm.new_cache(1, 32, num_pages=4)

"""The paged 4-bit KV cache on the GPU against the oracle in 64 bits.

The append must match the oracle bit for bit (integer work on correctly rounded divisions).  Attention
is compared with fp64 attention over the values the cache stands for.  Its error is bounded by the
output's rounding, u |o| (u = 2^-8 bf16, 2^-11 f16, 2^-24 f32), plus what moves the probabilities:
    c = r + 2^-19 (1 + max|s|) + n 2^-27
with r the rounding of p in the product with V (one fp16 part, 2^-11, for bf16 outputs; two parts, 2^-21,
otherwise; the prefill kernel's bf16 / fp16 p and cubic exponential, 2^-8 + 2^-13 or 2^-11 + 2^-13), the
second term fp32 scores and the approximate exponential, the third the additions' truncation over n keys;
each scaled by sum_j p_j |v_j|.
"""

import numpy as np
import pytest

import oracle
from helpers import to_np, torch_dtype

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import _lib, engine  # noqa: E402

UNIT = {"bfloat16": 2.0**-8, "float16": 2.0**-11, "float32": 2.0**-24}
P_PAGES = {"bfloat16": 2.0**-11, "float16": 2.0**-21, "float32": 2.0**-21}
P_PREFILL = {"bfloat16": 2.0**-8 + 2.0**-13, "float16": 2.0**-11 + 2.0**-13}


class Cache:
    """A pool whose pages hold garbage (NaN scales) until written, with scattered page tables."""

    def __init__(self, lens, kv_heads, dim, page, *, seed=0, extra_slots=1, extra_pages=3, stride_pages=None):
        rng = np.random.default_rng(seed)
        self.lens, self.page, self.dim = np.asarray(lens), page, dim
        need = -(-self.lens // page)
        slots = int(need.max(initial=0)) + extra_slots
        pages = int(need.sum()) + extra_pages
        order = rng.permutation(pages)
        table = np.full((len(lens), slots), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n]
            at += n
        self.pool = engine.int4_pool(pages, kv_heads, dim, page_size=page)
        self.pool.fill_(255)
        self.table = torch.from_numpy(table).cuda()
        self.kv_lens = torch.from_numpy(self.lens.astype(np.int32)).cuda()
        most = max(1, int(self.lens.max(initial=0)))
        self.k = rng.standard_normal((len(lens), kv_heads, most, dim))
        self.v = rng.standard_normal((len(lens), kv_heads, most, dim)) * np.exp(rng.uniform(-2, 2, (1, kv_heads, 1, dim)))
        self.pool_table = table

    def fill(self, dtype):
        """Append each row's tokens; returns the values the cache then stands for."""
        k = torch.from_numpy(self.k).to("cuda", torch_dtype(dtype))
        v = torch.from_numpy(self.v).to("cuda", torch_dtype(dtype))
        keys, values = [], []
        for r, n in enumerate(self.lens):
            if n:
                engine.kv_append_int4(k[r:r + 1, :, :n], v[r:r + 1, :, :n], self.pool, self.table[r:r + 1],
                                      page_size=self.page)
            keys.append(oracle.dequantize_int4(*oracle.quantize_int4(to_np(k[r, :, :n]))))
            values.append(oracle.dequantize_int4(*oracle.quantize_int4(to_np(v[r, :, :n]))))
        return keys, values


def check_attention(cache, dtype, q_heads, q_len, *, causal=True, seed=1, scale=None, path=None, monkeypatch=None):
    if path:
        monkeypatch.setenv("TS_INT4_KERNEL", path)
    keys, values = cache.fill(dtype)
    rng = np.random.default_rng(seed)
    q = torch.from_numpy(rng.standard_normal((len(cache.lens), q_len, q_heads, cache.dim))).to("cuda", torch_dtype(dtype))
    q = q.permute(0, 2, 1, 3)  # the strides of a projection seen as heads
    kw = dict(page_size=cache.page, is_causal=causal, scale=scale, max_len=max(1, int(cache.lens.max(initial=0))))
    if path:
        expect = {"pages": "decode", "prefill": "tcgen05"}[path]
        assert engine.attention_int4_path(q, cache.pool, cache.table, cache.kv_lens, **kw) == expect
    out, lse = engine.attention_int4(q, cache.pool, cache.table, cache.kv_lens, need_lse=True, **kw)
    again, _ = engine.attention_int4(q, cache.pool, cache.table, cache.kv_lens, **kw)
    torch.cuda.synchronize()
    engine.check_device_status()
    assert torch.equal(out, again)
    ref, ref_lse, spread = oracle.attention_int4(to_np(q).astype(np.float64), keys, values, cache.lens,
                                                 is_causal=causal, scale=scale)
    r = (P_PREFILL if path == "prefill" else P_PAGES)[dtype]
    top = max(1.0, float(np.abs(ref_lse[np.isfinite(ref_lse)]).max(initial=0)) + 10)
    c = r + 2.0**-19 * (1 + top) + int(cache.lens.max(initial=0)) * 2.0**-27
    err = np.abs(to_np(out).astype(np.float64) - ref)
    assert (err <= UNIT[dtype] * np.abs(ref) + c * spread + 1e-7).all(), float((err / (spread + 1e-9)).max())
    got = to_np(lse).astype(np.float64)
    assert np.array_equal(np.isneginf(got), np.isneginf(ref_lse))
    finite = np.isfinite(ref_lse)
    assert (np.abs(got[finite] - ref_lse[finite]) <= 2.0**-19 * (1 + top) + (1e-3 if path == "prefill" else 0)).all()
    return out


@pytest.mark.parametrize("group, q_len", [(1, 1), (5, 1), (2, 5)])
@pytest.mark.parametrize("dim, page", [(32, 16), (64, 32), (96, 16), (128, 64), (256, 32)])
def test_fp32_attention_keeps_fp32_precision(dim, page, group, q_len):
    """The error's norm against the output's: q in two fp16 parts, the scores' sums, the exponential and p in two
    parts each move a probability by at most 2^-22 of itself (scores of size one); independent, they add up to
    2^-21.  The n additions' truncation is the 2^-27 each of the other bounds here."""
    c = Cache([40, 33, 37], 2, dim, page, seed=dim)
    c.v = np.random.default_rng(dim + 1).standard_normal(c.v.shape)
    keys, values = c.fill("float32")
    q = torch.from_numpy(np.random.default_rng(3).standard_normal((3, 2 * group, q_len, dim))).cuda().float()
    out, _ = engine.attention_int4(q, c.pool, c.table, c.kv_lens, page_size=page)
    engine.check_device_status()
    ref, _, _ = oracle.attention_int4(to_np(q).astype(np.float64), keys, values, c.lens, is_causal=True, scale=None)
    assert np.linalg.norm(to_np(out) - ref) <= (2.0**-21 + 40 * 2.0**-27) * np.linalg.norm(ref)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dim, page, heads", [(32, 16, 1), (64, 32, 3), (96, 16, 2), (128, 64, 8), (256, 32, 2)])
def test_append_and_gather_match_the_oracle(dtype, dim, page, heads):
    rng = np.random.default_rng(dim + page)
    lens, steps = np.array([0, 5, page - 1, 2 * page + 3]), page + 7
    c = Cache(lens + steps, heads, dim, page, seed=dim)
    x = rng.standard_normal((2, 4, steps, heads, dim)) * np.exp(rng.uniform(-12, 6, (2, 4, steps, heads, 1)))
    x[0, 0, 0, 0, :3] = [np.inf, -np.inf, np.nan]
    x[1, 1, 1] = 0.0
    t = torch.from_numpy(x).to("cuda", torch_dtype(dtype)).permute(0, 1, 3, 2, 4)
    start = torch.from_numpy(lens.astype(np.int32)).cuda()
    stop = torch.empty_like(start)
    engine.kv_append_int4(t[0], t[1], c.pool, c.table, page_size=page, positions=start, positions_out=stop)
    assert stop.tolist() == (lens + steps).tolist()
    k, v = engine.kv_gather_int4(c.pool, c.table, steps, page_size=page, dtype=torch.float32, starts=start)
    half, _ = engine.kv_gather_int4(c.pool, c.table, steps, page_size=page, dtype=torch.bfloat16, starts=start)
    torch.cuda.synchronize()
    engine.check_device_status()
    for got, given in ((k, t[0]), (v, t[1])):
        ref = oracle.dequantize_int4(*oracle.quantize_int4(to_np(given)))
        np.testing.assert_array_equal(got.cpu().numpy(), ref)
    assert torch.equal(half.float(), k)  # every stored value is a bf16 number
    # the stored bytes, not only what the gather makes of them
    for r in range(4):
        slot, at = divmod(int(lens[r]), page)
        block = c.pool[int(c.table[r, slot]), heads - 1].cpu().numpy()
        keys, values = oracle.unpack_block(block, page, dim)
        np.testing.assert_array_equal(keys[at], k[r, heads - 1, 0].cpu().numpy())
        np.testing.assert_array_equal(values[at], v[r, heads - 1, 0].cpu().numpy())


def test_append_of_unaligned_strided_rows():
    base = torch.randn(2, 5, 3, 2 * 64 + 1, device="cuda", dtype=torch.bfloat16)
    x = base[..., 1::2].permute(0, 2, 1, 3)  # channel stride 2, odd offsets
    c = Cache([5, 5], 3, 64, 16)
    engine.kv_append_int4(x, x, c.pool, c.table, page_size=16)
    k, v = engine.kv_gather_int4(c.pool, c.table, 5, page_size=16, dtype=torch.float16)
    ref = oracle.dequantize_int4(*oracle.quantize_int4(to_np(x)))
    np.testing.assert_array_equal(k.double().cpu().numpy(), ref)
    assert torch.equal(k, v)


def test_gather_zeroes_past_the_lengths():
    c = Cache([0, 3, 40], 2, 32, 16)
    keys, _ = c.fill("float32")
    k, v = engine.kv_gather_int4(c.pool, c.table, 45, page_size=16, dtype=torch.float32, kv_lens=c.kv_lens)
    for r, n in enumerate(c.lens):
        np.testing.assert_array_equal(k[r, :, :n].cpu().numpy(), keys[r])
        assert not k[r, :, n:].any() and not v[r, :, n:].any()
    engine.check_device_status()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_head_dims(dtype, dim):
    check_attention(Cache([1, 130, 0, 65], 2, dim, 32, seed=dim), dtype, 4, 1)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("group, q_len", [(1, 1), (1, 3), (8, 1), (3, 7), (5, 4), (2, 33)])
def test_attention_groups_and_tokens(dtype, page, causal, group, q_len, monkeypatch):
    lens = [0, 1, 2, 15, 16, 17, 63, 64, 65, 300]
    check_attention(Cache(lens, 2, 64, page, seed=page), dtype, 2 * group, q_len, causal=causal, path="pages",
                    monkeypatch=monkeypatch)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("group, q_len", [(1, 1), (4, 1), (4, 5)])
def test_attention_splits_long_rows(dtype, group, q_len):
    c = Cache([4097, 1, 9000, 0], 1, 128, 64, seed=7)
    q = torch.zeros(4, group, q_len, 128, device="cuda", dtype=torch_dtype(dtype))
    assert engine.attention_int4_workspace_bytes(q, c.pool, c.table, c.kv_lens, page_size=64, max_len=9000) > 0
    check_attention(c, dtype, group, q_len)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens, q_len", [([150, 0, 64, 257], 40), ([300, 128], 129), ([1000], 300)])
def test_attention_prefill_route(dtype, dim, causal, lens, q_len, monkeypatch):
    check_attention(Cache(lens, 2, dim, 32, seed=dim), dtype, 4, q_len, causal=causal, path="prefill",
                    monkeypatch=monkeypatch)


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5, 1e-30])
def test_attention_scales(scale):
    check_attention(Cache([70, 9], 2, 64, 16), "bfloat16", 2, 1, scale=scale)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_attention_of_extreme_queries(dtype):
    """Rows of queries whose magnitudes span the type, one of them non-finite: it alone turns NaN."""
    c = Cache([90], 1, 64, 16)
    keys, values = c.fill(dtype)
    q = torch.randn(1, 6, 1, 64, device="cuda", dtype=torch.float64, generator=torch.Generator("cuda").manual_seed(3))
    q *= torch.tensor([1e-38, 1e-20, 1.0, 1e4, 1e18, 1.0], device="cuda").view(1, 6, 1, 1)
    q = q.to(torch_dtype(dtype))
    q[0, 5, 0, 7] = float("inf")
    out, lse = engine.attention_int4(q, c.pool, c.table, c.kv_lens, page_size=16, need_lse=True)
    ref, _, spread = oracle.attention_int4(to_np(q[:, :5]).astype(np.float64), keys, values, c.lens)
    err = np.abs(to_np(out[:, :5]).astype(np.float64) - ref)
    # a score s carries a relative error of 2^-20, which at |s| beyond 2^20 moves p by any factor unless
    # one key stands alone: the two largest rows are held to the value of their top key
    top = np.abs(to_np(q)).max(axis=-1)[0, :5, 0] * 64 * 8
    bound = UNIT[dtype] * np.abs(ref) + spread * (2.0**-11 + np.minimum(1, top * 2.0**-19))[None, :, None, None]
    assert (err[:, :3] <= bound[:, :3]).all()
    assert np.isfinite(to_np(out[:, :5])).all() and torch.isnan(out[:, 5]).all() and torch.isnan(lse[:, 5]).all()


def test_attention_reads_pages_beyond_4_gib():
    """Pages whose byte offsets pass 32 bits."""
    pages, heads, dim, page = 60000, 8, 128, 64
    pool = engine.int4_pool(pages, heads, dim, page_size=page)
    table = torch.tensor([[59999, 7, 58255], [3, 59998, -1]], dtype=torch.int32, device="cuda")
    lens = np.array([150, 70])
    x = torch.randn(2, 2, heads, 150, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(1)).bfloat16()
    kv_lens = torch.from_numpy(lens.astype(np.int32)).cuda()
    for r, n in enumerate(lens):
        engine.kv_append_int4(x[0, r:r + 1, :, :n], x[1, r:r + 1, :, :n], pool, table[r:r + 1], page_size=page)
    q = torch.randn(2, heads, 1, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).bfloat16()
    out, _ = engine.attention_int4(q, pool, table, kv_lens, page_size=page, max_len=150)
    k, _ = engine.kv_gather_int4(pool, table, 150, page_size=page, dtype=torch.bfloat16, kv_lens=kv_lens)
    engine.check_device_status()
    keys, values = ([oracle.dequantize_int4(*oracle.quantize_int4(to_np(y[r, :, :n]))) for r, n in enumerate(lens)]
                    for y in x)
    np.testing.assert_array_equal(to_np(k[0]), keys[0])
    ref, _, spread = oracle.attention_int4(to_np(q).astype(np.float64), keys, values, lens)
    assert (np.abs(to_np(out) - ref) <= 2.0**-8 * np.abs(ref) + 2.0**-10 * spread).all()


def test_out_tensors_streams_and_graphs():
    c = Cache([100, 33], 2, 64, 16)
    c.fill("bfloat16")
    q = torch.randn(2, 4, 1, 64, device="cuda", dtype=torch.bfloat16)
    kw = dict(page_size=16, max_len=100)
    want, want_lse = engine.attention_int4(q, c.pool, c.table, c.kv_lens, need_lse=True, **kw)
    torch.cuda.synchronize()
    out = torch.zeros(2, 1, 4, 64, device="cuda", dtype=torch.bfloat16).permute(0, 2, 1, 3)
    lse = torch.zeros(2, 4, 1, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got, got_lse = engine.attention_int4(q, c.pool, c.table, c.kv_lens, out=out, lse=lse, need_lse=True, **kw)
    side.synchronize()
    assert got.data_ptr() == out.data_ptr() and torch.equal(got, want) and torch.equal(got_lse, want_lse)
    graph = torch.cuda.CUDAGraph()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    with torch.cuda.graph(graph):
        engine.attention_int4(q, c.pool, c.table, c.kv_lens, out=out, workspace=ws, **kw)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("rows, heads, start", [(3, 2, 11), (16, 8, 700)])
def test_calls_in_a_row_see_one_anothers_writes(rows, heads, start):
    """The kernels of one call start while those of the call before it end: a chain in which every call reads what
    the one before it wrote gives the same bits as with a synchronisation after each, and from a graph."""
    dim, page, steps = 64, 16, 12
    slots = (start + steps) // page + 2
    pages = rows * slots + rows

    def chain(after):
        gen = torch.Generator(device="cuda").manual_seed(5)
        pool = torch.zeros_like(engine.int4_pool(pages, heads, dim, page_size=page, layers=1))
        refs, counters = engine.kv_pages_state(pages)
        table = torch.full((rows, slots), -1, dtype=torch.int32, device="cuda")
        lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        prompt = torch.randn(2, rows, heads, start, dim, generator=gen, device="cuda").half()
        x = torch.randn(rows, heads, 1, dim, generator=gen, device="cuda").half()
        parents = torch.arange(rows, device="cuda", dtype=torch.int32) // 2
        engine.kv_pages_reserve(pool, table, lens, start, refs, counters, page_size=page)
        engine.kv_append_int4(prompt[0], prompt[1], pool[0], table, page_size=page, positions=lens)
        lens = lens + start
        torch.cuda.synchronize()

        def run():
            t, n, token, outs = table, lens, x, []
            for step in range(steps):
                engine.kv_pages_reserve(pool, t, n, 1, refs, counters, page_size=page)
                after()
                engine.kv_append_int4(token, token * 0.5, pool[0], t, page_size=page, positions=n)
                after()
                n = n + 1
                token, _ = engine.attention_int4(token, pool[0], t, n, page_size=page, max_len=start + steps)
                after()
                again, _ = engine.attention_int4(token * 2, pool[0], t, n, page_size=page, max_len=start + steps)
                after()
                outs.append(again)
                token = token + again
                if step % 4 == 3:
                    t, n = engine.kv_pages_fork(t, n, parents, refs, counters, page_size=page)
                    after()
                    engine.kv_pages_compact(pool, t, refs, counters)
                    after()
                    key, value = engine.kv_gather_int4(pool[0], t, start, page_size=page, dtype=torch.float16, kv_lens=n)
                    after()
                    outs.append(key + value)
            return [o.clone() for o in outs] + [t, n, refs, counters]

        return run

    expect = chain(torch.cuda.synchronize)()
    torch.cuda.synchronize()
    assert expect[-1][2].item() == 0 and torch.isfinite(expect[0]).all()
    for _ in range(3):
        got = chain(lambda: None)()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(expect, got))
    graph, run = torch.cuda.CUDAGraph(), chain(lambda: None)
    with torch.cuda.graph(graph):
        got = run()
    graph.replay()
    torch.cuda.synchronize()
    engine.check_device_status()
    assert all(torch.equal(a, b) for a, b in zip(expect, got))


def test_refusals_on_device_tensors():
    c = Cache([10, 20], 2, 64, 16)
    q = torch.zeros(2, 4, 1, 64, device="cuda", dtype=torch.bfloat16)
    x = torch.zeros(2, 2, 3, 64, device="cuda", dtype=torch.bfloat16)
    attn = lambda **kw: engine.attention_int4(**{**dict(  # noqa: E731
        q=q, pool=c.pool, page_table=c.table, kv_lens=c.kv_lens, page_size=16), **kw})
    append = lambda **kw: engine.kv_append_int4(**{**dict(  # noqa: E731
        key=x, value=x, pool=c.pool, page_table=c.table, page_size=16), **kw})
    for bad in (dict(page_size=32), dict(q=q[:1]), dict(q=q[:, :3]), dict(q=q[0]), dict(kv_lens=c.kv_lens.long()),
                dict(kv_lens=c.kv_lens[:1]), dict(page_table=c.table.long()), dict(page_table=c.table.t()),
                dict(max_len=10**6), dict(max_len=-1), dict(out=q[:1]), dict(need_lse=True, lse=q[..., 0])):
        with pytest.raises(ValueError):
            attn(**bad)
    for bad in (dict(q=q.double()), dict(q=q.long())):
        with pytest.raises((TypeError, _lib.EngineError)):
            attn(**bad)
    for bad in (dict(key=x[:1]), dict(value=x[:, :1]), dict(positions=c.kv_lens.long()), dict(page_size=16.5)):
        with pytest.raises((ValueError, TypeError, _lib.EngineError)):
            append(**bad)
    with pytest.raises(TypeError):
        append(value=x.half())
    with pytest.raises(TypeError):
        append(pool=c.pool.char())
    with pytest.raises(_lib.EngineError) as error:
        append(position=47)
    assert error.value.status == _lib.ERR_CAPACITY
    with pytest.raises(ValueError):
        engine.kv_gather_int4(c.pool, c.table, -1, page_size=16, dtype=torch.bfloat16)
    assert engine.kv_gather_int4(c.pool, c.table, 0, page_size=16, dtype=torch.bfloat16)[0].shape == (2, 2, 0, 64)


def test_a_missing_page_is_reported_and_nothing_is_written():
    c = Cache([16, 16], 1, 32, 16)
    before = c.pool.clone()
    x = torch.ones(2, 1, 1, 32, device="cuda", dtype=torch.bfloat16)
    engine.kv_append_int4(x, x, c.pool, c.table, page_size=16, position=16)  # slot 1 has no page
    status, site = engine.device_status()
    assert status == _lib.ERR_PAGE and site == 0x301
    assert torch.equal(before, c.pool)
    table = c.table.clone()
    table[0, 0] = 10**6
    q = torch.ones(2, 1, 1, 32, device="cuda", dtype=torch.bfloat16)
    engine.attention_int4(q, c.pool, table, c.kv_lens, page_size=16)
    with pytest.raises(_lib.EngineError, match="page table entry"):
        engine.check_device_status()
    engine.check_device_status()

"""Attention over 4-bit pages whose scales reach the ends of the format's range.

A scale lies in [2^-20, 9216], so a cached value reaches 64512 (what an infinity is stored as).  The bounds are
those of test_gpu_int4_cache: an error of the probabilities counts with sum_j p_j |v_j| of its channel, so a
group of ordinary values is held to ordinary errors beside one of huge ones.
"""

import numpy as np
import pytest

import oracle
from helpers import to_np, torch_dtype
from test_gpu_int4_cache import Cache, check_attention

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402

# Largest |x| of a group: scales of 2^-20, 1, 896, 928 (the first whose 72-fold passes fp16), 9216, and saturated.
PEAKS = [1e-9, 7.0, 7 * 896.0, 7 * 928.0, 64512.0, np.inf]


def spread_values(c, seed):
    """V whose groups have the peaks above: the first group of a head keeps one for all tokens, the others change
    from token to token; the last three tokens of a row are huge in a head that is ordinary elsewhere."""
    rng = np.random.default_rng(seed)
    v = rng.uniform(-1, 1, c.v.shape)
    rows, heads, tokens, dim = v.shape
    groups = v.reshape(rows, heads, tokens, dim // 32, 32)
    groups[..., 5] = np.sign(groups[..., 5])  # the group's largest
    with np.errstate(invalid="ignore"):
        for h in range(heads):
            peak = rng.choice(PEAKS, (rows, tokens, dim // 32))
            peak[:, :, 0] = PEAKS[h % len(PEAKS)]
            if h == heads - 1:
                peak[:] = 7.0
                for r, n in enumerate(c.lens):
                    peak[r, max(0, n - 3):n] = 64512.0
            full = np.isinf(peak)
            groups[:, h] *= np.where(full, 1e5, peak)[..., None]
            groups[:, h, :, :, 5] = np.where(full, np.copysign(np.inf, groups[:, h, :, :, 5]), groups[:, h, :, :, 5])
    c.v = np.where(np.isinf(v), v, np.clip(v, -64512, 64512))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dim, page", [(64, 16), (96, 32), (128, 64), (256, 32)])
@pytest.mark.parametrize("group, q_len", [(1, 1), (3, 1), (2, 4), (3, 5), (4, 5)])
def test_values_over_the_whole_range(dtype, dim, page, group, q_len, monkeypatch):
    """One, two and three column tiles, columns held twice, rows of one warp and rows whose parts are merged."""
    c = Cache([70, 1, 0, 333, 16], 4, dim, page, seed=dim + group)
    spread_values(c, seed=dim)
    check_attention(c, dtype, 4 * group, q_len, path="pages", monkeypatch=monkeypatch)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("group, q_len", [(1, 1), (4, 5)])
def test_values_over_the_whole_range_in_long_rows(dtype, group, q_len):
    c = Cache([4100, 9001], 2, 128, 64, seed=3)
    spread_values(c, seed=4)
    check_attention(c, dtype, 2 * group, q_len)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_over_the_whole_range_on_the_prefill_route(dtype, dim, monkeypatch):
    c = Cache([150, 0, 64, 257], 4, dim, 32, seed=dim)
    spread_values(c, seed=dim + 1)
    check_attention(c, dtype, 8, 40, path="prefill", monkeypatch=monkeypatch)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("group, q_len", [(1, 1), (2, 5)])
def test_keys_over_the_whole_range(dtype, group, q_len):
    """Groups of tiny, ordinary and huge keys, the queries' channels scaled against them: ordinary scores."""
    dim, page = 128, 32
    c = Cache([90, 37], 2, dim, page, seed=9)
    peaks = np.repeat([1e-9, 1.0, 6400.0, 64512.0], 32)
    c.k = np.clip(c.k * peaks / 4, -64512, 64512)
    keys, values = c.fill(dtype)
    rng = np.random.default_rng(1)
    q = rng.standard_normal((2, 2 * group, q_len, dim)) / np.maximum(peaks, 1.0)
    q = torch.from_numpy(q).to("cuda", torch_dtype(dtype))
    out, lse = engine.attention_int4(q, c.pool, c.table, c.kv_lens, page_size=page, need_lse=True)
    engine.check_device_status()
    ref, ref_lse, spread = oracle.attention_int4(to_np(q).astype(np.float64), keys, values, c.lens)
    top = float(np.abs(ref_lse[np.isfinite(ref_lse)]).max()) + 10
    r, unit = {"bfloat16": (2.0**-11, 2.0**-8), "float16": (2.0**-21, 2.0**-11), "float32": (2.0**-21, 2.0**-24)}[dtype]
    bound = unit * np.abs(ref) + (r + 2.0**-19 * (1 + top) + 90 * 2.0**-27) * spread + 1e-7
    assert (np.abs(to_np(out).astype(np.float64) - ref) <= bound).all()
    finite = np.isfinite(ref_lse)
    assert (np.abs(to_np(lse).astype(np.float64)[finite] - ref_lse[finite]) <= 2.0**-19 * (1 + top)).all()


@pytest.mark.parametrize("path", ["pages", "prefill"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("group, q_len", [(1, 3), (3, 7), (1, 40)])
def test_queries_that_see_no_key_may_hold_anything(path, dtype, group, q_len, monkeypatch):
    """The first tokens of a chunk longer than its row: zeros and -inf, like a row without tokens, beside queries
    that are as before."""
    if path == "prefill" and dtype == "float32":
        pytest.skip("the prefill kernel takes half types")
    c = Cache([0, 2, 1, 90], 2, 64, 16, seed=2)
    c.fill(dtype)
    monkeypatch.setenv("TS_INT4_KERNEL", path)
    kw = dict(page_size=16, max_len=90, need_lse=True)
    q = torch.randn(4, 2 * group, q_len, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    q = q.to(torch_dtype(dtype))
    want, want_lse = engine.attention_int4(q, c.pool, c.table, c.kv_lens, **kw)
    odd = q.clone()
    for r, n in enumerate(c.lens):
        blind = max(0, q_len - int(n))
        odd[r, :, :blind, ::3] = float("nan")
        odd[r, :, :blind, 1::3] = float("inf")
    got, got_lse = engine.attention_int4(odd, c.pool, c.table, c.kv_lens, **kw)
    engine.check_device_status()
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse)
    assert not got[0].any() and not got[2, :, :-1].any() and torch.isneginf(got_lse[1, :, : q_len - 2]).all()

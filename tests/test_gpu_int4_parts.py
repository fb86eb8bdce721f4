"""Attention over 4-bit pages in several launches: batches past 1024 rows, lines of work past the limit of one
launch (lowered here by TS_INT4_LINE), rows of q and out that no wide access can take."""

import numpy as np
import pytest

import oracle
from helpers import to_np, torch_dtype
from test_gpu_int4_cache import Cache, check_attention

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("group, q_len", [(1, 1), (3, 7), (2, 33)])
@pytest.mark.parametrize("line", [50, 90])
def test_a_line_of_work_in_parts(dtype, causal, group, q_len, line, monkeypatch):
    """Rows and query tokens split over launches: each part sees its own keys, lengths, LSE and strides."""
    lens = [0, 1, 2, 17, 64, 300, 65]
    c = Cache(lens, 2, 64, 32, seed=q_len)
    q = torch.zeros(len(lens), 2 * group, q_len, 64, device="cuda", dtype=torch_dtype(dtype))
    need = lambda: engine.attention_int4_workspace_bytes(q, c.pool, c.table, c.kv_lens, page_size=32)  # noqa: E731
    monkeypatch.setenv("TS_INT4_KERNEL", "pages")
    whole = need()
    monkeypatch.setenv("TS_INT4_LINE", str(line))
    assert need() < whole
    check_attention(c, dtype, 2 * group, q_len, causal=causal, path="pages", monkeypatch=monkeypatch)


def test_a_line_too_long_for_one_token_is_refused(monkeypatch):
    from tensorsmith_b200 import _lib

    c = Cache([300], 2, 64, 32)
    q = torch.zeros(1, 2, 1, 64, device="cuda")
    monkeypatch.setenv("TS_INT4_LINE", "10")
    with pytest.raises(_lib.EngineError) as error:
        engine.attention_int4(q, c.pool, c.table, c.kv_lens, page_size=32)
    assert error.value.status == _lib.ERR_UNSUPPORTED


def test_the_prefill_route_asks_for_no_more_than_the_pool(monkeypatch):
    """64 rows, one of which may hold 131072 tokens: dequantised whole, the batch would take 34 GB."""
    pool = engine.int4_pool(600, 8, 128, page_size=64)
    table = torch.full((64, 2048), -1, dtype=torch.int32, device="cuda")
    q = torch.zeros(64, 32, 64, 128, device="cuda", dtype=torch.bfloat16)
    args = (q, pool, table, torch.full((64,), 500, dtype=torch.int32, device="cuda"))
    kw = dict(page_size=64, max_len=131072)
    assert engine.attention_int4_path(*args, **kw) == "decode"  # the padding would cost more than it saves
    assert engine.attention_int4_workspace_bytes(*args, **kw) < 1 << 28
    monkeypatch.setenv("TS_INT4_KERNEL", "prefill")
    assert engine.attention_int4_path(*args, **kw) == "tcgen05"
    assert engine.attention_int4_workspace_bytes(*args, **kw) <= max(1 << 30, pool.numel())


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("q_len", [40, 200])
@pytest.mark.parametrize("dim, bound, parts", [(128, 1 << 20, "rows"), (64, 1 << 22, "heads")])
def test_the_prefill_route_in_parts(dtype, q_len, dim, bound, parts, monkeypatch):
    """Rows or KV heads one after the other in a workspace that holds NaN where nothing of a row is due."""
    lens = [300, 40, 0, 129]
    c = Cache(lens, 2, dim, 64, seed=q_len)
    keys, values = c.fill(dtype)
    table = torch.full((4, bound // 64), -1, dtype=torch.int32, device="cuda")
    table[:, : c.table.shape[1]] = c.table
    q = torch.from_numpy(np.random.default_rng(0).standard_normal((4, q_len, 6, dim))).to("cuda", torch_dtype(dtype))
    q = q.permute(0, 2, 1, 3)
    monkeypatch.setenv("TS_INT4_KERNEL", "prefill")
    args, kw = (q, c.pool, table, c.kv_lens), dict(page_size=64, max_len=bound)
    need = engine.attention_int4_workspace_bytes(*args, **kw)
    assert need == {"rows": 2, "heads": 1}[parts] * 4 * bound * dim
    workspace = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    out, lse = engine.attention_int4(*args, **kw, need_lse=True, workspace=workspace)
    engine.check_device_status()
    short = dict(page_size=64, max_len=300)
    whole, whole_lse = engine.attention_int4(q, c.pool, c.table, c.kv_lens, **short, need_lse=True)
    assert torch.equal(out, whole) and torch.equal(lse, whole_lse)
    ref, ref_lse, spread = oracle.attention_int4(to_np(q).astype(np.float64), keys, values, lens)
    unit = {"bfloat16": 2.0**-8, "float16": 2.0**-11}[dtype]
    # the bounds of test_gpu_int4_cache for the prefill kernel
    top = float(np.abs(ref_lse[np.isfinite(ref_lse)]).max()) + 10
    bound = unit * np.abs(ref) + (unit + 2.0**-13 + 2.0**-19 * (1 + top) + 300 * 2.0**-27) * spread + 1e-7
    assert (np.abs(to_np(out).astype(np.float64) - ref) <= bound).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dim, page", [(32, 16), (64, 16), (96, 32), (128, 64)])
@pytest.mark.parametrize("group", [1, 2, 7])
def test_several_waves_of_short_rows(dtype, dim, page, group):
    """A block a pair, many blocks an SM one after the other; every call gives the same bits."""
    lens = np.random.default_rng(group).integers(0, 60, 300)
    lens[:4] = [0, 60, 17, 1]
    c = Cache(lens, 4, dim, page, seed=dim)
    out = check_attention(c, dtype, 4 * group, 1)
    q = np.random.default_rng(1).standard_normal((300, 1, 4 * group, dim))  # as check_attention draws it
    q = torch.from_numpy(q).to("cuda", torch_dtype(dtype)).permute(0, 2, 1, 3)
    for _ in range(20):
        again, _ = engine.attention_int4(q, c.pool, c.table, c.kv_lens, page_size=page, max_len=60)
        assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("most, group, q_len", [(40, 2, 1), (90, 2, 1), (90, 3, 4)])
def test_more_rows_than_a_launch_takes(dtype, most, group, q_len):
    """1100 rows: the second launch starts at its own lengths, table rows, outputs and LSE (most <= 64: a block a
    pair, else a shared line)."""
    lens = np.random.default_rng(most).integers(0, most + 1, 1100)
    lens[[0, 1023, 1024, 1099]] = [most, 1, most, 2]
    check_attention(Cache(lens, 1, 32, 16, seed=1), dtype, group, q_len)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("dim", [64, 96, 256])
@pytest.mark.parametrize("lens, group, q_len", [([37, 5], 1, 1), ([700, 2000, 0], 3, 1), ([700, 90], 3, 7)])
def test_rows_that_no_wide_access_takes(dtype, dim, lens, group, q_len):
    """Queries and outputs with a channel stride of two from an odd element on, a strided LSE: the same bits."""
    c = Cache(lens, 2, dim, 32, seed=dim)
    c.fill(dtype)
    rows, heads = len(lens), 2 * group
    kw = dict(page_size=32, max_len=max(lens), need_lse=True)
    args = (c.pool, c.table, c.kv_lens)
    q = torch.randn(rows, heads, q_len, dim, device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    q = q.to(torch_dtype(dtype))
    want, want_lse = engine.attention_int4(q, *args, **kw)
    wide = torch.zeros(rows, q_len, heads, 2 * dim + 1, device="cuda", dtype=q.dtype)
    odd = wide[..., 1::2].permute(0, 2, 1, 3)
    odd.copy_(q)
    into = torch.full((rows, heads, q_len, 2 * dim + 1), 7.0, device="cuda", dtype=q.dtype)
    lse = torch.zeros(heads, rows, q_len, 3, device="cuda")[..., 1].permute(1, 0, 2)
    got, got_lse = engine.attention_int4(odd, *args, out=into[..., 1::2], lse=lse, **kw)
    engine.check_device_status()
    assert torch.equal(got, want) and torch.equal(got_lse, want_lse) and (into[..., ::2] == 7).all()

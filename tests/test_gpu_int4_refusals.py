"""Arguments of the 4-bit cache's calls that are refused before anything is launched."""

import pytest

from test_gpu_int4_cache import Cache
from test_gpu_kv_pages import Pages

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import _lib, engine  # noqa: E402


def test_workspaces_elsewhere_or_scattered():
    c = Cache([300, 200], 2, 64, 16)
    c.fill("bfloat16")
    q = torch.randn(2, 4, 1, 64, device="cuda", dtype=torch.bfloat16)
    p = Pages([20, 5], 12, 16)
    args = dict(page_size=16)
    calls = [lambda ws: engine.attention_int4(q, c.pool, c.table, c.kv_lens, workspace=ws, **args),
             lambda ws: engine.kv_pages_reserve(p.pool, p.table, p.lens, 1, p.refs, p.counters, workspace=ws, **args),
             lambda ws: engine.kv_pages_compact(p.pool, p.table, p.refs, p.counters, workspace=ws)]
    for call in calls:
        for bad in (torch.empty(1 << 22, dtype=torch.uint8), torch.empty(1, device="cuda").expand(1 << 22),
                    torch.empty(1 << 22, 2, dtype=torch.uint8, device="cuda")[:, 0]):
            with pytest.raises(ValueError, match="workspace"):
                call(bad)
        call(torch.empty(1 << 22, dtype=torch.uint8, device="cuda"))
        call(torch.empty(1, dtype=torch.uint8))  # too small to be used: a new one takes its place
    torch.cuda.synchronize()
    engine.check_device_status()


def test_tables_whose_rows_overlap():
    p = Pages([20, 5], 12, 16)
    shared = p.table[:1].expand(2, -1)
    index = torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlap"):
        engine.kv_pages_reserve(p.pool, shared, p.lens, 1, p.refs, p.counters, page_size=16)
    with pytest.raises(ValueError, match="overlap"):
        engine.kv_pages_fork(p.table, p.lens, index, p.refs, p.counters, page_size=16, table_out=shared)
    with pytest.raises(ValueError, match="overlap"):
        engine.kv_pages_compact(p.pool, shared, p.refs, p.counters)
    p.check()
    # rows that only read the same pages may share a table row
    c = Cache([40], 1, 64, 16)
    c.fill("bfloat16")
    q = torch.randn(1, 1, 1, 64, device="cuda", dtype=torch.bfloat16)
    one, _ = engine.attention_int4(q, c.pool, c.table, c.kv_lens, page_size=16)
    two, _ = engine.attention_int4(q.expand(2, -1, -1, -1), c.pool, c.table.expand(2, -1), c.kv_lens.repeat(2), page_size=16)
    assert torch.equal(two[0], one[0]) and torch.equal(two[1], one[0])


def test_tokens_before_the_first_are_reported():
    """A read-back from a negative start has no page for its first tokens, with lengths given or without."""
    c = Cache([20], 1, 64, 16)
    keys, _ = c.fill("float32")
    for lens in (None, c.kv_lens):
        k, _ = engine.kv_gather_int4(c.pool, c.table, 8, page_size=16, dtype=torch.float32, kv_lens=lens,
                                     starts=torch.tensor([-3], dtype=torch.int32, device="cuda"))
        assert engine.device_status() == (_lib.ERR_PAGE, 0x301)
        assert not k[0, :, :3].any() and (k[0, :, 3:].cpu().double().numpy() == keys[0][:, :5]).all()

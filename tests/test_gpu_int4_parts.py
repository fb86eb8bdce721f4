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

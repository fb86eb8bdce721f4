"""The 4-bit cache's definitions and refusals that need no GPU."""

import ctypes

import numpy as np
import pytest

import oracle
from tensorsmith_b200 import _lib, engine

torch = pytest.importorskip("torch")


def test_scale_has_five_bits_and_covers_the_group():
    rng = np.random.default_rng(0)
    amax = np.exp(rng.uniform(-40, 20, 20000)).astype(np.float32)
    s = oracle.int4_scale(amax)
    mant, _ = np.frexp(s)
    assert np.array_equal(mant * 32, np.round(mant * 32))
    inside = (amax / 7 >= 2.0**-20) & (amax / 7 <= 9216)
    assert (s[inside] >= np.float32(amax[inside] / np.float32(7))).all()
    assert (s[inside] <= amax[inside].astype(np.float64) / 7 * (1 + 1 / 16)).all()


def test_values_are_exact_in_both_half_types():
    scales = [2.0**e * m / 16 for e in range(-20, 14) for m in range(16, 32) if 2.0**e * m / 16 <= 9216]
    values = np.array([n * s for s in scales for n in range(-7, 8)])
    assert np.array_equal(values.astype(np.float16).astype(np.float64), values)
    got = torch.from_numpy(values).to(torch.bfloat16).double().numpy()
    assert np.array_equal(got, values)


@pytest.mark.parametrize("dim", [32, 64, 96, 128, 256])
def test_pack_round_trip(dim):
    rng = np.random.default_rng(dim)
    x = rng.standard_normal((2, 16, dim)) * np.exp(rng.uniform(-3, 3, (2, 16, 1)))
    (kn, ks), (vn, vs) = oracle.quantize_int4(x[0]), oracle.quantize_int4(x[1])
    block = oracle.pack_block(kn, ks, vn, vs)
    assert block.size == _lib.lib().ts_kv4_block_bytes(dim, 16) == 2 * 16 * (dim // 2 + dim // 16)
    k, v = oracle.unpack_block(block, 16, dim)
    assert np.array_equal(k, oracle.dequantize_int4(kn, ks)) and np.array_equal(v, oracle.dequantize_int4(vn, vs))
    step = np.repeat(ks, 32, axis=-1)
    assert (np.abs(k - x[0].astype(np.float32)) <= step * (0.5 + 1e-6)).all()


def test_quantiser_saturates_and_drops_nan():
    x = np.zeros((1, 64), np.float32)
    x[0, :4] = [np.inf, -np.inf, np.nan, 1e30]
    n, s = oracle.quantize_int4(x)
    assert s[0, 0] == 9216 and n[0, :4].tolist() == [7, -7, 0, 7] and s[0, 1] == 2.0**-20 and not n[0, 4:].any()


def test_ctypes_layout(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc unavailable")
    src = tmp_path / "probe.c"
    fields = {"ts_kv4_cache": _lib.Kv4Cache, "ts_page_pool": _lib.PagePool}
    lines = [f'printf("{s}.{f} %zu\\n", offsetof({s}, {f}));' for s, c in fields.items() for f, _ in c._fields_]
    lines += [f'printf("{s} %zu\\n", sizeof({s}));' for s in fields]
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "ts_attn.h"\nint main(void) {' + "\n".join(lines)
                   + "return 0; }")
    exe = tmp_path / "probe"
    include = Path(__file__).resolve().parent.parent / "include"
    subprocess.run([gcc, "-I", str(include), str(src), "-o", str(exe)], check=True)
    got = dict(x.rsplit(" ", 1) for x in subprocess.run([str(exe)], capture_output=True, text=True).stdout.split("\n") if x)
    assert engine._ATTN_STRUCT.size == ctypes.sizeof(_lib.AttnParams)
    assert engine._KV4_STRUCT.size == ctypes.sizeof(_lib.Kv4Cache)
    assert engine._POOL_STRUCT.size == ctypes.sizeof(_lib.PagePool)
    p = _lib.AttnParams.from_buffer_copy(engine._ATTN_STRUCT.pack(*range(1, 43)))
    assert (p.q.data, p.o.stride[3], p.lse, p.dtype, p.value_dim, p.scale, p.is_causal, p.causal_offset, p.kv_lens,
            p.mask_kind, p.mask_stride[3]) == (1, 20, 21, 25, 32, 33.0, 34, 35, 36, 37, 42)
    for s, c in fields.items():
        assert int(got[s]) == ctypes.sizeof(c)
        for f, _ in c._fields_:
            assert int(got[f"{s}.{f}"]) == getattr(c, f).offset, f


def _cache(**kw):
    args = dict(pool=4096, page_stride=2 * 9216, table=4096, table_stride=4, batch=2, slots=4, pages=8, kv_heads=2,
                head_dim=128, page_size=64)
    args.update(kw)
    return _lib.Kv4Cache(**args)


def _params(**kw):
    p = _lib.AttnParams()
    args = dict(dtype=_lib.BF16, batch=2, q_heads=4, kv_heads=2, q_len=1, kv_len=256, head_dim=128, value_dim=128,
                scale=0.1, is_causal=1, kv_lens=4096, mask_kind=0)
    args.update(kw)
    for name, value in args.items():
        setattr(p, name, value)
    p.q.data = p.o.data = 4096
    return p


# Arguments the entry points refuse before anything is launched (the addresses are never read).
@pytest.mark.parametrize("cache, params, status", [
    (dict(head_dim=100), {}, _lib.ERR_UNSUPPORTED),
    (dict(head_dim=288), {}, _lib.ERR_UNSUPPORTED),
    (dict(page_size=48), {}, _lib.ERR_UNSUPPORTED),
    (dict(pool=None), {}, _lib.ERR_INVALID_ARGUMENT),
    (dict(pool=4104), {}, _lib.ERR_INVALID_ARGUMENT),
    (dict(table=None), {}, _lib.ERR_INVALID_ARGUMENT),
    (dict(page_stride=9216), {}, _lib.ERR_INVALID_ARGUMENT),
    (dict(page_stride=2 * 9216 + 8), {}, _lib.ERR_INVALID_ARGUMENT),
    (dict(slots=0), {}, _lib.ERR_INVALID_ARGUMENT),
    (dict(pages=0), {}, _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(kv_len=257), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(kv_len=0), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(q_heads=3), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(q_len=0), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(batch=3), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(kv_lens=None), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(value_dim=64), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(scale=float("nan")), _lib.ERR_INVALID_ARGUMENT),
    ({}, dict(dtype=_lib.F64), _lib.ERR_UNSUPPORTED),
    ({}, dict(mask_kind=1), _lib.ERR_UNSUPPORTED),
])
def test_attention_refusals(cache, params, status):
    c, p = _cache(**cache), _params(**params)
    assert _lib.lib().ts_attn_int4(ctypes.byref(p), ctypes.byref(c), None, 0, None) == status
    assert _lib.lib().ts_attn_int4_workspace_size(ctypes.byref(p), ctypes.byref(c)) == 0


def test_attention_refuses_a_missing_workspace():
    c, p = _cache(slots=4096, pages=9000, table_stride=4096), _params(kv_len=4096 * 64)
    need = _lib.lib().ts_attn_int4_workspace_size(ctypes.byref(p), ctypes.byref(c))
    assert need > 0
    assert _lib.lib().ts_attn_int4(ctypes.byref(p), ctypes.byref(c), None, 0, None) == _lib.ERR_WORKSPACE
    assert _lib.lib().ts_attn_int4(ctypes.byref(p), ctypes.byref(c), 4096, need - 1, None) == _lib.ERR_WORKSPACE


def test_append_and_gather_refusals():
    h = _lib.lib()
    view, none = _lib.View4(4096, (ctypes.c_int64 * 4)(1, 1, 1, 1)), _lib.View4()
    ok = ctypes.byref(_cache())
    assert h.ts_kv_append_int4(view, view, _lib.BF16, 0, ok, 0, None, None, None) == _lib.ERR_CAPACITY
    assert h.ts_kv_append_int4(view, view, _lib.BF16, 1, ok, 256, None, None, None) == _lib.ERR_CAPACITY
    assert h.ts_kv_append_int4(view, view, _lib.BF16, 1, ok, -1, None, None, None) == _lib.ERR_CAPACITY
    assert h.ts_kv_append_int4(view, none, _lib.BF16, 1, ok, 0, None, None, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_append_int4(view, view, _lib.F64, 1, ok, 0, None, None, None) == _lib.ERR_UNSUPPORTED
    assert h.ts_kv_append_int4(view, view, _lib.BF16, 1, None, 0, None, None, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_gather_int4(ok, None, None, view, view, _lib.BF16, 257, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_gather_int4(ok, None, None, none, view, _lib.BF16, 1, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_gather_int4(ok, None, None, view, view, _lib.I8, 1, None) == _lib.ERR_UNSUPPORTED


def test_page_refusals():
    h = _lib.lib()
    pool = _lib.PagePool(4096, 1 << 20, 1024, 1024, 2, 8)
    bad = _lib.PagePool(4096, 1 << 20, 1016, 1024, 2, 8)
    other = _lib.PagePool(4096, 1 << 20, 1024, 512, 2, 8)
    a = 4096
    assert h.ts_kv_pages_copy(ctypes.byref(pool), ctypes.byref(bad), a, a, 1, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_pages_copy(ctypes.byref(pool), ctypes.byref(other), a, a, 1, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_pages_copy(ctypes.byref(pool), ctypes.byref(pool), None, a, 1, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_pages_fork(a, 4, a, 2, a, a, 4, 8192, 2, 4, 16, a, 8, a, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_pages_fork(a, 4, a, 2, a, 8192, 4, 8192, 0, 4, 16, a, 8, a, None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_pages_reserve(ctypes.byref(pool), a, 4, a, 2, 4, 16, -1, None, a, a, a, 1 << 20,
                                 None) == _lib.ERR_INVALID_ARGUMENT
    assert h.ts_kv_pages_reserve(ctypes.byref(pool), a, 4, a, 2, 4, 16, 1, None, a, a, a, 8,
                                 None) == _lib.ERR_WORKSPACE
    assert h.ts_kv_pages_compact(ctypes.byref(pool), a, 4, a, 4, 2, 4, a, a, a, None, 0, None) == _lib.ERR_WORKSPACE
    assert h.ts_kv_pages_compact(ctypes.byref(pool), a, 4, None, 4, 2, 4, a, a, a, a, 1 << 20,
                                 None) == _lib.ERR_INVALID_ARGUMENT


def test_python_refusals():
    assert engine.int4_block_bytes(128, 64) == 9216
    for dim, page in ((100, 64), (128, 48), (0, 16), (512, 16)):
        with pytest.raises(ValueError):
            engine.int4_block_bytes(dim, page)
    cpu = torch.zeros(4, 2, 9216, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        engine.kv_gather_int4(cpu, torch.zeros(1, 2, dtype=torch.int32), 1, page_size=64, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        engine.int4_pool(0, 1, 64, device="cpu")


def test_page_oracle_shares_copies_and_closes_up():
    """A worked example: two rows of a 4-token page size; the oracle's own behaviour."""
    pool = np.arange(8, dtype=np.int64).reshape(1, 8, 1) * 10
    o = oracle.PagesOracle([[3, 5, -1], [2, -1, -1]], [6, 4], [0, 0, 1, 1, 0, 1, 0, 0], pool, 4)
    o.fork([0, 0, 1])
    assert o.table.tolist() == [[3, 5, -1], [3, 5, -1], [2, -1, -1]] and o.refs.tolist() == [0, 0, 1, 2, 0, 2, 0, 0]
    assert o.reserve([1, 1, 1])  # row 0 copies page 5 to page 0, row 1 keeps it, row 2 gets page 1
    assert o.table.tolist() == [[3, 0, -1], [3, 5, -1], [2, 1, -1]] and o.refs.tolist() == [1, 1, 1, 2, 0, 1, 0, 0]
    assert o.pool[0, 0, 0] == 50
    o.compact()
    assert o.table.tolist() == [[3, 0, -1], [3, 4, -1], [2, 1, -1]] and o.refs.tolist() == [1, 1, 1, 2, 1, 0, 0, 0]
    assert not o.reserve([100, 0, 0])


def test_attention_refuses_a_line_of_work_past_32_bits():
    """64 heads of 2^25 stages for one token; half as many heads, or many tokens of a shorter row, run in parts."""
    def cache(heads, tokens):
        return _cache(slots=tokens // 64, table_stride=tokens // 64, kv_heads=heads, page_stride=heads * 9216)

    most = 0x7FFFFF00
    for heads, kv_len, q_len, ok in ((64, most, 1, False), (8, most, 1, True), (8, most // 2, 4096, True)):
        c = cache(heads, kv_len)
        p = _params(dtype=_lib.F32, q_heads=heads, kv_heads=heads, kv_len=kv_len, q_len=q_len)
        need = _lib.lib().ts_attn_int4_workspace_size(ctypes.byref(p), ctypes.byref(c))
        assert (need > 0) == ok
        assert _lib.lib().ts_attn_int4(ctypes.byref(p), ctypes.byref(c), None, 0, None) == (
            _lib.ERR_WORKSPACE if ok else _lib.ERR_UNSUPPORTED)


def test_append_refuses_to_advance_positions_in_place():
    h, ok = _lib.lib(), ctypes.byref(_cache())
    view = _lib.View4(4096, (ctypes.c_int64 * 4)(1, 1, 1, 1))
    # no steps: refused as such once the positions have passed
    for positions, out, status in ((4096, 4096, _lib.ERR_INVALID_ARGUMENT), (4096, 4100, _lib.ERR_INVALID_ARGUMENT),
                                   (4100, 4096, _lib.ERR_INVALID_ARGUMENT), (4096, 4104, _lib.ERR_CAPACITY),
                                   (None, 4096, _lib.ERR_CAPACITY), (4096, None, _lib.ERR_CAPACITY)):
        assert h.ts_kv_append_int4(view, view, _lib.BF16, 0, ok, 0, positions, out, None) == status


def test_page_calls_refuse_an_unaligned_workspace():
    h, a = _lib.lib(), 4096
    pool = ctypes.byref(_lib.PagePool(4096, 1 << 20, 1024, 1024, 2, 8))
    assert h.ts_kv_pages_reserve(pool, a, 4, a, 2, 4, 16, 1, None, a, a, a + 2, 1 << 20, None) == _lib.ERR_WORKSPACE
    assert h.ts_kv_pages_compact(pool, a, 4, a, 4, 2, 4, a, a, a, a + 1, 1 << 20, None) == _lib.ERR_WORKSPACE


def test_page_calls_refuse_tables_whose_rows_overlap():
    h, a, bad = _lib.lib(), 4096, _lib.ERR_INVALID_ARGUMENT
    pool = ctypes.byref(_lib.PagePool(4096, 1 << 20, 1024, 1024, 2, 8))
    for stride in (0, 3):  # of two rows with four slots
        assert h.ts_kv_pages_fork(a, 4, a, 2, a, 8192, stride, 8192, 2, 4, 16, a, 8, a, None) == bad
        # refused for the table, before the workspace that is missing
        assert h.ts_kv_pages_reserve(pool, a, stride, a, 2, 4, 16, 1, None, a, a, None, 0, None) == bad
        assert h.ts_kv_pages_compact(pool, a, stride, a, stride, 2, 4, a, a, a, None, 0, None) == bad
    assert h.ts_kv_pages_reserve(pool, a, 0, a, 1, 4, 16, 1, None, a, a, None, 0, None) == _lib.ERR_WORKSPACE

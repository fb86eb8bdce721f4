"""CPU checks of the C ABI's windowed, tree, cache-closing and log-probability calls: struct layouts, and refusals
before anything is launched (no GPU calls)."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from tensorsmith_b200 import _lib

HEADER = Path(__file__).resolve().parent.parent / "include" / "ts_attn.h"
FAKE = 1 << 20  # an address that is never read
STRUCTS = {"ts_window": _lib.Window, "ts_tree": _lib.Tree, "ts_kv_keep_params": _lib.KvKeepParams,
           "ts_token_logprobs": _lib.TokenLogprobs}
BAD, UNSUPPORTED, WORKSPACE = _lib.ERR_INVALID_ARGUMENT, _lib.ERR_UNSUPPORTED, _lib.ERR_WORKSPACE


def test_layouts(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("gcc unavailable")
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "ts_attn.h"', "int main(void) {"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("{name} %zu\\n", sizeof({name}));')
        lines += [f'printf("{name}.{f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    lines.append(f'printf("nodes %d\\ntop %d\\n", TS_TREE_MAX_NODES, TS_TOP_TOKENS_MAX); return 0; }}')
    (tmp_path / "probe.c").write_text("\n".join(lines))
    subprocess.run(["gcc", "-I", str(HEADER.parent), str(tmp_path / "probe.c"), "-o", str(tmp_path / "probe")], check=True)
    out = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout
    c = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for name, cls in STRUCTS.items():
        assert int(c[name]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(c[f"{name}.{f}"]) == getattr(cls, f).offset, f
    assert (int(c["nodes"]), int(c["top"])) == (_lib.TREE_MAX_NODES, _lib.TOP_TOKENS_MAX)


def problem(**kw):
    p = _lib.AttnParams()
    for name in "qkvo":
        view = getattr(p, name)
        view.data = FAKE
        view.stride = (ctypes.c_int64 * 4)(4096, 1024, 64, 1)
    p.lse, p.dtype, p.scale, p.is_causal = FAKE, _lib.F32, 1.0, 1
    p.batch = p.q_heads = p.kv_heads = 1
    p.q_len = p.kv_len = p.head_dim = p.value_dim = 16
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_window_refusals():
    lib = _lib.lib()
    good = _lib.Window(4, 1)
    assert lib.ts_attn_window_path(ctypes.byref(problem()), ctypes.byref(good)) == _lib.PATH_SIMT
    cases = [(problem(), _lib.Window(0, 0), BAD), (problem(), _lib.Window(-1, 0), BAD),
             (problem(), _lib.Window(3, -1), BAD), (problem(is_causal=0), good, BAD), (problem(batch=0), good, BAD),
             (problem(q_heads=3, kv_heads=2), good, BAD), (problem(causal_offset=-1), good, BAD),
             (problem(scale=float("nan")), good, BAD), (problem(dtype=7), good, UNSUPPORTED),
             (problem(head_dim=257), good, UNSUPPORTED), (problem(mask_kind=1, mask=FAKE), good, UNSUPPORTED),
             (problem(batch=70000), good, UNSUPPORTED), (problem(kv_len=(1 << 30) + 1), good, UNSUPPORTED),
             (problem(causal_offset=(1 << 62) + 1), good, BAD)]
    for p, w, status in cases:
        assert lib.ts_attn_fwd_window(ctypes.byref(p), ctypes.byref(w), FAKE, 1 << 40, None) == status
        assert lib.ts_attn_fwd_window_workspace_size(ctypes.byref(p), ctypes.byref(w)) == 0
        assert lib.ts_attn_window_path(ctypes.byref(p), ctypes.byref(w)) == status
        b = _lib.AttnBwdParams()
        b.fwd = p
        for name in ("dout", "dq", "dk", "dv"):
            getattr(b, name).data = FAKE
        assert lib.ts_attn_bwd_window(ctypes.byref(b), ctypes.byref(w), FAKE, 1 << 40, None) == status
        assert lib.ts_attn_bwd_window_workspace_size(ctypes.byref(b), ctypes.byref(w)) == 0
    assert lib.ts_attn_fwd_window(None, ctypes.byref(good), FAKE, 1 << 40, None) == BAD
    assert lib.ts_attn_fwd_window(ctypes.byref(problem()), None, FAKE, 1 << 40, None) == BAD
    b = _lib.AttnBwdParams()
    b.fwd = problem()
    assert lib.ts_attn_bwd_window(ctypes.byref(b), ctypes.byref(good), FAKE, 1 << 40, None) == BAD  # no gradients' views
    for name in ("dout", "dq", "dk", "dv"):
        getattr(b, name).data = FAKE
    need = lib.ts_attn_bwd_window_workspace_size(ctypes.byref(b), ctypes.byref(good))
    assert need > 0
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 8, need)):
        assert lib.ts_attn_bwd_window(ctypes.byref(b), ctypes.byref(good), ws, size, None) == WORKSPACE
    b.fwd.lse = None
    assert lib.ts_attn_bwd_window(ctypes.byref(b), ctypes.byref(good), FAKE, need, None) == BAD


def test_tree_refusals():
    lib = _lib.lib()

    def call(p, t, ws=FAKE, size=1 << 40):
        return lib.ts_attn_tree(ctypes.byref(p), ctypes.byref(t), ws, size, None)

    good = _lib.Tree(None, 0, 0, 0)
    tree = _lib.Tree(FAKE, 16, 0, 0)
    with_lens = lambda **kw: problem(kv_lens=FAKE, **kw)  # noqa: E731
    cases = [(problem(), good, BAD), (with_lens(), _lib.Tree(None, 0, -1, 0), BAD),
             (with_lens(), _lib.Tree(None, 0, 4, -1), BAD), (with_lens(kv_len=0), good, BAD),
             (with_lens(q_heads=3, kv_heads=2), good, BAD), (with_lens(dtype=9), good, UNSUPPORTED),
             (with_lens(q_len=65), tree, UNSUPPORTED), (with_lens(mask_kind=1, mask=FAKE), good, UNSUPPORTED),
             (with_lens(q_len=1 << 30, batch=2), good, UNSUPPORTED), (with_lens(value_dim=300), good, UNSUPPORTED)]
    for p, t, status in cases:
        assert call(p, t) == status
        assert lib.ts_attn_tree_path(ctypes.byref(p), ctypes.byref(t)) == status
        assert lib.ts_attn_tree_workspace_size(ctypes.byref(p), ctypes.byref(t)) == 0
    need = lib.ts_attn_tree_workspace_size(ctypes.byref(with_lens()), ctypes.byref(tree))
    assert need > 0
    for ws, size in ((None, need), (FAKE, need - 1), (FAKE + 4, need)):
        assert call(with_lens(), tree, ws, size) == WORKSPACE
    # the causal fields are not the tree's: nothing they hold is refused
    assert lib.ts_attn_tree_path(ctypes.byref(with_lens(is_causal=0, causal_offset=-5)), ctypes.byref(tree)) == _lib.PATH_SIMT
    for args in ((None, 4, FAKE, 2, 4, FAKE), (FAKE, 4, None, 2, 4, FAKE), (FAKE, 4, FAKE, 0, 4, FAKE),
                 (FAKE, 4, FAKE, 2, 0, FAKE), (FAKE, 4, FAKE, 2, 4, None)):
        assert lib.ts_tree_positions(*args, None) == BAD
    view = _lib.View4(FAKE, (ctypes.c_int64 * 4)(64, 64, 16, 1))
    rope = lambda dtype=_lib.F32, batch=1, rot=16, pos=FAKE: lib.ts_rope_at(  # noqa: E731
        view, view, dtype, batch, 1, 4, 16, rot, pos, FAKE, 0, None)
    assert (rope(dtype=6), rope(batch=0), rope(rot=3), rope(rot=18), rope(pos=None), rope(batch=1 << 17)) == (
        UNSUPPORTED, BAD, BAD, BAD, BAD, UNSUPPORTED)


def test_keep_refusals():
    lib = _lib.lib()

    def params(**kw):
        p = _lib.KvKeepParams()
        p.keys = (ctypes.c_void_p * 2)(FAKE, FAKE)
        p.values = (ctypes.c_void_p * 2)(FAKE, FAKE)
        p.key_stride = p.value_stride = (ctypes.c_int64 * 4)(256, 64, 16, 1)
        p.layers, p.batch, p.heads, p.head_dim, p.value_dim, p.capacity, p.nodes = 2, 1, 1, 16, 16, 4, 3
        p.base = p.path = p.counts = FAKE
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    strided = (ctypes.c_int64 * 4)(256, 64, 16, 2)
    cases = [(dict(layers=0), BAD), (dict(batch=0), BAD), (dict(head_dim=0), BAD), (dict(capacity=-1), BAD),
             (dict(nodes=0), BAD), (dict(base=None), BAD), (dict(path=None), BAD), (dict(counts=None), BAD),
             (dict(key_stride=strided), BAD), (dict(value_stride=strided), BAD), (dict(dtype=9), UNSUPPORTED),
             (dict(batch=70000), UNSUPPORTED), (dict(values=(ctypes.c_void_p * 2)(FAKE, None)), BAD),
             (dict(keys=None), BAD)]
    for kw, status in cases:
        assert lib.ts_kv_keep(ctypes.byref(params(**kw)), None) == status, kw
    assert lib.ts_kv_keep(None, None) == BAD


def test_logprob_refusals():
    lib = _lib.lib()

    def params(**kw):
        p = _lib.TokenLogprobs()
        p.logits, p.stride, p.dtype, p.rows, p.vocab, p.top = FAKE, 50, _lib.BF16, 4, 50, 2
        p.targets = p.logprob = p.entropy = p.norm = p.top_logprobs = p.top_indices = FAKE
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    both = [(dict(logits=None), BAD), (dict(rows=0), BAD), (dict(vocab=0, top=0), BAD), (dict(top=-1), BAD),
            (dict(top=51), BAD), (dict(top=33), UNSUPPORTED), (dict(dtype=_lib.F64), UNSUPPORTED),
            (dict(dtype=_lib.I8), UNSUPPORTED), (dict(logits=FAKE + 1), BAD), (dict(stride=-50), BAD)]
    backward = lambda p, grad=FAKE + 4096, stride=50: lib.ts_token_logprobs_bwd(  # noqa: E731
        ctypes.byref(p), FAKE, FAKE, FAKE, grad, stride, None)
    for kw, status in both:
        assert lib.ts_token_logprobs_fwd(ctypes.byref(params(**kw)), None) == status, kw
        assert backward(params(**kw)) == status, kw
    for kw in (dict(targets=None), dict(top_logprobs=None), dict(top_indices=None)):
        assert lib.ts_token_logprobs_fwd(ctypes.byref(params(**kw)), None) == BAD
    for kw in (dict(targets=None), dict(norm=None), dict(entropy=None), dict(top_indices=None)):
        assert backward(params(**kw)) == BAD
    assert backward(params(), grad=None) == BAD and backward(params(), grad=FAKE) == BAD
    assert backward(params(), stride=49) == BAD
    assert lib.ts_token_logprobs_fwd(None, None) == BAD

"""CPU checks of sizes that the windowed, tree and log-probability calls of the C ABI refuse (no GPU calls)."""

import ctypes

import pytest

from tensorsmith_b200 import _lib
from test_more_abi import FAKE, UNSUPPORTED, problem


@pytest.mark.parametrize("dtype", [_lib.F32, _lib.F64, _lib.BF16])
def test_longest_cache_of_a_tree(dtype):
    """As under a window, caches hold 2^30 keys at most: a tile's end behind them is still a 32-bit number."""
    lib = _lib.lib()
    for parents, window, sinks in ((FAKE, 0, 0), (None, 0, 0), (None, 5, 2**31 - 1)):
        tree = _lib.Tree(parents, 16, window, sinks)
        status = lambda n: lib.ts_attn_tree_path(ctypes.byref(problem(kv_len=n, kv_lens=FAKE, dtype=dtype)), ctypes.byref(tree))  # noqa: E731
        assert status(1 << 30) >= 0
        for keys in ((1 << 30) + 1, 2**31 - 100, 2**31 - 1):
            p = problem(kv_len=keys, kv_lens=FAKE, dtype=dtype)
            assert status(keys) == UNSUPPORTED
            assert lib.ts_attn_tree(ctypes.byref(p), ctypes.byref(tree), FAKE, 1 << 40, None) == UNSUPPORTED
            assert lib.ts_attn_tree_workspace_size(ctypes.byref(p), ctypes.byref(tree)) == 0

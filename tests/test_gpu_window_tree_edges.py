"""Windows and drafted trees where they can go wrong beside sizes and masks: head dimensions of half a quad."""

import random

import pytest

from plain64 import DTYPES
from test_gpu_tree import check, random_tree
from test_gpu_window import run

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402

NAN = float("nan")


def nan_everywhere(dtype, dim):
    """Windowed and tree calls whose operands are NaN: what blocks of the same shape find in shared memory."""
    q = torch.full((4, 4, 300, dim), NAN, dtype=DTYPES[dtype], device="cuda")
    out, lse = engine.forward(q, q, q, is_causal=True, window=100)
    engine.backward(q, q, q, out, lse, q, is_causal=True, window=100)
    lens = torch.full((4,), 300, dtype=torch.int32, device="cuda")
    engine.attention_tree(q[:, :, :5], q, q, lens)


# Two channels of a quad, alone and behind whole quads, in each class of head dimensions.
@pytest.mark.parametrize("dim,value_dim", [(2, 2), (6, 6), (66, 66), (130, 130), (254, 10), (64, 6), (6, 64), (12, 130)])
def test_f64_half_quads(dim, value_dim):
    wide = max(dim, value_dim)
    room = 64 if wide <= 64 else 128 if wide <= 128 else 256
    nan_everywhere("f64", room)
    run("f64", 2, 4, 2, 70, dim, 30, 3, value_dim=value_dim, path="simt")
    rng = random.Random(dim)
    nan_everywhere("f64", room)
    check("f64", 4, 2, dim, [9, 200, 131], [random_tree(rng, 7, b) for b in range(3)], value_dim=value_dim, path="simt")

"""The append's quantiser over every scale of the format: the corrected reciprocal of half types and the division
of fp32 must give the oracle's correctly rounded quotients, bit for bit."""

import numpy as np
import pytest

import oracle
from helpers import to_np, torch_dtype

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402

SCALES = [2.0**e * m / 16 for e in range(-20, 14) for m in range(16, 32) if 2.0**e * m / 16 <= 9216]


def groups_of(values):
    """Rows of 32: the largest value of each scale with 31 of its others, signs alternating."""
    rows = []
    for scale, x in zip(SCALES, values):
        x = np.resize(x, (-(-len(x) // 31), 31)) * np.where(np.arange(31) % 2, -1, 1)
        rows.append(np.concatenate([np.full((len(x), 1), 7 * scale), x], axis=1))
    return np.concatenate(rows)


def check(rows, dtype):
    dim, page = 64, 64
    tokens = -(-len(rows) * 32 // dim // page) * page
    x = torch.from_numpy(np.resize(rows, (tokens, dim // 32, 32)).reshape(1, 1, tokens, dim)).to("cuda", torch_dtype(dtype))
    pool = engine.int4_pool(tokens // page, 1, dim, page_size=page)
    table = torch.arange(tokens // page, dtype=torch.int32, device="cuda")[None]
    engine.kv_append_int4(x, -x, pool, table, page_size=page)
    k, v = engine.kv_gather_int4(pool, table, tokens, page_size=page, dtype=torch.float32)
    engine.check_device_status()
    n, scale = oracle.quantize_int4(to_np(x))
    np.testing.assert_array_equal(to_np(k), oracle.dequantize_int4(n, scale))
    np.testing.assert_array_equal(to_np(v), oracle.dequantize_int4(-n, scale))
    return scale


def test_every_scale_and_every_11_bit_value():
    """All fp16 values of the four binades below 8 scales: smaller ones have a quotient below a half."""
    values = []
    for scale in SCALES:
        top = np.floor(np.log2(scale)) + 2
        x = np.concatenate([2.0 ** (top - b) * (1 + np.arange(1024) / 1024) for b in range(4)])
        values.append(x[x <= 7 * scale])
    scale = check(groups_of(values), "float16")
    assert set(SCALES) <= set(np.unique(scale).tolist())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_every_scale_and_random_values(dtype):
    """With values at and beside the halves, where a quotient one unit off would round the other way."""
    rng = np.random.default_rng(0)
    values = []
    for scale in SCALES:
        halves = (np.arange(7) + 0.5) * scale
        near = np.concatenate([np.nextafter(halves.astype(np.float32), np.float32(d)) for d in (0, np.inf)])
        values.append(np.concatenate([halves, near, rng.uniform(0, 7 * scale, 500)]))
    check(groups_of(values), dtype)

"""Attention under a sliding window with sinks against fp64, forward and backward, on both kernel families."""

import pytest

from plain64 import DTYPES, Attention, window_seen, within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402


@pytest.fixture(autouse=True, params=["chosen", "split", "tile", "pair"])
def route(request, monkeypatch):
    """The way the engine chooses, the one along the keys, and a block for one or two query tiles."""
    if request.param != "chosen":
        monkeypatch.setenv("TS_WINDOW_KERNEL", request.param)


def heads(gen, rows, tokens, n, dim, dtype):
    """[B, H, T, D] as the projections give it: a view of [B, T, H, D]."""
    return torch.randn(rows, tokens, n, dim, generator=gen, device="cuda").to(DTYPES[dtype]).permute(0, 2, 1, 3)


def run(dtype, rows, q_heads, kv_heads, tokens, dim, window, sinks, offset=0, lens=None, capacity=None, value_dim=None,
        scale=None, path=None, grad=True, seed=1):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    keys = capacity or tokens + offset
    q = heads(gen, rows, tokens, q_heads, dim, dtype)
    k, v = heads(gen, rows, keys, kv_heads, dim, dtype), heads(gen, rows, keys, kv_heads, value_dim or dim, dtype)
    g = heads(gen, rows, tokens, q_heads, value_dim or dim, dtype)
    if lens is not None:
        lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    rule = dict(window=window, sinks=sinks, causal_offset=offset, kv_lens=lens, scale=scale)
    if path:
        assert engine.window_path(q, k, v, **rule) == path
    out, lse = engine.forward(q, k, v, is_causal=True, **rule)
    torch.cuda.synchronize()
    engine.check_device_status()
    ref = Attention(q, k, v, window_seen(rows, tokens, keys, window, sinks, offset, lens), scale,
                    cubic=engine.window_path(q, k, v, **rule) == "tcgen05")
    ref.check(out, lse)
    if grad:
        got = engine.backward(q, k, v, out, lse, g, is_causal=True, **rule)
        torch.cuda.synchronize()
        engine.check_device_status()
        want, bounds = ref.backward(g)
        for x, y, bound, name in zip(got, want, bounds, ("dq", "dk", "dv")):
            within(x, y, bound, name)
    return q, k, v, g, out, lse


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 72, 96, 128])
def test_head_dimensions(dtype, dim):
    run(dtype, 2, 4, 2, 300, dim, 70, 3, path="tcgen05")


# Windows around the tiles of 128 keys and 64 queries, sinks within and over a tile, one token to several tiles.
@pytest.mark.parametrize("tokens,window,sinks", [
    (1, 1, 0), (2, 1, 1), (127, 5, 0), (129, 128, 1), (256, 129, 130), (257, 1, 0), (385, 127, 127), (513, 300, 0),
    (700, 64, 260), (640, 700, 5), (1000, 999, 1000), (900, 256, 128), (300, 40, 2**31 - 1)])
def test_window_edges(tokens, window, sinks):
    run("bf16", 1, 2, 1, tokens, 64, window, sinks, path="tcgen05")


@pytest.mark.parametrize("tokens,window,sinks,offset", [(1, 40, 2, 500), (77, 33, 150, 1000), (300, 200, 0, 129),
                                                        (256, 1, 7, 4000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_chunk_behind_a_prefix(dtype, tokens, window, sinks, offset):
    run(dtype, 2, 4, 4, tokens, 64, window, sinks, offset=offset)


# Rows shorter than the queries leave some without a key; an empty row leaves all of them.
@pytest.mark.parametrize("dtype,dim", [("bf16", 128), ("f16", 64), ("f32", 40), ("f64", 64)])
def test_ragged_rows(dtype, dim):
    run(dtype, 5, 6, 2, 150, dim, 60, 9, lens=[400, 0, 1, 149, 151], capacity=420)


@pytest.mark.parametrize("dtype,dim,tokens,window,sinks", [
    ("f32", 64, 511, 128, 3), ("f32", 128, 200, 33, 40), ("f32", 200, 70, 50, 0), ("f32", 5, 40, 7, 2),
    ("f64", 128, 130, 31, 4), ("f64", 256, 40, 9, 1), ("f16", 256, 90, 40, 3), ("bf16", 33, 90, 40, 3),
    ("f32", 64, 1, 1, 0), ("f32", 64, 33, 1000, 0)])
def test_cuda_cores(dtype, dim, tokens, window, sinks):
    run(dtype, 2, 4, 2, tokens, dim, window, sinks, path="simt")


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f32", 32), ("f16", 256)])
def test_many_keys(dtype, dim):
    """A few queries behind more than a million keys: what the sinks and the last keys alone give, gradients of zero
    everywhere else."""
    tokens, window, sinks, keys = 5, 300, 3, 1_200_001
    gen = torch.Generator(device="cuda").manual_seed(6)
    make = lambda h, t: torch.randn(1, h, t, dim, generator=gen, device="cuda").to(DTYPES[dtype])  # noqa: E731
    q, k, v, g = make(2, tokens), make(1, keys), make(1, keys), make(2, tokens)
    rule = dict(is_causal=True, window=window, sinks=sinks, causal_offset=keys - tokens)
    out, lse = engine.forward(q, k, v, **rule)
    dq, dk, dv = engine.backward(q, k, v, out, lse, g, **rule)
    seen = torch.cat([torch.arange(sinks), torch.arange(keys - tokens - window + 1, keys)]).cuda()
    ref = Attention(q, k[:, :, seen], v[:, :, seen],
                    window_seen(1, tokens, len(seen), window, sinks, len(seen) - tokens),
                    cubic=engine.window_path(q, k, v, window=window, sinks=sinks) == "tcgen05")
    ref.check(out, lse)
    want, bounds = ref.backward(g)
    for x, y, bound, name in zip((dq, dk[:, :, seen], dv[:, :, seen]), want, bounds, ("dq", "dk", "dv")):
        within(x, y, bound, name)
    dk[:, :, seen] = 0
    dv[:, :, seen] = 0
    assert not dk.any() and not dv.any()


@pytest.mark.parametrize("dtype", ["f32", "f64", "bf16"])
def test_nan_stays_in_its_row(dtype):
    """A query that is NaN, and a key that only two queries see: their outputs are NaN (on CUDA cores the LSE too)."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (heads(gen, 1, 200, 2, 64, dtype) for _ in range(3))
    clean, clean_lse = engine.forward(q, k, v, is_causal=True, window=2)
    q[0, 1, 17, 3] = float("nan")
    k[0, 0, 90, 0] = float("nan")
    out, lse = engine.forward(q, k, v, is_causal=True, window=2)
    gone = torch.zeros(2, 200, dtype=torch.bool, device="cuda")
    gone[1, 17] = gone[0, 90] = gone[0, 91] = True
    assert out[0][gone].isnan().all() and (dtype == "bf16" or lse[0][gone].isnan().all())
    assert torch.equal(out[0][~gone], clean[0][~gone]) and torch.equal(lse[0][~gone], clean_lse[0][~gone])


def test_value_dimension_and_scale():
    run("f32", 1, 2, 2, 100, 48, 30, 2, value_dim=80, path="simt")
    run("bf16", 1, 2, 2, 100, 64, 30, 2, value_dim=32, path="simt")
    run("bf16", 1, 2, 2, 300, 64, 30, 2, scale=-0.2, path="simt")
    run("f16", 1, 2, 2, 300, 64, 30, 2, scale=0.31, path="tcgen05")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_wide_window_is_the_causal_rule(dtype, monkeypatch):
    """A window over everything gives what the call without one gives (same kernels for half types)."""
    monkeypatch.setenv("TS_WINDOW_KERNEL", "pair")
    q, k, v, g, out, lse = run(dtype, 2, 4, 2, 300, 64, 2**31 - 1, 0)
    plain, plain_lse = engine.forward(q, k, v, is_causal=True)
    if dtype == "bf16":
        assert torch.equal(out, plain) and torch.equal(lse, plain_lse)
    else:
        assert torch.allclose(out, plain, atol=1e-5) and torch.allclose(lse, plain_lse, atol=1e-5)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradients_against_differences(dtype):
    """Directional differences of sum(out * g) in the fp64 forward agree with the engine's gradients."""
    q, k, v, g, out, lse = run(dtype, 1, 2, 1, 140, 32, 40, 5, seed=4)
    got = engine.backward(q, k, v, out, lse, g, is_causal=True, window=40, sinks=5)
    seen = window_seen(1, 140, 140, 40, 5)
    gen = torch.Generator(device="cuda").manual_seed(9)
    base = [x.double() for x in (q, k, v)]
    refs, bounds = Attention(q, k, v, seen).backward(g)
    for which in range(3):
        step = torch.randn(base[which].shape, generator=gen, device="cuda", dtype=torch.float64)
        value = []
        for sign in (1, -1):
            moved = list(base)
            moved[which] = base[which] + sign * 1e-5 * step
            value.append(float((Attention(*moved, seen).out * g.double()).sum()))
        slope = (value[0] - value[1]) / 2e-5
        # central differences err by the third derivative, far below the roundings of the gradient
        allowed = float((bounds[which] * step.abs()).sum()) + 1e-6
        assert abs(float((got[which].double() * step).sum()) - slope) <= allowed


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides_and_given_outputs(dtype):
    """Contiguous, [B, T, H, D] and padded views agree; given outputs are filled and nothing around them."""
    q, k, v, g, out, lse = run(dtype, 2, 4, 2, 150, 64, 40, 5, grad=False)
    kw = dict(is_causal=True, window=40, sinks=5)
    flat, _ = engine.forward(q.contiguous(), k.contiguous(), v.contiguous(), **kw)
    assert torch.equal(flat, out)
    room = torch.full((2, 4, 152, 80), 7.0, dtype=q.dtype, device="cuda")
    into, _ = engine.forward(q, k, v, out=room[:, :, :150, :64], **kw)
    assert torch.equal(into, out)
    assert (room[:, :, 150:] == 7).all() and (room[:, :, :, 64:] == 7).all()
    wide = torch.zeros(2, 4, 150, 96, dtype=q.dtype, device="cuda")
    wide[..., 1:65] = q  # rows that start off the 16-byte grid
    odd, _ = engine.forward(wide[..., 1:65], k, v, **kw)
    Attention(q, k, v, window_seen(2, 150, 150, 40, 5), cubic=dtype == "bf16").check(odd)


def test_values_out_of_the_window_may_be_anything():
    """Key tiles that no query sees are not read: what they hold, NaN included, changes nothing."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    q = heads(gen, 1, 100, 2, 64, "bf16")
    k, v = (heads(gen, 1, 1500, 2, 64, "bf16").contiguous() for _ in range(2))
    kw = dict(is_causal=True, causal_offset=1400, window=100, sinks=4)
    out, _ = engine.forward(q, k, v, **kw)
    k[:, :, 128:1280], v[:, :, 128:1280] = float("nan"), float("inf")
    again, _ = engine.forward(q, k, v, **kw)
    assert torch.equal(out, again)


def test_streams_and_graphs():
    """On a side stream, and captured and replayed with new inputs."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    for dtype in ("bf16", "f32"):
        q, k, v, g = (heads(gen, 1, 200, 2, 64, dtype).contiguous() for _ in range(4))
        kw = dict(is_causal=True, window=50, sinks=2)

        def step():
            out, lse = engine.forward(q, k, v, **kw)
            return (out, lse, *engine.backward(q, k, v, out, lse, g, **kw))

        want = step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept = step()
        for x in (q, k, v, g):
            x.neg_()
        graph.replay()
        after = step()
        torch.cuda.synchronize()
        for i in (0, 1, 3, 4):  # dq on the tensor cores adds in no fixed order
            assert torch.equal(got[i], want[i]) and torch.equal(kept[i], after[i])
        assert torch.allclose(got[2].float(), want[2].float(), atol=2e-2)
        assert torch.allclose(kept[2].float(), after[2].float(), atol=2e-2)
    engine.check_device_status()


def test_refusals():
    q = torch.zeros(1, 2, 8, 64, device="cuda")
    for kw in (dict(window=0), dict(window=-3), dict(window=4, sinks=-1), dict(window=2**31), dict(window=1, sinks=2**31)):
        with pytest.raises(ValueError, match="window"):
            engine.forward(q, q, q, is_causal=True, **kw)
    with pytest.raises(ValueError, match="is_causal"):
        engine.forward(q, q, q, window=4)
    with pytest.raises(ValueError, match="mask"):
        engine.forward(q, q, q, is_causal=True, window=4, mask=torch.ones(8, 8, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="dropout"):
        engine.forward(q, q, q, is_causal=True, window=4, dropout=(0.1, 1, 0))
    with pytest.raises(ValueError, match="sinks"):
        engine.forward(q, q, q, is_causal=True, sinks=4)
    out, lse = engine.forward(q, q, q, is_causal=True, window=4)
    with pytest.raises(ValueError, match="sinks"):
        engine.backward(q, q, q, out, lse, q, is_causal=True, sinks=4)

"""Windows and drafted trees where they can go wrong beside sizes and masks: head dimensions of half a quad, NaN through
the join of many partial results, slots that nobody sees, more
queries than a grid's second dimension has tiles, positions in a column."""

import random

import pytest

from plain64 import DTYPES, Attention, tree_seen, window_seen, within
from test_gpu_tree import check, random_tree
from test_gpu_window import run

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402

NAN = float("nan")


def make(dtype, *shape, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=gen, device="cuda").to(DTYPES[dtype])


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


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("keys", [300, 20011])
@pytest.mark.parametrize("nodes,tree", [(1, False), (3, True)])
def test_nan_through_the_join(dtype, keys, nodes, tree):
    """A NaN query, and NaN keys in a part of a row: NaN in what sees them, output and LSE, with few partial results
    and with many; nothing changes elsewhere, and a padded node and an empty row stay zero."""
    q, k, v = make(dtype, 3, 2, nodes, 64), make(dtype, 3, 1, keys, 64, seed=1), make(dtype, 3, 1, keys, 64, seed=2)
    lens = torch.tensor([keys, keys - 60, 0], dtype=torch.int32, device="cuda")
    parents = torch.tensor([[-1, 0, -2]] * 3, dtype=torch.int32, device="cuda") if tree else None
    clean, clean_lse = engine.attention_tree(q, k, v, lens, parents, need_lse=True)
    q[0, 1, 0, 5] = NAN
    if tree:
        q[0, 0, 2] = NAN  # of a padded node
    k[1, 0, keys // 2 : keys // 2 + keys // 10] = NAN
    out, lse = engine.attention_tree(q, k, v, lens, parents, need_lse=True)
    gone = torch.zeros(3, 2, nodes, dtype=torch.bool, device="cuda")
    gone[0, 1, 0] = True
    gone[1, :, : 2 if tree else 1] = True
    assert out[gone].isnan().all() and lse[gone].isnan().all()
    assert torch.equal(out[~gone], clean[~gone]) and torch.equal(lse[~gone], clean_lse[~gone])
    assert not clean[2].any() and (clean_lse[2] == -float("inf")).all()
    if tree:
        assert not clean[:, :, 2].any() and (clean_lse[:, :, 2] == -float("inf")).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_nan_through_a_split_window(dtype, monkeypatch):
    monkeypatch.setenv("TS_WINDOW_KERNEL", "split")
    q, k, v = make(dtype, 1, 2, 2, 64), make(dtype, 1, 1, 9001, 64, seed=1), make(dtype, 1, 1, 9001, 64, seed=2)
    kw = dict(is_causal=True, window=8000, sinks=4, causal_offset=8999)
    clean, clean_lse = engine.forward(q, k, v, **kw)
    q[0, 1, 1, 0] = NAN
    out, lse = engine.forward(q, k, v, **kw)
    assert out[0, 1, 1].isnan().all() and lse[0, 1, 1].isnan()
    out[0, 1, 1], lse[0, 1, 1] = clean[0, 1, 1], clean_lse[0, 1, 1]
    assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("dtype,dim", [("bf16", 64), ("f16", 128), ("bf16", 96), ("f32", 64), ("f32", 33), ("f64", 64),
                                       ("f64", 6), ("bf16", 256), ("f16", 20)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 200)])
def test_slots_of_padded_nodes_may_hold_anything(dtype, dim, window, sinks):
    """Slots below kv_lens that nobody sees: of padded nodes, of their children, of children of nodes before the cache."""
    rng = random.Random(dim)
    nodes = 40
    odd = [-2, nodes, 2**31 - 1, -(2**31)]
    trees = [random_tree(rng, nodes) for _ in range(6)]
    for tree in trees[1:]:
        for i in rng.sample(range(nodes), 6):
            tree[i] = rng.choice([*odd, i])
    lens = [170, 150, 128 + 20, 40, 25, 9000]  # nodes over a tile's border, at a row's start, of a row in many parts
    q, k, v, kv_lens, parents, out, lse = check(dtype, 4, 2, dim, lens, trees, window=window, sinks=sinks,
                                                capacity=9000)
    hidden = ~tree_seen(trees, lens, 9000).any(2)[:, 0].cuda()  # no node sees the slot
    for b, n in enumerate(lens):
        hidden[b, : max(n - nodes, 0)] = hidden[b, n:] = False
    assert hidden.any()
    for fill in (NAN, float("inf"), -float("inf")):
        for x in (k, v):
            x.masked_fill_(hidden[:, None, :, None], fill)
        again, again_lse = engine.attention_tree(q, k, v, kv_lens, parents, window=window or None, sinks=sinks,
                                                 need_lse=True)
        torch.cuda.synchronize()
        engine.check_device_status()
        assert torch.equal(again, out) and torch.equal(again_lse, lse)


def test_more_queries_than_a_grid_has_rows_of_tiles():
    """4.2 million queries, 65537 tiles of 64: the last of them, and keys that the first ones alone see."""
    tokens, keys, dim, window, sinks, last = 65536 * 64 + 70, 200, 8, 40, 2, 100
    q, g = make("bf16", 1, 1, tokens, dim), make("bf16", 1, 1, tokens, dim, seed=1)
    k, v = make("bf16", 1, 1, keys, dim, seed=2), make("bf16", 1, 1, keys, dim, seed=3)
    kw = dict(is_causal=True, window=window, sinks=sinks)
    out, lse = engine.forward(q, k, v, **kw)
    dq, dk, dv = engine.backward(q, k, v, out, lse, g, **kw)
    torch.cuda.synchronize()
    engine.check_device_status()
    for first, n in ((0, 400), (tokens - last, last)):
        some = slice(first, first + n)
        ref = Attention(q[:, :, some], k, v, window_seen(1, n, keys, window, sinks, first))
        ref.check(out[:, :, some], lse[:, :, some])
        want, bounds = ref.backward(g[:, :, some])
        within(dq[:, :, some], want[0], bounds[0], "dq")
        if first == 0:  # behind the sinks, a key is seen by the window's queries alone
            within(dk[:, :, sinks:], want[1][:, :, sinks:], bounds[1][:, :, sinks:], "dk")
            within(dv[:, :, sinks:], want[2][:, :, sinks:], bounds[2][:, :, sinks:], "dv")


def test_positions_of_one_column():
    """Positions [B, 1] are a row's, as [B] are: token t stands at positions[b] + t."""
    x = make("f32", 2, 3, 5, 64)
    positions = torch.tensor([7, 300], dtype=torch.int32, device="cuda")
    assert torch.equal(engine.rope(x, positions=positions[:, None]), engine.rope(x, positions=positions))


@pytest.mark.parametrize("tokens", [1, 5])
def test_positions_that_are_refused(tokens):
    x = make("f32", 2, 3, tokens, 64)
    cuda = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    for positions in (cuda(2, 1).cpu(), cuda(2, tokens).cpu(), cuda(2).cpu(), cuda(1), cuda(1, 1), cuda(2, tokens + 1),
                      cuda(0)):
        with pytest.raises(ValueError, match="positions"):
            engine.rope(x, positions=positions)


@pytest.mark.parametrize("nodes,group", [(2, 1), (5, 2), (20, 2), (31, 5), (32, 3), (33, 4), (64, 5)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_slots_of_padded_nodes_in_trees_of_any_size(dtype, nodes, group):
    rng = random.Random(nodes)
    trees = [random_tree(rng, nodes) for _ in range(5)]
    for tree in trees:
        for i in rng.sample(range(nodes), max(1, nodes // 6)):
            tree[i] = rng.choice([-2, nodes, i])
    lens = [nodes + 100, nodes - 1, 128, nodes + 3000, nodes + 127]
    q, k, v, kv_lens, parents, out, lse = check(dtype, 2 * group, 2, 64, lens, trees, capacity=3100)
    hidden = ~tree_seen(trees, lens, 3100).any(2)[:, 0].cuda()
    for b, n in enumerate(lens):
        hidden[b, : max(n - nodes, 0)] = hidden[b, n:] = False
    assert hidden.any()
    v.masked_fill_(hidden[:, None, :, None], NAN)
    again, again_lse = engine.attention_tree(q, k, v, kv_lens, parents, need_lse=True)
    assert torch.equal(again, out) and torch.equal(again_lse, lse)

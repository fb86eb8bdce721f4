"""Attention of drafted trees and chains over a KV cache against fp64, their positions, and the closing of the cache."""

import random

import pytest

from plain64 import DTYPES, Attention, tree_seen, window_seen

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402


def random_tree(rng, nodes, padded=0):
    """Every node's parent: -1 or an earlier node; the last ``padded`` ones are padding."""
    return [rng.randint(-1, i - 1) if i < nodes - padded else rng.choice([-2, nodes, i]) for i in range(nodes)]


def inputs(dtype, rows, q_heads, kv_heads, nodes, dim, capacity, lens, value_dim=None, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(DTYPES[dtype])  # noqa: E731
    q = make(rows, nodes, q_heads, dim).permute(0, 2, 1, 3)
    k, v = make(rows, kv_heads, capacity, dim), make(rows, kv_heads, capacity, value_dim or dim)
    for b, n in enumerate(lens):  # what lies behind a row's keys is nobody's business
        k[b, :, max(n, 0):], v[b, :, max(n, 0):] = float("nan"), float("nan")
    return q, k, v, torch.tensor(lens, dtype=torch.int32, device="cuda")


def check(dtype, q_heads, kv_heads, dim, lens, parents=None, nodes=None, window=0, sinks=0, capacity=None, path=None,
          value_dim=None, scale=None, seed=0):
    rows, nodes = len(lens), nodes or len(parents[0])
    capacity = capacity or max(lens)
    q, k, v, kv_lens = inputs(dtype, rows, q_heads, kv_heads, nodes, dim, capacity, lens, value_dim, seed)
    tree = None if parents is None else torch.tensor(parents, dtype=torch.int32, device="cuda")
    kw = dict(window=window or None, sinks=sinks, scale=scale)
    got_path = engine.attention_tree_path(q, k, v, kv_lens, tree, **kw)
    assert path in (None, got_path)
    out, lse = engine.attention_tree(q, k, v, kv_lens, tree, need_lse=True, **kw)
    torch.cuda.synchronize()
    engine.check_device_status()
    if parents is None:
        seen = window_seen(rows, nodes, capacity, window, sinks, lens=kv_lens)
    else:
        seen = tree_seen(parents, lens, capacity, window, sinks).cuda()
    for b, n in enumerate(lens):
        k[b, :, max(n, 0):], v[b, :, max(n, 0):] = 0, 0
    Attention(q, k, v, seen, scale, cubic=got_path == "tcgen05").check(out, lse)
    return q, k, v, kv_lens, tree, out, lse


@pytest.mark.parametrize("dtype,dim,path", [("bf16", 64, "tcgen05"), ("f16", 128, "tcgen05"), ("bf16", 96, "tcgen05"),
                                            ("f16", 8, "tcgen05"), ("f32", 64, "simt"), ("f32", 128, "simt"),
                                            ("f64", 64, "simt"), ("bf16", 256, "simt"), ("f16", 20, "simt"),
                                            ("f32", 33, "simt"), ("f32", 256, "simt"), ("f64", 256, "simt")])
def test_types_and_head_dimensions(dtype, dim, path):
    rng = random.Random(dim)
    lens = [9, 200, 131, 128, 700]
    check(dtype, 6, 3, dim, lens, [random_tree(rng, 9, b % 4) for b in range(5)], capacity=720, path=path)


# Nodes of one to 64, groups that fill a 128-row tile partly, wholly and more than once.
@pytest.mark.parametrize("nodes,group", [(1, 1), (1, 8), (2, 5), (7, 3), (16, 8), (33, 4), (64, 2), (64, 5), (63, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tree_sizes(dtype, nodes, group):
    rng = random.Random(nodes * 9 + group)
    lens = [nodes, nodes + 1, nodes + 127, nodes + 128, 500]
    check(dtype, 2 * group, 2, 64, lens, [random_tree(rng, nodes, min(b, nodes - 1)) for b in range(5)], capacity=520)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (3, 0), (20, 70), (130, 1), (127, 300), (1000, 2)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_tree_under_a_window(dtype, window, sinks):
    rng = random.Random(window)
    lens = [24, 25, 100, 290, 600]
    deep = [list(range(-1, 23)) for _ in range(2)] + [random_tree(rng, 24, b) for b in range(3)]
    check(dtype, 4, 2, 64, lens, deep, window=window, sinks=sinks)


@pytest.mark.parametrize("nodes,window,sinks", [(1, 0, 0), (1, 50, 3), (5, 0, 0), (5, 2, 1), (70, 40, 5), (200, 0, 0),
                                                (300, 129, 64)])
@pytest.mark.parametrize("dtype", ["f16", "f32", "f64"])
def test_chains(dtype, nodes, window, sinks):
    check(dtype, 4, 2, 64, [nodes, nodes + 60, 1000, nodes // 2, 0], nodes=nodes, window=window, sinks=sinks)


def test_rows_that_hold_less_than_the_tree():
    """Nodes without a slot do not exist, nor do their children; a row without a key is zeros."""
    chain = list(range(-1, 11))
    wide = [-1] * 12
    for dtype in ("bf16", "f32"):
        for lens in ([0, 1, 5, 12], [11, 0, 3, 13]):
            check(dtype, 2, 1, 64, lens, [chain, wide, [-1, 0, 0, 1, 1, 2, 2, 3, 3, 4, 4, 5], chain], capacity=40)


def test_every_entry_of_parents():
    """Whatever parents holds, nothing but the cache is read: all values around the valid ones."""
    nodes = 6
    values = [-(2**31), -3, -2, -1, 0, 1, 4, 5, 6, 7, 64, 2**31 - 1]
    rng = random.Random(3)
    rows = [[rng.choice(values) for _ in range(nodes)] for _ in range(40)]
    for dtype in ("bf16", "f32"):
        check(dtype, 2, 2, 32, [50 + b for b in range(40)], rows, capacity=100)


def test_value_dimension_scale_and_strides():
    rng = random.Random(5)
    trees = [random_tree(rng, 5) for _ in range(2)]
    check("f32", 4, 2, 48, [60, 90], trees, value_dim=72)
    check("f32", 4, 2, 48, [60, 90], trees, value_dim=7)
    check("bf16", 4, 2, 64, [60, 90], trees, scale=-0.3, path="simt")
    q, k, v, lens, tree, out, lse = check("bf16", 4, 2, 64, [60, 90], trees, capacity=100, path="tcgen05")
    # a cache in [B, T, H, D] order, parents with padded rows, an output inside a larger buffer
    k2, v2 = (x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (k, v))
    wide = torch.full((2, 9), -7, dtype=torch.int32, device="cuda")
    wide[:, :5] = tree
    room = torch.full((2, 4, 6, 72), 3.0, dtype=q.dtype, device="cuda")
    room_lse = torch.full((2, 4, 6), 3.0, device="cuda")
    got, got_lse = engine.attention_tree(q.contiguous(), k2, v2, lens, wide[:, :5], out=room[:, :, :5, :64], need_lse=True,
                                         lse=room_lse[:, :, :5])
    assert torch.equal(got, out) and torch.equal(got_lse, lse)
    assert (room[:, :, 5] == 3).all() and (room[..., 64:] == 3).all() and (room_lse[:, :, 5] == 3).all()


def test_one_long_row_among_short_ones():
    """Units that many CTAs share beside units of a tile."""
    rng = random.Random(7)
    for dtype in ("bf16", "f32"):
        check(dtype, 4, 1, 64, [20001, 6, 40, 0, 129, 9000], [random_tree(rng, 6) for _ in range(6)], capacity=20010)


def test_many_rows():
    rng = random.Random(8)
    lens = [rng.randint(0, 300) for _ in range(700)]
    for dtype in ("bf16", "f32"):
        check(dtype, 1, 1, 32, lens, [random_tree(rng, 3) for _ in lens], capacity=300)


def test_offsets_past_32_bits():
    """A cache whose last rows start more than 2^31 elements behind its first."""
    rows, capacity, dim = 3, 9_000_000, 128  # 3.4e9 elements, 6.9 GB each
    gen = torch.Generator(device="cuda").manual_seed(1)
    k = torch.zeros(rows, 1, capacity, dim, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    q = torch.randn(rows, 2, 2, dim, generator=gen, device="cuda").bfloat16()
    for b in range(rows):
        k[b, 0, -300:] = torch.randn(300, dim, generator=gen, device="cuda").bfloat16()
        v[b, 0, -300:] = torch.randn(300, dim, generator=gen, device="cuda").bfloat16()
    lens = torch.full((rows,), capacity, dtype=torch.int32, device="cuda")
    out, _ = engine.attention_tree(q, k, v, lens, window=250)
    torch.cuda.synchronize()
    engine.check_device_status()
    seen = window_seen(rows, 2, 300, 250, 0, lens=torch.full((rows,), 300, device="cuda"))
    Attention(q, k[:, :, -300:], v[:, :, -300:], seen).check(out)


def test_streams_graphs_and_workspaces():
    rng = random.Random(2)
    trees = [random_tree(rng, 8) for _ in range(3)]
    for dtype in ("bf16", "f32"):
        q, k, v, lens, tree, want, _ = check(dtype, 8, 2, 64, [500, 100, 1500], trees, capacity=1500)
        need = engine.attention_tree_workspace_bytes(q, k, v, lens, tree)
        ws = torch.empty(need, dtype=torch.uint8, device="cuda")
        for _ in range(3):  # calls behind one another in one workspace
            got, _ = engine.attention_tree(q, k, v, lens, tree, workspace=ws)
            assert torch.equal(got, want)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got, _ = engine.attention_tree(q, k, v, lens, tree)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            kept, _ = engine.attention_tree(q, k, v, lens, tree)
        tree.copy_(tree.flip(0))
        lens.sub_(30)
        graph.replay()
        after, _ = engine.attention_tree(q, k, v, lens, tree)
        assert torch.equal(kept, after)
    engine.check_device_status()


def test_positions():
    rng = random.Random(11)
    trees = [random_tree(rng, 20, b) for b in range(6)] + [list(range(-1, 19))]
    base = [5, 0, 100, 7, 1, 2, 30]
    got = engine.tree_positions(torch.tensor(trees, dtype=torch.int32, device="cuda"),
                                torch.tensor(base, dtype=torch.int32, device="cuda")).tolist()
    for b, tree in enumerate(trees):
        for i in range(20):
            depth, j = 0, i
            while depth >= 0 and tree[j] != -1:
                depth, j = (depth + 1, tree[j]) if 0 <= tree[j] < j else (-1, j)
                if depth < 0:
                    break
            assert got[b][i] == (base[b] + depth if depth >= 0 else -1)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16", "f64"])
def test_rope_of_every_token(dtype):
    """Per-token positions give, token by token, what one offset gives."""
    gen = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(2, 5, 3, 64, generator=gen, device="cuda").to(DTYPES[dtype]).permute(0, 2, 1, 3)
    positions = torch.tensor([[7, 0, 3, 1000, 3], [1, 2, 2, 5, 40000]], dtype=torch.int32, device="cuda")
    for inverse in (False, True):
        got = engine.rope(x, positions=positions, rotary_dim=48, inverse=inverse)
        for b in range(2):
            for t in range(5):
                one = engine.rope(x[b:b + 1, :, t:t + 1], offset=int(positions[b, t]), rotary_dim=48, inverse=inverse)
                assert torch.equal(got[b:b + 1, :, t:t + 1], one)
    with pytest.raises(ValueError, match="positions"):
        engine.rope(x, positions=positions[:, :4])


def keep_reference(caches, base, path, counts):
    for pair in caches:
        for cache in pair:
            for b in range(cache.shape[0]):
                slots = [base[b] + i for i in path[b][: counts[b]]]
                cache[b, :, base[b]: base[b] + len(slots)] = cache[b][:, slots]


@pytest.mark.parametrize("dtype,dim,value_dim", [("f32", 32, 32), ("bf16", 128, 128), ("f16", 10, 6), ("f64", 5, 8),
                                                 ("i8", 64, 64), ("i8", 13, 3), ("f32", 1, 1)])
@pytest.mark.parametrize("layers", [1, 3, 70])
def test_keep(dtype, dim, value_dim, layers):
    rng = random.Random(dim)
    rows, heads, nodes, base = 5, 3, 21, [0, 4, 30, 9, 11]
    taken = [sorted(rng.sample(range(nodes), n)) for n in (0, 1, 21, 9, 13)]
    path = torch.full((rows, nodes), nodes + 5, dtype=torch.int32)  # entries behind counts are not looked at
    for b, t in enumerate(taken):
        path[b, : len(t)] = torch.tensor(t)
    gen = torch.Generator(device="cuda").manual_seed(layers)

    def make(width):
        x = torch.randint(-100, 100, (rows, heads, 60, width + 2), generator=gen, device="cuda")
        return x.to(torch.int8 if dtype == "i8" else DTYPES[dtype])[..., :width]

    caches = [(make(dim), make(value_dim)) for _ in range(layers)]
    want = [tuple(t.clone() for t in pair) for pair in caches]
    keep_reference(want, base, [p.tolist() for p in path], [len(t) for t in taken])
    cuda = lambda x: torch.as_tensor(x, dtype=torch.int32).cuda()  # noqa: E731
    engine.kv_keep(caches, cuda(base), cuda(path), cuda([len(t) for t in taken]))
    for got, ref in zip(caches, want):
        for a, b in zip(got, ref):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_far_addresses(dtype):
    """Heads and rows that lie more than 2^31 elements apart, read by the attention and closed up behind a path."""
    far, nodes, dim, room = 2**31 + 64, 6, 64, 700
    store = torch.empty(far + 4 * room * dim, dtype=DTYPES[dtype], device="cuda")
    k = store.as_strided((1, 2, room, dim), (far, far, dim, 1))
    v = store[2 * room * dim :].as_strided((1, 2, room, dim), (far, far, dim, 1))
    gen = torch.Generator(device="cuda").manual_seed(2)
    for x in (k, v):
        x.copy_(torch.randn(1, 2, room, dim, generator=gen, device="cuda"))
    q = torch.randn(1, 4, nodes, dim, generator=gen, device="cuda").to(k.dtype)
    cuda = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    lens, parents = cuda([650]), cuda([[-1, 0, 0, 1, 3, 2]])
    out, lse = engine.attention_tree(q, k, v, lens, parents, need_lse=True)
    near, near_lse = engine.attention_tree(q, k.contiguous(), v.contiguous(), lens, parents, need_lse=True)
    assert torch.equal(out, near) and torch.equal(lse, near_lse)
    rows = [x.transpose(0, 1) for x in (k, v)]  # the heads as rows of a batch
    want = [x.contiguous() for x in rows]
    path, counts, base = cuda([[1, 3, 4], [0, 2, 5]]), cuda([3, 2]), cuda([644, 644])
    keep_reference([want], [644, 644], path.tolist(), [3, 2])
    engine.kv_keep([rows], base, path, counts)
    assert all(torch.equal(a, b) for a, b in zip(rows, want))


def test_keep_stays_inside():
    """Counts and entries that no tree gives move nothing outside the cache."""
    room = torch.arange(4 * 2 * 10 * 8, device="cuda", dtype=torch.float32).view(4, 2, 10, 8)
    k, v = room[:, :1], room[:, 1:]
    before = room.clone()
    cuda = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    engine.kv_keep([(k, v)], cuda([8, -1, 2**31 - 1, 0]), cuda([[1, 2, 9], [1, 2, 3], [1, 2, 3], [-5, 0, 2**31 - 1]]),
                   cuda([3, 3, 3, 99]))
    before[0, :, 8] = before[0, :, 9]  # the one move that is inside
    assert torch.equal(room, before)


def test_refusals():
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, device="cuda", dtype=dtype)  # noqa: E731
    q, k, lens, tree = z(2, 4, 3, 64), z(2, 2, 9, 64), z(2, dtype=torch.int32), z(2, 3, dtype=torch.int32)
    call = engine.attention_tree
    call(q, k, k, lens, tree)
    bad = [
        (ValueError, (q[0], k, k, lens), {}), (ValueError, (q.cpu(), k, k, lens), {}),
        (TypeError, (q, k.half(), k, lens), {}), (ValueError, (q, k[..., :32], k, lens), {}),
        (ValueError, (q[:, :3], k, k, lens), {}), (ValueError, (q[:, :, :0], k, k, lens), {}),
        (ValueError, (q, k[:, :, :0], k[:, :, :0], lens), {}), (ValueError, (q, k, k, lens.long()), {}),
        (ValueError, (q, k, k, lens[:1]), {}), (ValueError, (q, k, k, lens, tree.long()), {}),
        (ValueError, (q, k, k, lens, tree[:, :2]), {}), (ValueError, (q, k, k, lens, tree.t().contiguous().t()), {}),
        (ValueError, (z(2, 4, 65, 64), k, k, lens, z(2, 65, dtype=torch.int32)), {}),
        (ValueError, (q, k, k, lens), dict(window=0)), (ValueError, (q, k, k, lens), dict(window=2, sinks=-1)),
        (ValueError, (q, k, k, lens), dict(sinks=2)), (ValueError, (q, k, k, lens), dict(scale=float("nan"))),
        (ValueError, (q, k, k, lens), dict(out=z(2, 4, 3, 32))), (ValueError, (q, k, k, lens), dict(need_lse=True, lse=z(2, 4, 4))),
        (ValueError, (q, k, k, lens), dict(workspace=torch.zeros(1 << 24, dtype=torch.uint8))),
        (TypeError, (q.to(torch.int32), k.to(torch.int32), k.to(torch.int32), lens), {}),
    ]
    for error, args, kw in bad:
        with pytest.raises(error):
            call(*args, **kw)
    with pytest.raises(ValueError):
        engine.tree_positions(tree.long(), lens)
    with pytest.raises(ValueError):
        engine.tree_positions(tree, lens[:1])
    v, layer = torch.zeros_like(k), (k.clone(), k.clone())
    engine.kv_keep([(k, v), layer], lens, tree, lens)
    for caches in ([(k, k)], [(k, v), (v, k)], [layer, layer]):  # two walks along one memory
        with pytest.raises(ValueError, match="once"):
            engine.kv_keep(caches, lens, tree, lens)
    for args in (([], lens, tree, lens), ([(k, k[:1])], lens, tree, lens), ([(k, k.half())], lens, tree, lens),
                 ([(k, k), (k[:, :, :8], k)], lens, tree, lens), ([(k, k)], lens.long(), tree, lens),
                 ([(k, k)], lens, tree[:1], lens), ([(k, k)], lens, tree, lens[:1]),
                 ([(k.transpose(2, 3), k.transpose(2, 3))], lens, tree, lens), ([(k.cpu(), k.cpu())], lens, tree, lens)):
        with pytest.raises(ValueError):
            engine.kv_keep(*args)

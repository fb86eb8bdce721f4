"""Cases that time attention with a sliding window and sinks (training, prompt chunks, one token over
a cache), attention of a tree of drafted tokens over a KV cache, the closing of a cache behind the
accepted path, and the log probabilities of given tokens with entropy and top alternatives.

Where ``own`` is false the operators run in their plain form, elementary torch operations in 32 bits;
where it is true, the engine's entry points run on the same state.

What the operators mean.

  window, sinks   a query at position i sees the keys j <= i with i - j < window or j < sinks.
  tree            row b's cache holds kv_lens[b] keys, the last T of them drafted tokens: node i sits
                  in slot kv_lens[b] - T + i and its parent is node parents[b, i] < i, or the last
                  committed token (-1).  A node sees every committed key, its ancestors and itself;
                  any other entry of parents marks a padded node, whose output is zero and which, like
                  its children, nobody sees.  With parents absent the drafted tokens are a chain.
                  Under a window, a node's position is the number of committed tokens plus its depth.
  keep            slot base[b] + path[b, k] moves to slot base[b] + k for the k < counts[b] accepted
                  nodes (ascending), keys and values of every layer.
  log probability logprob = x[target] - log sum exp x, entropy = -sum p log p, and the largest logits'
                  log probabilities in descending order, equal ones by index.
"""

import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
MAX_SCORES = 1 << 28  # elements of one block of scores in the plain forms


def engine():
    """The package's array-level entry points (only where ``own`` is true)."""
    root = os.path.join(os.getcwd(), "custom-ml-library_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from tensorsmith_b200 import engine as entry_points

    return entry_points


# -- cases -----------------------------------------------------------------------------------


def listed():
    return [
        # A training step's attention over long documents, window and first tokens, grouped heads.
        dict(op="window", name="window_train", dtype="bf16", grad=True, rows=1, q_heads=16, kv_heads=8, dim=128,
             q_len=16384, offset=0, window=4096, sinks=4),
        # A chunk of two prompts against what earlier chunks left in the cache; odd lengths.
        dict(op="window", name="window_chunk", dtype="f16", grad=False, rows=2, q_heads=8, kv_heads=8, dim=64,
             q_len=1001, offset=14999, window=2048, sinks=65),
        # A small model trained in fp32, as the library's own transformer is by default.
        dict(op="window", name="window_f32", dtype="f32", grad=True, rows=2, q_heads=4, kv_heads=2, dim=64, q_len=511,
             offset=0, window=128, sinks=3),
        # A handful of drafts in one short conversation with a small model: latency alone counts.
        dict(op="tree", name="tree_short", dtype="bf16", rows=1, q_heads=4, kv_heads=4, dim=64, nodes=8, chain=False,
             lo=37, hi=37, window=0, sinks=0),
        # A serving batch, 16 drafted tokens a row over ragged caches with shared heads.
        dict(op="tree", name="tree_batch", dtype="bf16", rows=32, q_heads=32, kv_heads=8, dim=128, nodes=16,
             chain=False, lo=500, hi=8192, window=0, sinks=0),
        # One token of two very long conversations, of which a window and the first tokens are seen.
        dict(op="tree", name="decode_window", dtype="f16", rows=2, q_heads=16, kv_heads=2, dim=128, nodes=1,
             chain=True, lo=60001, hi=131072, window=32768, sinks=4),
        # A small fp32 evaluation with an uneven head size, a wide tree and odd lengths.
        dict(op="tree", name="tree_f32", dtype="f32", rows=3, q_heads=6, kv_heads=3, dim=96, nodes=33, chain=False,
             lo=40, hi=701, window=0, sinks=0),
        # The cache of a small model closed up behind the accepted path.
        dict(op="keep", name="keep_small", dtype="f32", rows=4, kv_heads=4, dim=32, layers=4, nodes=8, lo=20, hi=200),
        # The same for a serving batch and a model of many layers.
        dict(op="keep", name="keep_large", dtype="bf16", rows=64, kv_heads=8, dim=128, layers=32, nodes=63, lo=60,
             hi=190),
        # The next tokens of a serving batch with the alternatives that an answer reports.
        dict(op="logprob", name="logprob_decode", dtype="f32", grad=False, rows=17, vocab=50257, top=20),
        # Documents scored by a model with a large vocabulary.
        dict(op="logprob", name="logprob_score", dtype="bf16", grad=False, rows=4096, vocab=128256, top=5),
        # A training loss with an entropy term: both gradients, an odd vocabulary, ignored targets.
        dict(op="logprob", name="logprob_train", dtype="bf16", grad=True, rows=4095, vocab=50257, top=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["window", "window", "tree", "tree", "keep", "logprob", "logprob"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([32, 64, 64, 96, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 1, 2, 4, 5, 8])
    if op == "window":
        grad = rng.random() < 0.5
        rows = _log(rng, 1, 8)
        q_len = _log(rng, 1, 2000 if dtype == "f32" else 16000)
        offset = 0 if rng.random() < 0.5 else _log(rng, 1, 16000)
        # all scores of the largest listed case at most, in fp32 a sixteenth of them
        most = 4.2e9 / (16 if dtype == "f32" else 1)
        while rows * kv_heads * group * q_len * (q_len + offset) * dim > most * 128:
            if rows > 1:
                rows = rows // 2
            elif offset:
                offset = offset // 2
            else:
                q_len = q_len * 2 // 3
        window = _log(rng, 1, q_len + offset)
        return dict(op=op, dtype=dtype, grad=grad, rows=rows, q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim,
                    q_len=q_len, offset=offset, window=window, sinks=rng.choice([0, 0, 1, 4, rng.randint(1, 200)]))
    if op == "tree":
        rows = _log(rng, 1, 64)
        nodes = 1 if rng.random() < 0.25 else _log(rng, 2, 64)
        hi = _log(rng, nodes, 131072)
        hi = max(nodes, min(hi, int(2.6e8 / (rows * kv_heads * dim)), int(1.3e8 / (rows * kv_heads * group * nodes))))
        window = 0 if rng.random() < 0.6 else _log(rng, 1, hi)
        return dict(op=op, dtype=dtype, rows=rows, q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, nodes=nodes,
                    chain=rng.random() < 0.3, lo=rng.randint(nodes, hi), hi=hi, window=window,
                    sinks=rng.randint(0, 70) if window else 0)
    if op == "keep":
        nodes, lo = _log(rng, 1, 64), rng.randint(0, 100)
        layers = _log(rng, 1, 32)
        rows = max(1, min(_log(rng, 1, 64), int(8e8 / (layers * kv_heads * dim * 264))))
        return dict(op=op, dtype=dtype, rows=rows, kv_heads=kv_heads, dim=dim, layers=layers, nodes=nodes, lo=lo,
                    hi=lo + rng.randint(0, 100))
    vocab = _log(rng, 32, 260000)
    rows = max(1, min(_log(rng, 1, 8192), int(4e8 / vocab)))
    return dict(op=op, dtype=dtype, grad=rng.random() < 0.4, rows=rows, vocab=vocab,
                top=rng.choice([0, 1, 5, 20, rng.randint(0, 32)]))


def _lengths(case):
    """One length a row, evenly spread over [lo, hi]."""
    n, lo, hi = case["rows"], case["lo"], case["hi"]
    return [lo + (hi - lo) * i // (n - 1) if n > 1 else hi for i in range(n)]


# -- inputs ----------------------------------------------------------------------------------


def _heads(gen, rows, tokens, heads, dim, dtype):
    """A projection [rows, tokens, heads, dim] seen as [rows, heads, tokens, dim]."""
    x = torch.randn(rows, tokens, heads, dim, generator=gen, device="cuda")
    return x.to(dtype).permute(0, 2, 1, 3)


def _tree(gen, rows, nodes):
    """Drafted trees: a root, children of random earlier nodes, some rows with fewer nodes (padding)."""
    at = torch.arange(nodes, device="cuda")
    pick = torch.rand(rows, nodes, generator=gen, device="cuda").pow(0.5)  # later parents more often
    parents = torch.minimum((pick * at).int(), (at - 1).clamp(min=0).int())
    parents[:, 0] = -1
    used = nodes - torch.randint(0, nodes // 4 + 1, (rows, 1), generator=gen, device="cuda")
    return torch.where(at < used, parents, -2).int().contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = dict(case)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    if op == "window":
        rows, heads, dim = case["rows"], case["kv_heads"], case["dim"]
        state["q"] = _heads(gen, rows, case["q_len"], case["q_heads"], dim, dtype)
        for name in ("k", "v"):
            state[name] = _heads(gen, rows, case["q_len"] + case["offset"], heads, dim, dtype)
        if case["grad"]:
            state["g"] = _heads(gen, rows, case["q_len"], case["q_heads"], dim, dtype)
    elif op == "tree":
        rows, heads, dim, nodes = case["rows"], case["kv_heads"], case["dim"], case["nodes"]
        order = torch.randperm(rows, generator=gen, device="cuda")
        state["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[order].contiguous()
        state["q"] = _heads(gen, rows, nodes, case["q_heads"], dim, dtype)
        for name in ("k", "v"):  # caches are [rows, heads, capacity, dim]
            cache = torch.empty(rows, heads, case["hi"], dim, dtype=dtype, device="cuda")
            for row in cache:
                row.copy_(torch.randn(row.shape, generator=gen, device="cuda"))
            state[name] = cache
        state["parents"] = None if case["chain"] else _tree(gen, rows, nodes)
    elif op == "keep":
        rows, nodes = case["rows"], case["nodes"]
        capacity = case["hi"] + nodes
        state["caches"] = [
            tuple(torch.randn(rows, case["kv_heads"], capacity, case["dim"], generator=gen, device="cuda").to(dtype)
                  for _ in range(2)) for _ in range(case["layers"])]
        state["base"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
        # about a third of the drafted nodes is accepted
        taken = torch.rand(rows, nodes, generator=gen, device="cuda") < 0.35
        state["counts"] = taken.sum(1).int()
        order = torch.where(taken, torch.arange(nodes, device="cuda"), nodes).sort(1).values
        state["path"] = order.clamp(max=nodes - 1).int().contiguous()
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.empty(rows, vocab, dtype=dtype, device="cuda")
        for part in logits.split(max(1, (1 << 26) // vocab)):
            part.copy_(3 * torch.randn(part.shape, generator=gen, device="cuda"))
        state["logits"] = logits
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        state["targets"] = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.05, -100, targets)
        if case["grad"]:
            for name in ("g_logprob", "g_entropy"):
                state[name] = torch.randn(rows, generator=gen, device="cuda") / rows
    return state


# -- the plain forms -------------------------------------------------------------------------


def _seen(case, first, tokens, keys, device):
    """[tokens, keys] truth values: what the queries at the positions from ``first`` see."""
    at = first + torch.arange(tokens, device=device)[:, None]
    key = torch.arange(keys, device=device)
    return (key <= at) & ((at - key < case["window"]) | (key < case["sinks"]))


def _window(s):
    group = s["q_heads"] // s["kv_heads"]
    scale = s["dim"] ** -0.5
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    rows, heads, tokens, dim = q.shape
    keys = k.shape[2]
    k_all, v_all = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    out = torch.empty(rows, heads, tokens, dim, device=q.device)
    if s["grad"]:
        g = s["g"].float()
        dq, dk, dv = torch.empty_like(out), torch.zeros_like(k_all), torch.zeros_like(v_all)
    block = max(1, min(tokens, MAX_SCORES // (rows * heads * keys)))
    for i in range(0, tokens, block):
        part = slice(i, min(tokens, i + block))
        seen = _seen(s, s["offset"] + i, part.stop - i, keys, q.device)
        score = (q[:, :, part] @ k_all.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, -torch.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        p /= p.sum(-1, keepdim=True)
        out[:, :, part] = p @ v_all
        if s["grad"]:
            dv += p.transpose(-1, -2) @ g[:, :, part]
            dp = g[:, :, part] @ v_all.transpose(-1, -2)
            dp -= (g[:, :, part] * out[:, :, part]).sum(-1, keepdim=True)
            ds = dp.mul_(p).mul_(scale)
            dq[:, :, part] = ds @ k_all
            dk += ds.transpose(-1, -2) @ q[:, :, part]
    dtype = s["q"].dtype
    if not s["grad"]:
        return out.to(dtype)
    fold = lambda x: x.view(rows, -1, group, keys, dim).sum(2).to(dtype)  # the query heads of a key head
    return out.to(dtype), dq.to(dtype), fold(dk), fold(dv)


def _ancestors(parents):
    """([rows, nodes, nodes] truth values: node j is node i or an ancestor of it, depths, padded nodes)."""
    rows, nodes = parents.shape
    seen = torch.zeros(rows, nodes, nodes, dtype=torch.bool, device=parents.device)
    depth = torch.zeros(rows, nodes, dtype=torch.long, device=parents.device)
    live = torch.zeros(rows, nodes, dtype=torch.bool, device=parents.device)
    every = torch.arange(rows, device=parents.device)
    for i in range(nodes):
        up = parents[:, i].long()
        inner = (up >= 0) & (up < i)
        above = up.clamp(0, nodes - 1)
        ok = (up == -1) | (inner & live[every, above])
        live[:, i] = ok
        depth[:, i] = torch.where(inner & ok, depth[every, above] + 1, 0)
        seen[:, i] = seen[every, above] & (inner & ok)[:, None]
        seen[:, i, i] = ok
    return seen, depth, live


def _tree_seen(s, keys):
    """[rows, nodes, keys] truth values: what every node sees of its row's cache."""
    lens, nodes = s["lens"].long(), s["nodes"]
    device = lens.device
    parents = s["parents"]
    if parents is None:
        parents = (torch.arange(nodes, device=device) - 1).expand(len(lens), nodes)
    seen, depth, live = _ancestors(parents)
    base = (lens - nodes)[:, None]
    key = torch.arange(keys, device=device)
    node = (key - base).clamp(0, nodes - 1)  # the node in a slot
    drafted = (key >= base) & (key < base + nodes)
    at = (base + depth)[:, :, None]
    where = torch.where(drafted, base + depth.gather(1, node), key)  # a slot's position
    visible = torch.where(drafted[:, None], seen.gather(2, node[:, None].expand(-1, nodes, -1)),
                          (key < base)[:, None] & live[:, :, None])
    if s["window"]:
        visible &= (at - where[:, None] < s["window"]) | (where < s["sinks"])[:, None]
    return visible


def _tree_attention(s):
    rows, heads, nodes, dim = s["q"].shape
    kv_heads, keys = s["k"].shape[1], s["k"].shape[2]
    q = s["q"].float().reshape(rows, kv_heads, -1, dim)
    score = (q @ s["k"].float().transpose(-1, -2)).mul_(dim ** -0.5).view(rows, heads, nodes, keys)
    score.masked_fill_(~_tree_seen(s, keys)[:, None], -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.view(rows, kv_heads, -1, keys) @ s["v"].float()).view(rows, heads, nodes, dim)
    return (out / torch.where(total == 0, 1.0, total)).to(s["q"].dtype)


def _keep(s):
    rows, nodes = s["path"].shape
    place = torch.arange(nodes, device="cuda")
    kept = place < s["counts"][:, None]
    row, k = torch.nonzero(kept, as_tuple=True)
    src = (s["base"][row] + s["path"][row, k]).long()
    dst = (s["base"][row] + k).long()
    for pair in s["caches"]:
        for cache in pair:
            cache[row, :, dst] = cache[row, :, src]
    return [cache for pair in s["caches"] for cache in pair]


def _logprob(s):
    rows, vocab = s["logits"].shape
    logprob, entropy = (torch.empty(rows, device="cuda") for _ in range(2))
    values = torch.empty(rows, s["top"], device="cuda")
    picks = torch.empty(rows, s["top"], dtype=torch.long, device="cuda")
    grad = torch.empty_like(s["logits"]) if s["grad"] else None
    step = max(1, MAX_SCORES // vocab)
    for i in range(0, rows, step):
        part = slice(i, min(rows, i + step))
        given = s["logits"][part].float()
        x = given - given.amax(-1, keepdim=True)
        e = torch.exp(x)
        total = e.sum(-1, keepdim=True)
        lp = x - torch.log(total)
        p = e / total
        h = -(p * lp).sum(-1)
        target = s["targets"][part]
        ignored = target == -100
        at = target.clamp(min=0)[:, None]
        logprob[part] = torch.where(ignored, 0.0, lp.gather(1, at)[:, 0])
        entropy[part] = h
        if s["top"]:  # a stable order: equal logits by index
            picks[part] = torch.sort(given, dim=-1, descending=True, stable=True).indices[:, : s["top"]]
            values[part] = lp.gather(1, picks[part])
        if s["grad"]:
            gl = torch.where(ignored, 0.0, s["g_logprob"][part])[:, None]
            d = -p * (gl + s["g_entropy"][part][:, None] * (lp + h[:, None]))
            d.scatter_add_(1, at, gl)
            grad[part] = d.to(grad.dtype)
    return (logprob, entropy, values, picks) + ((grad,) if s["grad"] else ())


def run(s):
    op = s["op"]
    if not own:
        return {"window": _window, "tree": _tree_attention, "keep": _keep, "logprob": _logprob}[op](s)
    e = engine()
    if op == "window":
        rule = dict(is_causal=True, causal_offset=s["offset"], window=s["window"], sinks=s["sinks"])
        out, lse = e.forward(s["q"], s["k"], s["v"], need_lse=s["grad"], **rule)
        if not s["grad"]:
            return out
        return (out, *e.backward(s["q"], s["k"], s["v"], out, lse, s["g"], **rule))
    if op == "tree":
        return e.attention_tree(s["q"], s["k"], s["v"], s["lens"], s["parents"], window=s["window"] or None,
                                sinks=s["sinks"])[0]
    if op == "keep":
        e.kv_keep(s["caches"], s["base"], s["path"], s["counts"])
        return [cache for pair in s["caches"] for cache in pair]
    r = e.token_logprobs(s["logits"], s["targets"], top=s["top"])
    out = (r.logprob, r.entropy, r.top_logprobs, r.top_indices)
    if s["grad"]:
        out += (e.token_logprobs_backward(s["logits"], s["targets"], r, s["g_logprob"], s["g_entropy"]),)
    return out


# -- what a pass cannot do without -----------------------------------------------------------


def _pairs(case):
    """Query-key pairs under the window, of one head."""
    total = 0
    window, sinks, offset, tokens = case["window"], case["sinks"], case["offset"], case["q_len"]
    for i in range(offset, offset + tokens):
        near = min(i + 1, window)
        total += near + max(0, min(sinks, i + 1 - near))
    return total


def work(case):
    op, size = case["op"], SIZES[case["dtype"]]
    if op == "window":
        pairs = _pairs(case) * case["rows"] * case["q_heads"]
        q = case["rows"] * case["q_heads"] * case["q_len"] * case["dim"] * size
        first = max(case["sinks"], 0)
        low = max(0, case["offset"] - case["window"] + 1)  # keys that some query sees
        keys = case["q_len"] + case["offset"] - max(0, low - min(first, low))
        kv = 2 * case["rows"] * case["kv_heads"] * keys * case["dim"] * size
        if not case["grad"]:
            return {"bytes": 2 * q + kv, "flops": 4 * case["dim"] * pairs}
        return {"bytes": 4 * q + 2 * kv, "flops": 14 * case["dim"] * pairs}
    if op == "tree":
        io = 2 * case["rows"] * case["q_heads"] * case["nodes"] * case["dim"] * size
        keys = 0
        for n in _lengths(case):
            seen = n
            if case["window"]:
                seen = min(n, case["window"] + case["nodes"] - 1 + case["sinks"])
            keys += seen
        pairs = keys * case["q_heads"] * case["nodes"]
        return {"bytes": io + 2 * keys * case["kv_heads"] * case["dim"] * size, "flops": 4 * case["dim"] * pairs}
    if op == "keep":
        moved = 0.35 * case["nodes"] * case["rows"] * case["kv_heads"] * case["layers"] * 2
        return {"bytes": 2 * moved * case["dim"] * size + 4 * case["rows"] * case["nodes"], "flops": 0}
    values = case["rows"] * case["vocab"]
    # read once, and once more written where there is a gradient (which needs the sums first, but a row fits on chip)
    return {"bytes": values * size * (2 if case["grad"] else 1) + case["rows"] * (24 + 12 * case["top"]),
            "flops": values * (12 if case["grad"] else 6)}


# -- the operators in 64 bits ----------------------------------------------------------------


def _exact_window(case, s):
    group, dim = case["q_heads"] // case["kv_heads"], case["dim"]
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    out = torch.zeros_like(q)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    tokens, keys = case["q_len"], case["q_len"] + case["offset"]
    for b in range(case["rows"]):
        for h in range(case["q_heads"]):
            hk = h // group
            for i in range(0, tokens, 2048):
                n = min(2048, tokens - i)
                low, high = case["offset"] + i, case["offset"] + i + n - 1  # positions of the block
                near = max(0, low - case["window"] + 1)
                cols = torch.cat((torch.arange(min(case["sinks"], near)), torch.arange(near, high + 1))).to(q.device)
                dist = torch.arange(low, high + 1, device=q.device)[:, None] - cols
                hidden = (dist < 0) | ((dist >= case["window"]) & (cols >= case["sinks"]))
                kk, vv = k[b, hk, cols], v[b, hk, cols]
                p = torch.softmax((q[b, h, i:i + n] @ kk.T / math.sqrt(dim)).masked_fill(hidden, -math.inf), -1)
                o = p @ vv
                out[b, h, i:i + n] = o
                if case["grad"]:
                    g = s["g"][b, h, i:i + n].double()
                    ds = p * (g @ vv.T - (g * o).sum(1, keepdim=True)) / math.sqrt(dim)
                    dq[b, h, i:i + n] = ds @ kk
                    dk[b, hk].index_add_(0, cols, ds.T @ q[b, h, i:i + n])
                    dv[b, hk].index_add_(0, cols, p.T @ g)
    return (out, dq, dk, dv) if case["grad"] else out


def _exact_tree(case, s):
    q = s["q"].double()
    group, nodes = case["q_heads"] // case["kv_heads"], case["nodes"]
    out = torch.zeros_like(q)
    for b, n in enumerate(s["lens"].tolist()):
        base = n - nodes
        parents = list(range(-1, nodes - 1)) if s["parents"] is None else s["parents"][b].tolist()
        chains = []  # every node's path from the root, or None
        for i, up in enumerate(parents):
            if up == -1:
                chains.append([i])
            else:
                chains.append(chains[up] + [i] if 0 <= up < i and chains[up] is not None else None)
        hidden = torch.ones(nodes, n, dtype=torch.bool)
        for i, chain in enumerate(chains):
            if chain is None:
                continue
            at = base + len(chain) - 1
            low = max(0, at - case["window"] + 1) if case["window"] else 0
            hidden[i, min(low, base):base] = False
            hidden[i, : min(case["sinks"], base)] = False
            for d, j in enumerate(chain):
                if base + d >= low or base + d < case["sinks"]:
                    hidden[i, base + j] = False
        hidden = hidden.to(q.device)
        dead = torch.tensor([chain is None for chain in chains], device=q.device)
        for hk in range(case["kv_heads"]):
            k, v = s["k"][b, hk, :n].double(), s["v"][b, hk, :n].double()
            mine = q[b, hk * group:(hk + 1) * group]
            score = (mine @ k.T / math.sqrt(case["dim"])).masked_fill(hidden, -math.inf)
            p = torch.softmax(score, -1).masked_fill(dead[:, None], 0.0)
            out[b, hk * group:(hk + 1) * group] = p @ v
    return out


def _exact_logprob(case, s):
    rows, vocab = s["logits"].shape
    logprob, entropy = (torch.empty(rows, dtype=torch.float64, device="cuda") for _ in range(2))
    top = torch.empty(rows, case["top"], dtype=torch.float64, device="cuda")
    grad = torch.empty(rows, vocab, dtype=torch.float64, device="cuda") if case["grad"] else None
    for i in range(0, rows, max(1, (1 << 26) // vocab)):
        part = slice(i, min(rows, i + max(1, (1 << 26) // vocab)))
        lp = torch.log_softmax(s["logits"][part].double(), -1)
        p = lp.exp()
        entropy[part] = -(p * lp).sum(1)
        target = s["targets"][part]
        real = target != -100
        picked = lp[torch.arange(len(target), device="cuda"), target.clamp(min=0)]
        logprob[part] = torch.where(real, picked, 0.0)
        if case["top"]:
            top[part] = torch.topk(lp, case["top"], dim=1).values
        if case["grad"]:
            gl = s["g_logprob"][part].double() * real
            ge = s["g_entropy"][part].double()
            d = -p * gl[:, None] - ge[:, None] * p * (lp + entropy[part][:, None])
            d[torch.arange(len(target), device="cuda"), target.clamp(min=0)] += gl
            grad[part] = d
    return (logprob, entropy, top, None) + ((grad,) if case["grad"] else ())


def exact(case, seed):
    op = case["op"]
    if op == "keep":
        return None  # moved bytes
    s = prepare(case, seed)
    return {"window": _exact_window, "tree": _exact_tree, "logprob": _exact_logprob}[op](case, s)

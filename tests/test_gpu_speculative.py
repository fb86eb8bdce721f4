"""The new operators together, as a model uses them: drafted trees checked over caches and closed behind the accepted
path, sliding windows in training and cached decoding, log probabilities as a loss.

Tolerances are those of the fp32 transformer tests: logits rtol 2e-4 / atol 2e-5, gradients rtol 1e-3 / atol 1e-5.
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine, nn, no_grad  # noqa: E402


def model(window=None, sinks=0, layers=3, vocab=61, max_seq_len=96):
    np.random.seed(11)
    config = nn.TransformerConfig(vocab, dim=64, num_heads=4, num_kv_heads=2, num_layers=layers, hidden_dim=96,
                                  max_seq_len=max_seq_len, window=window, sinks=sinks)
    return nn.TransformerLM(config, device="cuda")


def close(a, b):
    np.testing.assert_allclose(a.detach().cpu().numpy(), b.detach().cpu().numpy(), rtol=2e-4, atol=2e-5)


def full(lm, tokens):
    with no_grad(), torch.no_grad():
        return lm.eval()(torch.tensor([tokens], device="cuda"))[0]


def path_of(parents, node):
    path = [node]
    while parents[path[-1]] != -1:
        path.append(parents[path[-1]])
    return path[::-1]


@pytest.mark.parametrize("window,sinks", [(None, 0), (7, 2), (1, 0), (30, 5)])
@pytest.mark.parametrize("quantized", [False, True])
def test_tree_step_keep_and_go_on(window, sinks, quantized):
    """Logits of every node are those of its path alone; after the path is kept the rows go on, each at its length."""
    lm = model(window, sinks)
    rng = np.random.default_rng(5)
    prompt = rng.integers(0, 61, (2, 20))
    parents = [[-1, 0, 0, 1, 1, 2, 5], [-1, -1, 0, 1, 3, 4, -2]]
    drafts = rng.integers(0, 61, (2, 7))
    paths, counts = [[0, 2, 5, 6], [1, 3, 0, 0]], [4, 2]
    with no_grad(), torch.no_grad():
        lm.eval()
        caches = lm.new_cache(2, quantized=quantized)
        lm(torch.tensor(prompt), caches=caches)
        logits = lm(torch.tensor(drafts), caches=caches, parents=parents)
        nn.keep_drafts(caches, 7, paths, counts)
        assert [c.lengths.tolist() for c in caches] == [[24, 22]] * 3
        more = torch.tensor(rng.integers(0, 61, (2, 3)))
        after = lm(more, caches=caches)
        assert caches[0].lengths.tolist() == [27, 25]
    for b in range(2):
        for node in range(7):
            if parents[b][node] == -2:
                continue
            ids = path_of(parents[b], node)
            text = [*prompt[b], *drafts[b][ids]]
            want = full(lm, text)[-1]
            if quantized:  # int8 rows: the reference's own tolerance for its quantised cache
                np.testing.assert_allclose(logits[b, node].cpu().numpy(), want.cpu().numpy(), rtol=0.08, atol=0.02)
            else:
                close(logits[b, node], want)
        kept = [*prompt[b], *drafts[b][paths[b][: counts[b]]], *more[b].tolist()]
        want = full(lm, kept)[-3:]
        if quantized:
            np.testing.assert_allclose(after[b].cpu().numpy(), want.cpu().numpy(), rtol=0.08, atol=0.02)
        else:
            close(after[b], want)


def test_greedy_speculation_gives_greedy_text():
    """Trees of guesses, right and wrong ones, checked by argmax: the text is that of plain greedy decoding."""
    lm = model(max_seq_len=80)
    prompt = torch.tensor([[3, 9, 27, 1, 44]], device="cuda")
    want = lm.generate(prompt, 30, temperature=0)[0].tolist()
    rng = np.random.default_rng(0)
    text = prompt[0].tolist()
    with no_grad(), torch.no_grad():
        lm.eval()
        caches = lm.new_cache(1)
        text.append(int(lm(prompt, caches=caches)[0, -1].argmax()))
        steps = 0
        while len(text) < len(want):
            # the root is the last sure token; below it a chain of guesses with wrong siblings
            known = want[len(text): len(text) + int(rng.integers(0, 4))]
            tokens, parents, last = [text[-1]], [-1], 0
            for guess in known:
                tokens += [(guess + 1) % 61, guess]
                parents += [last, last]
                last = len(tokens) - 1
            choice = lm(torch.tensor([tokens]), caches=caches, parents=[parents])[0].argmax(-1).tolist()
            path = [0]
            while True:
                below = [i for i, up in enumerate(parents) if up == path[-1] and tokens[i] == choice[path[-1]]]
                if not below:
                    break
                path.append(below[0])
            nn.keep_drafts(caches, len(tokens), [path])
            text += [tokens[i] for i in path[1:]] + [choice[path[-1]]]
            steps += 1
    assert text[: len(want)] == want and steps < 30


@pytest.mark.parametrize("window,sinks", [(5, 0), (9, 3), (64, 0)])
def test_windowed_model_cached_and_whole(window, sinks):
    lm = model(window, sinks)
    tokens = torch.randint(0, 61, (2, 50), generator=torch.Generator().manual_seed(3))
    with no_grad(), torch.no_grad():
        whole = lm.eval()(tokens)
        for cuts in ((0, 50), (0, 20, 21, 22, 50), (0, 1, 2, 40, 50)):
            caches = lm.new_cache(2)
            parts = [lm(tokens[:, a:b], caches=caches) for a, b in zip(cuts, cuts[1:])]
            close(torch.cat(parts, 1), whole)
        wide = model(None)
        wide.load_state_dict(lm.state_dict())
        assert (torch.allclose(whole, wide.eval()(tokens), rtol=2e-4, atol=2e-5)) == (window >= 50)
    text = lm.generate(tokens[:, :10], 12, temperature=0)
    assert torch.equal(text, lm.generate(tokens[:, :10], 12, temperature=0, use_cache=False))


def test_windowed_training_gradients():
    """One training step of a windowed model against the same model with the mask in torch operations."""
    lm = model(6, 2, layers=2).train()
    tokens = torch.randint(0, 61, (2, 33), generator=torch.Generator().manual_seed(4)).cuda()
    result = lm.token_logprobs(tokens[:, :-1], tokens[:, 1:], top=3)
    weight = torch.linspace(0.5, 1.5, 64, device="cuda").view(2, 32)
    loss = -(result.logprob * weight).mean() - 0.1 * result.entropy.mean() + 0.01 * result.top_logprobs.sum()
    loss.backward()
    got = {n: p.grad.clone() for n, p in lm.named_parameters()}
    for p in lm.parameters():
        p.grad = None

    at = torch.arange(32, device="cuda")
    dist = at[:, None] - at
    seen = (dist >= 0) & ((dist < 6) | (at < 2))

    def rope(x):
        inv = engine.rope_inv_freq(16, 10000.0, x.device)
        angle = at[:, None] * inv
        c, s = angle.cos(), angle.sin()
        even, odd = x[..., 0::2], x[..., 1::2]
        return torch.stack((even * c - odd * s, odd * c + even * s), -1).flatten(-2)

    def attention(block, h):
        m = block.attention
        q, k, v = (f(h).view(2, 32, n, 16).transpose(1, 2) for f, n in ((m.q_proj, 4), (m.k_proj, 2), (m.v_proj, 2)))
        q, k, v = rope(q), rope(k).repeat_interleave(2, 1), v.repeat_interleave(2, 1)
        p = torch.softmax((q @ k.transpose(-1, -2) / 4).masked_fill(~seen, -torch.inf), -1)
        return m.out_proj((p @ v).transpose(1, 2).reshape(2, 32, 64))

    x = lm.token_embedding_weight[tokens[:, :-1]]
    for block in lm.blocks:
        x = x + attention(block, block.attention_norm(x))
        x = x + block.ffn(block.ffn_norm(x))
    lp = torch.log_softmax(lm.final_norm(x) @ lm.output_weight.T, -1)
    picked = lp.gather(-1, tokens[:, 1:, None])[..., 0]
    entropy = -(lp.exp() * lp).sum(-1)
    want = -(picked * weight).mean() - 0.1 * entropy.mean() + 0.01 * lp.topk(3).values.sum()
    np.testing.assert_allclose(float(loss), float(want), rtol=2e-5)
    want.backward()
    for name, p in lm.named_parameters():
        np.testing.assert_allclose(got[name].cpu().numpy(), p.grad.cpu().numpy(), rtol=1e-3, atol=1e-5, err_msg=name)


def test_token_logprobs_as_the_loss():
    """Their negated mean over the targets that count is the model's loss, with the same gradients; half types, shared
    and broadcast gradients."""
    lm = model(layers=1)
    tokens = torch.randint(0, 61, (3, 20), generator=torch.Generator().manual_seed(6)).cuda()
    targets = tokens.roll(-1, 1).clone()
    targets[:, -1] = -100
    want = lm.loss(tokens, targets)
    want.backward()
    ref = [p.grad.clone() for p in lm.parameters()]
    for p in lm.parameters():
        p.grad = None
    got = -lm.token_logprobs(tokens, targets).logprob.sum() / (targets != -100).sum()
    got.backward()
    np.testing.assert_allclose(float(got), float(want), rtol=1e-5)
    for p, r in zip(lm.parameters(), ref):
        np.testing.assert_allclose(p.grad.cpu().numpy(), r.cpu().numpy(), rtol=1e-3, atol=1e-6)
    x = torch.randn(7, 90, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    t = torch.arange(7, device="cuda")
    r = nn.token_logprobs(x, t, top=2)
    assert not r.top_indices.requires_grad and r.logprob.dtype == torch.float32
    (r.logprob.sum() + r.entropy.mean()).backward()
    y = x.detach().double().requires_grad_()
    lp = torch.log_softmax(y, -1)
    (lp[t, t].sum() - (lp.exp() * lp).sum(-1).mean()).backward()
    # one rounding of the gradient to bf16 (2^-8), fp32 sums below it
    assert (x.grad.double() - y.grad).abs().le(2.0 ** -8 * y.grad.abs() + 1e-6).all()
    with torch.no_grad():
        assert torch.equal(nn.token_logprobs(x, t).logprob, r.logprob)


def test_sdpa_window():
    """nn.scaled_dot_product_attention under a window: forward and VJP on the tape."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    q, k, v = (torch.randn(2, h, 40, 32, generator=gen, device="cuda") for h in (4, 2, 2))
    t = [nn.attention.Tensor(x.clone(), requires_grad=True, device="cuda") for x in (q, k, v)]
    out = nn.scaled_dot_product_attention(*t, is_causal=True, enable_gqa=True, window=9, sinks=2)
    o, lse = engine.forward(q, k, v, is_causal=True, window=9, sinks=2)
    assert torch.equal(out._data, o)
    out.sum().backward() if hasattr(out, "sum") else out.backward(torch.ones_like(o))
    for x, g in zip(t, engine.backward(q, k, v, o, lse, torch.ones_like(o), is_causal=True, window=9, sinks=2)):
        assert torch.allclose(x._grad if isinstance(x._grad, torch.Tensor) else x._grad._data, g, atol=1e-6)


def test_refusals():
    with pytest.raises(ValueError, match="window"):
        nn.TransformerConfig(8, window=0)
    with pytest.raises(ValueError, match="sinks"):
        nn.TransformerConfig(8, sinks=2)
    with pytest.raises(ValueError, match="dropout"):
        nn.TransformerConfig(8, window=4, dropout=0.1)
    q = nn.attention.Tensor(torch.zeros(1, 2, 4, 32), device="cuda")
    for kw in (dict(window=3), dict(window=0, is_causal=True), dict(sinks=3, is_causal=True), dict(window=2.5, is_causal=True),
               dict(window=3, is_causal=True, dropout_p=0.5),
               dict(window=3, is_causal=True, attn_mask=nn.attention.Tensor(torch.ones(4, 4, dtype=torch.bool), device="cuda"))):
        with pytest.raises(ValueError):
            nn.scaled_dot_product_attention(q, q, q, **kw)
    lm = model(window=4)
    with pytest.raises(ValueError, match="paged"):
        lm.new_cache(1, quantized="int4")
    tokens = torch.zeros(2, 3, dtype=torch.long)
    with no_grad(), torch.no_grad():
        lm.eval()
        with pytest.raises(ValueError, match="caches"):
            lm(tokens, parents=[[-1, 0, 1]] * 2)
        caches = lm.new_cache(2)
        with pytest.raises(ValueError, match="parents"):
            lm(tokens, caches=caches, parents=[[-1, 0]] * 2)
        with pytest.raises(ValueError, match="mask"):
            lm(tokens, caches=caches, parents=[[-1, 0, 1]] * 2, attn_mask=torch.ones(3, 3, dtype=torch.bool, device="cuda"))
        assert [c.length for c in caches] == [0, 0, 0]
        lm(tokens, caches=caches, parents=[[-1, 0, 1]] * 2)
        for args in ((3, [[0, 1]]), (4, [[0], [0]]), (3, [[1, 0], [0, 1]]), (3, [[0, 3], [0, 1]]), (3, [[0.5], [0]]),
                     (3, [[0], [0]], [2, 0]), (3, [[0], [0]], [1])):
            with pytest.raises(ValueError):
                nn.keep_drafts(caches, *args)
        with pytest.raises(ValueError):
            nn.keep_drafts([], 0, [[0]])
        caches[1].truncate(2)
        with pytest.raises(ValueError, match="position"):
            nn.keep_drafts(caches, 1, [[0], [0]])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("captured", [False, True])
def test_two_streams_at_once(dtype, captured):
    """A decoding loop on each of two streams, eager or as graphs replayed side by side, gives what it gives alone."""
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def work(seed):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        make = lambda *s: torch.randn(*s, generator=gen, device="cuda").to(dtype)  # noqa: E731
        q, k, v, x = make(3, 8, 6, 64), make(3, 2, 900, 64), make(3, 2, 900, 64), make(18, 20011)
        lens, tree = ints([800, 77, 301]), ints([[-1, 0, 0, 1, 2, 2]] * 3)
        path, counts = ints([[0, 2, 5], [0, 1, 3], [0, 0, 0]]), ints([3, 3, 1])
        keys, values, goal = k.clone(), v.clone(), torch.arange(18, device="cuda")

        def step():
            keys.copy_(k)
            values.copy_(v)
            o, lse = engine.attention_tree(q, keys, values, lens, tree, need_lse=True)
            w, _ = engine.forward(q, keys, values, is_causal=True, kv_lens=lens, window=200, sinks=3)
            engine.kv_keep([(keys, values)], lens - 6, path, counts)
            lp = engine.token_logprobs(x, goal, top=3)
            return [o, lse, w, keys, values, *lp, engine.token_logprobs_backward(x, goal, lp, lp.logprob)]

        return step

    steps = [work(1), work(2)]
    want = [[t.clone() for t in step()] for step in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in steps]
    got = [None, None]
    if captured:
        graphs = [torch.cuda.CUDAGraph() for _ in steps]
        for i, (graph, step) in enumerate(zip(graphs, steps)):
            with torch.cuda.graph(graph, stream=streams[i]):
                got[i] = step()
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                if captured:
                    graphs[i].replay()
                else:
                    got[i] = steps[i]()
    torch.cuda.synchronize()
    engine.check_device_status()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_a_failed_step_gives_ragged_rows_back():
    """A layer that fails leaves every row of every cache at its own length."""
    lm = model()
    tokens = torch.zeros(2, 3, dtype=torch.long)
    with no_grad(), torch.no_grad():
        lm.eval()
        caches = lm.new_cache(2)
        lm(tokens, caches=caches, parents=[[-1, 0, 1]] * 2)
        nn.keep_drafts(caches, 3, [[0, 1, 2], [0, 1, 2]], [3, 1])
        broken = lm.blocks[2].ffn.forward
        lm.blocks[2].ffn.forward = lambda x: 1 / 0
        with pytest.raises(ZeroDivisionError):
            lm(tokens, caches=caches)
        lm.blocks[2].ffn.forward = broken
        assert [c.lengths.tolist() for c in caches] == [[3, 1]] * 3

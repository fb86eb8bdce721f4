"""Log probabilities of tokens, entropies, alternatives and their gradient against fp64.

Bounds: a difference x - m of logits is off by 2^-24 of itself, its exponential by that much times itself and a few
steps (2^-22 relative for the approximation); so is, relative to the largest, every term of the sums, whose n additions
in fp32 (a few hundred a thread, then a tree) add n 2^-24 at most.  With d the spread of a row's logits
(-inf apart), rho = 2^-24 (3 d + n_thread + 64) bounds the relative error of a probability and the absolute one of
log sum; the log probability and the entropy round a handful of times more at their own size.
"""

import math

import pytest

from plain64 import DTYPES, half_step, within

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
from tensorsmith_b200 import engine  # noqa: E402


def reference(logits, targets, top, ignore=-100):
    x = logits.double()
    none = (x == -math.inf).all(-1)
    x = x.masked_fill(none[..., None], 0.0)
    lp = torch.log_softmax(x, -1)
    p = lp.exp()
    entropy = -(p * lp.masked_fill(p == 0, 0)).sum(-1)
    lp = lp.masked_fill(none[..., None], -math.inf)
    p = p.masked_fill(none[..., None], 0.0)
    real = targets != ignore
    at = targets.masked_fill(~real, 0)
    logprob = lp.gather(-1, at[..., None])[..., 0].masked_fill(~real, 0.0)
    order = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[..., :top]
    finite = x.masked_fill(torch.isinf(x), float("nan"))
    spread = (x.amax(-1) - finite.nan_to_num(math.inf).amin(-1)).clamp(0, 200)
    rho = 2.0 ** -24 * (3 * spread + x.shape[-1] / 128 + 64)
    return dict(lp=lp, p=p, logprob=logprob, entropy=entropy.masked_fill(none, 0.0), indices=order,
                values=lp.gather(-1, order), rho=rho, none=none, real=real, at=at)


def equal_or_within(got, want, bound, what):
    inf = torch.isinf(want)
    assert torch.equal(got.double()[inf], want[inf]), what
    within(got.masked_fill(inf, 0), want.masked_fill(inf, 0), bound.expand_as(want).masked_fill(inf, 0), what)


def check(logits, targets, top=0, grads=True, ignore=-100, seed=0):
    r = reference(logits, targets, top, ignore)
    got = engine.token_logprobs(logits, targets, top=top, ignore_index=ignore)
    torch.cuda.synchronize()
    e = 2.0 ** -24
    size = r["logprob"].abs().nan_to_num(posinf=0)
    equal_or_within(got.logprob, r["logprob"], r["rho"] + 8 * e * (1 + size), "logprob")
    # entropy = log s - t / s: t's terms carry d as a factor
    log_s = r["values"][..., 0].abs() if top else r["lp"].amax(-1).abs()
    within(got.entropy, r["entropy"], r["rho"] * (2 + r["entropy"].abs()) + 8 * e * (1 + r["entropy"] + log_s.nan_to_num(posinf=0)),
           "entropy")
    if top:
        assert torch.equal(got.top_indices, r["indices"])
        equal_or_within(got.top_logprobs, r["values"],
                        r["rho"][..., None] + 8 * e * (1 + r["values"].abs().nan_to_num(posinf=0)), "alternatives")
    if not grads:
        return got
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda like: torch.randn(like.shape, generator=gen, device="cuda")  # noqa: E731
    gl, ge, gt = draw(got.logprob), draw(got.entropy), draw(got.top_logprobs)
    for use in ((gl, None, None), (None, ge, None), (gl, ge, gt if top else None)):
        d = engine.token_logprobs_backward(logits, targets, got, *use, ignore_index=ignore)
        torch.cuda.synchronize()
        p, lp, u = r["p"], r["lp"].masked_fill(r["p"] == 0, 0), half_step(logits.dtype)
        a, b, t = (torch.zeros_like(r["entropy"]) if x is None else x.double() for x in (use[0], use[1], None))
        a = a * r["real"]
        total = a + (use[2].double().sum(-1) if use[2] is not None else 0)
        want = -p * (total[..., None] + b[..., None] * (lp + r["entropy"][..., None]))
        own = torch.zeros_like(want).scatter_add_(-1, r["at"][..., None], a[..., None])
        if use[2] is not None:
            own.scatter_add_(-1, r["indices"], use[2].double())
        want = (want + own).masked_fill(r["none"][..., None], 0.0)
        sizes = (a.abs() + (use[2].double().abs().sum(-1) if use[2] is not None else 0))[..., None]
        inner = sizes + b.abs()[..., None] * (lp.abs() + r["entropy"][..., None])
        rho = (r["rho"] * (4 + r["entropy"]))[..., None]
        bound = p * inner * (4 * rho + 64 * e) + 8 * e * own.abs() + u * want.abs()
        bound = bound + (2.0 ** -25 if logits.dtype == torch.float16 else 1e-37)
        within(d, want, bound, "gradient")
    return got


def make(rows, vocab, dtype, spread=3.0, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = (spread * torch.randn(rows, vocab, generator=gen, device="cuda")).to(DTYPES[dtype])
    t = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
    t[::7] = -100
    return x, t


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 33, 127, 255, 1000, 4095, 4097, 8193, 50257])
def test_vocabularies(dtype, vocab):
    x, t = make(9, vocab, dtype, seed=vocab)
    check(x, t, top=min(5, vocab))


@pytest.mark.parametrize("rows", [1, 2, 147, 149, 700])
@pytest.mark.parametrize("vocab", [50, 3001])
def test_row_counts(rows, vocab):
    check(*make(rows, vocab, "bf16", seed=rows), top=3)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("top", [0, 1, 2, 31, 32])
def test_top(dtype, top):
    for vocab in (32, 40, 300, 700, 33000, 260001):
        check(*make(3, vocab, dtype, seed=vocab), top=top, grads=vocab < 1000)


def test_few_long_rows():
    for rows in (1, 3, 20):
        check(*make(rows, 260000, "f32", seed=rows), top=8)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ties_go_to_the_lowest_index(dtype):
    """Constant rows, rows of few values, rising, falling and repeating ones: more candidates than any buffer."""
    n = 40011
    at = torch.arange(n, device="cuda")
    rows = [torch.zeros(n), torch.ones(n) * -5, (at % 2).cpu().float(), (at % 3 == 2).cpu().float() * 7,
            at.cpu().float() / 1000, -at.cpu().float() / 1000, (at // 512).cpu().float(), (at % 512 < 9).cpu().float(),
            (at >= n - 40).cpu().float(), -(at < 33).cpu().float(), (at % 4096 == 17).cpu().float()]
    x = torch.stack(rows).to("cuda", DTYPES[dtype])
    t = torch.arange(len(rows), device="cuda")
    for top in (1, 9, 32):
        check(x, t, top=top, grads=top == 9)
    check(torch.zeros(4, 300, device="cuda", dtype=DTYPES[dtype]), t[:4], top=32)
    # -0 and 0 are equal
    z = torch.zeros(1, 100, device="cuda", dtype=DTYPES[dtype])
    z[0, ::2] = -0.0
    assert engine.token_logprobs(z, t[:1], top=4).top_indices.tolist() == [[0, 1, 2, 3]]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [70, 5003])
def test_masked_logits(dtype, vocab):
    """-inf and the type's lowest value: one survivor, some, none at all; masked targets and alternatives."""
    x, t = make(8, vocab, dtype, seed=3)
    t[:] = torch.arange(8, device="cuda") * 3
    low = torch.finfo(DTYPES[dtype]).min
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 3] = 2.0
    x[2, 40:] = -math.inf
    x[3] = low
    x[4, 20:] = low
    x[5] = -math.inf
    x[5, 15] = low
    x[6, 18] = -math.inf
    x[7, :] = low
    x[7, 21:24] = -math.inf
    check(x, t, top=7)


@pytest.mark.parametrize("vocab", [70, 5003])
def test_nan_and_inf(vocab):
    x, t = make(4, vocab, "f32", seed=5)
    x[0, 9] = float("nan")
    x[1, 60] = math.inf
    got = engine.token_logprobs(x, t.clamp(min=0), top=3)
    assert torch.isnan(got.logprob[0]) and torch.isnan(got.entropy[0]) and torch.isnan(got.entropy[1])
    assert got.top_indices[0, 0] == 9 and got.top_indices[1, 0] == 60
    assert torch.isfinite(got.logprob[2:]).all() and torch.isfinite(got.entropy[2:]).all()


def test_large_logits():
    """Differences are taken before exponentials: far logits lose nothing."""
    x, t = make(5, 2000, "f32", seed=1)
    for shift in (1000.0, -1000.0):
        got = engine.token_logprobs(x + shift, t, top=2)
        ref = reference(x + shift, t, 2)
        within(got.logprob, ref["logprob"], ref["rho"] + 8 * 2.0 ** -24 * 20, "logprob")
    check(x * 3e4, t, top=4, grads=False)
    check((x * 1e37).clamp(-3e38, 3e38), t, top=4, grads=False)


def test_targets():
    x, t = make(6, 90, "bf16")
    t[:] = torch.tensor([5, 90, -1, -100, 89, 2**40], device="cuda")
    got = engine.token_logprobs(x, t)
    assert torch.isnan(got.logprob).tolist() == [False, True, True, False, False, True] and got.logprob[3] == 0
    assert torch.isfinite(got.entropy).all()
    d = engine.token_logprobs_backward(x, t, got, torch.ones(6, device="cuda"))
    assert torch.isnan(d[1]).any() and torch.isfinite(d[[0, 3, 4]]).all() and (d[3] == 0).all()
    t[:] = torch.tensor([5, 7, 7, 89, 0, 7], device="cuda")
    check(x, t, top=3, ignore=7)


def test_shapes_and_strides():
    x, t = make(12, 501, "f16")
    want = engine.token_logprobs(x, t, top=3)
    shaped = engine.token_logprobs(x.view(3, 4, 501), t.view(3, 4), top=3)
    assert shaped.logprob.shape == (3, 4) and shaped.top_indices.shape == (3, 4, 3)
    assert torch.equal(shaped.logprob.view(-1), want.logprob)
    room = torch.full((12, 520), 99.0, device="cuda", dtype=x.dtype)
    room[:, 7:508] = x
    for view in (room[:, 7:508], x.t().contiguous().t(), x[:1].expand(12, -1)):
        check(view, t, top=3)
    empty = engine.token_logprobs(x[:0], t[:0], top=2)
    assert empty.logprob.shape == (0,) and empty.top_indices.shape == (0, 2)
    assert engine.token_logprobs_backward(x[:0], t[:0], empty).shape == (0, 501)
    assert torch.allclose(want.lse.double(), torch.logsumexp(x.double(), -1), atol=1e-5)


def test_gradients_against_differences():
    x, t = make(3, 60, "f32", seed=8)
    got = engine.token_logprobs(x, t, top=2)
    gen = torch.Generator(device="cuda").manual_seed(1)
    gl, ge, gt, step = (torch.randn(s, generator=gen, device="cuda").double() for s in ((3,), (3,), (3, 2), (3, 60)))

    def value(y):
        r = reference(y, t, 2)
        return float((r["logprob"] * gl).sum() + (r["entropy"] * ge).sum()
                     + (r["lp"].gather(-1, got.top_indices) * gt).sum())

    slope = (value(x.double() + 1e-6 * step) - value(x.double() - 1e-6 * step)) / 2e-6
    d = engine.token_logprobs_backward(x, t, got, gl.float(), ge.float(), gt.float())
    assert abs(float((d.double() * step).sum()) - slope) < 1e-4


@pytest.mark.parametrize("vocab", [999, 20011])
def test_far_rows(vocab):
    """Rows more than 2^31 elements apart."""
    far = 2**31 + 5
    store = torch.empty(far + vocab, dtype=torch.float16, device="cuda")
    x = store.as_strided((2, vocab), (far, 1))
    x.copy_(torch.randn(2, vocab, generator=torch.Generator(device="cuda").manual_seed(8), device="cuda"))
    t, g = torch.tensor([3, vocab - 1], device="cuda"), torch.ones(2, device="cuda")
    near = x.contiguous()
    a, b = engine.token_logprobs(x, t, top=5), engine.token_logprobs(near, t, top=5)
    # the two layouts start at other offsets from a vector's boundary, and sum in another order
    assert torch.equal(a.top_indices, b.top_indices) and torch.allclose(a.logprob, b.logprob, atol=1e-5)
    da = engine.token_logprobs_backward(x, t, a, g, g)
    db = engine.token_logprobs_backward(near, t, a, g, g)
    assert torch.equal(da, db)


def test_streams_and_graphs():
    x, t = make(50, 7001, "bf16")
    g = torch.ones(50, device="cuda")

    def step():
        r = engine.token_logprobs(x, t, top=4)
        return (*r, engine.token_logprobs_backward(x, t, r, g, g))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    x.copy_(x.flip(0))
    graph.replay()
    after = step()
    for a, b, c, d in zip(want, got, kept, after):
        assert torch.equal(a, b) and torch.equal(c, d)


def test_refusals():
    x, t = make(4, 30, "f32")
    for error, args, kw in (
            (TypeError, (x.double(), t), {}), (TypeError, (x.long(), t), {}), (ValueError, (x.cpu(), t), {}),
            (ValueError, (x, t.cpu()), {}), (ValueError, (x, t.int()), {}), (ValueError, (x, t[:3]), {}),
            (ValueError, (x[:, :0], t), {}), (ValueError, (x, t), dict(top=31)), (ValueError, (x, t), dict(top=-1)),
            (ValueError, (x.repeat(1, 9), t), dict(top=33)), (ValueError, (x[0, 0], t[0]), {})):
        with pytest.raises(error):
            engine.token_logprobs(*args, **kw)
    r = engine.token_logprobs(x, t, top=2)
    for bad in ((t.float()[:3],), (t.double(),), (None, x), (None, None, x), (t.float().cpu(),)):
        with pytest.raises(ValueError):
            engine.token_logprobs_backward(x, t, r, *bad)
    with pytest.raises(ValueError):
        engine.token_logprobs_backward(x[:3], t[:3], r)

"""fp64 attention under any visibility, with bounds on what the engine's roundings may change.

``u`` is half a step of the storage type.  Rounded values are the probabilities (to the type of V, on the tensor
cores), dS, the outputs and gradients themselves, and the output that enters delta; each is off by at most u times
its value.  A probability p = 2^(s - lse) also carries the error of its score, a sum of D products in fp32 (at most
D 2^-24 times the sum of their magnitudes, and as much for its part in the LSE), of the exponential and of the sum of
the row (a few steps of fp32 and n 2^-24 for n keys).  The tensor-core forward takes one exponential pair in eight
from a cubic with a relative error of 7.5e-5.  f16 probabilities below 2^-14 of the reference are subnormal: off by
2^-25.
"""

import math

import torch

DTYPES = {"f32": torch.float32, "f64": torch.float64, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def _fp32(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


class Attention:
    """q [B, Hq, T, D], k, v [B, Hkv, K, D / Dv] (storage type), seen [B, 1 or Hq, T, K] truth values."""

    def __init__(self, q, k, v, seen, scale=None, cubic=True):
        self.dtype = q.dtype
        self.group = q.shape[1] // k.shape[1]
        self.scale = 1 / math.sqrt(q.shape[3]) if scale is None else scale
        up = lambda x: x.double().repeat_interleave(self.group, 1)  # noqa: E731
        self.q, self.k, self.v = q.double(), up(k), up(v)
        none = ~seen.any(-1, keepdim=True)
        s = (self.q @ self.k.transpose(-1, -2)) * self.scale
        s = s.masked_fill(~seen, -math.inf)
        self.lse = torch.where(none[..., 0], -math.inf, torch.logsumexp(s, -1))
        self.p = torch.where(none, 0.0, torch.exp(s - torch.where(none, 0.0, self.lse[..., None])))
        self.out = self.p @ self.v
        half = self.dtype in (torch.float16, torch.bfloat16)
        self.u = half_step(self.dtype)
        e = _fp32(self.dtype)
        dim, keys = q.shape[3], k.shape[2]
        size = (self.q.abs() @ self.k.abs().transpose(-1, -2)).masked_fill(~seen, 0).amax(-1, keepdim=True)
        # relative error of a probability before it is rounded
        self.rho = e * (2 * dim * abs(self.scale) * size + 2 * size * abs(self.scale) + keys + 32)
        self.cubic = 7.5e-5 if half and cubic else 0.0
        self.round_p = self.u if half and cubic else 0.0  # the CUDA-core kernels keep P in fp32
        tiny = 2.0 ** -25 * keys * self.v.abs().amax() if self.dtype == torch.float16 else 0.0
        spread = self.p @ self.v.abs()
        self.out_bound = (self.rho + self.cubic + self.round_p + e * keys) * spread + self.u * self.out.abs() + tiny
        # the LSE in fp32: the sum's relative error, and a step of its own size
        self.lse_bound = (self.rho[..., 0] + self.cubic) + 4 * e * (1 + self.lse.abs().nan_to_num(posinf=0))

    def fold(self, x):
        b, h, n, d = x.shape
        return x.view(b, h // self.group, self.group, n, d).sum(2)

    def backward(self, g):
        g = g.double()
        u, e, p = self.u, _fp32(self.dtype), self.p
        half = self.dtype in (torch.float16, torch.bfloat16)
        dp = g @ self.v.transpose(-1, -2)
        delta = (g * self.out).sum(-1, keepdim=True)
        ds = p * (dp - delta) * self.scale
        # of dS: p's error, the output's rounding in delta, dots of fp32
        spread = g.abs() @ self.v.abs().transpose(-1, -2)
        rho = self.rho + self.cubic * 0 + 8 * e
        dim = g.shape[-1]
        delta_err = (g.abs() * (self.out_bound + u * self.out.abs())).sum(-1, keepdim=True)
        ds_err = rho * ds.abs() + p * abs(self.scale) * (delta_err + 2 * dim * e * (spread + (g * self.out).abs().sum(-1, keepdim=True)))
        ds_err = ds_err + (u if half else e) * (ds.abs() + ds_err)
        p_err = (rho + (u if half else e)) * p
        if self.dtype == torch.float16:
            ds_err, p_err = ds_err + 2.0 ** -25, p_err + 2.0 ** -25
        if half is False:
            n = max(p.shape[-1], p.shape[-2]) * self.group
            ds_err, p_err = ds_err + e * n * ds.abs(), p_err + e * n * p
        q, k = self.q, self.k
        dq, dk, dv = ds @ k, self.fold(ds.transpose(-1, -2) @ q), self.fold(p.transpose(-1, -2) @ g)
        tiny = 2.0 ** -25 if self.dtype == torch.float16 else 0.0
        bounds = (ds_err @ k.abs() + u * dq.abs() + tiny,
                  self.fold(ds_err.transpose(-1, -2) @ q.abs()) + u * dk.abs() + tiny,
                  self.fold(p_err.transpose(-1, -2) @ g.abs()) + u * dv.abs() + tiny)
        slack = 1 + 2.0 ** -6  # of the products of two errors
        return (dq, dk, dv), tuple(b * slack for b in bounds)

    def check(self, out, lse=None):
        within(out, self.out, self.out_bound, "out")
        if lse is not None:
            none = torch.isinf(self.lse)
            assert torch.equal(torch.isinf(lse), none), "LSE: rows that see nothing"
            within(lse.masked_fill(none, 0), self.lse.masked_fill(none, 0), self.lse_bound.masked_fill(none, 0), "lse")


def within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    err = (got.double() - want).abs()
    over = err - bound
    worst = int(over.argmax())
    assert float(over.max()) <= 0, (
        f"{what}: off by {float(err.view(-1)[worst]):.3e}, allowed {float(bound.expand_as(err).reshape(-1)[worst]):.3e}, "
        f"value {float(want.reshape(-1)[worst]):.3e}; {int((over > 0).sum())} of {err.numel()}")


def window_seen(rows, tokens, keys, window, sinks, offset=0, lens=None, device="cuda"):
    """[B, 1, T, K]: what queries see under a window (0: none); with ``lens`` the queries end row b's keys."""
    key = torch.arange(keys, device=device)
    if lens is None:
        at = (offset + torch.arange(tokens, device=device)).expand(rows, tokens)
        seen = torch.ones(rows, 1, keys, dtype=torch.bool, device=device)
    else:
        lens = lens.long().clamp(0, keys)
        at = lens[:, None] - tokens + torch.arange(tokens, device=device)
        seen = (key < lens[:, None])[:, None]
    dist = at[:, :, None] - key
    seen = seen & (dist >= 0)
    if window:
        seen = seen & ((dist < window) | (key < sinks))
    return seen[:, None]


def tree_seen(parents, lens, keys, window=0, sinks=0):
    """[B, 1, T, K] of drafted trees, node by node from the definition (parents: list of lists; lens: list)."""
    rows, nodes = len(parents), len(parents[0])
    seen = torch.zeros(rows, nodes, keys, dtype=torch.bool)
    for b in range(rows):
        base = min(lens[b], keys) - nodes
        for i in range(nodes):
            path, j = [], i
            while True:
                path.append(j)
                up = parents[b][j]
                if base + j < 0 or not (up == -1 or 0 <= up < j):
                    path = None
                    break
                if up == -1:
                    break
                j = up
            if path is None:
                continue
            at = base + len(path) - 1
            for key in range(max(base, 0)):
                seen[b, i, key] = not window or at - key < window or key < sinks
            for d, j in enumerate(path):  # d steps above node i
                seen[b, i, base + j] = not window or d < window or at - d < sinks
    return seen[:, None]

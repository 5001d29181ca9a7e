"""The gated delta rule and causal attention from their definitions, in 64 bits, and
inputs for their tests."""
from __future__ import annotations

import math

import torch

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def delta_ref(q, k, v, g, beta, scale=None, init=None, cu=None):
    """(o, final states) token by token, in 64 bits; differentiable.  cu: a list of row
    numbers of a packed batch; rows of no sequence are zero."""
    q, k, v, g, beta = (t.double() for t in (q, k, v, g, beta))
    B, H, N, Dv = v.shape
    Dk = k.shape[-1]
    q, k = (t.repeat_interleave(H // t.shape[1], 1) for t in (q, k))
    scale = Dk ** -0.5 if scale is None else scale
    seqs = [(b, 0, N) for b in range(B)] if cu is None else [(0, a, b) for a, b in zip(cu[:-1], cu[1:])]
    rows = [[v.new_zeros(H, Dv)] * N for _ in range(B)]
    finals = []
    for s, (b, first, end) in enumerate(seqs):
        S = v.new_zeros(H, Dk, Dv) if init is None else init[s].double()
        for t in range(first, end):
            S = g[b, :, t].exp()[:, None, None] * S
            kt = k[b, :, t, :, None]
            u = beta[b, :, t, None] * (v[b, :, t] - (kt * S).sum(1))
            S = S + kt * u[:, None, :]
            rows[b][t] = scale * (q[b, :, t, :, None] * S).sum(1)
        finals.append(S)
    o = torch.stack([torch.stack(r, 1) if N else v.new_zeros(H, 0, Dv) for r in rows]) if B else v.new_zeros(v.shape)
    return o, torch.stack(finals) if finals else v.new_zeros(0, H, Dk, Dv)


def attention_ref(q, k, v, scale=None, cu=None):
    """Causal attention row block by row block, in 64 bits; differentiable."""
    q, k, v = (t.double() for t in (q, k, v))
    B, H, N, Dk = q.shape
    k, v = (t.repeat_interleave(H // t.shape[1], 1) for t in (k, v))
    scale = Dk ** -0.5 if scale is None else scale
    seqs = [(b, 0, N) for b in range(B)] if cu is None else [(0, a, b) for a, b in zip(cu[:-1], cu[1:])]
    parts = [[] for _ in range(B)]
    for b in range(B):
        at = 0
        for bb, first, end in seqs:
            if bb != b or end <= first:
                continue
            parts[b].append(v.new_zeros(H, first - at, v.shape[-1]))
            x = scale * (q[b, :, first:end, None, :] * k[b, :, None, first:end, :]).sum(-1)
            x = x.masked_fill(torch.ones(end - first, end - first, dtype=torch.bool, device=q.device).triu(1), -math.inf)
            parts[b].append(torch.softmax(x, -1) @ v[b, :, first:end])
            at = end
        parts[b].append(v.new_zeros(H, N - at, v.shape[-1]))
    return torch.stack([torch.cat(p, 1) for p in parts]) if B else q.new_zeros(*q.shape[:3], v.shape[-1])


def unit(x):
    return x / x.square().sum(-1, keepdim=True).add(1e-6).sqrt()


def delta_inputs(B, Hk, H, N, Dk, Dv, dtype, seed=0, layout="heads", device="cpu"):
    """q, k of unit length, normal v, log decays of a memory of 2 to 200 tokens, beta in (0, 1)."""
    gen = torch.Generator().manual_seed(seed)

    def rows(heads, width, f=lambda x: x):
        if layout == "tokens":
            return f(torch.randn(B, N, heads, width, generator=gen)).to(dtype).to(device).transpose(1, 2)
        return f(torch.randn(B, heads, N, width, generator=gen)).to(dtype).to(device)

    q, k, v = rows(Hk, Dk, unit), rows(Hk, Dk, unit), rows(H, Dv)
    g = -torch.exp(-0.7 - 4.5 * torch.rand(B, N, H, generator=gen)).to(device).transpose(1, 2)
    beta = torch.sigmoid(torch.randn(B, N, H, generator=gen)).to(device).transpose(1, 2)
    return q, k, v, g, beta


def assert_near(x, ref, what, slack=1.0, terms=0.0):
    """x against the 64-bit ref.  x was rounded once to its type: half a step of the value.
    16-bit types' outputs come from products kept to 2^-16 of their terms; over up to
    64 + 128 terms of either sign that is within 2^-16 sqrt(192), 2^-12, of the largest
    value.  32-bit results add rounding errors of 2^-24 over the same sums and up to
    300 tokens: 2^-24 sqrt(192 * 300) = 1.4e-5.  In the 2-norm a quarter of either.  terms: the size of what a result is the
    difference of, where that is more than the result itself."""
    dtype = x.dtype
    half = torch.finfo(dtype).eps / 2
    x, ref = x.detach().double().cpu(), ref.detach().double().cpu()
    assert x.shape == ref.shape, (what, tuple(x.shape), tuple(ref.shape))
    if not ref.numel():
        return
    assert torch.isfinite(x).all(), f"{what}: not finite"
    top, norm = max(float(ref.abs().max()), terms), float(ref.norm())
    most = (1.4e-5 if dtype == torch.float32 else 2.0 ** -12) * slack
    off = ((x - ref).abs() - half * ref.abs()).max()
    assert float(off) <= most * top, f"{what}: {float(off):.3e} beyond half a step, largest value {top:.3e}"
    rel = float((x - ref).norm()) / max(norm, terms) if max(norm, terms) else float(x.norm())
    assert rel <= half + most / 4, f"{what}: relative error {rel:.3e}"

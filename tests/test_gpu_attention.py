"""Causal attention's kernel against its definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

import kilat_amd
from tests.mixer_cases import DTYPES, assert_near, attention_ref

pytestmark = pytest.mark.gpu

# (B, Hk, H, N, Dk, Dv, layout)
SHAPES = [
    (1, 1, 1, 1, 64, 64, "heads"),
    (2, 3, 3, 2, 32, 16, "tokens"),
    (2, 2, 2, 63, 64, 64, "heads"),
    (1, 2, 4, 64, 64, 64, "tokens"),
    (3, 1, 2, 65, 16, 48, "tokens"),
    (1, 2, 2, 127, 128, 128, "heads"),
    (1, 2, 8, 128, 64, 128, "heads"),
    (2, 1, 3, 300, 96, 80, "tokens"),
    (1, 1, 1, 200, 1, 1, "heads"),
    (1, 2, 2, 129, 7, 20, "tokens"),
    (1, 1, 2, 257, 100, 33, "tokens"),
]


def inputs(shape, dname, dev, seed=0, sharp=1.0):
    B, Hk, H, N, Dk, Dv, layout = shape
    gen = torch.Generator().manual_seed(seed)

    def rows(heads, width, f=1.0):
        if layout == "tokens":
            return (f * torch.randn(B, N, heads, width, generator=gen)).to(DTYPES[dname]).to(dev).transpose(1, 2)
        return (f * torch.randn(B, heads, N, width, generator=gen)).to(DTYPES[dname]).to(dev)

    print("  ", shape, dname, flush=True)
    return rows(H, Dk, sharp), rows(Hk, Dk), rows(Hk, Dv)


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(hip_device, kdecay_lib, shape, dname):
    for sharp, scale in ((1.0, None), (6.0, 0.5)):
        x = inputs(shape, dname, hip_device, sharp=sharp)
        o = kilat_amd.causal_attention(*x, scale=scale)
        assert o.dtype == x[0].dtype
        # Probabilities are operands of the second product: rounded to the type once more, half
        # a step of each term (fp32: three terms, none).  The row's terms, of either sign,
        # add to at most its values' size.
        ref = attention_ref(*(t.cpu() for t in x), scale=scale)
        size = attention_ref(x[0].cpu(), x[1].cpu(), x[2].cpu().abs(), scale=scale)
        half = torch.finfo(o.dtype).eps / 2
        # fp32 scores of size |x| are off by 2^-24 |x| sqrt(Dk) each, the probabilities by as much
        # relative: 2^-24 * 100 * 12 covers scores up to 100.
        most = half * ref.abs() + (0 if o.dtype == torch.float32 else half) * size + 2.0 ** -24 * 1200 * size
        off = (o.cpu().double() - ref).abs()
        assert bool((off <= most).all()), float((off - most).max())
        assert torch.equal(kilat_amd.causal_attention(*x, scale=scale), o)


@pytest.mark.parametrize("dname", ["bf16", "f32"])
@pytest.mark.parametrize("cu,N", [([0, 1, 65, 65, 200, 264, 300], 300), ([5, 5, 70, 133], 150), ([7, 7, 7], 20),
                                  ([0, 128, 256, 257], 400)], ids=str)
def test_packed(hip_device, kdecay_lib, cu, N, dname):
    """Rows of no sequence are zero; rows of one sequence alone change its rows alone."""
    x = inputs((1, 2, 4, N, 64, 48, "tokens"), dname, hip_device, seed=1)
    for cut in (torch.tensor(cu, dtype=torch.int32, device=hip_device), torch.tensor(cu, device=hip_device)):
        o = kilat_amd.causal_attention(*x, cu_seqlens=cut)
        ref = attention_ref(*(t.cpu() for t in x), cu=cu)
        size = attention_ref(x[0].cpu(), x[1].cpu(), x[2].cpu().abs(), cu=cu)
        half = torch.finfo(o.dtype).eps / 2
        most = half * ref.abs() + (0 if dname == "f32" else half) * size + 2.0 ** -24 * 1200 * size
        assert bool(((o.cpu().double() - ref).abs() <= most).all())
        assert not o[:, :, : cu[0]].any() and not o[:, :, cu[-1]:].any()
    y = [t.clone() for t in x]
    for t in y:
        t[:, :, cu[-2]:] = float("nan")
    p = kilat_amd.causal_attention(*y, cu_seqlens=cut)
    assert torch.equal(p[:, :, : cu[-2]], o[:, :, : cu[-2]]) and not p[:, :, cu[-1]:].any()


@pytest.mark.parametrize("cu", [[-5, 40, 900], [60, 20, 80], [0, 2**31 - 1], [-(2**31), -7]], ids=str)
def test_row_numbers_out_of_range_stay_in_bounds(hip_device, kdecay_lib, cu):
    x = inputs((1, 1, 2, 100, 32, 32, "heads"), "bf16", hip_device)
    ref = kilat_amd.causal_attention(*x)
    kilat_amd.causal_attention(*x, cu_seqlens=torch.tensor(cu, dtype=torch.int32, device=hip_device))
    torch.cuda.synchronize()
    assert torch.equal(kilat_amd.causal_attention(*x), ref)


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("which", ["v nan", "v inf", "k nan", "k inf", "q nan"])
@pytest.mark.parametrize("at", [0, 63, 100, 190])
def test_values_that_are_not_finite_reach_no_earlier_row(hip_device, kdecay_lib, which, at, dname):
    x = inputs((1, 2, 2, 230, 64, 64, "tokens"), dname, hip_device, seed=2)
    o = kilat_amd.causal_attention(*x)
    y = [t.clone() for t in x]
    y["qkv".index(which[0])][:, 0, at, 17] = float("inf") if "inf" in which else float("nan")
    p = kilat_amd.causal_attention(*y)
    assert torch.equal(p[:, 1], o[:, 1]) and torch.equal(p[:, 0, :at], o[:, 0, :at])
    if which[0] == "q":
        assert p[:, 0, at].isnan().all() and torch.equal(p[:, 0, at + 1:], o[:, 0, at + 1:])
    elif which[0] == "v":
        assert not p[:, 0, at:, 17].isfinite().any()
        keep = [c for c in range(64) if c != 17]
        assert torch.equal(p[:, 0][..., keep], o[:, 0][..., keep])
    elif "nan" in which:
        assert p[:, 0, at:].isnan().all()


def test_scores_far_apart(hip_device, kdecay_lib):
    """Scores of thousands, of the lowest value and equal ones: the maximum is always subtracted."""
    q, k, v = inputs((1, 1, 1, 200, 64, 64, "heads"), "f32", hip_device, seed=3)
    big = torch.linspace(-3000, 3000, 200, device=hip_device)
    k = torch.zeros_like(k)
    k[0, 0, :, 0] = big
    q = torch.zeros_like(q)
    q[..., 0] = 8.0  # scores are k's first channel: each row's own key is the highest by 30
    assert_near(kilat_amd.causal_attention(q, k, v), v.cpu().double(), "own value")
    k.zero_()
    mean = v.cpu().double().cumsum(2) / torch.arange(1, 201).view(1, 1, -1, 1)
    assert_near(kilat_amd.causal_attention(q, k, v), mean, "mean")
    k.fill_(torch.finfo(torch.float32).min / 1e3)  # scores of -3e36 throughout
    assert_near(kilat_amd.causal_attention(q / 8, k, v), mean, "mean of lowest")


def test_layouts(hip_device, kdecay_lib):
    q, k, v = inputs((2, 2, 4, 150, 40, 24, "heads"), "bf16", hip_device, seed=4)
    plain = kilat_amd.causal_attention(q, k, v)

    def off(t, by):
        buf = torch.zeros(t.numel() + by, dtype=t.dtype, device=t.device)
        return buf[by:].view(t.shape).copy_(t)

    for by in (1, 2, 4):
        assert torch.equal(kilat_amd.causal_attention(off(q, by), off(k, by), off(v, by)), plain)
    turned = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    assert torch.equal(kilat_amd.causal_attention(*turned), plain)
    neg = torch._neg_view(-v)
    assert torch.equal(kilat_amd.causal_attention(q, k, neg), plain)
    o = kilat_amd.causal_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k, v)
    assert o.stride(1) < o.stride(2) and torch.equal(o, plain)  # laid out like q
    e = kilat_amd.causal_attention(q, k[:, :1].expand(-1, 4, -1, -1), v[:, :1].expand(-1, 4, -1, -1))
    assert torch.equal(e, kilat_amd.causal_attention(q, k[:, :1], v[:, :1]))


@pytest.mark.parametrize("B,N", [(0, 5), (2, 0), (0, 0)])
def test_empty(hip_device, kdecay_lib, B, N):
    q, k, v = inputs((B, 1, 2, N, 32, 16, "heads"), "bf16", hip_device)
    assert kilat_amd.causal_attention(q, k, v).shape == (B, 2, N, 16)


def test_rows_past_32_bit_offsets(hip_device, kdecay_lib):
    far = 2**31 + 64
    buf = torch.zeros(far + 66 * 64, dtype=torch.bfloat16, device=hip_device)
    q, k, v = inputs((1, 2, 2, 66, 64, 64, "heads"), "bf16", hip_device, seed=5)
    w = buf.as_strided((1, 2, 66, 64), (far + 66 * 64, far, 64, 1))
    for i in range(3):
        x = [q, k, v]
        w.copy_(x[i])
        x[i] = w
        assert torch.equal(kilat_amd.causal_attention(*x), kilat_amd.causal_attention(q, k, v))


def test_streams_and_graphs(hip_device, kdecay_lib):
    x = inputs((2, 2, 4, 300, 64, 64, "tokens"), "bf16", hip_device, seed=6)
    cu = torch.tensor([0, 100, 290], dtype=torch.int32, device=hip_device)
    pk = [t[:1].clone() for t in x]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kilat_amd.causal_attention(*x)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = kilat_amd.causal_attention(*x), kilat_amd.causal_attention(*pk, cu_seqlens=cu)
    for seed in range(3):
        y = inputs((2, 2, 4, 300, 64, 64, "tokens"), "bf16", hip_device, seed=7 + seed)
        cu.copy_(torch.tensor([0, 50 + seed, 200 + seed]))
        for a, b in zip(x, y):
            a.copy_(b)
        ref = kilat_amd.causal_attention(*y), kilat_amd.causal_attention(*pk, cu_seqlens=cu)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref)), seed


def test_gradients_are_refused(hip_device, kdecay_lib):
    q, k, v = inputs((1, 1, 1, 10, 32, 32, "heads"), "bf16", hip_device)
    with pytest.raises(RuntimeError, match="no backward"):
        kilat_amd.causal_attention(q, k.requires_grad_(), v)
    with torch.no_grad():
        kilat_amd.causal_attention(q, k, v)

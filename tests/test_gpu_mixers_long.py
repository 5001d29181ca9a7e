"""The mixers where their work is divided otherwise than in a small call: long sequences of
few heads in pieces, keys in two parts, many workgroups, many sequences; and a hybrid
layer's mixers together."""
from __future__ import annotations

import ctypes

import pytest
import torch

import kilat_amd
from kilat_amd import _lib
from tests.mixer_cases import DTYPES, assert_near, attention_ref, delta_ref
from tests.test_gpu_attention import inputs
from tests.test_gpu_delta import case, check_grads, grads_of, kernel
from tests.test_mixers import problem

pytestmark = pytest.mark.gpu


def attention_near(x, cu=None, **kw):
    """The bounds of test_gpu_attention."""
    o = kilat_amd.causal_attention(*x, cu_seqlens=None if cu is None else torch.tensor(cu, device=x[0].device), **kw)
    ref = attention_ref(*(t.cpu() for t in x), cu=cu, **kw)
    size = attention_ref(x[0].cpu(), x[1].cpu(), x[2].cpu().abs(), cu=cu, **kw)
    half = torch.finfo(o.dtype).eps / 2
    most = half * ref.abs() + (0 if o.dtype == torch.float32 else half) * size + 2.0 ** -24 * 1200 * size
    assert bool(((o.cpu().double() - ref).abs() <= most).all())
    return o


# ---------------------------------------------------------------------------
# The gated delta scan in pieces
# ---------------------------------------------------------------------------
PIECES = [
    (1, 1, 1, 512, 64, 64, "heads"),
    (1, 1, 2, 1100, 64, 48, "tokens"),
    (1, 2, 2, 1025, 128, 96, "heads"),
    (2, 1, 3, 900, 80, 40, "tokens"),
    (1, 1, 1, 1537, 24, 16, "tokens"),
]


def test_these_are_in_pieces(kdecay_lib):
    """By the workspace: a stream of a short grid needs more of it than one of many."""
    kdecay_lib.kdelta_scan_workspace_bytes.restype = ctypes.c_size_t
    for B, Hk, H, N, Dk, Dv, _ in PIECES:
        for dtype in (_lib.KDECAY_BF16, _lib.KDECAY_F16, _lib.KDECAY_F32):
            need = [kdecay_lib.kdelta_scan_workspace_bytes(ctypes.byref(
                problem(B=b, sequences=b, Hk=Hk, H=H, N=N, Dk=Dk, Dv=Dv, dtype=dtype))) / b for b in (B, 4096)]
            assert need[0] > 1.01 * need[1], (B, H, N, Dk, Dv, dtype)


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", PIECES, ids=str)
def test_scan_in_pieces(hip_device, kdecay_lib, shape, dname):
    B, Hk, H, N, Dk, Dv, _ = shape
    x = case(hip_device, shape, dname, seed=1)
    init = torch.randn(B, H, Dk, Dv, generator=torch.Generator().manual_seed(2)).to(hip_device)
    for S0 in (None, init):
        o, S = kilat_amd.gated_delta_scan(*x, initial_state=S0, return_final_state=True)
        ro, rS = delta_ref(*(t.cpu() for t in x), init=None if S0 is None else S0.cpu())
        assert_near(o, ro, "o")
        assert_near(S, rS, "final state")
    again = kilat_amd.gated_delta_scan(*x, initial_state=init, return_final_state=True)
    assert torch.equal(again[0], o) and torch.equal(again[1], S)


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", PIECES[1:4], ids=str)
def test_backward_of_pieces(hip_device, kdecay_lib, shape, dname):
    B, Hk, H, N, Dk, Dv, _ = shape
    x = case(hip_device, shape, dname, seed=3)
    gen = torch.Generator().manual_seed(4)
    do = torch.randn(B, H, N, Dv, generator=gen).to(DTYPES[dname]).to(hip_device)
    init, dS = (torch.randn(B, H, Dk, Dv, generator=gen).to(hip_device) for _ in range(2))
    a = check_grads(hip_device, x, init, do, dS)
    assert all(torch.equal(s, t) for s, t in zip(a, grads_of(x, init, do, dS, kernel())))


@pytest.mark.parametrize("dname", ["bf16", "f32"])
def test_packed_pieces(hip_device, kdecay_lib, dname):
    """Sequences of no, one and many pieces in one batch."""
    cu, N = [3, 3, 4, 70, 1100, 1100, 2000], 2040
    x = case(hip_device, (1, 1, 2, N, 64, 32, "tokens"), dname, seed=5)
    gen = torch.Generator().manual_seed(6)
    init, dS = (torch.randn(len(cu) - 1, 2, 64, 32, generator=gen).to(hip_device) for _ in range(2))
    do = torch.randn(1, 2, N, 32, generator=gen).to(DTYPES[dname]).to(hip_device)
    cut = torch.tensor(cu, dtype=torch.int32, device=hip_device)
    o, S = kilat_amd.gated_delta_scan(*x, initial_state=init, cu_seqlens=cut, return_final_state=True)
    ro, rS = delta_ref(*(t.cpu() for t in x), init=init.cpu(), cu=cu)
    assert_near(o, ro, "o")
    assert_near(S, rS, "final state")
    assert not o[:, :, :3].any() and not o[:, :, 2000:].any()
    check_grads(hip_device, x, init, do, dS, cu=cu)


@pytest.mark.parametrize("which", ["v", "k", "q", "g", "state"])
def test_values_that_are_not_finite_in_pieces(hip_device, kdecay_lib, which):
    x = [t.clone() for t in case(hip_device, (1, 2, 2, 1000, 64, 64, "tokens"), "bf16", seed=7)]
    init = torch.randn(1, 2, 64, 64, device=hip_device)
    o = kilat_amd.gated_delta_scan(*x, initial_state=init)
    if which == "state":
        init[:, 0, 3, 17] = float("nan")
    elif which == "g":
        x[3][:, 0, 600] = float("nan")
    else:
        x["qkv".index(which)][:, 0, 600, 17] = float("nan")
    p = kilat_amd.gated_delta_scan(*x, initial_state=init)
    ref = delta_ref(*(t.cpu() for t in x), init=init.cpu())[0]
    assert torch.equal(p.cpu().isfinite(), ref.isfinite()) and torch.equal(p[:, 1], o[:, 1])
    assert_near(torch.where(ref.isfinite(), p.cpu(), 0.0), torch.where(ref.isfinite(), ref, 0.0), "o")


def test_two_captured_graphs_in_pieces(hip_device, kdecay_lib):
    """Two graphs of one pool, replayed in turn and on two streams at once."""
    xs = [case(hip_device, (1, 1, 2, 1100, 64, 64, "heads"), "bf16", seed=s) for s in (8, 9)]
    run = lambda x: kilat_amd.gated_delta_scan(*x, return_final_state=True)  # noqa: E731
    for x in xs:
        run(x)
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(run(x))
        graphs.append(g)
    for seed in range(3):
        refs = []
        for i, x in enumerate(xs):
            z = case(hip_device, (1, 1, 2, 1100, 64, 64, "heads"), "bf16", seed=20 + 2 * seed + i)
            for a, b in zip(x, z):
                a.copy_(b)
            refs.append(run(x))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for out, ref in zip(outs, refs):
            assert all(torch.equal(a, b) for a, b in zip(out, ref)), seed


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dname", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [(9, 4, 8, 1000, 64, 64, "tokens"), (33, 2, 16, 130, 64, 128, "heads"),
                                   (26, 1, 4, 641, 128, 40, "heads"), (17, 2, 8, 500, 120, 128, "tokens")], ids=str)
def test_attention_of_many_workgroups(hip_device, kdecay_lib, shape, dname):
    x = inputs(shape, dname, hip_device, seed=3)
    o = attention_near(x)
    assert torch.equal(kilat_amd.causal_attention(*x), o)


@pytest.mark.parametrize("dname", ["bf16", "f16"])
@pytest.mark.parametrize("which", ["v nan", "v inf", "k nan"])
@pytest.mark.parametrize("at", [0, 63, 100, 190])
def test_values_that_are_not_finite_in_many_workgroups(hip_device, kdecay_lib, which, at, dname):
    x = inputs((40, 8, 8, 230, 64, 64, "tokens"), dname, hip_device, seed=4)
    o = kilat_amd.causal_attention(*x)
    y = [t.clone() for t in x]
    y["qkv".index(which[0])][3, 2, at, 17] = float("inf") if "inf" in which else float("nan")
    p = kilat_amd.causal_attention(*y)
    assert torch.equal(p[3, 2, :at], o[3, 2, :at])
    if which[0] == "v":
        assert not p[3, 2, at:, 17].isfinite().any()
        p[3, 2, at:, 17] = o[3, 2, at:, 17]
        assert torch.equal(p, o)
    else:
        assert not p[3, 2, at:].isfinite().any()
        p[3, 2] = o[3, 2]
        assert torch.equal(p, o)


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.3])
def test_scales(hip_device, kdecay_lib, scale, dname):
    attention_near(inputs((2, 2, 2, 200, 64, 64, "tokens"), dname, hip_device, seed=5), scale=scale)


# cu_seqlens: more sequences than a wavefront has lanes; more than 64 times as many; rows before the first.
MANY = {
    "100": [0] + [13 * i + (i % 7) for i in range(1, 101)],
    "64": [2] + [30 * i for i in range(1, 65)],
    "65": [2] + [30 * i for i in range(1, 66)],
    "5000": [0] + [i // 3 for i in range(1, 5001)],
    "behind": [700, 700, 900],
}


@pytest.mark.parametrize("name", list(MANY))
def test_many_sequences(hip_device, kdecay_lib, name):
    cu = MANY[name]
    N = cu[-1] + 11
    x = inputs((1, 1, 2, N, 64, 32, "tokens"), "bf16", hip_device, seed=6)
    junk = [torch.full((1 << 20,), float("nan"), device=hip_device) for _ in range(4)]
    del junk  # what the allocator gives next
    o = attention_near(x, cu=cu)
    assert not o[:, :, : cu[0]].any() and not o[:, :, cu[-1]:].any()
    y = case(hip_device, (1, 1, 2, N, 32, 32, "tokens"), "bf16", seed=7)
    cut = torch.tensor(cu, dtype=torch.int32, device=hip_device)
    p, S = kilat_amd.gated_delta_scan(*y, cu_seqlens=cut, return_final_state=True)
    rp, rS = delta_ref(*(t.cpu() for t in y), cu=cu)
    assert_near(p, rp, "o")
    assert_near(S, rS, "final state")


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dname", ["bf16", "f16"])
def test_a_hybrid_layer(hip_device, kdecay_lib, dname):
    """One packed batch of prompts through all three mixers as views of one projection, then tokens
    one at a time through the delta rule's state; captured, and replayed on other rows."""
    cu, N, H, D = [0, 5, 140, 141, 400], 410, 4, 64
    dtype, gen = DTYPES[dname], torch.Generator().manual_seed(8)
    cut = torch.tensor(cu, dtype=torch.int32, device=hip_device)
    fused = torch.empty(1, N, 3 * H, D, dtype=dtype, device=hip_device)
    gates = torch.empty(1, N, 2, H, device=hip_device)
    one = torch.empty(3, len(cu) - 1, H, D, dtype=dtype, device=hip_device)
    lam = torch.full((H,), 0.9, device=hip_device)

    def fill():
        x = torch.randn(1, N, 3 * H, D, generator=gen)
        x[:, :, : 2 * H] /= x[:, :, : 2 * H].norm(dim=-1, keepdim=True)
        fused.copy_(x)
        gates[:, :, 0] = -torch.rand(1, N, H, generator=gen).to(hip_device)
        gates[:, :, 1] = torch.rand(1, N, H, generator=gen).to(hip_device)
        one.copy_(torch.randn(3, len(cu) - 1, H, D, generator=gen) / 8)

    def layer():
        q, k, v = (fused[:, :, i * H:(i + 1) * H].transpose(1, 2) for i in range(3))
        g, beta = (gates[:, :, i].transpose(1, 2) for i in range(2))
        a = kilat_amd.causal_attention(q, k, v, cu_seqlens=cut)
        d, S = kilat_amd.gated_delta_scan(q, k, v, g, beta, cu_seqlens=cut, return_final_state=True)
        y = kilat_amd.triton_global_decay(lam, v)
        b = gates[0, : len(cu) - 1]
        s, S2 = kilat_amd.gated_delta_step(*one, b[:, 0], b[:, 1], S)
        return a, d, S, y, s, S2

    fill()
    torch.cuda.synchronize()
    s, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        layer()  # (the decay scan's workspace belongs to the stream)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=s):
        out = layer()
    for _ in range(3):
        fill()
        eager = layer()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))
        q, k, v = (fused[:, :, i * H:(i + 1) * H].transpose(1, 2).cpu() for i in range(3))
        g, beta = (gates[:, :, i].transpose(1, 2).cpu() for i in range(2))
        rd, rS = delta_ref(q, k, v, g, beta, cu=cu)
        assert_near(out[1], rd, "o")
        assert_near(out[2], rS, "states")
        b = gates[0, : len(cu) - 1].cpu()
        rs, rS2 = delta_ref(*(t.cpu()[:, :, None] for t in one), b[:, 0, :, None], b[:, 1, :, None], init=out[2].cpu())
        assert_near(out[4], rs[:, :, 0], "step")
        assert_near(out[5], rS2, "states after the step")
        attention_near((fused[:, :, :H].transpose(1, 2), fused[:, :, H:2 * H].transpose(1, 2),
                        fused[:, :, 2 * H:].transpose(1, 2)), cu=cu)

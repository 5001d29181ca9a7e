"""The gated delta rule's kernels against its definition in 64 bits."""
from __future__ import annotations

import pytest
import torch

import kilat_amd
from tests.mixer_cases import DTYPES, assert_near, delta_inputs, delta_ref, unit

pytestmark = pytest.mark.gpu

# (B, Hk, H, N, Dk, Dv, layout): one token to a few chunks of 64, head dims on and off
# the tiles of 16 and 32, shared key heads, views of projections.
SHAPES = [
    (1, 1, 1, 1, 64, 64, "heads"),
    (2, 3, 3, 2, 32, 16, "tokens"),
    (2, 2, 2, 63, 64, 64, "heads"),
    (1, 2, 4, 64, 64, 64, "tokens"),
    (3, 1, 2, 65, 16, 48, "tokens"),
    (1, 2, 2, 130, 128, 128, "heads"),
    (2, 1, 3, 257, 96, 80, "tokens"),
    (1, 1, 1, 100, 1, 1, "heads"),
    (1, 2, 2, 70, 7, 20, "tokens"),
    (1, 1, 2, 129, 100, 256, "tokens"),
    (1, 1, 1, 192, 80, 200, "heads"),
]


def on(dev, *ts):
    return [t.to(dev) for t in ts]


def case(dev, shape, dname, seed=0):
    *sizes, layout = shape
    print("  ", shape, dname, flush=True)
    return delta_inputs(*sizes, DTYPES[dname], seed=seed, layout=layout, device=dev)


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_scan(hip_device, kdecay_lib, shape, dname):
    x = case(hip_device, shape, dname)
    B, Hk, H, N, Dk, Dv, _ = shape
    init = torch.randn(B, H, Dk, Dv, generator=torch.Generator().manual_seed(1)).to(hip_device)
    for S0, scale in ((None, None), (init, 0.7)):
        o, S = kilat_amd.gated_delta_scan(*x, initial_state=S0, scale=scale, return_final_state=True)
        ro, rS = delta_ref(*(t.cpu() for t in x), scale=scale, init=None if S0 is None else S0.cpu())
        assert o.dtype == x[2].dtype and o.shape == x[2].shape and S.dtype == torch.float32
        assert_near(o, ro, "o")
        assert_near(S, rS, "final state")
    assert torch.equal(kilat_amd.gated_delta_scan(*x, initial_state=init, scale=0.7), o)  # the same bits again


def grads_of(x, init, do, dS, f):
    leaves = [t.detach().clone().requires_grad_() for t in (*x, *(() if init is None else (init,)))]
    o, S = f(*leaves[:5], None if init is None else leaves[5])
    loss = [o], [do]
    if dS is not None:
        loss[0].append(S), loss[1].append(dS)
    return torch.autograd.grad(loss[0], leaves, loss[1])


def kernel(cu=None, scale=None):
    def f(q, k, v, g, beta, init):
        return kilat_amd.gated_delta_scan(q, k, v, g, beta, initial_state=init, scale=scale, return_final_state=True,
                                          cu_seqlens=cu)
    return f


def oracle(cu=None, scale=None):
    return lambda q, k, v, g, beta, init: delta_ref(q, k, v, g, beta, scale, init, cu)


NAMES = ("dq", "dk", "dv", "dg", "dbeta", "dinit")


def check_grads(dev, x, init, do, dS, cu=None, scale=None, slack=4.0):
    """Gradients' sums have three times the scan's terms, of both signs: slack."""
    cud = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=dev)
    got = grads_of(x, init, do, dS, kernel(cud, scale))
    host = [None if t is None else t.cpu().double() for t in (init, do, dS)]
    ref = grads_of([t.cpu().double() for t in x], *host, oracle(cu, scale))
    # dg_t is the sum, over the tokens from t to its chunk's end, of q.dq + k.(the reading part of
    # dk) - k.(the writing part): the first token's is exactly 0 where there is no state
    # before it, a difference of terms as large as |q.dq|, each rounded at 2^-24.
    terms = float((ref[0] * x[0].cpu().double()).sum(-1).abs().max())
    for name, a, b, src in zip(NAMES, got, ref, (*x, init)):
        assert a.dtype == src.dtype
        assert_near(a, b, name, slack, terms if name == "dg" else 0.0)
    return got


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(hip_device, kdecay_lib, shape, dname):
    x = case(hip_device, shape, dname, seed=2)
    B, Hk, H, N, Dk, Dv, _ = shape
    gen = torch.Generator().manual_seed(3)
    do = torch.randn(B, H, N, Dv, generator=gen).to(DTYPES[dname]).to(hip_device)
    init, dS = (torch.randn(B, H, Dk, Dv, generator=gen).to(hip_device) for _ in range(2))
    check_grads(hip_device, x, None, do, None)
    a = check_grads(hip_device, x, init, do, dS, scale=0.7)
    b = grads_of(x, init, do, dS, kernel(scale=0.7))
    assert all(torch.equal(s, t) for s, t in zip(a, b))  # no order of arrival in any sum


# ---------------------------------------------------------------------------
# Packed batches
# ---------------------------------------------------------------------------
PACKED = {
    "uneven": ([0, 1, 65, 65, 200, 264, 300], 300),
    "spare rows": ([5, 5, 70, 133], 150),
    "one": ([0, 90], 90),
    "empty": ([7, 7, 7], 20),
    "chunks": ([0, 64, 128, 129], 256),
}


@pytest.mark.parametrize("dname", ["bf16", "f32"])
@pytest.mark.parametrize("name", list(PACKED))
def test_packed(hip_device, kdecay_lib, name, dname):
    """Sequences of one batch in one tensor: their values are those of each alone, and rows
    of none are zero whatever the memory held."""
    cu, N = PACKED[name]
    x = case(hip_device, (1, 2, 4, N, 64, 48, "tokens"), dname, seed=5)
    gen = torch.Generator().manual_seed(6)
    init, dS = (torch.randn(len(cu) - 1, 4, 64, 48, generator=gen).to(hip_device) for _ in range(2))
    do = torch.randn(1, 4, N, 48, generator=gen).to(DTYPES[dname]).to(hip_device)
    junk = [torch.full((1 << 22,), float("nan"), device=hip_device) for _ in range(4)]
    del junk  # what the allocator gives next
    for cut in (torch.tensor(cu, dtype=torch.int32, device=hip_device), torch.tensor(cu, device=hip_device)):
        o, S = kilat_amd.gated_delta_scan(*x, initial_state=init, cu_seqlens=cut, return_final_state=True)
        ro, rS = delta_ref(*(t.cpu() for t in x), init=init.cpu(), cu=cu)
        assert_near(o, ro, "o")
        assert_near(S, rS, "final state")
        assert not o[:, :, : cu[0]].any() and not o[:, :, cu[-1]:].any()
    if cu[-1] > cu[0]:
        got = check_grads(hip_device, x, init, do, dS, cu=cu)
    else:
        got = grads_of(x, init, do, dS, kernel(cut))
        assert torch.equal(got[5], dS)
    for t in got[:5]:
        assert not t[:, :, : cu[0]].any() and not t[:, :, cu[-1]:].any()


def test_packed_rows_of_other_sequences_do_not_count(hip_device, kdecay_lib):
    """NaN in the rows of one sequence, and behind the last one, changes no bit of the others."""
    cu = [0, 70, 100, 240]
    x = case(hip_device, (1, 2, 2, 260, 64, 64, "tokens"), "bf16", seed=7)
    do = torch.randn(1, 2, 260, 64, device=hip_device).bfloat16()
    cud = torch.tensor(cu, dtype=torch.int32, device=hip_device)
    ref = grads_of(x, None, do, None, kernel(cud))
    o = kilat_amd.gated_delta_scan(*x, cu_seqlens=cud)
    y = [t.clone() for t in x]
    for t in (*y, do):
        t[:, :, 70:100] = float("nan")
        t[:, :, 240:] = float("nan")
    p = kilat_amd.gated_delta_scan(*y, cu_seqlens=cud)
    got = grads_of(y, None, do, None, kernel(cud))
    for a, b in zip((o, *ref), (p, *got)):
        assert torch.equal(a[:, :, :70], b[:, :, :70]) and torch.equal(a[:, :, 100:240], b[:, :, 100:240])
        assert not b[:, :, 240:].any()


@pytest.mark.parametrize("cu", [[-5, 40, 900], [60, 20, 80], [0, 2**31 - 1], [-(2**31), -7]], ids=str)
def test_row_numbers_out_of_range_stay_in_bounds(hip_device, kdecay_lib, cu):
    """Row numbers are taken as inside 0..N on the device; whatever they are the call
    returns, and the next one is right."""
    x = case(hip_device, (1, 1, 2, 100, 32, 32, "heads"), "bf16")
    cud = torch.tensor(cu, dtype=torch.int32, device=hip_device)
    kilat_amd.gated_delta_scan(*x, cu_seqlens=cud)
    grads_of(x, None, torch.ones_like(x[2]), None, kernel(cud))
    torch.cuda.synchronize()
    assert_near(kilat_amd.gated_delta_scan(*x), delta_ref(*(t.cpu() for t in x))[0], "o")


# ---------------------------------------------------------------------------
# Values
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dname", ["bf16", "f32"])
def test_gates_at_their_ends(hip_device, kdecay_lib, dname):
    """g = -inf, the type's lowest value and 0; beta 0 and 1; repeated keys."""
    q, k, v, g, beta = case(hip_device, (1, 2, 2, 150, 64, 32, "heads"), dname, seed=8)
    g, beta = g.clone(), beta.clone()
    g[:, 0, 20], g[:, 0, 90:93], g[:, 1, 5] = float("-inf"), torch.finfo(torch.float32).min, -1000.0
    g[:, 1, 64:] = 0.0
    beta[:, :, 30:40], beta[:, 1, 40:] = 0.0, 1.0
    k = k.clone()
    k[:, 1, 70:100] = k[:, 1, 70:71]
    k[:, 0, 100:] = 0.0
    x = (q, k, v, g, beta)
    o, S = kilat_amd.gated_delta_scan(*x, return_final_state=True)
    ro, rS = delta_ref(*(t.cpu() for t in x))
    assert_near(o, ro, "o")
    assert_near(S, rS, "final state")
    do = torch.randn(1, 2, 150, 32, device=hip_device).to(v.dtype)
    finite = [t if t is not g else g.clamp(min=-200.0) for t in x]  # 64-bit autograd has 0 * inf at -inf
    check_grads(hip_device, finite, None, do, None)
    for a, b in zip(grads_of(x, None, do, None, kernel()), grads_of(finite, None, do, None, kernel())):
        assert torch.equal(a, b)


def test_keys_all_alike_without_decay(hip_device, kdecay_lib):
    """(I + A)^-1 of the worst chunk: A is all ones below the diagonal.  u_t is v_t - v_{t-1}, and
    the state k v_t' the sum of the chunk's 64 k u_t', that cancel but for the last: each
    is rounded at 2^-24 of its own size, so the sum's terms set the error."""
    q, k, v, g, beta = case(hip_device, (1, 1, 1, 256, 64, 64, "heads"), "f32", seed=9)
    k, g, beta = k[:, :, :1].expand_as(k), torch.zeros_like(g), torch.ones_like(beta)
    o, S = kilat_amd.gated_delta_scan(q, k, v, g, beta, return_final_state=True)
    ro, rS = delta_ref(*(t.cpu() for t in (q, k, v, g, beta)))
    u = v[:, :, 1:] - v[:, :, :-1]
    terms = float(u[:, :, -64:].abs().sum(2).max() * k.abs().max())
    assert_near(o, ro, "o", terms=terms / 8)  # over scale = 1/8
    assert_near(S, rS, "final state", terms=terms)


def test_strong_decay_keeps_near_tokens(hip_device, kdecay_lib):
    """Sums of log decays of thousands: what counts are differences of a few."""
    q, k, v, g, beta = case(hip_device, (1, 1, 2, 128, 64, 64, "heads"), "f32", seed=10)
    g = g.clone()
    g[:, :, ::2] = -100.0  # every token's state lives for one more token
    o, S = kilat_amd.gated_delta_scan(q, k, v, g, beta, return_final_state=True)
    ro, rS = delta_ref(*(t.cpu() for t in (q, k, v, g, beta)))
    assert_near(o, ro, "o")
    assert_near(S, rS, "final state")


@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("which", ["v nan", "v inf", "k nan", "q nan", "beta nan", "g nan", "state nan"])
def test_values_that_are_not_finite_reach_later_tokens_only(hip_device, kdecay_lib, which, dname):
    x = [t.clone() for t in case(hip_device, (1, 2, 2, 200, 64, 64, "tokens"), dname, seed=11)]
    init = torch.randn(1, 2, 64, 64, device=hip_device)
    o = kilat_amd.gated_delta_scan(*x, initial_state=init)
    bad = float("inf") if "inf" in which else float("nan")
    name = which.split()[0]
    y, init2 = [t.clone() for t in x], init.clone()
    if name == "state":
        init2[:, 0, 3, 17] = bad
    elif name in ("g", "beta"):
        y[3 if name == "g" else 4][:, 0, 100] = bad
    else:
        y["qkv".index(name)][:, 0, 100, 17] = bad
    p = kilat_amd.gated_delta_scan(*y, initial_state=init2)
    ref = delta_ref(*(t.cpu() for t in y), init=init2.cpu())[0]
    # The same tokens, heads and columns as by the formula (which has inf where the sum of
    # the split terms of an inf is NaN).
    assert torch.equal(p.cpu().isfinite(), ref.isfinite())
    assert torch.equal(p[:, 1], o[:, 1])  # the other head: not a bit
    assert_near(torch.where(ref.isfinite(), p.cpu(), 0.0), torch.where(ref.isfinite(), ref, 0.0), "o")


# ---------------------------------------------------------------------------
# Layouts, types, empties
# ---------------------------------------------------------------------------
def test_layouts(hip_device, kdecay_lib):
    """Channels that are not adjacent, rows off the vector grid, expanded heads and
    batches, lazily negated views."""
    q, k, v, g, beta = case(hip_device, (2, 2, 2, 70, 40, 24, "heads"), "bf16", seed=12)
    plain = kilat_amd.gated_delta_scan(q, k, v, g, beta)

    def off(t, by):  # the same values `by` elements into a buffer
        buf = torch.zeros(t.numel() + by, dtype=t.dtype, device=t.device)
        return buf[by:].view(t.shape).copy_(t)

    for by in (1, 2, 3, 4):
        assert torch.equal(kilat_amd.gated_delta_scan(off(q, by), off(k, by), off(v, by), g, beta), plain)
    turned = [t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v)]
    assert torch.equal(kilat_amd.gated_delta_scan(*turned, g, beta), plain)
    wide = [torch.zeros(2, 2, 70, 3 * t.shape[-1] + 1, dtype=t.dtype, device=t.device)[..., 1:1 + t.shape[-1]].copy_(t)
            for t in (q, k, v)]
    assert torch.equal(kilat_amd.gated_delta_scan(*wide, g, beta), plain)
    neg = torch._neg_view(-v)
    assert neg.is_neg() and torch.equal(kilat_amd.gated_delta_scan(q, k, neg, g, beta), plain)
    one = kilat_amd.gated_delta_scan(q[:1, :1].expand(2, 2, -1, -1), k[:1, :1].expand(2, 2, -1, -1), v,
                                     g[:, :1].expand(-1, 2, -1), beta)
    two = kilat_amd.gated_delta_scan(q[:1, :1].expand(2, 2, -1, -1).contiguous(), k[:1, :1].repeat(2, 2, 1, 1), v,
                                     g[:, :1].repeat(1, 2, 1), beta)
    assert torch.equal(one, two)
    o = kilat_amd.gated_delta_scan(q, k, v.transpose(1, 2).contiguous().transpose(1, 2), g, beta)
    assert o.stride(1) < o.stride(2) and torch.equal(o, plain)  # laid out like v
    for t in (torch.float64, torch.bfloat16):
        p = kilat_amd.gated_delta_scan(q, k, v, g.to(t), beta.to(t))
        assert torch.equal(p, kilat_amd.gated_delta_scan(q, k, v, g.to(t).float(), beta.to(t).float()))


def test_gradients_of_broadcast_and_converted_inputs(hip_device, kdecay_lib):
    q, k, v, g, beta = case(hip_device, (2, 1, 4, 70, 32, 32, "heads"), "f32", seed=13)
    leaves = [q[:1], k, v, g[:, :1].double(), beta[..., :1].bfloat16()]
    do = torch.randn_like(v)

    def run(f, leaves, do):
        xs = [t.detach().clone().requires_grad_() for t in leaves]
        y = [xs[0].expand(2, -1, -1, -1), xs[1], xs[2], xs[3].expand(-1, 4, -1), xs[4].expand(-1, -1, 70)]
        return torch.autograd.grad(f(*y), xs, do)

    got = run(lambda *y: kilat_amd.gated_delta_scan(*y), leaves, do)
    ref = run(lambda *y: delta_ref(*y)[0], [t.cpu().double() for t in leaves], do.cpu().double())
    for a, b, t, name in zip(got, ref, leaves, NAMES):
        assert a.dtype == t.dtype and a.shape == t.shape
        # sums over the broadcast dimension on top, in the leaf's type (bfloat16: 70 additions of half a step)
        assert_near(a.float() if a.dtype == torch.bfloat16 else a.float(), b, name,
                    70 * 2.0 ** -8 / 1.4e-5 if a.dtype == torch.bfloat16 else 8.0)


def test_gradient_against_differences(hip_device, kdecay_lib):
    """The loss along one direction of every input, by central differences in 64 bits."""
    x = case(hip_device, (1, 2, 4, 90, 48, 40, "heads"), "f32", seed=14)
    gen = torch.Generator().manual_seed(15)
    do = torch.randn(1, 4, 90, 40, generator=gen)
    got = [t.cpu().double() for t in grads_of(x, None, do.to(hip_device), None, kernel())]
    host = [t.cpu().double() for t in x]
    for i, (t, d) in enumerate(zip(host, got)):
        way = torch.randn(t.shape, generator=gen, dtype=torch.float64)
        loss = lambda e: float((delta_ref(*host[:i], t + e * way, *host[i + 1:])[0] * do).sum())  # noqa: B023,E731
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        # differences are off by (1e-5)^2 of a third derivative and 2^-53 / 1e-5 of the loss; the
        # kernel by 2^-24 sqrt(192 * 300) of the gradient, in the 2-norm along a unit direction
        assert abs(slope - float((d * way).sum())) <= 1e-6 * abs(slope) + 1.4e-5 * float(d.norm()) * 4, NAMES[i]


@pytest.mark.parametrize("B,N", [(0, 5), (2, 0), (0, 0)])
def test_empty(hip_device, kdecay_lib, B, N):
    x = [t.requires_grad_() for t in case(hip_device, (B, 1, 2, N, 32, 16, "heads"), "bf16")]
    init = torch.randn(B, 2, 32, 16, device=hip_device, requires_grad=True)
    o, S = kilat_amd.gated_delta_scan(*x, initial_state=init, return_final_state=True)
    assert o.shape == x[2].shape and torch.equal(S, init)
    gr = torch.autograd.grad((o, S), (*x, init), (torch.ones_like(o), 2 * torch.ones_like(S)))
    assert [t.shape for t in gr] == [t.shape for t in (*x, init)] and torch.equal(gr[5], 2 * torch.ones_like(S))
    with torch.no_grad():
        assert not kilat_amd.gated_delta_scan(*x, return_final_state=True)[1].any()


def test_rows_past_32_bit_offsets(hip_device, kdecay_lib):
    """The last head's rows lie 2^31 elements and more into the buffer."""
    N, H = 66, 2
    far = 2**31 + 64
    buf = torch.zeros(far + N * 64, dtype=torch.bfloat16, device=hip_device)
    x = case(hip_device, (1, H, H, N, 64, 64, "heads"), "bf16", seed=16)
    v = buf.as_strided((1, H, N, 64), (far + N * 64, far, 64, 1))
    v.copy_(x[2])
    o = kilat_amd.gated_delta_scan(x[0], x[1], v, x[3], x[4])
    assert torch.equal(o, kilat_amd.gated_delta_scan(*x))


# ---------------------------------------------------------------------------
# The node, streams, graphs
# ---------------------------------------------------------------------------
def test_only_what_is_asked(hip_device, kdecay_lib):
    """A gradient of one input, of the final state alone, of o alone; none under no_grad."""
    x = case(hip_device, (1, 1, 2, 100, 32, 32, "heads"), "f32", seed=17)
    every = grads_of(x, None, torch.ones_like(x[2]), None, kernel())
    for i in range(5):
        y = [t.clone().requires_grad_() if j == i else t for j, t in enumerate(x)]
        assert torch.equal(torch.autograd.grad(kilat_amd.gated_delta_scan(*y).sum(), y[i])[0], every[i])
    y = [t.clone().requires_grad_() for t in x]
    o, S = kilat_amd.gated_delta_scan(*y, return_final_state=True)
    got = torch.autograd.grad(S.sum(), y, allow_unused=True)
    host = [t.cpu().double().requires_grad_() for t in x]
    ref = torch.autograd.grad(delta_ref(*host)[1].sum(), host, allow_unused=True)
    for a, b, name in zip(got, ref, NAMES):
        assert_near(a, b if b is not None else torch.zeros_like(a).cpu().double(), name, 4.0)
    with torch.no_grad():
        assert not kilat_amd.gated_delta_scan(*y).requires_grad
    with torch.inference_mode():
        z = kilat_amd.gated_delta_scan(*x)
    w = x[4].clone().requires_grad_()
    with torch.inference_mode():
        made = x[2].clone()
    torch.autograd.grad(kilat_amd.gated_delta_scan(x[0], x[1], made, x[3], w).sum(), w)
    assert torch.equal(z, kilat_amd.gated_delta_scan(*x))


def test_node_refusals(hip_device, kdecay_lib):
    x = [t.requires_grad_() for t in case(hip_device, (1, 1, 1, 70, 32, 32, "heads"), "f32")]
    o = kilat_amd.gated_delta_scan(*x)
    torch.autograd.grad(o.sum(), x)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(o.sum(), x)
    w = x[2] * 1
    o = kilat_amd.gated_delta_scan(x[0], x[1], w, x[3], x[4])
    w.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(o.sum(), x)
    import torch.autograd.forward_ad as fwad

    with fwad.dual_level(), pytest.raises(RuntimeError):
        kilat_amd.gated_delta_scan(x[0], x[1], fwad.make_dual(x[2].detach(), torch.ones_like(x[2])), x[3], x[4])


def test_another_stream(hip_device, kdecay_lib):
    x = case(hip_device, (2, 2, 4, 500, 64, 64, "tokens"), "bf16", seed=18)
    do = torch.randn_like(x[2])
    ref = grads_of(x, None, do, None, kernel())
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        with torch.cuda.stream(s):
            outs.append(grads_of(x, None, do, None, kernel()))
    torch.cuda.synchronize()
    for got in outs:
        assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_captured(hip_device, kdecay_lib):
    """The scan with its backward and a step in one graph, replayed on new inputs with
    eager work between the replays."""
    x = case(hip_device, (2, 1, 2, 150, 64, 64, "heads"), "bf16", seed=19)
    one = [t[:, :, 0].contiguous() for t in x]
    do = torch.randn_like(x[2])

    def run(y, one):
        o, S = kilat_amd.gated_delta_scan(*y, return_final_state=True)
        grads = torch.autograd.grad(o, y, do)
        return (o.detach(), *grads, *kilat_amd.gated_delta_step(*one, S))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = [t.clone().requires_grad_() for t in x]
        run(y, one)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            out = run(y, one)
    for seed in range(3):
        z = case(hip_device, (2, 1, 2, 150, 64, 64, "heads"), "bf16", seed=20 + seed)
        ref = run([t.clone().requires_grad_() for t in z], one)
        with torch.no_grad():
            for a, b in zip(y, z):
                a.copy_(b)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref)), seed


# ---------------------------------------------------------------------------
# One token
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dname", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("B,Hk,H,Dk,Dv", [(1, 6, 6, 64, 64), (3, 2, 4, 128, 128), (2, 1, 3, 7, 5), (1, 1, 1, 1, 1),
                                          (2, 2, 2, 100, 256), (5, 1, 2, 33, 36)])
def test_step(hip_device, kdecay_lib, B, Hk, H, Dk, Dv, dname):
    q, k, v, g, beta = (t[:, :, 0] for t in case(hip_device, (B, Hk, H, 1, Dk, Dv, "heads"), dname, seed=21))
    S = torch.randn(B, H, Dk, Dv, device=hip_device)
    ro, rS = delta_ref(*(t.cpu()[:, :, None] for t in (q, k, v, g, beta)), init=S.cpu())
    o, S1 = kilat_amd.gated_delta_step(q, k, v, g, beta, S)
    assert o.dtype == v.dtype
    assert_near(o, ro[:, :, 0], "out")
    assert_near(S1, rS, "state")
    o32, _ = kilat_amd.gated_delta_step(q, k, v, g, beta, S, out_dtype=torch.float32)
    assert o32.dtype == torch.float32 and torch.equal(o32.to(v.dtype), o)
    T = S.clone()
    out = torch.empty_like(v)
    r = kilat_amd.gated_delta_step(q, k, v, g, beta, T, new_state=T, out=out)
    assert r[0] is out and r[1] is T and torch.equal(T, S1) and torch.equal(out, o)
    # a state off the 16-byte grid, inputs that are not contiguous, other float types
    buf = torch.zeros(S.numel() + 1, device=hip_device)[1:].view(S.shape).copy_(S)
    wide = torch.zeros(B, H, 3 * Dv, dtype=v.dtype, device=hip_device)[..., Dv:2 * Dv].copy_(v)
    o2, S2 = kilat_amd.gated_delta_step(q, k, wide, g.double(), beta.double(), buf, new_state=buf)
    assert S2 is buf and torch.equal(S2, S1) and torch.equal(o2, o)


def test_step_outputs_that_share_memory(hip_device, kdecay_lib):
    """new_state overlapping the state by part, and out in the state's memory: through copies."""
    q, k, v, g, beta = (t[:, :, 0] for t in case(hip_device, (4, 2, 2, 1, 64, 64, "heads"), "f32", seed=22))
    n = 4 * 2 * 64 * 64
    buf = torch.randn(n + 64 * 64, device=hip_device)
    S, late = buf[:n].view(4, 2, 64, 64), buf[64 * 64:].view(4, 2, 64, 64)
    o, S1 = kilat_amd.gated_delta_step(q, k, v, g, beta, S)
    o2, S2 = kilat_amd.gated_delta_step(q, k, v, g, beta, S, new_state=late)
    assert torch.equal(S2, S1) and torch.equal(o2, o)
    T = S1.clone()
    o3, S3 = kilat_amd.gated_delta_step(q, k, v, g, beta, T)
    out = T.view(-1)[: o3.numel()].view(o3.shape)
    o4, S4 = kilat_amd.gated_delta_step(q, k, v, g, beta, T, out=out)
    assert torch.equal(S4, S3) and torch.equal(o4, o3)
    o5, _ = kilat_amd.gated_delta_step(q, k, v, g, beta, S1, out=v)
    assert o5 is v and torch.equal(v, o3)


@pytest.mark.parametrize("dname", ["bf16", "f32"])
def test_prefill_then_steps(hip_device, kdecay_lib, dname):
    """As they are used: a packed prefill, a second chunk from its states, then tokens one by
    one, against one pass over everything."""
    lens, more, steps = [70, 3, 129], 64, 5
    total = max(lens) + more + steps
    x = case(hip_device, (3, 2, 4, total, 64, 64, "heads"), dname, seed=23)
    cu = torch.tensor([0, *torch.tensor(lens).cumsum(0)], device=hip_device)
    packed = [torch.cat([t[b, :, :n] for b, n in enumerate(lens)], 1)[None] for t in x]
    o, S = kilat_amd.gated_delta_scan(*packed, cu_seqlens=cu, return_final_state=True)
    at = torch.tensor(lens, device=hip_device)[:, None] + torch.arange(more, device=hip_device)
    pick = [torch.stack([t[b][:, at[b]] for b in range(3)]) for t in x]
    o2, S = kilat_amd.gated_delta_scan(*pick, initial_state=S, return_final_state=True)
    for b, n in enumerate(lens):
        ro = delta_ref(*(t[b:b + 1, :, : n + more + steps].cpu() for t in x))[0]
        assert_near(o[:, :, int(cu[b]):int(cu[b]) + n], ro[:, :, :n], "prefill")
        assert_near(o2[b:b + 1], ro[:, :, n:n + more], "second chunk")
    for s in range(steps):
        one = [torch.stack([t[b, :, n + more + s] for b, n in enumerate(lens)]) for t in x]
        y, S = kilat_amd.gated_delta_step(*one, S, new_state=S)
        for b, n in enumerate(lens):
            ro = delta_ref(*(t[b:b + 1, :, : n + more + s + 1].cpu() for t in x))[0]
            assert_near(y[b], ro[0, :, -1], "token")

"""The gated delta rule's and causal attention's public functions and C ABI without a GPU:
what they refuse, and their oracles against forms written another way."""
from __future__ import annotations

import ctypes
import os
import re
import subprocess

import pytest
import torch

import kilat_amd
from kilat_amd import _build, _lib
from tests.mixer_cases import attention_ref, delta_inputs, delta_ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def inputs(B=2, Hk=1, H=2, N=3, Dk=8, Dv=4, dtype=torch.float32):
    return list(delta_inputs(B, Hk, H, N, Dk, Dv, dtype))


def test_cpu_tensors_are_refused(kdecay_lib):
    x = inputs()
    with pytest.raises(RuntimeError, match="HIP"):
        kilat_amd.gated_delta_scan(*x)
    with pytest.raises(RuntimeError, match="HIP"):
        kilat_amd.gated_delta_step(*(t[:, :, 0] for t in x), torch.zeros(2, 2, 8, 4))
    with pytest.raises(RuntimeError, match="HIP"):
        kilat_amd.causal_attention(torch.zeros(1, 2, 3, 4), torch.zeros(1, 1, 3, 4), torch.zeros(1, 1, 3, 4))


SCAN_REFUSALS = {
    "q is no tensor": (lambda x, kw: x.__setitem__(0, [1.0]), TypeError),
    "float64": (lambda x, kw: x.__setitem__(slice(0, 3), [t.double() for t in x[:3]]), TypeError),
    "integers": (lambda x, kw: x.__setitem__(slice(0, 3), [t.long() for t in x[:3]]), TypeError),
    "two types": (lambda x, kw: x.__setitem__(1, x[1].half()), TypeError),
    "three dimensions": (lambda x, kw: x.__setitem__(2, x[2][0]), ValueError),
    "q unlike k": (lambda x, kw: x.__setitem__(0, x[0][..., :4]), ValueError),
    "rows of v": (lambda x, kw: x.__setitem__(2, x[2][:, :, :2]), ValueError),
    "batch of v": (lambda x, kw: x.__setitem__(2, x[2][:1]), ValueError),
    "heads": (lambda x, kw: x.__setitem__(slice(0, 2), [t.expand(-1, 3, -1, -1) for t in x[:2]]), ValueError),
    "no heads": (lambda x, kw: x.__setitem__(slice(0, 2), [t[:, :0] for t in x[:2]]), ValueError),
    "wide keys": (lambda x, kw: x.__setitem__(slice(0, 2), [torch.zeros(2, 1, 3, 129)] * 2), ValueError),
    "wide values": (lambda x, kw: x.__setitem__(2, torch.zeros(2, 2, 3, 257)), ValueError),
    "no channels": (lambda x, kw: x.__setitem__(2, x[2][..., :0]), ValueError),
    "g": (lambda x, kw: x.__setitem__(3, x[3][:, :1]), ValueError),
    "g of integers": (lambda x, kw: x.__setitem__(3, x[3].long()), TypeError),
    "beta": (lambda x, kw: x.__setitem__(4, x[4][..., None]), ValueError),
    "state": (lambda x, kw: kw.__setitem__("initial_state", torch.zeros(2, 2, 4, 8)), ValueError),
    "state of integers": (lambda x, kw: kw.__setitem__("initial_state", torch.zeros(2, 2, 8, 4).long()), TypeError),
    "packed batch of two": (lambda x, kw: kw.__setitem__("cu_seqlens", torch.tensor([0, 3])), ValueError),
    "cu_seqlens of floats": (lambda x, kw: kw.__setitem__("cu_seqlens", torch.tensor([0.0, 3.0])), TypeError),
    "cu_seqlens of one": (lambda x, kw: kw.__setitem__("cu_seqlens", torch.tensor([0])), ValueError),
    "cu_seqlens is a list": (lambda x, kw: kw.__setitem__("cu_seqlens", [0, 3]), TypeError),
}


@pytest.mark.parametrize("name", list(SCAN_REFUSALS))
def test_scan_refusals(kdecay_lib, name):
    x, kw = inputs(), {}
    change, error = SCAN_REFUSALS[name]
    change(x, kw)
    with pytest.raises(error):
        kilat_amd.gated_delta_scan(*x, **kw)


def test_packed_states_are_per_sequence(kdecay_lib):
    x = inputs(B=1)
    with pytest.raises(ValueError, match="initial_state"):
        kilat_amd.gated_delta_scan(*x, cu_seqlens=torch.tensor([0, 1, 3]), initial_state=torch.zeros(1, 2, 8, 4))


def test_step_refusals(kdecay_lib):
    q, k, v, g, beta = (t[:, :, 0] for t in inputs())
    S = torch.zeros(2, 2, 8, 4)
    step = kilat_amd.gated_delta_step
    for args, error in (((q, k, v, g, beta, S[0]), ValueError), ((q[:1], k[:1], v, g, beta, S), ValueError),
                        ((q, k, v[..., :2], g, beta, S), ValueError), ((q, k, v, g[:1], beta, S), ValueError),
                        ((q, k, v, g, beta[:, :1], S), ValueError), ((q, k.half(), v, g, beta, S), TypeError),
                        ((q, k, v, g, beta, S.long()), TypeError), ((q, k, v, g, beta, None), TypeError),
                        ((q[..., :4], k[..., :4], v, g, beta, S), ValueError)):
        with pytest.raises(error):
            step(*args)


def test_attention_refusals(kdecay_lib):
    q, k, v = torch.zeros(1, 4, 3, 8), torch.zeros(1, 2, 3, 8), torch.zeros(1, 2, 3, 5)
    f = kilat_amd.causal_attention
    for args, error in (((q[0], k, v), ValueError), ((q, k[:, :, :2], v), ValueError), ((q, k, v[:, :1]), ValueError),
                        ((q, k[..., :4], v), ValueError), ((q[:, :3], k, v), ValueError), ((q, k[:, :0], v[:, :0]), ValueError),
                        ((q, k.half(), v), TypeError), ((q.double(), k.double(), v.double()), TypeError),
                        ((torch.zeros(1, 4, 3, 129), torch.zeros(1, 2, 3, 129), v), ValueError),
                        ((q, k, torch.zeros(1, 2, 3, 129)), ValueError), ((q, k, 1.0), TypeError)):
        with pytest.raises(error):
            f(*args)
    with pytest.raises(ValueError):
        f(q.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1), cu_seqlens=torch.tensor([0, 3]))


# ---------------------------------------------------------------------------
# The C ABI
# ---------------------------------------------------------------------------
def test_headers_match_the_library(kdecay_lib):
    out = subprocess.run(["nm", "-D", "--defined-only", _build.LIBRARY], capture_output=True, text=True, check=True)
    exported = set(re.findall(r"\bT (k(?:delta|attn)_\w+)", out.stdout))
    declared = set()
    for name in ("kdelta.h", "kattn.h"):
        text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", name)).read(), flags=re.S)
        declared |= set(re.findall(r"\b(k(?:delta|attn)_\w+)\s*\(", text))
    assert exported == declared


class Problem(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "g", "beta", "cu", "init")] + [
        (n, ctypes.c_int64 * c) for n, c in (("qs", 4), ("ks", 4), ("vs", 4), ("gs", 3), ("bs", 3))] + [
        (n, ctypes.c_int64) for n in ("B", "Hk", "H", "N", "Dk", "Dv", "sequences")] + [
        ("scale", ctypes.c_float), ("dtype", ctypes.c_int)]


class Attention(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("q", "k", "v", "cu")] + [
        (n, ctypes.c_int64 * 4) for n in ("qs", "ks", "vs")] + [
        (n, ctypes.c_int64) for n in ("B", "Hk", "H", "N", "Dk", "Dv", "sequences")] + [
        ("scale", ctypes.c_float), ("dtype", ctypes.c_int)]


FAKE = 0x10000  # never dereferenced on the host


def problem(kind=Problem, **kw):
    p = kind(q=FAKE, k=FAKE, v=FAKE, B=1, Hk=1, H=2, N=100, Dk=64, Dv=64, sequences=1, scale=0.125, dtype=_lib.KDECAY_BF16)
    if kind is Problem:
        p.g = p.beta = FAKE
    for name in ("qs", "ks", "vs"):
        getattr(p, name)[:] = [12800, 6400, 64, 1]
    for name, x in kw.items():
        setattr(p, name, x)
    return p


BAD = [dict(B=-1), dict(dtype=_lib.KDECAY_F64), dict(dtype=9), dict(Dk=0), dict(Dk=129), dict(Dv=300), dict(Hk=0), dict(Hk=3),
       dict(H=70000, Hk=1), dict(sequences=2), dict(cu=FAKE, B=2, sequences=2), dict(cu=FAKE, sequences=0), dict(q=None),
       dict(qs=(ctypes.c_int64 * 4)(1, 1, 1, 2))]


@pytest.mark.parametrize("kw", BAD, ids=str)
def test_abi_rejects_bad_problems(kdecay_lib, kw):
    """Nothing is launched (there is no GPU here), and the message says why."""
    st = (ctypes.c_int64 * 4)(12800, 6400, 64, 1)
    lib = kdecay_lib
    lib.kdelta_scan_workspace_bytes.restype = ctypes.c_size_t
    fake, big = ctypes.c_void_p(FAKE), ctypes.c_size_t(1 << 40)
    assert lib.kdelta_scan_fwd(ctypes.byref(problem(**kw)), fake, st, None, None, fake, big, None) < 0
    assert lib.kdecay_last_error_string()
    assert lib.kdelta_scan_bwd(ctypes.byref(problem(**kw)), fake, st, None, fake, fake, st, fake, st, fake, st, fake, fake,
                               None, fake, big, None) < 0
    assert lib.kattn_fwd(ctypes.byref(problem(Attention, **kw)), fake, st, None) < 0
    assert lib.kdelta_scan_workspace_bytes(ctypes.byref(problem(**kw))) == 0 or kw.get("q", 1) is None or "qs" in kw


def test_abi_rejects_bad_buffers(kdecay_lib):
    st = (ctypes.c_int64 * 4)(12800, 6400, 64, 1)
    lib, fake = kdecay_lib, ctypes.c_void_p(FAKE)
    for name in ("kdelta_scan_workspace_bytes", "kdelta_scan_bwd_workspace_bytes", "kdelta_scan_saved_floats"):
        getattr(lib, name).restype = ctypes.c_size_t
    p = ctypes.byref(problem())
    need, need_b = lib.kdelta_scan_workspace_bytes(p), lib.kdelta_scan_bwd_workspace_bytes(p)
    assert 0 < need < need_b and lib.kdelta_scan_saved_floats(p) >= 2 * 2 * 64 * 64
    small, enough = ctypes.c_size_t(need - 1), ctypes.c_size_t(need)
    assert lib.kdelta_scan_fwd(p, fake, st, None, None, fake, small, None) == _lib.KDECAY_EWORKSPACE
    assert lib.kdelta_scan_fwd(p, fake, st, None, None, None, enough, None) == _lib.KDECAY_EWORKSPACE
    assert lib.kdelta_scan_fwd(p, fake, st, None, None, ctypes.c_void_p(FAKE + 4), enough, None) == _lib.KDECAY_EWORKSPACE
    assert lib.kdelta_scan_fwd(p, None, st, None, None, fake, enough, None) == _lib.KDECAY_EINVAL
    assert lib.kdelta_scan_fwd(p, fake, st, None, ctypes.c_void_p(FAKE + 4), fake, enough, None) == _lib.KDECAY_ELAYOUT
    assert lib.kdelta_scan_fwd(None, fake, st, None, None, fake, enough, None) == _lib.KDECAY_EINVAL
    assert lib.kattn_fwd(None, fake, st, None) == _lib.KDECAY_EINVAL
    step = lambda **kw: lib.kdelta_step(*(kw.get(n, fake) for n in "qkv"), kw.get("dtype", 1), fake, fake, fake, fake, fake,  # noqa: E731
                                        kw.get("out", 1), *(ctypes.c_int64(kw.get(n, d)) for n, d in
                                                            (("B", 1), ("Hk", 1), ("H", 2), ("Dk", 64), ("Dv", 64))),
                                        ctypes.c_float(1.0), None)
    for kw, code in ((dict(B=-1), _lib.KDECAY_EINVAL), (dict(dtype=3), _lib.KDECAY_EDTYPE), (dict(out=2), _lib.KDECAY_EDTYPE),
                     (dict(Dk=129), _lib.KDECAY_ESHAPE), (dict(Dv=0), _lib.KDECAY_ESHAPE), (dict(Hk=4), _lib.KDECAY_ESHAPE),
                     (dict(q=None), _lib.KDECAY_EINVAL), (dict(B=0), 0)):
        assert step(**kw) == code, kw


def test_abi_takes_rows_of_whole_vectors_only(kdecay_lib):
    """Head dims that are no multiples of 8, rows and bases off 16 bytes: refused by both headers' functions."""
    st, fake, big = (ctypes.c_int64 * 4)(12800, 6400, 64, 1), ctypes.c_void_p(FAKE), ctypes.c_size_t(1 << 40)
    off = (ctypes.c_int64 * 4)(12800, 6400, 68, 1)
    for kw, code in ((dict(Dk=20), _lib.KDECAY_ESHAPE), (dict(Dv=12), _lib.KDECAY_ESHAPE), (dict(q=FAKE + 2), _lib.KDECAY_ELAYOUT),
                     (dict(k=FAKE + 8), _lib.KDECAY_ELAYOUT), (dict(vs=off), _lib.KDECAY_ELAYOUT),
                     (dict(qs=off), _lib.KDECAY_ELAYOUT)):
        assert kdecay_lib.kdelta_scan_fwd(ctypes.byref(problem(**kw)), fake, st, None, None, fake, big, None) == code, kw
        assert kdecay_lib.kattn_fwd(ctypes.byref(problem(Attention, **kw)), fake, st, None) == code, kw
    assert kdecay_lib.kdelta_scan_fwd(ctypes.byref(problem()), fake, off, None, None, fake, big, None) == _lib.KDECAY_ELAYOUT
    assert kdecay_lib.kattn_fwd(ctypes.byref(problem(Attention)), fake, off, None) == _lib.KDECAY_ELAYOUT
    assert kdecay_lib.kattn_fwd(ctypes.byref(problem(Attention)), ctypes.c_void_p(FAKE + 4), st, None) == _lib.KDECAY_ELAYOUT


# ---------------------------------------------------------------------------
# The oracles
# ---------------------------------------------------------------------------
def test_delta_oracle_is_the_recurrence_by_matrices():
    """S_t as a product of the matrices that the rule's definition names."""
    q, k, v, g, beta = inputs(B=1, Hk=2, H=2, N=9, Dk=5, Dv=3)
    o, S = delta_ref(q, k, v, g, beta, scale=0.3)
    for h in range(2):
        M = torch.zeros(5, 3, dtype=torch.float64)
        for t in range(9):
            kt, b, a = k[0, h, t].double(), float(beta[0, h, t]), float(g[0, h, t].double().exp())
            M = a * (torch.eye(5, dtype=torch.float64) - b * torch.outer(kt, kt)) @ M + b * torch.outer(kt, v[0, h, t].double())
            assert torch.allclose(o[0, h, t], 0.3 * q[0, h, t].double() @ M, rtol=0, atol=1e-13)
        assert torch.allclose(S[0, h], M, rtol=0, atol=1e-13)


def test_oracles_of_packed_batches_are_those_of_each_sequence():
    q, k, v, g, beta = inputs(B=1, N=12)
    o, S = delta_ref(q, k, v, g, beta, cu=[1, 4, 4, 10])
    assert not o[:, :, 0].any() and not o[:, :, 10:].any() and not S[1].any()
    p, T = delta_ref(*(t[:, :, 4:10] for t in (q, k, v, g, beta)))
    assert torch.equal(o[:, :, 4:10], p) and torch.equal(S[2], T[0])
    k2 = k.expand(-1, 2, -1, -1)
    a = attention_ref(k2, k, v[:, :1], cu=[1, 4, 4, 10])
    assert not a[:, :, 0].any() and not a[:, :, 10:].any()
    x = torch.nn.functional.scaled_dot_product_attention(k2[:, :, 4:10].double(), k2[:, :, 4:10].double(),
                                                         v[:, :1, 4:10].expand(-1, 2, -1, -1).double(), is_causal=True)
    assert torch.allclose(a[:, :, 4:10], x, rtol=0, atol=1e-13)

"""The mixers that stand next to the decay scan in a hybrid layer, as measurable cases.

Four kinds of pass, each through the package's public functions:
  scan   the gated delta rule over whole sequences (``gated_delta_scan``): o and
         the final state of a prefill
  train  the same scan and its backward: o, dq, dk, dv, dg and dbeta
  step   one token of the gated delta rule for a batch (``gated_delta_step``)
  attn   causal attention over whole prompts (``causal_attention``)

With ``own`` false a pass is computed from elementary torch operations.

Inputs are synthetic: unit keys and queries (as these layers normalise them),
normal values, write strengths beta = sigmoid of a normal, and log decays g whose
scale per head runs from a memory of a few tokens to one of several thousand.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}

CHUNK = 64  # tokens that the plain form of the scan takes at a time

# The most work of a drawn case: that of the largest listed one of its kind.
MOST_SCAN = 16 * 65536 * 128 * 128
MOST_TRAIN = 8 * 12 * 4096 * 64 * 64
# (For attention the pairs of rows, masked or not.)
MOST_ATTN = 16 * 16384 * 16384
# Elements of q, k, v and o together that one drawn case may have.
MOST_ELEMENTS = 16 * 65536 * 128 * 4


def _scan(name, B, Hk, H, N, Dk, Dv, dtype, **more):
    return dict({"name": name, "kind": "scan", "B": B, "Hk": Hk, "H": H, "N": N, "Dk": Dk, "Dv": Dv, "dtype": dtype,
                 "layout": "heads", "packed": 0, "spare": 0, "carry": False}, **more)


def _attn(name, B, Hk, H, N, Dk, Dv, dtype, **more):
    return dict({"name": name, "kind": "attn", "B": B, "Hk": Hk, "H": H, "N": N, "Dk": Dk, "Dv": Dv, "dtype": dtype,
                 "layout": "heads", "packed": 0, "spare": 0}, **more)


def listed():
    return [
        # One user decoding: a single sequence's token in one layer of the
        # 12-head model with half of its heads recurrent.  Launch and host cost.
        {"name": "step_one", "kind": "step", "B": 1, "Hk": 6, "H": 6, "Dk": 64, "Dv": 64, "dtype": "bf16",
         "in_place": False},
        # A serving pool's token: 256 sequences, the states updated in place.
        {"name": "step_pool", "kind": "step", "B": 256, "Hk": 12, "H": 12, "Dk": 64, "Dv": 64, "dtype": "bf16",
         "in_place": True},
        # Prefill of one layer of that model: 8 sequences of 1024 tokens, as
        # the projections leave them.
        _scan("scan_layer", 8, 6, 6, 1024, 64, 64, "bf16", layout="tokens"),
        # A packed prefill batch: 24 prompts of different lengths in 16384
        # rows, some rows behind the last prompt unused.
        _scan("scan_packed", 1, 12, 12, 16384, 64, 64, "bf16", layout="tokens", packed=24, spare=37),
        # Chunked prefill in fp16 from carried states: heads of 80 channels,
        # two value heads for each key head, a ragged length.
        _scan("scan_carry_f16", 4, 8, 16, 2047, 80, 80, "f16", layout="tokens", carry=True),
        # One long document: 65536 tokens, 16 heads of 128 channels.
        _scan("scan_long", 1, 16, 16, 65536, 128, 128, "bf16"),
        # A small fp32 training pass (the fp32 parity configuration's sizes).
        _scan("train_f32_small", 2, 6, 6, 1024, 64, 64, "f32", kind="train"),
        # A training pass at the headline workload's sizes.
        _scan("train_bf16", 8, 12, 12, 4096, 64, 64, "bf16", kind="train"),
        # Training with 768 value channels in 8 heads of 96, two of them for
        # each key head of 64, as the projections lay them out, ragged length.
        _scan("train_grouped", 4, 4, 8, 3001, 64, 96, "bf16", layout="tokens", kind="train"),
        # The recall heads of the 12-head model's layer: 8 prompts of 1024.
        _attn("attn_layer", 8, 6, 6, 1024, 64, 64, "bf16", layout="tokens"),
        # A packed prefill batch in fp16 with grouped heads: 24 prompts.
        _attn("attn_packed_f16", 1, 4, 12, 16384, 64, 64, "f16", layout="tokens", packed=24, spare=37),
        # One long prompt, 16 heads of 128 channels over 4 key heads.
        _attn("attn_long", 1, 4, 16, 16384, 128, 128, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """One more case: any batch, heads, length, head dims, type and layout."""
    kind = rng.choice(["scan", "scan", "scan", "train", "train", "attn", "attn", "attn", "step"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    Hk = rng.randint(1, 12)
    H = Hk * rng.choice([1, 1, 2, 4]) if Hk <= 4 else Hk
    Dk = rng.choice([24, 32, 48, 64, 64, 64, 64, 80, 96, 100, 112, 128, 128])
    Dv = Dk if rng.random() < 0.7 else rng.choice([32, 64, 96, 128])
    if kind == "step":
        return {"kind": "step", "B": _log_int(rng, 1, 512), "Hk": Hk, "H": H, "Dk": Dk, "Dv": Dv, "dtype": dtype,
                "in_place": rng.random() < 0.5}
    packed = rng.choice([0, 0, _log_int(rng, 1, 64)])
    if kind == "attn":
        N = _log_int(rng, 1, 16384)
        most = min(MOST_ATTN // (H * N * N), MOST_ELEMENTS // 4 // (2 * H * (Dk + Dv) * N))
    else:
        N = _log_int(rng, 1, 65536 if kind == "scan" else 8192)
        least = MOST_SCAN if kind == "scan" else MOST_TRAIN
        while least < H * N * Dk * Dv:
            N //= 2
        most = min(least // (H * N * Dk * Dv), MOST_ELEMENTS // (2 * H * (Dk + Dv) * N))
    if dtype == "f32" or kind == "train":
        most //= 2
    B = 1 if packed else _log_int(rng, 1, max(1, min(256, most)))
    case = {"kind": kind, "B": B, "Hk": Hk, "H": H, "N": N, "Dk": Dk, "Dv": Dv, "dtype": dtype,
            "layout": rng.choice(["heads", "tokens"]), "packed": min(packed, N),
            "spare": rng.choice([0, rng.randint(1, 80)]) if packed else 0}
    if kind != "attn":
        case["carry"] = kind == "scan" and rng.random() < 0.4
    return case


def _lengths(case, seed):
    """Lengths of the packed sequences: uneven, their sum N, none empty."""
    g = torch.Generator().manual_seed(seed)
    cuts = (torch.randperm(case["N"] - 1, generator=g)[: case["packed"] - 1] + 1).sort().values.tolist()
    edges = [0, *cuts, case["N"]]
    return [b - a for a, b in zip(edges[:-1], edges[1:])]


def _rows(case, g, heads, width, dtype=torch.float32):
    """Normal [B, heads, N, width], contiguous ("heads") or a view of a
    projection's [B, N, heads * width] ("tokens")."""
    B, N = case["B"], case["N"] + case["spare"]
    if case["layout"] == "tokens":
        return torch.randn(B, N, heads, width, generator=g, device="cuda").to(dtype).permute(0, 2, 1, 3)
    return torch.randn(B, heads, N, width, generator=g, device="cuda").to(dtype)


def _unit(x, dtype):
    return (x * x.square().sum(-1, keepdim=True).add(1e-6).rsqrt()).to(dtype)


def _gates(case, g, shape):
    """g (log decay) and beta, [B, H] or [B, H, N], for heads of 4 to 4000 tokens' memory."""
    H = case["H"]
    span = torch.exp(torch.linspace(math.log(0.25), math.log(0.00025), H, device="cuda")).reshape(1, H, *[1] * (len(shape) - 2))
    noise = torch.rand(*shape, generator=g, device="cuda")
    return -span * (0.2 + 1.6 * noise), torch.sigmoid(torch.randn(*shape, generator=g, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    B, Hk, H, Dk, Dv = (case[x] for x in ("B", "Hk", "H", "Dk", "Dv"))
    state = {"case": case}
    if case["kind"] == "step":
        state["q"] = _unit(torch.randn(B, Hk, Dk, generator=gen, device="cuda"), dtype)
        state["k"] = _unit(torch.randn(B, Hk, Dk, generator=gen, device="cuda"), dtype)
        state["v"] = torch.randn(B, H, Dv, generator=gen, device="cuda").to(dtype)
        state["g"], state["beta"] = _gates(case, gen, (B, H))
        state["state"] = torch.randn(B, H, Dk, Dv, generator=gen, device="cuda")
        return state
    if case["packed"]:
        state["lengths"] = _lengths(case, seed)
        state["cu"] = torch.tensor([0, *state["lengths"]]).cumsum(0).to(device="cuda", dtype=torch.int32)
    if case["kind"] == "attn":
        state["q"] = _rows(case, gen, H, Dk, dtype)
        state["k"] = _rows(case, gen, Hk, Dk, dtype)
        state["v"] = _rows(case, gen, Hk, Dv, dtype)
        return state
    state["q"], state["k"] = _unit(_rows(case, gen, Hk, Dk), dtype), _unit(_rows(case, gen, Hk, Dk), dtype)
    state["v"] = _rows(case, gen, H, Dv, dtype)
    state["g"], state["beta"] = _gates(case, gen, (B, H, case["N"] + case["spare"]))
    if case["carry"]:
        state["carry"] = torch.randn(case["packed"] or B, H, Dk, Dv, generator=gen, device="cuda")
    if case["kind"] == "train":
        state["do"] = _rows(case, gen, H, Dv, dtype)
        for x in ("q", "k", "v", "g", "beta"):
            state[x].requires_grad_()
    return state


# ---------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------
def _heads(x, H):
    """Key heads repeated for the value heads that share them, in 32 bits."""
    return x.float().repeat_interleave(H // x.shape[1], dim=1)


def _inverse(A):
    """(I + A)^-1 of strictly lower triangular [..., n, C, C], C a power of two, by halves."""
    C = A.shape[-1]
    T = torch.ones(*A.shape[:-2], C, 1, 1, device=A.device)
    s = 1
    while s < C:
        blocks = A.reshape(*A.shape[:-2], C // (2 * s), 2 * s, C // (2 * s), 2 * s)
        low = torch.diagonal(blocks, dim1=-4, dim2=-2).movedim(-1, -3)[..., s:, :s].contiguous()
        T1, T2 = T[..., 0::2, :, :].contiguous(), T[..., 1::2, :, :].contiguous()
        X = -torch.matmul(torch.matmul(T2, low), T1)
        T = torch.cat([torch.cat([T1, torch.zeros_like(X)], -1), torch.cat([X, T2], -1)], -2)
        s *= 2
    return T[..., 0, :, :]


def _delta(q, k, v, g, beta, S):
    """o and the final state of [B, H, N, ...] in 32 bits, CHUNK tokens at a time."""
    B, H, N, Dk = q.shape
    pad = -N % CHUNK
    n = (N + pad) // CHUNK

    def chunks(x):
        x = torch.cat([x, x.new_zeros(B, H, pad, *x.shape[3:])], 2) if pad else x
        return x.reshape(B, H, n, CHUNK, *x.shape[3:])

    q, k, v, beta = chunks(q * Dk ** -0.5), chunks(k), chunks(v), chunks(beta)
    G = chunks(g.double()).cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    fade = torch.where(lower, G[..., :, None] - G[..., None, :], -math.inf).exp().float()  # 0 above the diagonal
    kt = k.transpose(-1, -2).contiguous()
    T = _inverse((beta[..., None] * fade * torch.matmul(k, kt)).tril(-1))
    P = fade * torch.matmul(q, kt)
    since, left = G.exp().float()[..., None], (G[..., -1:] - G).exp().float()[..., None]
    whole = G[..., -1].exp().float()[..., None, None]
    kw = (k * left).transpose(-1, -2).contiguous()
    outs = []
    for c in range(n):
        R = beta[:, :, c, :, None] * (v[:, :, c] - since[:, :, c] * torch.matmul(k[:, :, c], S))
        U = torch.matmul(T[:, :, c], R)
        outs.append(since[:, :, c] * torch.matmul(q[:, :, c], S) + torch.matmul(P[:, :, c], U))
        S = whole[:, :, c] * S + torch.matmul(kw[:, :, c], U)
    return torch.cat(outs, 2)[:, :, :N], S


def _unpack(lengths, total, device):
    """Indices that lay packed rows out as [sequences, longest] (rows past a
    sequence's end: any), which of them are rows, and the way back."""
    n = torch.tensor(lengths, device=device)
    t = torch.arange(max(lengths), device=device)
    real = t[None, :] < n[:, None]
    first = n.cumsum(0) - n
    return (first[:, None] + t[None, :]).clamp(max=total - 1), real, real.reshape(-1).nonzero()[:, 0]


def _plain_scan(state, q, k, v, g, beta):
    case = state["case"]
    H, Dk, Dv = case["H"], case["Dk"], case["Dv"]
    q, k, v, g, beta = _heads(q, H), _heads(k, H), v.float(), g, beta
    if not case["packed"]:
        S = state["carry"] if case["carry"] else torch.zeros(case["B"], H, Dk, Dv, device=q.device)
        return _delta(q, k, v, g, beta, S)
    total = case["N"] + case["spare"]
    at, real, back = _unpack(state["lengths"], total, q.device)

    def lay(x):
        x = x[0][:, at].transpose(0, 1)  # [sequences, H, longest, ...]
        return torch.where(real[:, None, :].reshape(len(at), 1, -1, *[1] * (x.dim() - 3)), x, 0.0)

    S = state["carry"] if case["carry"] else torch.zeros(len(at), H, Dk, Dv, device=q.device)
    o, S = _delta(lay(q), lay(k), lay(v), lay(g), lay(beta), S)
    o = o.transpose(1, 2).reshape(-1, H, Dv)[back].transpose(0, 1)[None]
    return torch.cat([o, o.new_zeros(1, H, case["spare"], Dv)], 2), S


def _plain_step(state):
    H = state["case"]["H"]
    q, k, v = _heads(state["q"], H), _heads(state["k"], H), state["v"].float()
    S = state["g"].exp()[..., None, None] * state["state"]
    u = state["beta"][..., None] * (v - (k[..., None] * S).sum(2))
    S = S + k[..., None] * u[:, :, None, :]
    o = (q[..., None] * S).sum(2) * state["case"]["Dk"] ** -0.5
    if state["case"]["in_place"]:
        S = state["state"].copy_(S)
    return o.to(state["v"].dtype), S


def _plain_attn(state):
    case = state["case"]
    H, N = case["H"], case["N"] + case["spare"]
    q, k, v = state["q"].float(), _heads(state["k"], H), _heads(state["v"], H)
    t = torch.arange(N, device=q.device)
    seen = t[:, None] >= t[None, :]
    if case["packed"]:
        seq = (t[:, None] >= state["cu"][None, 1:]).sum(1)  # the sequence of each row
        seen = seen & (seq[:, None] == seq[None, :])
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) * case["Dk"] ** -0.5
    x = torch.where(seen, x, -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp()
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    if case["packed"]:
        o = torch.where((seq < case["packed"])[:, None], o, 0.0)  # rows behind the last sequence
    return o.to(state["q"].dtype)


def _plain(state):
    kind = state["case"]["kind"]
    if kind == "step":
        return _plain_step(state)
    if kind == "attn":
        return _plain_attn(state)
    leaves = [state[x] for x in ("q", "k", "v", "g", "beta")]
    o, S = _plain_scan(state, *leaves)
    o = o.to(state["v"].dtype)
    if kind == "scan":
        return o, S
    grads = torch.autograd.grad(o, leaves, state["do"])
    return {"o": o.detach(), **{"d" + x: t for x, t in zip(("q", "k", "v", "g", "beta"), grads)}}


def run(state):
    if not own:
        return _plain(state)
    import kilat_amd

    case = state["case"]
    if case["kind"] == "step":
        return kilat_amd.gated_delta_step(state["q"], state["k"], state["v"], state["g"], state["beta"], state["state"],
                                          new_state=state["state"] if case["in_place"] else None)
    if case["kind"] == "attn":
        return kilat_amd.causal_attention(state["q"], state["k"], state["v"], cu_seqlens=state.get("cu"))
    leaves = [state[x] for x in ("q", "k", "v", "g", "beta")]
    if case["kind"] == "scan":
        return kilat_amd.gated_delta_scan(*leaves, initial_state=state.get("carry"), return_final_state=True,
                                          cu_seqlens=state.get("cu"))
    o = kilat_amd.gated_delta_scan(*leaves, cu_seqlens=state.get("cu"))
    grads = torch.autograd.grad(o, leaves, state["do"])
    return {"o": o.detach(), **{"d" + x: t for x, t in zip(("q", "k", "v", "g", "beta"), grads)}}


def work(case):
    """Bytes: each input read once and each output written once (a training
    pass is two calls: q, k, v, g and beta in, o out; those and do in, their
    gradients out).  Flops of the scan: the recurrence's own (two products with
    the state and a rank-one update of it per token, 6 Dk Dv and the decay);
    of its backward two and a half times that.  Of attention: two products over
    the pairs that are not masked."""
    es, B, Hk, H, Dk, Dv = SIZES[case["dtype"]], *(case[x] for x in ("B", "Hk", "H", "Dk", "Dv"))
    if case["kind"] == "step":
        return {"bytes": B * (2 * Hk * Dk * es + 2 * H * Dv * es + 8 * H + 8 * H * Dk * Dv), "flops": 7 * B * H * Dk * Dv}
    rows = B * case["N"]
    if case["kind"] == "attn":
        pairs = rows * (case["N"] / max(1, case["packed"]) + 1) / 2
        return {"bytes": rows * (H + Hk) * (Dk + Dv) * es, "flops": pairs * H * 2 * (Dk + Dv)}
    read = rows * (2 * Hk * Dk * es + H * Dv * es + 8 * H)
    if case["kind"] == "train":
        return {"bytes": 3 * read + 2 * rows * H * Dv * es, "flops": 25 * rows * H * Dk * Dv}
    states = (case["packed"] or B) * H * Dk * Dv * 4 * (2 if case["carry"] else 1)
    return {"bytes": read + rows * H * Dv * es + states, "flops": 7 * rows * H * Dk * Dv}


# ---------------------------------------------------------------------------
# In 64 bits, from the definitions
# ---------------------------------------------------------------------------
def _sequences(case, state):
    """(batch entry, first row, rows) of every sequence."""
    if not case["packed"]:
        return [(b, 0, case["N"]) for b in range(case["B"])]
    first, out = 0, []
    for n in state["lengths"]:
        out.append((0, first, n))
        first += n
    return out


def _by_time(case, state, name):
    """A [B, heads, rows, ...] input as [longest, sequences, H, ...] in 64 bits, zero past a sequence's end."""
    x, seqs = state[name].detach().double(), _sequences(case, state)
    if x.shape[1] != case["H"]:
        x = x[:, torch.arange(case["H"], device=x.device) // (case["H"] // x.shape[1])]
    out = x.new_zeros(max(n for _, _, n in seqs), len(seqs), case["H"], *x.shape[3:])
    for s, (b, first, n) in enumerate(seqs):
        out[:n, s] = x[b, :, first:first + n].transpose(0, 1)
    return out


def _by_row(case, state, x, heads):
    """The way back, shared heads' rows added up."""
    out = x.new_zeros(case["B"], heads, case["N"] + case["spare"], *x.shape[3:])
    x = x.reshape(x.shape[0], x.shape[1], heads, case["H"] // heads, *x.shape[3:]).sum(3)
    for s, (b, first, n) in enumerate(_sequences(case, state)):
        out[b, :, first:first + n] = x[:n, s].transpose(0, 1)
    return out


def _exact_scan(case, state):
    q, k, v, g, beta = (_by_time(case, state, x) for x in ("q", "k", "v", "g", "beta"))
    q = q / math.sqrt(case["Dk"])
    a = g.exp()[..., None, None]
    T, train = q.shape[0], case["kind"] == "train"
    S = state["carry"].double() if case["carry"] else q.new_zeros(*q.shape[1:], case["Dv"])
    o, us = torch.empty_like(v), torch.empty_like(v)
    before = torch.empty(T, *S.shape, dtype=S.dtype, device=S.device) if train else None
    for t in range(T):
        if train:
            before[t] = S
        S = a[t] * S  # past a sequence's end g, k and beta are zero: the state stays
        u = beta[t, ..., None] * (v[t] - torch.matmul(k[t, ..., None, :], S)[..., 0, :])
        S = S + k[t, ..., None] * u[..., None, :]
        o[t], us[t] = torch.matmul(q[t, ..., None, :], S)[..., 0, :], u
    if not train:
        return _by_row(case, state, o, case["H"]), S
    do = _by_time(case, state, "do")
    dq, dk, dv, dg, db = (torch.zeros_like(x) for x in (q, k, v, g, beta))
    dS = torch.zeros_like(S)
    for t in range(T - 1, -1, -1):
        kt, qt, u, old = k[t, ..., None], q[t, ..., None], us[t, ..., None], a[t] * before[t]
        new = old + kt * us[t, ..., None, :]
        dq[t] = torch.matmul(new, do[t, ..., None])[..., 0]
        dS = dS + qt * do[t, ..., None, :]
        du = torch.matmul(kt.transpose(-1, -2), dS)[..., 0, :]
        x = torch.matmul(kt.transpose(-1, -2), old)[..., 0, :]
        dx = -beta[t, ..., None] * du
        dv[t] = -dx
        db[t] = (du * (v[t] - x)).sum(-1)
        dk[t] = torch.matmul(dS, u)[..., 0] + torch.matmul(old, dx[..., None])[..., 0]
        dS = dS + kt * dx[..., None, :]
        dg[t] = (dS * old).sum((-1, -2))
        dS = a[t] * dS
    dq = dq / math.sqrt(case["Dk"])
    return {"o": _by_row(case, state, o, case["H"]), "dq": _by_row(case, state, dq, case["Hk"]),
            "dk": _by_row(case, state, dk, case["Hk"]), "dv": _by_row(case, state, dv, case["H"]),
            "dg": _by_row(case, state, dg, case["H"]), "dbeta": _by_row(case, state, db, case["H"])}


def _exact_attn(case, state):
    q, k, v = (state[x].double() for x in ("q", "k", "v"))
    out = q.new_zeros(*q.shape[:3], case["Dv"])
    for b, first, n in _sequences(case, state):
        future = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1)
        for h in range(case["H"]):
            j = h // (case["H"] // case["Hk"])
            rows = slice(first, first + n)
            x = torch.mm(q[b, h, rows], k[b, j, rows].t().contiguous()) / math.sqrt(case["Dk"])
            x = torch.softmax(x.masked_fill_(future, -math.inf), -1)
            out[b, h, rows] = torch.mm(x, v[b, j, rows])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(case, state)
    if case["kind"] != "step":
        return _exact_scan(case, state)
    q, k = (state[x].double().repeat_interleave(case["H"] // case["Hk"], 1) for x in ("q", "k"))
    S = state["g"].double().exp()[..., None, None] * state["state"].double()
    err = state["v"].double() - torch.matmul(k[..., None, :], S)[..., 0, :]
    S = S + k[..., None] * (state["beta"].double()[..., None] * err)[..., None, :]
    return torch.matmul(q[..., None, :], S)[..., 0, :] / math.sqrt(case["Dk"]), S

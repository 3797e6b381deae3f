"""The gated delta rule on packed and served sequences, and the group norm
behind its heads and on channels-last maps.

Kinds (``case["op"]``):
  delta_step    one token for each of S sequences: the matrix states advance in
                their cache (S rows of a larger one, in shuffled order)
  delta_prompt  prompts of different lengths, packed without padding: from zero
                or from the states that an earlier piece left, into the cache
  delta_train   packed sequences, forward and backward, gradients of every
                input, of the initial states and through the final ones
  norm          group norm, channels last, with SiLU or a SiLU gate
  norm_train    the same, forward and backward

q and k are unit normal and normalised by the operator, as behind a conv; the
decays are exp(-A dt) with A in [1, 16] and dt log-uniform in [1e-3, 1e-1], the
writing strengths sigmoids of normals.  Sequence lengths are a random cut of the
packed tokens; where there are several, one sequence has a single token and, of
four or more, one has none.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
CHUNK = 64
L2_EPS = 1e-6
EPS = 1e-5


def listed():
    return [
        # one user's next token in a d_model = 768 layer of 12 heads: nothing but latency
        {"name": "delta_step_one", "op": "delta_step", "dtype": "bfloat16", "S": 1, "HK": 12, "HV": 12, "DK": 128, "DV": 128},
        # a serving batch, odd heads, keys shared by two value heads
        {"name": "delta_step_odd", "op": "delta_step", "dtype": "float32", "S": 33, "HK": 5, "HV": 10, "DK": 40, "DV": 100},
        # a full decode batch: the states are all the traffic
        {"name": "delta_step_full", "op": "delta_step", "dtype": "bfloat16", "S": 512, "HK": 12, "HV": 12, "DK": 128, "DV": 128},
        # two short prompts: the latency of the first token
        {"name": "delta_prompt_short", "op": "delta_prompt", "dtype": "float32", "S": 2, "T": 392, "HK": 12, "HV": 12, "DK": 64, "DV": 64},
        # a step of a scheduler that packs prompts, and pieces of long ones, of many users
        {"name": "delta_prompt_ragged", "op": "delta_prompt", "dtype": "bfloat16", "S": 23, "T": 8191, "HK": 12, "HV": 12, "DK": 128, "DV": 128},
        # one long document
        {"name": "delta_prompt_long", "op": "delta_prompt", "dtype": "bfloat16", "S": 1, "T": 32768, "HK": 12, "HV": 12, "DK": 128, "DV": 128},
        # odd sizes throughout, keys shared
        {"name": "delta_train_odd", "op": "delta_train", "dtype": "float32", "S": 5, "T": 3111, "HK": 5, "HV": 10, "DK": 40, "DV": 100},
        # a training batch of packed documents
        {"name": "delta_train_packed", "op": "delta_train", "dtype": "bfloat16", "S": 8, "T": 16384, "HK": 12, "HV": 12, "DK": 128, "DV": 128},
        # the heads' norm and gate behind a serving batch's step
        {"name": "norm_heads_step", "op": "norm", "dtype": "bfloat16", "N": 64, "P": 1, "G": 12, "C": 1536, "gate": True},
        # the same in the training batch above
        {"name": "norm_heads_train", "op": "norm_train", "dtype": "bfloat16", "N": 16384, "P": 1, "G": 12, "C": 1536, "gate": True},
        # 14 x 14 patch maps of 32 images, 384 channels
        {"name": "norm_patches_train", "op": "norm_train", "dtype": "float32", "N": 32, "P": 196, "G": 32, "C": 384, "gate": False},
        # a few large maps (224 x 224, 128 channels): one pass for the sums, one for the values
        {"name": "norm_large_map", "op": "norm", "dtype": "bfloat16", "N": 4, "P": 50176, "G": 32, "C": 128, "gate": False},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta_step", "delta_prompt", "delta_train", "norm", "norm_train"])
    case = {"op": op, "dtype": rng.choice(["float32", "bfloat16"])}
    if op.startswith("norm"):
        case["G"] = rng.choice([1, 4, 8, 12, 32])
        case["C"] = case["G"] * _spread(rng, 2, 1536 // case["G"])
        case["P"] = 1 if rng.random() < 0.5 else _spread(rng, 2, 4096)
        case["N"] = _spread(rng, 1, max(1, min(16384, 12_000_000 // (case["P"] * case["C"]))))
        case["gate"] = rng.random() < 0.5
        return case
    whole = rng.random() < 0.5  # half of them whole multiples of 32, as models have them
    for name in ("DK", "DV"):
        d = _spread(rng, 16, 128)
        case[name] = (d + 31) // 32 * 32 if whole else d
    case["HK"] = rng.randint(1, 6)
    case["HV"] = case["HK"] * rng.choice([1, 1, 2])
    if op == "delta_step":
        case["S"] = _spread(rng, 1, 500)
    else:
        case["T"] = _spread(rng, 64, 12000)
        case["S"] = _spread(rng, 1, max(2, min(64, case["T"] // 16)))
    return case


def _lengths(case, gen):
    """A random cut of T tokens into S sequences."""
    T, S = case["T"], case["S"]
    if S == 1:
        return [T]
    fixed = [1] if S < 4 else [1, 0]
    left, n = T - sum(fixed), S - len(fixed)
    share = torch.rand(n, generator=gen, dtype=torch.float64) + 0.1
    cut = [0] + (torch.cumsum(share, 0) / share.sum() * left).round().long().tolist()
    cut[-1] = left
    lens = [b - a for a, b in zip(cut, cut[1:])] + fixed
    order = torch.randperm(S, generator=gen).tolist()
    return [lens[i] for i in order]


LEAVES = {"delta_train": ("q", "k", "v", "g", "beta", "initial"), "norm_train": ("x", "weight", "bias", "z")}


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt, op = TYPES[case["dtype"]], case["op"]

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEV).to(dtype)

    st = {"op": op}
    if op.startswith("norm"):
        shape = (case["N"], case["C"]) if case["P"] == 1 else (case["N"], case["P"], case["C"])
        st["groups"] = case["G"]
        # channels of different means and widths, as behind a conv or a product
        st["x"] = (rand(*shape) * (1 + 0.2 * rand(case["C"])) + 0.5 * rand(case["C"])).to(dt)
        st["weight"], st["bias"] = 1 + 0.1 * rand(case["C"]), 0.1 * rand(case["C"])
        st["z"] = rand(*shape, dtype=dt) if case["gate"] else None
        if op == "norm_train":
            st["dy"] = rand(*shape, dtype=dt)
            for k in LEAVES[op]:
                if st[k] is not None:
                    st[k].requires_grad_(True)
        return st
    S, HK, HV, DK, DV = (case[k] for k in ("S", "HK", "HV", "DK", "DV"))
    T = S if op == "delta_step" else case["T"]
    st["q"], st["k"], st["v"] = rand(T, HK, DK, dtype=dt), rand(T, HK, DK, dtype=dt), rand(T, HV, DV, dtype=dt)
    A = 1 + 15 * torch.rand(HV, generator=gen, device=DEV)
    step = torch.exp(math.log(1e-3) + math.log(100.0) * torch.rand(T, HV, generator=gen, device=DEV))
    st["g"], st["beta"] = -A * step, torch.sigmoid(rand(T, HV)).to(dt)
    if op == "delta_train":
        st["initial"] = rand(S, HV, DK, DV)
        st["do"], st["dfinal"] = rand(T, HV, DV, dtype=dt), rand(S, HV, DK, DV)
        for k in LEAVES[op]:
            st[k].requires_grad_(True)
    else:  # a cache of a few more rows than there are sequences
        M = S + max(3, S // 16)
        st["states"] = rand(M, HV, DK, DV)
        st["slots"] = torch.randperm(M, generator=host)[:S].int().to(DEV)
    if op != "delta_step":
        lens = _lengths(case, host)
        st["max_len"] = max(lens)
        st["offsets"] = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
        if op == "delta_prompt":  # every other prompt is at its first piece
            st["fresh"] = (torch.arange(S) % 2 == 0).to(DEV)
    return st


# ------------------------------------------------------------ plain forms

def _unit(x):
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + L2_EPS)


def _chunks(offsets, T):
    """Of packed sequences cut into chunks: each chunk's sequence, whether it is its first, the chunk's
    tokens (clamped) and which of them are there; each sequence's last chunk, and which sequences are empty."""
    off = offsets.long()
    lens = off[1:] - off[:-1]
    upto = torch.cumsum((lens + CHUNK - 1) // CHUNK, 0)
    S = lens.shape[0]
    c = torch.arange(T // CHUNK + S, device=off.device)
    seq = (c[:, None] >= upto[None, :]).sum(1)
    there = seq < S
    seq = seq.clamp(max=S - 1)
    nth = c - (upto[seq] - (lens[seq] + CHUNK - 1) // CHUNK)
    pos = nth[:, None] * CHUNK + torch.arange(CHUNK, device=off.device)
    valid = there[:, None] & (pos < lens[seq][:, None])
    return seq, there & (nth == 0), (off[seq][:, None] + pos).clamp(max=T - 1), valid, (upto - 1).clamp(min=0), lens == 0


def _inverse(A):
    """(I + A)^-1 of strictly lower triangles, by blocks of doubled size."""
    n = A.shape[-1]
    i = torch.arange(n, device=A.device)
    inv, b = torch.eye(n, device=A.device).expand_as(A), 1
    while b < n:
        low = (i[:, None] // (2 * b) == i[None, :] // (2 * b)) & (i[:, None] // b > i[None, :] // b)
        inv = inv - inv @ torch.where(low, A, 0.0) @ inv
        b *= 2
    return inv


def _delta_chunks(q, k, v, g, beta, h0, offsets):
    """o (T, HV, DV) and the final states, in 32 bits: products within the chunks, and the chunks' states by doubling spans."""
    T, HV, DV = v.shape
    r, scale = HV // q.shape[1], q.shape[-1] ** -0.5
    seq, first, tok, valid, last, empty = _chunks(offsets, T)
    there = valid[:, :, None, None]

    def rows(x):  # (chunks, heads, CHUNK, columns)
        return torch.where(there, x[tok], 0.0).transpose(1, 2)

    Q, K = (rows(_unit(x.float())).repeat_interleave(r, 1) for x in (q, k))
    V = rows(v.float())
    G = torch.cumsum(rows(g.float()[..., None])[..., 0].double(), -1)
    beta = rows(beta.float()[..., None])
    i = torch.arange(CHUNK, device=Q.device)
    lower = i[:, None] >= i[None, :]
    L = torch.exp(torch.where(lower, G[..., :, None] - G[..., None, :], 0.0)).float() * lower
    eG, eR, eC = (torch.exp(x).float()[..., None] for x in (G, G[..., -1:] - G, G[..., -1:]))
    Kt = K.transpose(-1, -2)
    inv = _inverse(beta * (K @ Kt) * L * (i[:, None] > i[None, :]))
    U, W = inv @ (beta * V), inv @ (beta * eG * K)
    Kr = (eR * K).transpose(-1, -2)
    E, M = Kr @ U, eC * torch.eye(Kt.shape[-2], device=Q.device) - Kr @ W
    # S[c] = M[c] S[c - 1] + E[c]; a sequence's first chunk starts from its initial state
    begin = first[:, None, None, None]
    start = h0[seq]
    E, M, n = E + torch.where(begin, M @ start, 0.0), torch.where(begin, 0.0, M), 1
    while n < E.shape[0]:
        E, M = torch.cat([E[:n], E[n:] + M[n:] @ E[:-n]]), torch.cat([M[:n], M[n:] @ M[:-n]])
        n *= 2
    before = torch.where(begin, start, torch.cat([E[:1], E[:-1]]))
    new = U - W @ before
    O = scale * (eG * (Q @ before) + ((Q @ Kt) * L) @ new)
    o = torch.zeros(T + 1, HV, DV, device=O.device).index_copy(
        0, torch.where(valid, tok, T).flatten(), O.transpose(1, 2).reshape(-1, HV, DV))[:T]
    return o, torch.where(empty[:, None, None, None], h0, E[last])


def _delta_prompt(st):
    slots = st["slots"].long()
    h0 = torch.where(st["fresh"][:, None, None, None], 0.0, st["states"][slots])
    o, final = _delta_chunks(st["q"], st["k"], st["v"], st["g"], st["beta"], h0, st["offsets"])
    st["states"][slots] = final
    return {"o": o.to(st["v"].dtype), "states": st["states"]}


def _delta_train(st):
    leaves = {k: st[k].detach().float().requires_grad_(True) for k in LEAVES["delta_train"]}
    o, final = _delta_chunks(*leaves.values(), st["offsets"])
    grads = torch.autograd.grad([o, final], list(leaves.values()), [st["do"].float(), st["dfinal"]])
    out = {"o": o.detach().to(st["v"].dtype), "final": final.detach()}
    out.update({"d" + k: g.to(st[k].dtype) for k, g in zip(leaves, grads)})
    return out


def _delta_step(st):
    slots = st["slots"].long()
    r, scale = st["v"].shape[1] // st["q"].shape[1], st["q"].shape[-1] ** -0.5
    q, k = (_unit(st[n].float()).repeat_interleave(r, 1) for n in ("q", "k"))
    h = torch.exp(st["g"])[:, :, None, None] * st["states"][slots]
    d = st["beta"].float()[..., None] * (st["v"].float() - (k[..., None] * h).sum(-2))
    h = h + k[..., None] * d[..., None, :]
    st["states"][slots] = h
    return {"o": (scale * (q[..., None] * h).sum(-2)).to(st["v"].dtype), "states": st["states"]}


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _norm_values(st):
    """Everything of the norm that its output and gradients need, in 32 bits."""
    x = st["x"].detach().float()
    f = {"shape": x.shape, "x": x.reshape(x.shape[0], -1, st["groups"], x.shape[-1] // st["groups"])}
    w, b = (st[k].detach().reshape(st["groups"], -1) for k in ("weight", "bias"))
    mean = f["x"].mean((1, 3), keepdim=True)
    f["c"] = f["x"] - mean
    f["rstd"] = 1 / torch.sqrt((f["c"] * f["c"]).mean((1, 3), keepdim=True) + EPS)
    f["xh"], f["w"] = f["c"] * f["rstd"], w
    f["n"] = f["xh"] * w + b
    if st["z"] is None:
        f["sn"] = _sigmoid(f["n"])
        f["y"] = f["n"] * f["sn"]
    else:
        f["z"] = st["z"].detach().float().reshape(f["x"].shape)
        f["sz"] = _sigmoid(f["z"])
        f["y"] = f["n"] * f["z"] * f["sz"]
    return f


def _norm(st):
    f = _norm_values(st)
    return {"y": f["y"].reshape(f["shape"]).to(st["x"].dtype)}


def _norm_train(st):
    f = _norm_values(st)
    dy = st["dy"].float().reshape(f["x"].shape)
    out = {"y": f["y"].reshape(f["shape"]).to(st["x"].dtype)}
    if st["z"] is None:
        dn = dy * f["sn"] * (1 + f["n"] * (1 - f["sn"]))
    else:
        dn = dy * f["z"] * f["sz"]
        dz = dy * f["n"] * f["sz"] * (1 + f["z"] * (1 - f["sz"]))
        out["dz"] = dz.reshape(f["shape"]).to(st["z"].dtype)
    h = dn * f["w"]
    dx = f["rstd"] * (h - h.mean((1, 3), keepdim=True) - f["xh"] * (h * f["xh"]).mean((1, 3), keepdim=True))
    out["dx"] = dx.reshape(f["shape"]).to(st["x"].dtype)
    out["dweight"], out["dbias"] = (dn * f["xh"]).sum((0, 1)).flatten(), dn.sum((0, 1)).flatten()
    return out


PLAIN = {"delta_step": _delta_step, "delta_prompt": _delta_prompt, "delta_train": _delta_train, "norm": _norm,
         "norm_train": _norm_train}


# ------------------------------------------------- the framework's operators

def _call(st):
    import mlx_vision_mamba_amd as mvm
    op = st["op"]
    if op.startswith("norm"):
        y = mvm.group_norm(st["x"], st["groups"], st["weight"], st["bias"], eps=EPS,
                           activation="silu" if st["z"] is None else None, z=st["z"])
        if op == "norm":
            return {"y": y}
        leaves = [k for k in LEAVES[op] if st[k] is not None]
        grads = torch.autograd.grad(y, [st[k] for k in leaves], st["dy"])
        return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}
    args = st["q"], st["k"], st["v"], st["g"], st["beta"]
    if op == "delta_step":
        o = mvm.gated_delta_rule_step(*args, st["states"], slots=st["slots"], qk_l2norm=True)
        return {"o": o, "states": st["states"]}
    if op == "delta_prompt":
        o = mvm.gated_delta_rule_prefill(*args, st["states"], st["offsets"], slots=st["slots"], fresh=st["fresh"],
                                         qk_l2norm=True, max_len=st["max_len"])
        return {"o": o, "states": st["states"]}
    o, final = mvm.gated_delta_rule_packed(*args, st["offsets"], initial_states=st["initial"], qk_l2norm=True,
                                           max_len=st["max_len"])
    leaves = LEAVES[op]
    grads = torch.autograd.grad([o, final], [st[k] for k in leaves], [st["do"], st["dfinal"]])
    return {"o": o.detach(), "final": final.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}


def run(state):
    return _call(state) if own else PLAIN[state["op"]](state)


# -------------------------------------------------------------------- work

def work(case):
    e, op = TYPES[case["dtype"]].itemsize, case["op"]
    if op.startswith("norm"):
        n, C = case["N"] * case["P"] * case["C"], case["C"]
        gate = 1 if case["gate"] else 0
        nbytes, flops = n * e * (2 + gate) + 8 * C, 15 * n
        if op == "norm_train":  # dy read, dx and dz written; the parameters' gradients
            nbytes += n * e * (2 + gate) + 8 * C
            flops += 30 * n
        return {"bytes": nbytes, "flops": flops}
    S, HK, HV, DK, DV = (case[k] for k in ("S", "HK", "HV", "DK", "DV"))
    T = S if op == "delta_step" else case["T"]
    acts = T * e * 2 * (HK * DK + HV * DV) + T * HV * (4 + e)  # q, k, v and o; g and beta
    states = 2 * S * HV * DK * DV * 4
    flops = T * HV * 6 * DK * DV  # S^T k, the outer product, S^T q
    if op == "delta_train":
        return {"bytes": 2 * (acts + states), "flops": 3 * flops}
    return {"bytes": acts + states, "flops": flops}


# ------------------------------------------------------ the values in 64 bits

SPAN = 128  # tokens of the backward whose states are held at once


def _exact_delta(st):
    """Token by token, all sequences side by side; gradients by the recurrence's adjoint."""
    op = st["op"]
    train = op == "delta_train"
    x = {k: st[k].detach().double() for k in ("q", "k", "v", "g", "beta")}
    r, scale = x["v"].shape[1] // x["q"].shape[1], x["q"].shape[-1] ** -0.5
    norm = {n: (x[n].square().sum(-1, keepdim=True) + L2_EPS).rsqrt() for n in ("q", "k")}
    S = st["initial"].shape[0] if train else st["slots"].shape[0]
    T, HV, DV = x["v"].shape
    off = torch.arange(S + 1, device=DEV) if op == "delta_step" else st["offsets"].long()
    lens = off[1:] - off[:-1]
    longest = int(lens.max())
    pos = torch.arange(longest, device=DEV)[:, None]
    tok = torch.where(pos < lens, off[:-1] + pos, T)  # (longest, S); T: none

    def rows(t):  # (longest, S, heads, ...), zeros where there is no token
        return torch.cat([t, torch.zeros_like(t[:1])])[tok]

    q, k = (rows(x[n] * norm[n]).repeat_interleave(r, 2) for n in ("q", "k"))
    v, a, beta = rows(x["v"]), rows(x["g"]).exp(), rows(x["beta"])
    if train:
        h0 = st["initial"].detach().double()
    else:
        h0 = st["states"][st["slots"].long()].double()
        if "fresh" in st:
            h0[st["fresh"]] = 0

    def advance(h, t):
        p = a[t][:, :, None, None] * h
        d = beta[t][..., None] * (v[t] - torch.matmul(k[t][..., None, :], p)[..., 0, :])
        return p, d, torch.addcmul(p, k[t][..., None], d[..., None, :])

    h, o, marks = h0, torch.empty_like(v), []
    for t in range(longest):
        if t % SPAN == 0:
            marks.append(h)
        h = advance(h, t)[2]
        o[t] = scale * torch.matmul(q[t][..., None, :], h)[..., 0, :]

    def packed(t):
        got = torch.zeros(T + 1, *t.shape[2:], dtype=t.dtype, device=DEV)
        got[tok.flatten()] = t.flatten(0, 1)
        return got[:T]

    if not train:
        states = st["states"].double()
        states[st["slots"].long()] = h
        return {"o": packed(o), "states": states}
    out = {"o": packed(o), "final": h}
    do, D = rows(st["do"].double()) * scale, st["dfinal"].double()
    dq, dk, dv, dg, db = (torch.zeros_like(t) for t in (q, k, v, a, beta))
    for m in reversed(range(len(marks))):
        hs = [marks[m]]
        ts = range(m * SPAN, min(longest, (m + 1) * SPAN))
        for t in ts:
            hs.append(advance(hs[-1], t)[2])
        for t in reversed(ts):
            p, d, _ = advance(hs[t - m * SPAN], t)
            live = (tok[t] < T)[:, None, None, None]
            now = hs[t - m * SPAN + 1]
            dq[t] = torch.matmul(now, do[t][..., None])[..., 0]
            Dt = D + q[t][..., None] * do[t][..., None, :]
            dd = torch.matmul(k[t][..., None, :], Dt)[..., 0, :]
            dk[t] = torch.matmul(Dt, d[..., None])[..., 0] - beta[t][..., None] * torch.matmul(p, dd[..., None])[..., 0]
            dv[t] = beta[t][..., None] * dd
            db[t] = (dd * (v[t] - torch.matmul(k[t][..., None, :], p)[..., 0, :])).sum(-1)
            dp = Dt - k[t][..., None] * dv[t][..., None, :]
            dg[t] = (dp * p).sum((-1, -2))
            D = torch.where(live, a[t][:, :, None, None] * dp, D)
    grads = {"v": packed(dv), "g": packed(dg), "beta": packed(db), "initial": D}
    for n, d in (("q", dq), ("k", dk)):
        d = packed(d).reshape(T, HV // r, r, -1).sum(2)
        unit = x[n] * norm[n]
        grads[n] = norm[n] * (d - unit * (unit * d).sum(-1, keepdim=True))
    out.update({"d" + n: grads[n] for n in LEAVES[op]})
    return out


def _exact_norm(st):
    """By autograd in 64 bits, groups as rows."""
    leaves = {k: st[k].detach().double().requires_grad_(True) for k in LEAVES["norm_train"] if st[k] is not None}
    x = leaves["x"]
    shape, C, G = x.shape, x.shape[-1], st["groups"]
    rows = x.reshape(shape[0], -1, G, C // G).transpose(1, 2).flatten(2)  # (N, G, values)
    var, mean = torch.var_mean(rows, -1, correction=0, keepdim=True)
    n = ((rows - mean) * (var + EPS).rsqrt()).reshape(shape[0], G, -1, C // G).transpose(1, 2).reshape(shape)
    n = n * leaves["weight"] + leaves["bias"]
    gate = leaves["z"] if "z" in leaves else n
    y = gate * torch.sigmoid(gate) * (n if "z" in leaves else 1)
    if st["op"] == "norm":
        return {"y": y.detach()}
    grads = torch.autograd.grad(y, list(leaves.values()), st["dy"].double())
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_norm(state) if case["op"].startswith("norm") else _exact_delta(state)

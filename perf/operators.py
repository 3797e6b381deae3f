"""Packed and served sequences through the Mamba block's recurrent operators.

Kinds (``case["op"]``):
  scan_step    one token for each of S sequences: the scan's states advance in
               their cache (S rows of a larger one, in shuffled order)
  conv_step    the same for the causal conv's window of earlier inputs
  scan_prompt  prompts of different lengths, packed without padding, through
               the scan: from zero or from the states that an earlier piece of
               the prompt left, the new states written to the cache
  conv_prompt  the same for the conv
  scan_train   packed sequences, forward and backward, gradients of every
               input, of the initial states and through the final ones
  conv_train   the same for the conv

Inputs follow the distributions of ``mlx_vision_mamba_amd.synthetic``: unit
normal activations, dt log-normal in about [1e-3, 1e-1] behind its softplus,
S4D-real A.  Sequence lengths are a random cut of the packed tokens; where
there are several, one sequence has a single token and, of four or more, one
has none.
"""

import math

import torch

own = False

DEV = "cuda"
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one user's next token: nothing but latency
        {"name": "scan_step_one", "op": "scan_step", "dtype": "float32", "S": 1, "D": 1536, "N": 16},
        # a serving batch of a d_model = 768 block
        {"name": "scan_step_batch", "op": "scan_step", "dtype": "bfloat16", "S": 64, "D": 1536, "N": 16},
        # a full decode batch: the states are all the traffic
        {"name": "scan_step_full", "op": "scan_step", "dtype": "bfloat16", "S": 1024, "D": 1536, "N": 16},
        # the conv before the first and the last of these
        {"name": "conv_step_one", "op": "conv_step", "dtype": "bfloat16", "S": 1, "D": 1536, "W": 4},
        {"name": "conv_step_full", "op": "conv_step", "dtype": "bfloat16", "S": 1024, "D": 1536, "W": 4},
        # a step of a scheduler that packs prompts, and pieces of long ones, of many users
        {"name": "conv_prompt_ragged", "op": "conv_prompt", "dtype": "bfloat16", "S": 23, "T": 8191, "D": 1536, "W": 4},
        # 32 sequences of 196 tokens on average, trained: a d_model = 384 block
        {"name": "conv_train_packed", "op": "conv_train", "dtype": "float32", "S": 32, "T": 6272, "D": 768, "W": 4},
        # two short prompts: the latency of the first token
        {"name": "scan_prompt_short", "op": "scan_prompt", "dtype": "float32", "S": 2, "T": 392, "D": 1536, "N": 16},
        {"name": "scan_prompt_ragged", "op": "scan_prompt", "dtype": "bfloat16", "S": 23, "T": 8191, "D": 1536, "N": 16},
        # one long document
        {"name": "scan_prompt_long", "op": "scan_prompt", "dtype": "bfloat16", "S": 1, "T": 32768, "D": 1536, "N": 16},
        # odd sizes throughout
        {"name": "scan_train_odd", "op": "scan_train", "dtype": "float32", "S": 5, "T": 3111, "D": 1000, "N": 16},
        # a training batch of packed documents
        {"name": "scan_train_packed", "op": "scan_train", "dtype": "bfloat16", "S": 8, "T": 16384, "D": 1536, "N": 16},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan_step", "conv_step", "scan_prompt", "conv_prompt", "scan_train", "conv_train"])
    case = {"op": op, "dtype": rng.choice(["float32", "bfloat16"]), "D": _spread(rng, 96, 1536)}
    if rng.random() < 0.5:  # half of them whole multiples of 32, as models have them
        case["D"] = (case["D"] + 31) // 32 * 32
    if op.startswith("scan"):
        case["N"] = rng.choice([16, 16, 16, 8, 4, 13])
    else:
        case["W"] = rng.choice([4, 4, 4, 3, 2])
    if op.endswith("step"):
        case["S"] = _spread(rng, 1, 1000)
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


def prepare(case, seed):
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt, D, S, op = TYPES[case["dtype"]], case["D"], case["S"], case["op"]

    def rand(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=DEV).to(dtype)

    st = {"op": op}
    rows = S if op.endswith("step") else case["T"]
    if op.startswith("scan"):
        N = case["N"]
        st["u"], st["z"] = rand(rows, D, dtype=dt), rand(rows, D, dtype=dt)
        st["delta"] = (0.5 * rand(rows, D)).to(dt)  # before its bias and the softplus
        st["B"], st["C"] = rand(rows, N, dtype=dt), rand(rows, N, dtype=dt)
        st["A_log"] = torch.log(torch.arange(1, N + 1, dtype=torch.float32, device=DEV)).repeat(D, 1)
        st["D"] = torch.ones(D, device=DEV)
        st["delta_bias"] = 0.3 * rand(D) - 4.6
        state = (D, N)
        state_type = torch.float32
    else:
        W = case["W"]
        st["x"] = rand(rows, D, dtype=dt)
        st["weight"], st["bias"] = rand(D, W) / W ** 0.5, 0.1 * rand(D)
        state = (W - 1, D)
        state_type = dt
    if op.endswith("train"):
        st["initial"] = rand(S, *state, dtype=state_type)
        st["dy"], st["dfinal"] = rand(rows, D, dtype=dt), rand(S, *state, dtype=state_type)
        for k in LEAVES[op]:
            st[k].requires_grad_(True)
    else:  # a cache of a few more rows than there are sequences
        M = S + max(3, S // 16)
        st["states"] = rand(M, *state, dtype=state_type)
        st["slots"] = torch.randperm(M, generator=host)[:S].int().to(DEV)
    if not op.endswith("step"):
        lens = _lengths(case, host)
        st["max_len"] = max(lens)
        st["offsets"] = torch.tensor([0] + lens).cumsum(0).int().to(DEV)
        if op.endswith("prompt"):  # every other prompt is at its first piece
            st["fresh"] = (torch.arange(S) % 2 == 0).to(DEV)
    return st


LEAVES = {"scan_train": ("u", "delta", "A_log", "B", "C", "D", "z", "delta_bias", "initial"),
          "conv_train": ("x", "weight", "bias", "initial")}


# ------------------------------------------------------------ plain forms

def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _recur(a, b):
    """h of h[t] = a[t] h[t-1] + b[t], h[-1] = 0, over the first axis, by doubling spans."""
    a, k = a.clone(), 1
    h = b.clone()
    while k < a.shape[0]:
        h[k:] = h[k:] + a[k:] * h[:-k]
        a[k:] = a[k:] * a[:-k]
        k *= 2
    return h


def _bounds(offsets, T):
    """Of packed sequences: each token's sequence, the first and last tokens (clamped, for the empty ones), which are empty."""
    off = offsets.long()
    tok = torch.arange(T, device=off.device)
    seq = (tok[:, None] >= off[None, 1:]).sum(1)
    return seq, off[:-1].clamp(max=T - 1), (off[1:] - 1).clamp(min=0), off[1:] == off[:-1]


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _scan_forward(st, h0):
    """Everything of the packed scan that its outputs and gradients need, in 32 bits."""
    f = {k: st[k].detach().float() for k in ("u", "delta", "B", "C", "z", "A_log", "D", "delta_bias")}
    T = f["u"].shape[0]
    f["A"] = -torch.exp(f["A_log"])
    f["raw"] = f["delta"] + f["delta_bias"]
    f["dl"] = _softplus(f["raw"])
    seq, first, last, empty = _bounds(st["offsets"], T)
    a = torch.exp(f["dl"][:, :, None] * f["A"])
    b = (f["dl"] * f["u"])[:, :, None] * f["B"][:, None, :]
    begin = (torch.arange(T, device=a.device) == first[seq])[:, None, None]
    start = h0[seq]                         # the state before a first token
    b = b + torch.where(begin, a * start, 0.0)
    f["h"] = _recur(torch.where(begin, 0.0, a), b)
    f["r"] = (f["h"] * f["C"][:, None, :]).sum(-1) + f["D"] * f["u"]
    f["sz"] = _sigmoid(f["z"])
    f["y"] = f["r"] * f["z"] * f["sz"]
    f["final"] = torch.where(empty[:, None, None], h0, f["h"][last])
    f.update(a=a, begin=begin, start=start, seq=seq, first=first, last=last, empty=empty)
    return f


def _scan_prompt(st):
    slots = st["slots"].long()
    h0 = torch.where(st["fresh"][:, None, None], 0.0, st["states"][slots])
    f = _scan_forward(st, h0)
    st["states"][slots] = f["final"]
    return {"y": f["y"].to(st["u"].dtype), "states": st["states"]}


def _scan_train(st):
    f = _scan_forward(st, st["initial"].detach())
    T, begin, empty = f["u"].shape[0], f["begin"], f["empty"]
    dy = st["dy"].float()
    silu = f["z"] * f["sz"]
    dr = dy * silu
    dz = dy * f["r"] * f["sz"] * (1 + f["z"] * (1 - f["sz"]))
    # the adjoint runs backwards: its factor at t is the decay of t + 1
    inject = dr[:, :, None] * f["C"][:, None, :]
    ends = (torch.arange(T, device=dr.device) == f["last"][f["seq"]])[:, None, None]
    inject = inject + torch.where(ends, st["dfinal"][f["seq"]], 0.0)
    after = torch.cat([f["a"][1:], f["a"][:1]])
    g = _recur(torch.where(ends, 0.0, after).flip(0), inject.flip(0)).flip(0)
    del inject, after
    before = torch.where(begin, f["start"], torch.cat([f["h"][:1], f["h"][:-1]]))
    ah = f["a"] * before
    gah = g * ah
    gB = (g * f["B"][:, None, :]).sum(-1)
    dA = (gah * f["dl"][:, :, None]).sum(0)
    ddl = (gah * f["A"]).sum(-1) + gB * f["u"]
    draw_ = ddl * _sigmoid(f["raw"])
    dh0 = torch.where(empty[:, None, None], st["dfinal"], (f["a"] * g)[f["first"]])
    grads = {"u": gB * f["dl"] + f["D"] * dr, "delta": draw_, "A_log": dA * f["A"],
             "B": (g * (f["dl"] * f["u"])[:, :, None]).sum(1), "C": (f["h"] * dr[:, :, None]).sum(1),
             "D": (dr * f["u"]).sum(0), "z": dz, "delta_bias": draw_.sum(0), "initial": dh0}
    out = {"y": f["y"].to(st["u"].dtype), "final": f["final"]}
    out.update({"d" + k: v.to(st[k].dtype) for k, v in grads.items()})
    return out


def _scan_step(st):
    slots = st["slots"].long()
    u, z, Bm, Cm = (st[k].float() for k in ("u", "z", "B", "C"))
    dl = _softplus(st["delta"].float() + st["delta_bias"])
    A = -torch.exp(st["A_log"])
    h = torch.exp(dl[:, :, None] * A) * st["states"][slots] + (dl * u)[:, :, None] * Bm[:, None, :]
    st["states"][slots] = h
    r = (h * Cm[:, None, :]).sum(-1) + st["D"] * u
    return {"y": (r * z * _sigmoid(z)).to(st["u"].dtype), "states": st["states"]}


def _conv_window(st, c0):
    """x~ of every (token, tap): the inputs W - 1 back to this one, earlier sequences' replaced by the states."""
    x = st["x"].detach().float()
    T, W = x.shape[0], st["weight"].shape[1]
    seq, first, last, empty = _bounds(st["offsets"], T)
    tok = torch.arange(T, device=x.device)
    taps = []
    for j in range(W):
        at = tok - (W - 1) + j
        pos = at - first[seq]             # < 0: row W - 1 + pos of the state
        tap = x[at.clamp(min=0)]
        if j < W - 1:
            tap = torch.where((pos < 0)[:, None], c0[seq, (W - 1 + pos).clamp(0, W - 2)], tap)
        taps.append(tap)
    return torch.stack(taps, 1)


def _conv_final(st, c0):
    """The last W - 1 inputs of each sequence, its initial state's rows where it has fewer."""
    x, W, off = st["x"].detach(), st["weight"].shape[1], st["offsets"].long()
    rows = torch.arange(W - 1, device=x.device)
    n = (off[1:] - off[:-1])[:, None]
    pos = n - (W - 1) + rows              # < 0: row W - 1 + pos of the old state
    old = torch.gather(c0, 1, (W - 1 + pos).clamp(0, W - 2)[:, :, None].expand_as(c0))
    return torch.where((pos < 0)[:, :, None], old, x[(off[:-1, None] + pos).clamp(0, x.shape[0] - 1)])


def _conv_prompt(st):
    slots = st["slots"].long()
    c0 = torch.where(st["fresh"][:, None, None], 0.0, st["states"][slots].float())
    pre = (_conv_window(st, c0) * st["weight"].t()).sum(1) + st["bias"]
    st["states"][slots] = _conv_final(st, c0.to(st["x"].dtype))
    return {"y": (pre * _sigmoid(pre)).to(st["x"].dtype), "states": st["states"]}


def _conv_train(st):
    c0 = st["initial"].detach().float()
    w, T, S, W = st["weight"].detach(), st["x"].shape[0], c0.shape[0], st["weight"].shape[1]
    win = _conv_window(st, c0)
    pre = (win * w.t()).sum(1) + st["bias"].detach()
    s = _sigmoid(pre)
    dpre = st["dy"].float() * s * (1 + pre * (1 - s))
    seq, first, _, _ = _bounds(st["offsets"], T)
    tok = torch.arange(T, device=dpre.device)
    # x~ laid out as the states' rows, then the tokens'
    dall = torch.zeros(S * (W - 1) + T, dpre.shape[1], device=dpre.device)
    for j in range(W):
        pos = tok - (W - 1) + j - first[seq]
        to = torch.where(pos < 0, seq * (W - 1) + W - 1 + pos, S * (W - 1) + tok - (W - 1) + j)
        dall[to] = dall[to] + dpre * w[:, j]  # each tap's rows are different ones
    off = st["offsets"].long()
    for r in range(W - 1):
        pos = (off[1:] - off[:-1]) - (W - 1) + r
        n = torch.arange(S, device=dpre.device)
        to = torch.where(pos < 0, n * (W - 1) + W - 1 + pos, S * (W - 1) + off[:-1] + pos)
        dall[to] = dall[to] + st["dfinal"][:, r].float()
    grads = {"x": dall[S * (W - 1):], "weight": (win * dpre[:, None]).sum(0).t(), "bias": dpre.sum(0),
             "initial": dall[:S * (W - 1)].reshape(c0.shape)}
    out = {"y": (pre * s).to(st["x"].dtype), "final": _conv_final(st, st["initial"].detach())}
    out.update({"d" + k: v.to(st[k].dtype) for k, v in grads.items()})
    return out


def _conv_step(st):
    slots = st["slots"].long()
    win = torch.cat([st["states"][slots], st["x"][:, None]], 1)
    st["states"][slots] = win[:, 1:]
    pre = (win.float() * st["weight"].t()).sum(1) + st["bias"]
    return {"y": (pre * _sigmoid(pre)).to(st["x"].dtype), "states": st["states"]}


PLAIN = {"scan_step": _scan_step, "conv_step": _conv_step, "scan_prompt": _scan_prompt, "conv_prompt": _conv_prompt,
         "scan_train": _scan_train, "conv_train": _conv_train}


# ------------------------------------------------- the framework's operators

def _call(st):
    import mlx_vision_mamba_amd as mvm
    op = st["op"]
    if op == "scan_step":
        y = mvm.selective_scan_step(st["u"], st["delta"], st["A_log"], st["B"], st["C"], st["D"], st["states"],
                                    slots=st["slots"], z=st["z"], delta_bias=st["delta_bias"], delta_softplus=True,
                                    a_is_log=True)
        return {"y": y, "states": st["states"]}
    if op == "conv_step":
        y = mvm.causal_conv_silu_step(st["x"], st["weight"], st["bias"], st["states"], slots=st["slots"])
        return {"y": y, "states": st["states"]}
    if op == "scan_prompt":
        y = mvm.selective_scan_prefill(st["u"], st["delta"], st["A_log"], st["B"], st["C"], st["D"], st["states"],
                                       st["offsets"], slots=st["slots"], fresh=st["fresh"], z=st["z"],
                                       delta_bias=st["delta_bias"], delta_softplus=True, a_is_log=True,
                                       max_len=st["max_len"])
        return {"y": y, "states": st["states"]}
    if op == "conv_prompt":
        y = mvm.causal_conv_silu_prefill(st["x"], st["weight"], st["bias"], st["states"], st["offsets"],
                                         slots=st["slots"], fresh=st["fresh"])
        return {"y": y, "states": st["states"]}
    if op == "scan_train":
        y, final = mvm.selective_scan_packed(st["u"], st["delta"], st["A_log"], st["B"], st["C"], st["D"],
                                             st["offsets"], z=st["z"], delta_bias=st["delta_bias"],
                                             delta_softplus=True, a_is_log=True, initial_states=st["initial"],
                                             max_len=st["max_len"])
    else:
        y, final = mvm.causal_conv_silu_packed(st["x"], st["weight"], st["bias"], st["offsets"],
                                               initial_states=st["initial"])
    leaves = LEAVES[op]
    grads = torch.autograd.grad([y, final], [st[k] for k in leaves], [st["dy"], st["dfinal"]])
    out = {"y": y.detach(), "final": final.detach()}
    out.update({"d" + k: g for k, g in zip(leaves, grads)})
    return out


def run(state):
    return _call(state) if own else PLAIN[state["op"]](state)


# -------------------------------------------------------------------- work

def work(case):
    e, D, S, op = TYPES[case["dtype"]].itemsize, case["D"], case["S"], case["op"]
    T = S if op.endswith("step") else case["T"]
    if op.startswith("scan"):
        N = case["N"]
        state, params = S * D * N * 4, D * (N + 2) * 4
        # u, delta, z and y; B and C; the states read and written
        nbytes = T * D * 4 * e + T * 2 * N * e + 2 * state + params
        flops = T * D * (7 * N + 15)
        if op == "scan_train":
            # dy read, du, ddelta and dz written; dB and dC; the states' and the parameters' gradients
            nbytes += T * D * 4 * e + T * 2 * N * e + 2 * state + params
            flops += T * D * (19 * N + 30)
    else:
        W = case["W"]
        state, params = S * (W - 1) * D * e, D * (W + 1) * 4
        nbytes = T * D * 2 * e + 2 * state + params
        flops = T * D * (2 * W + 5)
        if op == "conv_train":
            nbytes += T * D * 2 * e + 2 * state + params
            flops += T * D * (4 * W + 8)
    return {"bytes": nbytes, "flops": flops}


# ------------------------------------------------------ the values in 64 bits

def _one_scan(u, dl, A, B, C, h, H=None):
    """r (without D u) of one sequence token by token, from state h; each h_t kept in H."""
    r = torch.empty_like(u)
    for t0 in range(0, u.shape[0], 128):
        d = dl[t0:t0 + 128]
        a = torch.exp(d[:, :, None] * A)
        b = (d * u[t0:t0 + 128])[:, :, None] * B[t0:t0 + 128, None, :]
        hs = torch.empty_like(a)
        for i in range(d.shape[0]):
            torch.addcmul(b[i], a[i], h, out=hs[i])
            h = hs[i]
        r[t0:t0 + 128] = (hs * C[t0:t0 + 128, None, :]).sum(-1)
        if H is not None:
            H[t0:t0 + 128] = hs
    return r, h


def _exact_scan(st):
    op = st["op"]
    v = {k: st[k].detach().double() for k in ("u", "delta", "B", "C", "z", "A_log", "D", "delta_bias")}
    A = -v["A_log"].exp()
    raw = v["delta"] + v["delta_bias"]
    dl = torch.nn.functional.softplus(raw, threshold=200)
    sil = torch.nn.functional.silu(v["z"])
    if op == "scan_step":
        off = list(range(v["u"].shape[0] + 1))
    else:
        off = st["offsets"].tolist()
    train = op == "scan_train"
    S, T = len(off) - 1, v["u"].shape[0]
    if train:
        h0 = st["initial"].detach().double()
    else:
        h0 = st["states"][st["slots"].long()].double()
        if "fresh" in st:
            h0[st["fresh"]] = 0
    if op == "scan_step":  # all sequences at once: one token each
        h1 = torch.exp(dl[:, :, None] * A) * h0 + (dl * v["u"])[:, :, None] * v["B"][:, None, :]
        r = (h1 * v["C"][:, None, :]).sum(-1) + v["D"] * v["u"]
    else:
        r, h1 = torch.zeros_like(v["u"]), h0.clone()
        grads = {k: torch.zeros_like(v[k]) for k in v}
        dh0 = torch.zeros_like(h0)
        for i in range(S):
            s = slice(off[i], off[i + 1])
            n = off[i + 1] - off[i]
            u, d, B, C = v["u"][s], dl[s], v["B"][s], v["C"][s]
            H = torch.empty(n, *h0.shape[1:], dtype=torch.float64, device=u.device) if train else None
            part, h1[i] = _one_scan(u, d, A, B, C, h0[i], H)
            r[s] = part + v["D"] * u
            if not train:
                continue
            dr = st["dy"][s].double() * sil[s]
            c = st["dfinal"][i].double()
            for t0 in reversed(range(0, n, 128)):
                q = slice(t0, min(n, t0 + 128))
                a = torch.exp(d[q][:, :, None] * A)
                inj = dr[q][:, :, None] * C[q][:, None, :]
                G = torch.empty_like(a)
                for j in reversed(range(a.shape[0])):
                    torch.add(inj[j], c, out=G[j])
                    c = a[j] * G[j]
                hp = torch.cat([h0[i][None] if t0 == 0 else H[t0 - 1:t0], H[t0:q.stop - 1]])
                x = G * a * hp
                k = slice(off[i] + t0, off[i] + q.stop)
                gB = (G * B[q][:, None, :]).sum(-1)
                grads["u"][k] = gB * d[q] + v["D"] * dr[q]
                grads["delta"][k] = (x * A).sum(-1) + gB * u[q]
                grads["A_log"] += (x * d[q][:, :, None]).sum(0) * A
                grads["B"][k] = (G * (d[q] * u[q])[:, :, None]).sum(1)
                grads["C"][k] = (H[q] * dr[q][:, :, None]).sum(1)
            dh0[i] = c
        if train:
            dy, sg = st["dy"].double(), torch.sigmoid(v["z"])
            grads["delta"] = grads["delta"] * torch.sigmoid(raw)
            grads["delta_bias"] = grads["delta"].sum(0)
            grads["D"] = (dy * sil * v["u"]).sum(0)
            grads["z"] = dy * r * (sg + sil * (1 - sg))
            grads["initial"] = dh0
            out = {"y": r * sil, "final": h1}
            out.update({"d" + k: grads[k] for k in LEAVES[op]})
            return out
    states = st["states"].double()
    states[st["slots"].long()] = h1
    return {"y": r * sil, "states": states}


def _exact_conv(st):
    op, W = st["op"], st["weight"].shape[1]
    leaves = {k: st[k].detach().double().requires_grad_(True) for k in ("x", "weight", "bias")}
    x, w, b = leaves.values()
    off = list(range(x.shape[0] + 1)) if op == "conv_step" else st["offsets"].tolist()
    if op == "conv_train":
        c0 = leaves["initial"] = st["initial"].detach().double().requires_grad_(True)
    else:
        c0 = st["states"][st["slots"].long()].double()
        if "fresh" in st:
            c0[st["fresh"]] = 0
    if op == "conv_step":
        win = torch.cat([c0, x[:, None]], 1)
        ys, final = [torch.nn.functional.silu((win * w.t()).sum(1) + b)], win[:, 1:]
    else:
        ys, final = [], []
        for i in range(len(off) - 1):
            seq = torch.cat([c0[i], x[off[i]:off[i + 1]]])
            final.append(seq[seq.shape[0] - (W - 1):])
            n = off[i + 1] - off[i]
            ys.append(torch.nn.functional.silu(sum(w[:, j] * seq[j:j + n] for j in range(W)) + b))
        final = torch.stack(final)
    y = torch.cat(ys)
    if op == "conv_train":
        g = torch.autograd.grad([y, final], [leaves[k] for k in LEAVES[op]], [st["dy"].double(), st["dfinal"].double()])
        out = {"y": y.detach(), "final": final.detach()}
        out.update({"d" + k: v for k, v in zip(LEAVES[op], g)})
        return out
    states = st["states"].double()
    states[st["slots"].long()] = final.detach()
    return {"y": y.detach(), "states": states}


def exact(case, seed):
    state = prepare(case, seed)
    return _exact_scan(state) if case["op"].startswith("scan") else _exact_conv(state)

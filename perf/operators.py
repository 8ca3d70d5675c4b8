"""Sizes at which the sequence operators of the framework are measured: the gated delta rule (whole sequences forward,
forward + backward, and one token per agent against a pool of states) and the norms around a block with their gate and
residual scale.  `run` computes them in plain torch operations, or, where `own` is true, through hhrl_vae_amd.sequence."""
import math

import numpy as np
import torch

own = False

DT = {"f32": torch.float32, "bf16": torch.bfloat16}
CHUNK = 64


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one agent acting: a single token against its state, latency counts
        {"name": "delta_step_one", "op": "step", "dtype": "f32", "B": 1, "slots": 1, "Hk": 4, "Hv": 4, "K": 64, "V": 64},
        # a serving batch: one token for each of 192 sequences out of a pool of states, in any order
        {"name": "delta_step_pool", "op": "step", "dtype": "bf16", "B": 192, "slots": 256, "Hk": 16, "Hv": 32, "K": 128, "V": 128},
        # the framework's own window (10 steps, 128 hidden units) and batch, in its own precision, trained
        {"name": "delta_train_window", "op": "train", "dtype": "f32", "seqs": 64, "rows": 640, "ragged": False, "Hk": 1, "Hv": 1,
         "K": 128, "V": 128},
        # fp32 training over episodes of odd length with shared key heads and odd widths
        {"name": "delta_train_f32", "op": "train", "dtype": "f32", "seqs": 8, "rows": 8 * 509, "ragged": False, "Hk": 2, "Hv": 4,
         "K": 61, "V": 72},
        # prompts of different lengths packed behind each other, states kept for decoding
        {"name": "delta_prefill_ragged", "op": "prefill", "dtype": "bf16", "seqs": 13, "rows": 12345, "ragged": True, "Hk": 8, "Hv": 16,
         "K": 128, "V": 128},
        # one long sequence with few heads: little to do side by side
        {"name": "delta_prefill_long", "op": "prefill", "dtype": "bf16", "seqs": 1, "rows": 32768, "ragged": False, "Hk": 4, "Hv": 8,
         "K": 128, "V": 128},
        # a training step's sequences
        {"name": "delta_train", "op": "train", "dtype": "bf16", "seqs": 4, "rows": 4 * 4096, "ragged": False, "Hk": 16, "Hv": 16,
         "K": 128, "V": 128},
        # acting: norm after one block, residual sum, norm before the next for one row
        {"name": "norm_one_row", "op": "norm", "dtype": "f32", "M": 1, "H": 1, "D": 256, "post": "rms", "pre": "rms", "x": True, "y": True,
         "gate": "none", "gate_rows": 1},
        # a prompt's rows between two blocks of an odd width, fp32, gated by one row of channel gates per sequence
        {"name": "norm_block_f32", "op": "norm", "dtype": "f32", "M": 4 * 1021, "H": 1, "D": 1000, "post": "layer", "pre": "layer",
         "x": True, "y": True, "gate": "none", "gate_rows": 1021},
        # between two blocks of a wide model, trained: both norms, one learned gate per channel
        {"name": "norm_block_train", "op": "norm_train", "dtype": "bf16", "M": 8192, "H": 1, "D": 4096, "post": "rms", "pre": "rms",
         "x": True, "y": True, "gate": "none", "gate_rows": 8192},
        # the gated norm behind the delta rule, trained: one norm per head, a SiLU gate per element
        {"name": "norm_heads_train", "op": "norm_train", "dtype": "bf16", "M": 16384, "H": 16, "D": 128, "post": "rms", "pre": "none",
         "x": False, "y": True, "gate": "silu", "gate_rows": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "prefill", "train", "norm", "norm_train"])
    dt = rng.choice(["f32", "bf16"])
    if op in ("norm", "norm_train"):
        H = rng.choice([1, 1, rng.randint(2, 16)])
        D = _log(rng, 16, 8192) if H == 1 else _log(rng, 16, 256)
        top = 24 * 1024 * 1024
        M = _log(rng, 1, max(1, min(65536, top // (H * D))))
        x = rng.random() < 0.7
        c = {"op": op, "dtype": dt, "M": M, "H": H, "D": D, "post": rng.choice(["none", "rms", "layer"]),
             "pre": rng.choice(["none", "rms", "layer"]), "x": x, "y": (not x) or rng.random() < 0.8,
             "gate": rng.choice(["off", "none", "sigmoid", "silu"]), "gate_rows": 1}
        if not c["y"]:
            c["gate"] = "off"
        if c["gate"] != "off" and H == 1 and rng.random() < 0.5:
            c["gate_rows"] = rng.randint(1, M)
        return c
    Hk = rng.choice([1, 2, 3, 4, 8, 16])
    Hv = Hk * rng.choice([1, 1, 2, 3])
    if rng.random() < 0.5:
        K = V = rng.choice([64, 128])
    else:
        K, V = rng.randint(8, 128), rng.randint(8, 160)
    if op == "step":
        B = _log(rng, 1, max(1, min(512, 90000000 // (Hv * K * V))))
        return {"op": op, "dtype": dt, "B": B, "slots": B + rng.randint(0, B), "Hk": Hk, "Hv": Hv, "K": K, "V": V}
    top = (40000000 if dt == "bf16" else 12000000) // (Hv * max(K, V))
    if op == "train":
        top //= 2
    rows = _log(rng, 1, max(2, min(32768 if op == "prefill" else 8192, top)))
    seqs = min(rows, _log(rng, 1, 48))
    ragged = rng.random() < 0.6
    if not ragged:
        rows = rows // seqs * seqs
    return {"op": op, "dtype": dt, "seqs": seqs, "rows": rows, "ragged": ragged, "Hk": Hk, "Hv": Hv, "K": K, "V": V}


def work(case):
    el = 4 if case["dtype"] == "f32" else 2
    if case["op"] in ("norm", "norm_train"):
        n, D = case["M"] * case["H"] * case["D"], case["D"]
        gate = 0 if case["gate"] == "off" else n * el if case["gate_rows"] == 1 else -(-case["M"] // case["gate_rows"]) * D * 4
        ins = n * el * (int(case["x"]) + int(case["y"])) + gate
        outs = n * el * (1 + int(case["pre"] != "none"))
        par = 4 * D * sum({"none": 0, "rms": 1, "layer": 2}[case[k]] for k in ("post", "pre"))
        by, fl = ins + outs + par, 12 * n
        if case["op"] == "norm_train":
            by, fl = 2 * ins + 2 * outs + 2 * par, 36 * n
        return {"bytes": float(by), "flops": float(fl)}
    Hk, Hv, K, V = (case[k] for k in ("Hk", "Hv", "K", "V"))
    rows = case["B"] if case["op"] == "step" else case["rows"]
    state = 4 * Hv * K * V
    by = rows * (el * (2 * Hk * K + 2 * Hv * V) + 8 * Hv)
    fl = 6 * rows * Hv * K * V
    if case["op"] == "step":
        by += 2 * rows * state
    else:
        by += case["seqs"] * state * (1 if case["op"] == "prefill" else 0)
    if case["op"] == "train":
        by, fl = by + rows * (el * (2 * Hk * K + 2 * Hv * V) + 8 * Hv), 3 * fl
    return {"bytes": float(by), "flops": float(fl)}


# ----------------------------------------------------------------------------------------------------------- inputs
def _lens(case, seed):
    n, rows = case["seqs"], case["rows"]
    if not case["ragged"]:
        return [rows // n] * n
    r = np.random.RandomState(seed % (1 << 31))
    w = r.exponential(size=n) + 0.02
    if n > 2:
        w[r.randint(n)] = 0.0                       # a sequence without a token
    cut = np.floor(np.cumsum(w) / w.sum() * rows + 1e-9).astype(int)
    cut[-1] = rows
    return np.diff(np.concatenate([[0], cut])).tolist()


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = DT[case["dtype"]]
    rn = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    ru = lambda *s: torch.rand(*s, generator=gen, device="cuda")
    if case["op"] in ("norm", "norm_train"):
        M, H, D = case["M"], case["H"], case["D"]
        st = {"x": rn(M, H, D).to(dt) if case["x"] else None, "y": (0.5 + 1.5 * rn(M, H, D)).to(dt) if case["y"] else None, "gate": None}
        if case["gate"] != "off":
            st["gate"] = rn(M, H, D).to(dt) if case["gate_rows"] == 1 else 0.7 * rn(-(-M // case["gate_rows"]), H, D)
        for k in ("post", "pre"):
            used = case[k] != "none" and (k == "pre" or case["y"])
            st["w_" + k] = 1 + 0.2 * rn(D) if used else None
            st["b_" + k] = 0.2 * rn(D) if used and case[k] == "layer" else None
        if case["op"] == "norm_train":
            st["d_out"] = rn(M, H, D).to(dt)
            st["d_h"] = rn(M, H, D).to(dt) if case["pre"] != "none" else None
        return st
    Hk, Hv, K, V = (case[k] for k in ("Hk", "Hv", "K", "V"))
    rows = case["B"] if case["op"] == "step" else case["rows"]
    unit = lambda t: (t / t.norm(dim=-1, keepdim=True)).to(dt)
    st = {"q": unit(rn(rows, Hk, K)), "k": unit(rn(rows, Hk, K)), "v": rn(rows, Hv, V).to(dt),
          # log decays as a softplus of a projection times a rate per head gives them: most near 0, a few resets
          "g": -torch.nn.functional.softplus(rn(rows, Hv) - 3.0) * (0.2 + 4.0 * ru(Hv)), "beta": torch.sigmoid(rn(rows, Hv))}
    if case["op"] == "step":
        st["state"] = 0.3 * rn(case["slots"], Hv, K, V)
        st["slots"] = torch.from_numpy(np.random.RandomState(seed % (1 << 31)).permutation(case["slots"])[:rows].astype(np.int32)).cuda()
        return st
    lens = _lens(case, seed)
    st["lens"] = lens
    if case["ragged"]:
        st["starts"] = torch.from_numpy(np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)).cuda()
    if case["op"] == "train":
        st["d_o"] = rn(rows, Hv, V).to(dt)
    return st


def _seq_view(st, case, name):
    """[rows, ...] as the framework takes it: packed rows beside their starts, or [sequences, tokens, ...]."""
    t = st[name]
    return t if case["ragged"] else t.view(case["seqs"], case["rows"] // case["seqs"], *t.shape[1:])


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    dt, op = DT[case["dtype"]], case["op"]
    dev = torch.device("cuda", torch.cuda.current_device())
    new = lambda *s, dtype=dt: torch.zeros(*s, dtype=dtype, device=dev)
    if op == "step":
        st["state_out"] = torch.zeros_like(st["state"])
    if not own:
        if "lens" in st:
            st["pad"] = _padded_index(st["lens"], max(1, -(-max(st["lens"]) // CHUNK)) * CHUNK).cuda()
        return st
    from hhrl_vae_amd import sequence
    if op in ("norm", "norm_train"):
        M, H, D = case["M"], case["H"], case["D"]
        st["plan"] = sequence.BlockNorm(D, H=H, post=case["post"] if case["y"] else "none", pre=case["pre"], gate_act=case["gate"] if case["gate"] != "off" else "none",
                                        gate_rows=case["gate_rows"], alpha=ALPHA, scale=SCALE, eps=EPS, dtype=dt)
        st["out"], st["h"] = new(M, H, D), new(M, H, D) if case["pre"] != "none" else None
        if op == "norm_train":
            st["ws"] = st["plan"].workspace(M, dev)
            for k in ("x", "y", "gate", "w_post", "b_post", "w_pre", "b_pre"):
                st["d" + k] = torch.zeros_like(st[k]) if st[k] is not None else None
            st["par"] = [st["d" + k] for k in ("w_post", "b_post", "w_pre", "b_pre") if st["d" + k] is not None]
        return st
    Hk, Hv, K, V = (case[k] for k in ("Hk", "Hv", "K", "V"))
    st["plan"] = sequence.GatedDelta(Hk, Hv, K, V, dtype=dt)
    st["o"] = torch.zeros_like(st["v"])
    if op == "step":
        return st
    st["ws"] = st["plan"].workspace(case["seqs"], case["rows"], dev, no_backward=op == "prefill")
    if op == "prefill":
        st["s1"] = new(case["seqs"], Hv, K, V, dtype=torch.float32)
    else:
        for k in ("q", "k", "v", "g", "beta"):
            st["d" + k] = torch.zeros_like(st[k])
    st["views"] = {n: _seq_view(st, case, n) for n in ("q", "k", "v", "g", "beta", "o", "d_o", "dq", "dk", "dv", "dg", "dbeta") if n in st}
    return st


# -------------------------------------------------------------------------------------------------------------- run
def run(st):
    case = st["case"]
    if not own:
        return _plain(st, case)
    p = st["plan"]
    if case["op"] == "step":
        p.step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["o"], st["state"], state_out=st["state_out"], slots=st["slots"])
        return {"o": st["o"], "state": st["state_out"]}
    if case["op"] in ("norm", "norm_train"):
        args = {k: st[k] for k in ("x", "y", "gate", "w_post", "b_post", "w_pre", "b_pre")}
        p.fwd(out=st["out"], h=st["h"], **args)
        res = {"out": st["out"], "h": st["h"]}
        if case["op"] == "norm_train":
            if st["par"]:                             # (norms may have no parameters)
                torch._foreach_zero_(st["par"])       # parameter gradients are added to
            grads = {"d" + k: st["d" + k] for k in args}
            p.bwd(d_out=st["d_out"], d_h=st["d_h"], ws=st["ws"], **args, **grads)
            res.update(grads)
        return {k: v for k, v in res.items() if v is not None}
    w = st["views"]
    ins = [w[k] for k in ("q", "k", "v", "g", "beta")]
    if case["op"] == "prefill":
        p.fwd(*ins, w["o"], st["ws"], s1=st["s1"], starts=st.get("starts"), no_backward=True)
        return {"o": st["o"], "s1": st["s1"]}
    p.fwd(*ins, w["o"], st["ws"], starts=st.get("starts"))
    p.bwd(*ins, w["d_o"], w["dq"], w["dk"], w["dv"], w["dg"], w["dbeta"], st["ws"], starts=st.get("starts"))
    return {k: st[k] for k in ("o", "dq", "dk", "dv", "dg", "dbeta")}


# ------------------------------------------------------------------------------------------------------ plain forms
def _plain(st, case):
    if case["op"] == "step":
        return _plain_step(st, case)
    if case["op"] in ("norm", "norm_train"):
        return _plain_norm(st, case)
    return _plain_delta(st, case)


def _plain_step(st, case):
    rep = case["Hv"] // case["Hk"]
    q, k = (st[n].float().repeat_interleave(rep, dim=1) for n in ("q", "k"))
    slots = st["slots"].long()
    s = st["state"][slots] * st["g"].exp()[..., None, None]
    u = st["beta"][..., None] * (st["v"].float() - (s * k[..., None]).sum(-2))
    s = s + k[..., None] * u[..., None, :]
    o = (s * q[..., None]).sum(-2) * case["K"] ** -0.5
    st["state_out"][slots] = s
    return {"o": o.to(st["v"].dtype), "state": st["state_out"]}


def _padded_index(lens, T):
    idx = torch.full((len(lens), T), -1, dtype=torch.long)
    at = 0
    for i, n in enumerate(lens):
        idx[i, :n] = torch.arange(at, at + n)
        at += n
    return idx


def _plain_delta(st, case):
    """The chunked form: within a chunk the recurrence is a triangular system, between chunks only the state passes on."""
    C, rep, scale = CHUNK, case["Hv"] // case["Hk"], case["K"] ** -0.5
    pad = st["pad"]
    valid, idx = pad >= 0, pad.clamp(min=0)
    N, T = pad.shape
    nc = T // C

    def chunks(t, r=1):                                   # [rows, H, *] -> [N, H, nc, C, *], rows behind the end are 0
        t = t.float().repeat_interleave(r, dim=1)[idx.flatten()].view(N, nc, C, t.shape[1] * r, *t.shape[2:])
        t = t * valid.view(N, nc, C, *[1] * (t.dim() - 3))
        return t.movedim(3, 1)

    def rows(t):                                          # and back
        t = t.movedim(1, 3)
        return t.reshape(N * T, *t.shape[3:])[valid.flatten()]

    q, k, v = chunks(st["q"], rep), chunks(st["k"], rep), chunks(st["v"])
    g, beta = chunks(st["g"]), chunks(st["beta"])
    low = torch.ones(C, C, dtype=torch.bool, device=q.device).tril()
    G = g.double().cumsum(-1)                             # long sums and their differences in 64 bits
    D = (G[..., :, None] - G[..., None, :]).masked_fill(~low, -math.inf).exp().float()
    gam, tail = G.exp().float(), (G[..., -1:] - G).exp().float()
    last = gam[..., -1]
    kk = k @ k.transpose(-1, -2)
    A = (beta[..., None] * kk * D).tril(-1)
    M = torch.eye(C, device=q.device).expand_as(A).clone()
    for i in range(1, C):
        M[..., i, :i] = -(A[..., i:i + 1, :i] @ M[..., :i, :i])[..., 0, :]
    P = (q @ k.transpose(-1, -2)) * D
    S = torch.zeros(*q.shape[:2], case["K"], case["V"], device=q.device)
    o, vn = torch.empty_like(v), torch.empty_like(v)
    states = []
    for c in range(nc):
        states.append(S)
        X = v[:, :, c] - gam[:, :, c, :, None] * (k[:, :, c] @ S)
        vn[:, :, c] = M[:, :, c] @ (beta[:, :, c, :, None] * X)
        o[:, :, c] = scale * (gam[:, :, c, :, None] * (q[:, :, c] @ S) + P[:, :, c] @ vn[:, :, c])
        S = last[:, :, c, None, None] * S + k[:, :, c].transpose(-1, -2) @ (tail[:, :, c, :, None] * vn[:, :, c])
    dt = st["v"].dtype
    if case["op"] == "prefill":
        return {"o": rows(o).to(dt), "s1": S}
    do = chunks(st["d_o"])
    S0 = torch.stack(states, dim=2)
    dS0, Y = torch.empty_like(S0), torch.empty_like(v)    # dS0[c]: gradient of the state BEHIND chunk c
    dS = torch.zeros_like(S)
    for c in reversed(range(nc)):
        dS0[:, :, c] = dS
        Z = scale * P[:, :, c].transpose(-1, -2) @ do[:, :, c] + tail[:, :, c, :, None] * (k[:, :, c] @ dS)
        Y[:, :, c] = M[:, :, c].transpose(-1, -2) @ Z
        dS = last[:, :, c, None, None] * dS + scale * q[:, :, c].transpose(-1, -2) @ (gam[:, :, c, :, None] * do[:, :, c]) \
            - k[:, :, c].transpose(-1, -2) @ ((gam * beta)[:, :, c, :, None] * Y[:, :, c])
    S0t = S0.transpose(-1, -2)
    E2 = Y @ S0t
    dP = scale * (do @ vn.transpose(-1, -2)) * D
    dA = -(Y @ vn.transpose(-1, -2)) * D.tril(-1)
    Bm = dA * beta[..., None]
    dq = scale * gam[..., None] * (do @ S0t) + dP @ k
    dk_row = -(gam * beta)[..., None] * E2 + Bm @ k
    dk_col = tail[..., None] * (vn @ dS0.transpose(-1, -2)) + Bm.transpose(-1, -2) @ k + dP.transpose(-1, -2) @ q
    dbeta = (Y * v).sum(-1) - gam * (k * E2).sum(-1) + (dA * kk).sum(-1)
    dG = (q * dq).sum(-1) + (k * dk_row).sum(-1) - (k * dk_col).sum(-1)
    S1 = torch.cat([S0[:, :, 1:], S[:, :, None]], dim=2)
    dG[..., -1] += (dS0 * S1).sum((-1, -2))
    dg = dG.flip(-1).cumsum(-1).flip(-1)
    heads = lambda t: t.view(t.shape[0], case["Hk"], rep, t.shape[-1]).sum(2)
    return {"o": rows(o).to(dt), "dq": heads(rows(dq)).to(dt), "dk": heads(rows(dk_row + dk_col)).to(dt),
            "dv": rows(beta[..., None] * Y).to(dt), "dg": rows(dg), "dbeta": rows(dbeta)}


ALPHA, SCALE, EPS = 0.9, 0.7, 1e-5
NORM_OUTPUTS = ("out", "h", "dx", "dy", "dgate", "dw_post", "db_post", "dw_pre", "db_pre")


def _norm_stats(t, kind):
    """Normalised t and 1/sqrt(mean square + eps) of what is left of it."""
    if kind == "layer":
        t = t - t.mean(-1, keepdim=True)
    r = (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return t * r, r


def _norm_back(dn, n, r, kind):
    d = dn - n * (dn * n).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - dn.mean(-1, keepdim=True)
    return d * r


def _plain_norm(st, case):
    f = lambda k: st[k].float() if st.get(k) is not None else None
    dt = DT[case["dtype"]]
    x, y, gate = f("x"), f("y"), f("gate")
    M, H, D = case["M"], case["H"], case["D"]
    r = ALPHA * x if x is not None else 0.0
    n = ry = act = None
    if y is not None:
        n, ry = _norm_stats(y, case["post"]) if case["post"] != "none" else (y, None)
        b = n * st["w_post"] if case["post"] != "none" else n
        if st["b_post"] is not None:
            b = b + st["b_post"]
        if gate is not None:
            if case["gate_rows"] > 1:
                gate = gate.repeat_interleave(case["gate_rows"], dim=0)[:M]
            sg = torch.sigmoid(gate)
            act = {"none": gate, "sigmoid": sg, "silu": gate * sg}[case["gate"]]
            r = r + SCALE * act * b
        else:
            r = r + SCALE * b
    res = {"out": r.to(dt)}
    if case["pre"] != "none":
        m, rp = _norm_stats(r, case["pre"])
        h = m * st["w_pre"]
        if st["b_pre"] is not None:
            h = h + st["b_pre"]
        res["h"] = h.to(dt)
    if case["op"] == "norm":
        return res
    dr = f("d_out")
    if case["pre"] != "none":
        dh = f("d_h")
        res["dw_pre"] = (dh * m).sum((0, 1))
        if st["b_pre"] is not None:
            res["db_pre"] = dh.sum((0, 1))
        dr = dr + _norm_back(dh * st["w_pre"], m, rp, case["pre"])
    if x is not None:
        res["dx"] = (ALPHA * dr).to(dt)
    if y is not None:
        db = SCALE * dr
        if gate is not None:
            da = db * b
            db = db * act
            da = da * {"none": torch.ones_like(sg), "sigmoid": sg * (1 - sg), "silu": sg * (1 + gate * (1 - sg))}[case["gate"]]
            if case["gate_rows"] > 1:
                R = case["gate_rows"]
                da = torch.cat([da, da.new_zeros(-M % R, H, D)]).view(-1, R, H, D).sum(1)
            res["dgate"] = da.to(st["gate"].dtype)
        if case["post"] != "none":
            res["dw_post"] = (db * n).sum((0, 1))
            if st["b_post"] is not None:
                res["db_post"] = db.sum((0, 1))
            db = _norm_back(db * st["w_post"], n, ry, case["post"])
        res["dy"] = db.to(dt)
    return {k: res[k] for k in NORM_OUTPUTS if k in res}


# -------------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    st = _inputs(case, seed)
    if case["op"] in ("norm", "norm_train"):
        return _exact_norm(st, case)
    return _exact_delta(st, case)


def _exact_norm(st, case):
    train = case["op"] == "norm_train"
    leaf = {k: st[k].double().requires_grad_(train) for k in ("x", "y", "gate", "w_post", "b_post", "w_pre", "b_pre") if st[k] is not None}

    def norm(t, which):
        kind = case[which]
        if kind == "none":
            return t
        if kind == "layer":
            t = (t - t.mean(-1, keepdim=True)) / (t.var(-1, unbiased=False, keepdim=True) + EPS).sqrt()
        else:
            t = t / ((t * t).sum(-1, keepdim=True) / t.shape[-1] + EPS).sqrt()
        t = t * leaf["w_" + which]
        return t + leaf["b_" + which] if kind == "layer" else t

    terms = []
    if "x" in leaf:
        terms.append(ALPHA * leaf["x"])
    if "y" in leaf:
        b = norm(leaf["y"], "post") * SCALE
        if "gate" in leaf:
            a = leaf["gate"]
            a = a if case["gate"] == "none" else 1 / (1 + (-a).exp()) * (a if case["gate"] == "silu" else 1.0)
            b = b * a[torch.arange(case["M"], device=a.device) // case["gate_rows"]]
        terms.append(b)
    r = sum(terms)
    res = {"out": r}
    loss = (r * st["d_out"].double()).sum() if train else None
    if case["pre"] != "none":
        res["h"] = norm(r, "pre")
        if train:
            loss = loss + (res["h"] * st["d_h"].double()).sum()
    res = {k: v.detach() for k, v in res.items()}
    if train:
        loss.backward()
        for k in ("dw_pre", "db_pre", "dx", "dgate", "dw_post", "db_post", "dy"):
            if k[1:] in leaf:
                res[k] = leaf[k[1:]].grad
    if train:
        res = {k: res[k] for k in NORM_OUTPUTS if k in res}
    return res


def _exact_delta(st, case):
    """The recurrence itself, token by token; its gradient by the same recurrence run backwards."""
    dev, f64 = st["q"].device, torch.float64
    Hv, K, V, rep, scale = case["Hv"], case["K"], case["V"], case["Hv"] // case["Hk"], case["K"] ** -0.5
    wide = lambda t, r=1: t.to(f64).repeat_interleave(r, dim=1)
    q, k, v = wide(st["q"], rep), wide(st["k"], rep), wide(st["v"])
    a, beta = wide(st["g"]).exp(), wide(st["beta"])

    def step(S, q_, k_, v_, a_, b_):
        Sd = a_[..., None, None] * S
        u = b_[..., None] * (v_ - torch.matmul(k_[..., None, :], Sd)[..., 0, :])
        return Sd, u, Sd + k_[..., :, None] * u[..., None, :]

    if case["op"] == "step":
        slots = st["slots"].long()
        _, _, S = step(st["state"][slots].to(f64), q, k, v, a, beta)
        pool = torch.zeros_like(st["state"], dtype=f64)
        pool[slots] = S
        return {"o": scale * torch.matmul(q[..., None, :], S)[..., 0, :], "state": pool}
    lens = st["lens"]
    N, T = len(lens), max(lens)
    if T > 33000 or T * N * Hv * K * V > 1e13:
        return None
    idx = _padded_index(lens, max(T, 1)).to(dev)
    ok = (idx >= 0)
    at = idx.clamp(min=0)
    t_major = lambda t: (t[at] * ok.view(N, -1, *[1] * (t.dim() - 1))).transpose(0, 1).contiguous()
    qs, ks, vs, bs = t_major(q), t_major(k), t_major(v), t_major(beta)
    as_ = torch.where(ok.t()[..., None], t_major(a), torch.ones((), dtype=f64, device=dev))
    S = torch.zeros(N, Hv, K, V, dtype=f64, device=dev)
    o = torch.zeros_like(vs)
    keep = []
    for t in range(T):
        if t % 64 == 0 and case["op"] == "train":
            keep.append(S)
        _, _, S = step(S, qs[t], ks[t], vs[t], as_[t], bs[t])
        o[t] = scale * torch.matmul(qs[t][..., None, :], S)[..., 0, :]
    flat = lambda t: t.transpose(0, 1)[ok]
    if case["op"] == "prefill":
        return {"o": flat(o), "s1": S}
    dos = t_major(st["d_o"].to(f64))
    dq, dk, dv, da, db = (torch.zeros_like(t) for t in (qs, ks, vs, as_, bs))
    dS = torch.zeros_like(S)
    col = lambda t: t[..., :, None]
    for c in reversed(range(len(keep))):
        S, run_ = keep[c], []
        for t in range(64 * c, min(T, 64 * c + 64)):
            run_.append((t, S) + step(S, qs[t], ks[t], vs[t], as_[t], bs[t]))
            S = run_[-1][-1]
        for t, S_, Sd, u, Sn in reversed(run_):
            dS = dS + scale * qs[t][..., :, None] * dos[t][..., None, :]
            dq[t] = scale * torch.matmul(Sn, col(dos[t]))[..., 0]
            du = torch.matmul(ks[t][..., None, :], dS)[..., 0, :]
            dk[t] = torch.matmul(dS, col(u))[..., 0]
            dv[t] = bs[t][..., None] * du
            db[t] = (du * (vs[t] - torch.matmul(ks[t][..., None, :], Sd)[..., 0, :])).sum(-1)
            dk[t] -= torch.matmul(Sd, col(dv[t]))[..., 0]
            dSd = dS - ks[t][..., :, None] * dv[t][..., None, :]
            da[t] = (dSd * S_).sum((-1, -2))
            dS = as_[t][..., None, None] * dSd
    heads = lambda t: t.view(t.shape[0], case["Hk"], rep, K).sum(2)
    return {"o": flat(o), "dq": heads(flat(dq)), "dk": heads(flat(dk)), "dv": flat(dv), "dg": flat(da * as_), "dbeta": flat(db)}

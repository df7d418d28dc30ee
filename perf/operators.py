"""Cases of the sequence-torso operators: linear attention with a decay per head (an unroll with
its gradient, a prompt, single acting steps), the per-head norms of queries and keys with the
position rotation, and the gated feed-forward layer.

`run` computes a case in its plain form (elementary torch operations in 32 bits, rounded once at
the end) or, where `own` is set, through boonta_b200's entry points.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}


# ---- the cases -----------------------------------------------------------------------------


def listed():
    return [
        # 512 environments x 128 steps of one update of a recurrent policy, episodes ending inside
        {"name": "attention_train_rollout", "op": "attention", "grad": True, "batch": 512,
         "steps": 128, "heads": 4, "dk": 64, "dv": 64, "dtype": "bf16", "resets": 0.02},
        # few long sequences (an offline dataset's trajectories), an odd number of steps
        {"name": "attention_train_long", "op": "attention", "grad": True, "batch": 2,
         "steps": 8191, "heads": 16, "dk": 128, "dv": 128, "dtype": "bf16", "resets": 0.0},
        # a small policy trained in float32, feature counts off every tile
        {"name": "attention_train_f32", "op": "attention", "grad": True, "batch": 48,
         "steps": 100, "heads": 3, "dk": 48, "dv": 40, "dtype": "f32", "resets": 0.03},
        # contexts read before acting, the state handed on
        {"name": "attention_prompt", "op": "attention", "grad": False, "batch": 16,
         "steps": 2000, "heads": 8, "dk": 64, "dv": 128, "dtype": "bf16", "resets": 0.0},
        # one acting step of few environments: latency
        {"name": "attention_step_small", "op": "step", "batch": 64, "heads": 4, "dk": 64,
         "dv": 64, "dtype": "bf16", "resets": 0.02},
        # one acting step of 4096 environments: the state's bytes
        {"name": "attention_step_large", "op": "step", "batch": 4096, "heads": 8, "dk": 64,
         "dv": 64, "dtype": "bf16", "resets": 0.02},
        # a training pass over full sequences, fewer key heads than query heads
        {"name": "norm_train", "op": "norm", "grad": True, "batch": 4, "steps": 4096, "heads": 16,
         "kv_heads": 4, "dim": 128, "rotary": 128, "interleaved": False, "dtype": "bf16"},
        # one acting step: latency
        {"name": "norm_step", "op": "norm", "grad": False, "batch": 128, "steps": 1, "heads": 8,
         "kv_heads": 8, "dim": 64, "rotary": 64, "interleaved": False, "dtype": "bf16"},
        # float32, half of an odd-sized head rotated, neighbours paired
        {"name": "norm_train_f32", "op": "norm", "grad": True, "batch": 32, "steps": 129,
         "heads": 6, "kv_heads": 6, "dim": 80, "rotary": 40, "interleaved": True, "dtype": "f32"},
        # one acting step of few environments: the weights' bytes
        {"name": "glu_act", "op": "glu", "grad": False, "rows": 16, "inner": 512, "outer": 1408,
         "act": "silu", "dtype": "bf16"},
        # a training minibatch of 4 x 4096 steps
        {"name": "glu_train", "op": "glu", "grad": True, "rows": 16384, "inner": 1024,
         "outer": 2816, "act": "silu", "dtype": "bf16"},
        # a float32 minibatch, sizes off every tile
        {"name": "glu_train_f32", "op": "glu", "grad": True, "rows": 2000, "inner": 500,
         "outer": 1001, "act": "tanh", "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "step", "norm", "glu", "glu"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op in ("attention", "step"):
        c = {"op": op, "heads": rng.randint(1, 16), "dk": rng.choice([16, 32, 48, 64, 72, 96, 128]),
             "dv": rng.choice([16, 32, 40, 64, 80, 128]), "dtype": dtype,
             "resets": rng.choice([0.0, 0.01, 0.1])}
        if op == "step":
            c["batch"] = _log(rng, 1, min(4096, 2 ** 27 // (c["heads"] * c["dk"] * c["dv"])))
        else:
            tokens = 2 ** (25 if dtype == "bf16" else 23) // (c["heads"] * max(c["dk"], c["dv"]))
            c["steps"] = _log(rng, 1, min(8192, tokens))
            most = min(1024, tokens // c["steps"], 2 ** 26 // (c["heads"] * c["dk"] * c["dv"]))
            c["batch"] = _log(rng, 1, max(1, most))
            c["grad"] = rng.random() < 0.7
        return c
    if op == "norm":
        dim = rng.choice([32, 64, 80, 96, 128, 256])
        heads = rng.randint(1, 16)
        tokens = 2 ** 24 // (heads * dim)
        steps = _log(rng, 1, min(8192, tokens))
        return {"op": op, "grad": rng.random() < 0.6, "batch": _log(rng, 1, max(1, min(1024, tokens // steps))),
                "steps": steps, "heads": heads, "kv_heads": rng.randint(1, heads), "dim": dim,
                "rotary": rng.choice([dim, dim // 2]), "interleaved": rng.random() < 0.5, "dtype": dtype}
    grad = rng.random() < 0.6
    # relu's border makes float32 gradients differ by whole terms, so it is drawn for bf16
    return {"op": op, "grad": grad, "rows": _log(rng, 1, 16384 if dtype == "bf16" else 4096),
            "inner": _log(rng, 32, 1024), "outer": _log(rng, 32, 2816),
            "act": rng.choice(["silu", "tanh", "none"] + (["relu"] if dtype == "bf16" else [])),
            "dtype": dtype}


# ---- what a program has in hand before the call -----------------------------------------------


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def rand(*shape, dtype=dt, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=g) * std).to(dtype)

    s = {"case": case}
    if case["op"] in ("attention", "step"):
        B, H, dk, dv = case["batch"], case["heads"], case["dk"], case["dv"]
        lead = (B, case["steps"], H) if case["op"] == "attention" else (B, H)
        s |= {"q": rand(*lead, dk), "k": rand(*lead, dk), "v": rand(*lead, dv),
              "state": rand(B, H, dk, dv, dtype=torch.float32),
              # time constants from a few steps to a few thousand, one for each head
              "log_decay": torch.log1p(-torch.exp2(-torch.linspace(3, 11, H, device="cuda")))}
        r = torch.rand(lead[:-1], device="cuda", generator=g)
        s["reset"] = (r < case["resets"]) if case["resets"] else None
        if case.get("grad"):
            s["dout"] = rand(*lead, dv)
            s["dstate"] = rand(B, H, dk, dv, dtype=torch.float32)
    elif case["op"] == "norm":
        B, T, D = case["batch"], case["steps"], case["dim"]
        s |= {"q": rand(B, T, case["heads"], D), "k": rand(B, T, case["kv_heads"], D),
              "q_weight": 1 + rand(D, std=0.2), "k_weight": 1 + rand(D, std=0.2)}
        start = torch.randint(0, 100000, (B, 1), device="cuda", generator=g)
        s["positions"] = start + torch.arange(T, device="cuda")
        half = case["rotary"] // 2
        s["frequencies"] = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        if case["grad"]:
            s |= {"dq": rand(B, T, case["heads"], D), "dk": rand(B, T, case["kv_heads"], D)}
    else:
        M, K, N = case["rows"], case["inner"], case["outer"]
        s |= {"x": rand(M, K), "w_gate": rand(K, N, std=K ** -0.5), "w_up": rand(K, N, std=K ** -0.5)}
        if case["grad"]:
            s["dh"] = rand(M, N)
    return s


# ---- one pass ------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if own:
        return {"attention": _own_attention, "step": _own_step, "norm": _own_norm, "glu": _own_glu}[case["op"]](s)
    return {"attention": _attention, "step": _step, "norm": _norm, "glu": _glu}[case["op"]](s)


def _leaves(*tensors):
    return [t.detach().requires_grad_() for t in tensors]


def _own_attention(s):
    from boonta_b200.linear_attention import linear_attention

    if not s["case"]["grad"]:
        return linear_attention(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["reset"])
    q, k, v, state = _leaves(s["q"], s["k"], s["v"], s["state"])
    out, last = linear_attention(q, k, v, s["log_decay"], state, s["reset"])
    return (out.detach(), last.detach(),
            *torch.autograd.grad((out, last), (q, k, v, state), (s["dout"], s["dstate"])))


def _own_step(s):
    from boonta_b200.linear_attention import linear_attention_step

    return linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["reset"])


def _own_norm(s):
    from boonta_b200.rotary import qk_norm_rotary

    inter = s["case"]["interleaved"]
    if not s["case"]["grad"]:
        return qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"],
                              s["frequencies"], interleaved=inter)
    q, k, wq, wk = _leaves(s["q"], s["k"], s["q_weight"], s["k_weight"])
    yq, yk = qk_norm_rotary(q, k, wq, wk, s["positions"], s["frequencies"], interleaved=inter)
    return (yq.detach(), yk.detach(),
            *torch.autograd.grad((yq, yk), (q, k, wq, wk), (s["dq"], s["dk"])))


def _own_glu(s):
    from boonta_b200.glu import gated_linear_unit

    act = s["case"]["act"]
    if not s["case"]["grad"]:
        return gated_linear_unit(s["x"], s["w_gate"], s["w_up"], act)
    x, wg, wu = _leaves(s["x"], s["w_gate"], s["w_up"])
    h = gated_linear_unit(x, wg, wu, act)
    return (h.detach(), *torch.autograd.grad(h, (x, wg, wu), s["dh"]))


# ---- plain forms -----------------------------------------------------------------------------


def _chunks(x, n, c):
    """[B, T, H, D] -> [B, H, n, c, D], zero rows behind the last step."""
    b, t, h, d = x.shape
    x = torch.cat([x, x.new_zeros(b, n * c - t, h, d)], 1)
    return x.reshape(b, n, c, h, d).permute(0, 3, 1, 2, 4)


def _attention_forward(q, k, v, log_decay, state, reset):
    """Chunks of 64 steps: products within a chunk, the chunks' own sums of k v^T joined by
    their decays, and the queries' products with the state that enters their chunk."""
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    c = 64
    n = -(-T // c)
    dev = q.device
    seg = torch.zeros(B, T, dtype=torch.int32, device=dev) if reset is None else reset.int().cumsum(1)
    seg_c = torch.cat([seg, seg[:, -1:].expand(B, n * c - T)], 1).reshape(B, n, c)
    end = torch.cat([seg.new_zeros(B, 1), seg_c[:, :, -1]], 1)  # at the end of each chunk, 0 before the first
    i = torch.arange(c, device=dev)
    gap = i[:, None] - i
    weight = torch.where(gap >= 0, torch.exp(gap.clamp(min=0) * log_decay[:, None, None]), 0.0)
    same = seg_c[..., :, None] == seg_c[..., None, :]
    qc, kc, vc = (_chunks(x, n, c) for x in (q, k, v))
    p = (qc @ kc.transpose(-1, -2)) * (weight[None, :, None] * same[:, None])
    out = p @ vc
    keep = torch.exp((c - 1 - i) * log_decay[:, None])[None, :, None] * (seg_c == end[:, 1:, None])[:, None]
    local = (kc * keep[..., None]).transpose(-1, -2) @ vc
    m = torch.arange(n, device=dev)
    gap = m[:, None] - m
    join = torch.where(gap >= 0, torch.exp(gap.clamp(min=0) * c * log_decay[:, None, None]), 0.0)
    join = join[None] * (end[:, :-1, None] == end[:, None, :-1])[:, None]
    sums = torch.cat([state[:, :, None], local[:, :, :-1]], 2)
    enter = (join @ sums.reshape(B, H, n, dk * dv)).reshape(B, H, n, dk, dv)
    reach = torch.exp((i + 1) * log_decay[:, None])[None, :, None] * (seg_c == end[:, :-1, None])[:, None]
    out = out + (qc @ enter) * reach[..., None]
    out = out.permute(0, 2, 3, 1, 4).reshape(B, n * c, H, dv)[:, :T] * dk ** -0.5
    t = torch.arange(T, device=dev)
    left = torch.exp((T - 1 - t)[:, None] * log_decay) * (seg == seg[:, -1:])[..., None]
    last = (k * left[..., None]).permute(0, 2, 3, 1) @ v.transpose(1, 2)
    kept = torch.exp(T * log_decay) * (seg[:, -1:] == 0)
    return out, last + state * kept[..., None, None]


def _attention(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    dt = s["q"].dtype
    if not s["case"]["grad"]:
        out, last = _attention_forward(q, k, v, s["log_decay"], s["state"], s["reset"])
        return out.to(dt), last
    leaves = _leaves(q, k, v, s["state"])
    out, last = _attention_forward(*leaves[:3], s["log_decay"], leaves[3], s["reset"])
    g = torch.autograd.grad((out, last), leaves, (s["dout"].float(), s["dstate"]))
    return out.detach().to(dt), last.detach(), g[0].to(dt), g[1].to(dt), g[2].to(dt), g[3]


def _step(s):
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    state = s["state"] * torch.exp(s["log_decay"])[:, None, None]
    if s["reset"] is not None:
        state = torch.where(s["reset"][:, None, None, None], 0.0, state)
    state = state + k[..., :, None] * v[..., None, :]
    out = (q[..., None, :] @ state)[..., 0, :] * q.shape[-1] ** -0.5
    return out.to(s["q"].dtype), state


def _norm_one(x, w, cos, sin, interleaved):
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    half = cos.shape[-1]
    rot, rest = y[..., : 2 * half], y[..., 2 * half:]
    a, b = (rot[..., 0::2], rot[..., 1::2]) if interleaved else (rot[..., :half], rot[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    rot = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([rot, rest], -1)


def _norm(s):
    case = s["case"]
    angle = (s["positions"][..., None].double() * s["frequencies"])[:, :, None]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    x = [s[n].float() for n in ("q", "k", "q_weight", "k_weight")]
    dt = s["q"].dtype
    if not case["grad"]:
        return tuple(_norm_one(x[i], x[i + 2], cos, sin, case["interleaved"]).to(dt) for i in (0, 1))
    x = _leaves(*x)
    y = [_norm_one(x[i], x[i + 2], cos, sin, case["interleaved"]) for i in (0, 1)]
    g = torch.autograd.grad(y, x, (s["dq"].float(), s["dk"].float()))
    return tuple(t.detach().to(dt) for t in (*y, *g))


def _act(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "tanh":
        return torch.tanh(z)
    if name == "relu":
        return torch.relu(z)
    return z


def _glu(s):
    x, wg, wu = (s[n].float() for n in ("x", "w_gate", "w_up"))
    dt = s["x"].dtype
    if not s["case"]["grad"]:
        return (_act(s["case"]["act"], x @ wg) * (x @ wu)).to(dt)
    x, wg, wu = _leaves(x, wg, wu)
    h = _act(s["case"]["act"], x @ wg) * (x @ wu)
    return tuple(t.detach().to(dt) for t in (h, *torch.autograd.grad(h, (x, wg, wu), s["dh"].float())))


# ---- what a pass cannot do without --------------------------------------------------------------


def work(case):
    e = _BYTES[case["dtype"]]
    if case["op"] in ("attention", "step"):
        bh, dk, dv = case["batch"] * case["heads"], case["dk"], case["dv"]
        n = bh * case.get("steps", 1)
        grad = bool(case.get("grad"))
        row = 2 * dk + 2 * dv + ((2 * dk + 2 * dv) if grad else 0)  # q, k, v, out; dout, dq, dk, dv
        state = 4 * (4 if grad else 2) * bh * dk * dv
        masks = case["batch"] * case.get("steps", 1) if case["resets"] else 0
        return {"bytes": n * row * e + state + masks, "flops": n * dk * dv * (12 if grad else 4)}
    if case["op"] == "norm":
        tokens = case["batch"] * case["steps"]
        n = tokens * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": n * e * (4 if case["grad"] else 2) + tokens * 8, "flops": n * (20 if case["grad"] else 8)}
    M, K, N = case["rows"], case["inner"], case["outer"]
    if case["grad"]:
        return {"bytes": e * (2 * M * K + 2 * M * N + 4 * K * N), "flops": 12 * M * K * N}
    return {"bytes": e * (M * K + M * N + 2 * K * N), "flops": 4 * M * K * N}


# ---- the definitions in 64 bits -------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "step": _exact_step, "norm": _exact_norm,
            "glu": _exact_glu}[case["op"]](s)


def _exact_attention(s):
    """Every pair of steps written out: o_t = scale (sum_{j <= t} e^{(t-j) g} (q_t . k_j) v_j
    + e^{(t+1) g} S^T q_t), pairs across a reset dropped, a few (batch row, head) pairs at a time."""
    case = s["case"]
    B, T, H, dk = s["q"].shape
    dv, dev = s["v"].shape[-1], s["q"].device
    grad = case["grad"]
    scale = 1.0 / math.sqrt(dk)
    fold = lambda x: x.transpose(1, 2).reshape(B * H, T, -1)  # noqa: E731
    q, k, v = (fold(s[n]) for n in ("q", "k", "v"))
    do = fold(s["dout"]) if grad else None
    S = s["state"].reshape(B * H, dk, dv)
    dS = s["dstate"].reshape(B * H, dk, dv) if grad else None
    g = s["log_decay"].double().repeat(B)
    seg = torch.zeros(B, T, device=dev) if s["reset"] is None else s["reset"].double().cumsum(1)
    seg = seg.repeat_interleave(H, 0)
    t = torch.arange(T, device=dev, dtype=torch.float64)
    gap = t[:, None] - t
    f64 = dict(dtype=torch.float64, device=dev)
    out = torch.empty(B * H, T, dv, **f64)
    last = torch.empty(B * H, dk, dv, **f64)
    if grad:
        gq, gk, gv = (torch.empty(B * H, T, d, **f64) for d in (dk, dk, dv))
        g0 = torch.empty(B * H, dk, dv, **f64)
    at_once = max(1, 2 ** 26 // (T * T))
    for a in range(0, B * H, at_once):
        z = slice(a, min(B * H, a + at_once))
        Q, K, V, S0 = (x[z].double() for x in (q, k, v, S))
        sg, ld = seg[z], g[z][:, None]
        w = torch.exp(gap * ld[..., None]).masked_fill_((gap < 0) | (sg[:, :, None] != sg[:, None, :]), 0)
        w *= scale
        p = torch.bmm(Q, K.mT) * w
        into = torch.exp((t + 1) * ld) * (sg == 0) * scale
        outof = torch.exp((T - 1 - t) * ld) * (sg == sg[:, -1:])
        through = (torch.exp(T * ld) * (sg[:, -1:] == 0))[..., None]
        out[z] = torch.bmm(p, V) + into[..., None] * torch.bmm(Q, S0)
        last[z] = torch.bmm((outof[..., None] * K).mT, V) + through * S0
        if grad:
            DO, DS = do[z].double(), dS[z].double()
            dp = torch.bmm(DO, V.mT) * w
            gv[z] = torch.bmm(p.mT, DO) + outof[..., None] * torch.bmm(K, DS)
            gq[z] = torch.bmm(dp, K) + into[..., None] * torch.bmm(DO, S0.mT)
            gk[z] = torch.bmm(dp.mT, Q) + outof[..., None] * torch.bmm(V, DS.mT)
            g0[z] = torch.bmm((into[..., None] * Q).mT, DO) + through * DS
    back = lambda x: x.reshape(B, H, T, -1).transpose(1, 2)  # noqa: E731
    state = lambda x: x.reshape(B, H, dk, dv)  # noqa: E731
    if not grad:
        return back(out), state(last)
    return back(out), state(last), back(gq), back(gk), back(gv), state(g0)


def _exact_step(s):
    q, k, v, S, g = (s[n].double() for n in ("q", "k", "v", "state", "log_decay"))
    keep = torch.exp(g).expand(S.shape[:2])
    if s["reset"] is not None:
        keep = keep * (~s["reset"])[:, None]
    new = torch.einsum("bh,bhij->bhij", keep, S) + torch.einsum("bhi,bhj->bhij", k, v)
    return torch.einsum("bhi,bhij->bhj", q, new) / math.sqrt(q.shape[-1]), new


def _exact_norm(s):
    """The rotation as multiplication by e^{i angle} of the pairs taken as complex numbers."""
    case = s["case"]
    angle = s["positions"].double()[..., None] * s["frequencies"]
    turn = torch.polar(torch.ones_like(angle), angle)[:, :, None]
    half, inter = case["rotary"] // 2, case["interleaved"]

    def rotate(y, by):
        head = y[..., : 2 * half]
        pair = head.unflatten(-1, (half, 2)) if inter else head.unflatten(-1, (2, half)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * by)
        z = z if inter else z.transpose(-1, -2)
        return torch.cat([z.flatten(-2), y[..., 2 * half:]], -1)

    ys, dxs, dws = [], [], []
    for n in ("q", "k"):
        x, w = s[n].double(), s[n + "_weight"].double()
        r = 1 / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
        ys.append(rotate(x * r * w, turn))
        if case["grad"]:
            dy = rotate(s["d" + n].double(), turn.conj())
            dws.append((dy * x * r).sum((0, 1, 2)))
            u = dy * w
            dxs.append(r * u - x * r ** 3 * (u * x).sum(-1, keepdim=True) / x.shape[-1])
    return (*ys, *dxs, *dws)


def _exact_glu(s):
    act = s["case"]["act"]
    x, wg, wu = (s[n].double() for n in ("x", "w_gate", "w_up"))
    g, u = x.mm(wg), x.mm(wu)
    sig = 1 / (1 + torch.exp(-g))
    a = {"silu": lambda: g * sig, "tanh": lambda: torch.tanh(g), "relu": lambda: g * (g > 0), "none": lambda: g}[act]()
    if not s["case"]["grad"]:
        return a * u
    slope = {"silu": lambda: sig + a * (1 - sig), "tanh": lambda: 1 - a * a, "relu": lambda: (g > 0).double(),
             "none": lambda: torch.ones_like(g)}[act]()
    dh = s["dh"].double()
    dg, du = dh * u * slope, dh * a
    return a * u, dg.mm(wg.mT) + du.mm(wu.mT), x.mT.mm(dg), x.mT.mm(du)

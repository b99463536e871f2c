"""The operators a causal mixer with a selective state is made of, as cases that can be prepared, run and timed: the short causal
convolution, the selective state space scan (both for whole prompts, for single tokens, and with their gradients), and group norm with an
activation on channels that lie last.

`own` False: elementary torch operations in 32 bits, rounded once at the end.  `own` True: m2_amd's kernels, as a user calls them.

A case is a dict of plain values:

    kind      "conv", "scan": a prompt's forward; "conv_step", "scan_step": one token more for every sequence; "conv_train", "scan_train":
              forward and gradients of all inputs for given gradients of the outputs; "norm", "norm_train"
    f32       True: fp32 inputs; False: bf16
    B, L, C   sequences, positions, channels (steps: L = 1)
    K         "conv*": taps
    N, G      "scan*": states a channel, groups of channels that share B and C; "norm*": G groups of channels
    silu      "conv*": SiLU on the way out
    gate      "scan*": y * silu(z)
    act       "norm*": "", "silu" or "gelu"
    state     "conv*", "scan*": the sequences go on from a state that they bring along
    ragged    "conv*", "scan*": sequences of different lengths, padded to L; one of them empty where there are more than two
"""
from __future__ import annotations

import math

import torch

own = False


def _conv(name, kind, B, L, C, K, f32=False, silu=True, state=False, ragged=False):
    case = {"kind": kind, "B": B, "L": L, "C": C, "K": K, "f32": f32, "silu": silu, "state": state, "ragged": ragged}
    return dict(case, name=name) if name else case


def _scan(name, kind, B, L, C, N, G=1, f32=False, gate=True, state=False, ragged=False):
    case = {"kind": kind, "B": B, "L": L, "C": C, "N": N, "G": G, "f32": f32, "gate": gate, "state": state, "ragged": ragged}
    return dict(case, name=name) if name else case


def _norm(name, kind, B, L, C, G, f32=False, act="silu"):
    case = {"kind": kind, "B": B, "L": L, "C": C, "G": G, "f32": f32, "act": act}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one token of one sequence, twice the 768-wide model's channels: latency
        _conv("conv_step_1x1536", "conv_step", 1, 1, 1536, 4, state=True),
        # prompts of the longest training context
        _conv("conv_4x8192x1536", "conv", 4, 8192, 1536, 4),
        # training on padded texts that go on from an earlier part, fp32, twice the 960-wide model's channels
        _conv("conv_train_8x2049x1920_f32", "conv_train", 8, 2049, 1920, 3, f32=True, state=True, ragged=True),
        # one token of one sequence
        _scan("scan_step_1x1536x16", "scan_step", 1, 1, 1536, 16, state=True),
        # one token each of a batch that is served, twice the 1792-wide model's channels and many states: nothing but states
        _scan("scan_step_64x3584x64", "scan_step", 64, 1, 3584, 64, state=True),
        # a single long prompt
        _scan("scan_1x8192x1536x16", "scan", 1, 8192, 1536, 16),
        # a batch of long prompts: the compute-heavy end
        _scan("scan_4x8192x1536x16", "scan", 4, 8192, 1536, 16),
        # padded texts in fp32 that go on from states, odd sizes, groups of channels, no gate
        _scan("scan_5x1013x1002x61_f32", "scan", 5, 1013, 1002, 61, G=3, f32=True, gate=False, state=True, ragged=True),
        # a training batch
        _scan("scan_train_8x2048x1536x16", "scan_train", 8, 2048, 1536, 16),
        # heads of 64 channels of every token, behind a mixer
        _norm("norm_32768x1536_heads", "norm", 32768, 1, 1536, 24),
        # whole sequences in fp32, odd length
        _norm("norm_3x4001x960_f32", "norm", 3, 4001, 960, 20, f32=True, act=""),
        # training on sequences
        _norm("norm_train_8x2048x1536", "norm_train", 8, 2048, 1536, 32),
    ]


def _between(rng, low, high):
    """A whole number between two, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["conv", "conv_train", "conv_step", "scan", "scan", "scan_train", "scan_train", "scan_step", "norm", "norm_train"])
    f32 = rng.random() < 0.4
    size = 2 if f32 else 1
    while True:
        B, L, C = _between(rng, 1, 64), _between(rng, 1, 8192), rng.choice([768, 1536, 1920, 3584, _between(rng, 64, 4096)])
        if kind.endswith("step"):
            B, L = _between(rng, 1, 256), 1
        state, ragged = kind.endswith("step") or rng.random() < 0.4, L > 1 and rng.random() < 0.4
        if kind.startswith("conv"):
            if B * L * C * size <= 4 * 8192 * 1536 // (2 if kind == "conv_train" else 1):
                return _conv("", kind, B, L, C, rng.choice([4, 4, 3, rng.randint(1, 8)]), f32, rng.random() < 0.7, state, ragged)
        elif kind.startswith("scan"):
            N, G = rng.choice([16, 16, 64, _between(rng, 1, 128)]), rng.choice([1, 1, 1, 2, 4])
            C += -C % G
            if B * L * C * N * size <= {"scan": 4 * 8192 * 1536 * 16, "scan_train": 8 * 2048 * 1536 * 16, "scan_step": 256 * 4096 * 128}[kind]:
                return _scan("", kind, B, L, C, N, G, f32, rng.random() < 0.7, state, ragged)
        else:
            if rng.random() < 0.5:
                B, L = _between(rng, 1, 32768), 1
            G = rng.choice([1, 8, 20, 24, 32, _between(rng, 1, 64)])
            C += -C % G
            if B * L * C * size <= 32768 * 1536 // (2 if kind == "norm_train" else 1):
                return _norm("", kind, B, L, C, G, f32, rng.choice(["", "silu", "silu", "gelu"]))


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 9973 + 31)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device=dev)

    kind, B, L, C = case["kind"], case["B"], case["L"], case["C"]
    dtype = torch.float32 if case["f32"] else torch.bfloat16
    step, train = kind.endswith("step"), kind.endswith("train")
    s = {"case": case}
    if kind.startswith("norm"):
        shape = (B, C) if L == 1 else (B, L, C)
        # channels with means and sizes of their own
        s["x"] = (randn(*shape) * (0.5 + rand(C)) + 0.5 * randn(C)).to(dtype)
        s["weight"], s["bias"] = 1 + 0.2 * randn(C), 0.2 * randn(C)
        if train:
            s["gy"] = randn(*shape).to(dtype)
        return s
    s["lengths"] = None
    if case["ragged"]:
        s["lengths"] = torch.randint(L // 3, L + 1, (B,), generator=gen, device=dev)
        s["lengths"][0] = L
        if B > 2:
            s["lengths"][B // 2] = 0
    if kind.startswith("conv"):
        K = case["K"]
        # one half of an in-projection's result: rows lie two widths apart
        s["x"] = randn(B, L, 2 * C).to(dtype)[..., :C]
        s["weight"], s["bias"] = randn(C, K) / math.sqrt(K), 0.2 * randn(C)
        s["state"] = randn(B, K - 1, C).to(dtype) if case["state"] else None
        if step:
            s["x"], s["next"] = s["x"][:, 0], torch.empty_like(s["state"])
        if train:
            s["gy"], s["gstate"] = randn(B, L, C).to(dtype), randn(B, K - 1, C).to(dtype)
        return s
    N, G = case["N"], case["G"]
    s["x"] = torch.nn.functional.silu(randn(B, L, C)).to(dtype)
    s["dt"] = (0.5 * randn(B, L, C)).to(dtype)
    # step sizes of 0.001 to 0.1, spread over their logarithm, behind the softplus
    sizes = torch.exp(rand(C) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    s["dt_bias"] = sizes + torch.log(-torch.expm1(-sizes))
    # decays of 1 .. N, as a model starts with, moved a little by training
    s["A"] = -torch.arange(1, N + 1, device=dev, dtype=torch.float32) * torch.exp(0.1 * randn(C, N))
    # B and C behind a low-rank part in one projection's result
    low = C // 16
    proj = randn(B, L, low + 2 * G * N).to(dtype)
    s["Bm"], s["Cm"] = proj[..., low:low + G * N].unflatten(-1, (G, N)), proj[..., low + G * N:].unflatten(-1, (G, N))
    s["D"] = 1 + 0.2 * randn(C)
    s["z"] = randn(B, L, 2 * C).to(dtype)[..., C:] if case["gate"] else None
    s["state"] = 0.5 * randn(B, C, N) if case["state"] else None
    if step:
        for name in ("x", "dt", "z", "Bm", "Cm"):
            if s[name] is not None:
                s[name] = s[name][:, 0]
        s["next"] = torch.empty_like(s["state"])
    if train:
        s["gy"], s["gstate"] = randn(B, L, C).to(dtype), 0.1 * randn(B, C, N)
    return s


def _silu(x):
    return x / (1 + torch.exp(-x))


def _silu_slope(x):
    p = 1 / (1 + torch.exp(-x))
    return p * (1 + x * (1 - p))


def _valid(state, L):
    """(B, L, 1): positions that belong to a sequence; None: all."""
    if state["lengths"] is None:
        return None
    return (torch.arange(L, device=state["lengths"].device) < state["lengths"].unsqueeze(1)).unsqueeze(-1)


def _plain_conv(s):
    case, K = s["case"], s["case"]["K"]
    x, w, b = s["x"].float(), s["weight"], s["bias"]
    if case["kind"] == "conv_step":
        rows = torch.cat((s["state"].float(), x.unsqueeze(1)), 1)
        pre = b + (rows * w.t()).sum(1)
        return {"y": (_silu(pre) if case["silu"] else pre).to(s["x"].dtype), "state": rows[:, 1:].to(s["x"].dtype)}
    B, L, C = x.shape
    valid = _valid(s, L)
    before = s["state"].float() if s["state"] is not None else x.new_zeros(B, K - 1, C)
    rows = torch.cat((before, x), 1)
    pre = b + sum(w[:, k] * rows[:, k:k + L] for k in range(K))
    y = _silu(pre) if case["silu"] else pre
    if valid is not None:
        y = torch.where(valid, y, torch.zeros_like(y))
    first = s["lengths"] if valid is not None else torch.full((B,), L, device=x.device)
    at = (first.unsqueeze(1) + torch.arange(K - 1, device=x.device)).unsqueeze(-1).expand(B, K - 1, C)
    out = {"y": y.to(s["x"].dtype), "state": rows.gather(1, at).to(s["x"].dtype)}
    if case["kind"] == "conv_train":
        g = s["gy"].float()
        if case["silu"]:
            g = g * _silu_slope(pre)
        if valid is not None:
            g = torch.where(valid, g, torch.zeros_like(g))
        grad = torch.zeros_like(rows)
        for k in range(K):
            grad[:, k:k + L] += w[:, k] * g
        grad.scatter_add_(1, at, s["gstate"].float())
        out["grad_x"] = grad[:, K - 1:].to(s["x"].dtype)
        out["grad_weight"] = torch.stack([(g * rows[:, k:k + L]).sum((0, 1)) for k in range(K)], -1)
        out["grad_bias"] = g.sum((0, 1))
        if s["state"] is not None:
            out["grad_state"] = grad[:, :K - 1].to(s["x"].dtype)
    return out


def _softplus(x):
    return x.clamp_min(0) + torch.log1p(torch.exp(-x.abs()))


def _plain_scan(s):
    case = s["case"]
    dtype, step, train = s["x"].dtype, case["kind"] == "scan_step", case["kind"] == "scan_train"
    G, N = case["G"], case["N"]

    def first(t):
        """(L, B, ...) in 32 bits"""
        t = t.float()
        return t.unsqueeze(0) if step else t.transpose(0, 1)

    x, raw = first(s["x"]), first(s["dt"]) + s["dt_bias"]
    L, B, C = x.shape
    d = _softplus(raw)
    valid = None if step else _valid(s, L)
    if valid is not None:
        valid = valid.transpose(0, 1)
        d = torch.where(valid, d, torch.zeros_like(d))
    bm, cm = first(s["Bm"]).unsqueeze(3), first(s["Cm"]).unsqueeze(3)            # L, B, G, 1, N
    grouped = (L, B, G, C // G, N)
    a = torch.exp(d.unsqueeze(-1) * s["A"])
    h = ((d * x).view(L, B, G, C // G, 1) * bm).view(L, B, C, N)
    h0 = s["state"] if s["state"] is not None else x.new_zeros(B, C, N)
    last = h0
    for at, ht in zip(a.unbind(0), h.unbind(0)):
        last = ht.addcmul_(at, last)
    yv = (h.view(grouped) * cm).sum(-1).view(L, B, C) + s["D"] * x
    z = first(s["z"]) if s["z"] is not None else None
    y = yv * _silu(z) if z is not None else yv
    if valid is not None:
        y = torch.where(valid, y, torch.zeros_like(y))

    def back(t):
        return (t[0] if step else t.transpose(0, 1).contiguous()).to(dtype)

    out = {"y": back(y), "state": last.clone()}
    if train:
        u = first(s["gy"])
        if valid is not None:
            u = torch.where(valid, u, torch.zeros_like(u))
        if z is not None:
            out["grad_z"] = back(u * yv * _silu_slope(z))
            u = u * _silu(z)
        u5 = u.view(L, B, G, C // G, 1)
        out["grad_C"] = back((u5 * h.view(grouped)).sum(3))
        out["grad_D"] = (u * x).sum((0, 1))
        dh = (u5 * cm).view(L, B, C, N).clone()
        carry = s["gstate"]
        steps, decays = dh.unbind(0), a.unbind(0)
        for t in range(L - 1, -1, -1):
            carry = steps[t].add_(carry) if t == L - 1 else steps[t].addcmul_(decays[t + 1], carry)
        if s["state"] is not None:
            out["grad_state"] = a[0] * dh[0]
        into = (dh.view(grouped) * bm).sum(-1).view(L, B, C)
        out["grad_B"] = back((dh.view(grouped) * (d * x).view(L, B, G, C // G, 1)).sum(3))
        a[1:] *= h[:-1]                                   # from here on what a step keeps of the state before it
        a[0] *= h0
        a *= dh
        dd = (a * s["A"]).sum(-1) + x * into
        out["grad_A"] = (a * d.unsqueeze(-1)).sum((0, 1))
        g_raw = dd / (1 + torch.exp(-raw))
        if valid is not None:
            g_raw = torch.where(valid, g_raw, torch.zeros_like(g_raw))
        out["grad_dt"], out["grad_dt_bias"] = back(g_raw), g_raw.sum((0, 1))
        out["grad_x"] = back(d * into + s["D"] * u)
    return out


def _plain_norm(s):
    case, C, G = s["case"], s["case"]["C"], s["case"]["G"]
    shape = s["x"].shape
    x = s["x"].float().view(case["B"], -1, G, C // G)
    centred = x - x.mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-5)
    xh = centred * r
    w, b = s["weight"].view(G, -1), s["bias"].view(G, -1)
    pre = xh * w + b
    half = 0.5 * (1 + torch.erf(pre * math.sqrt(0.5)))
    y = {"": lambda: pre, "silu": lambda: _silu(pre), "gelu": lambda: pre * half}[case["act"]]()
    out = {"y": y.reshape(shape).to(s["x"].dtype)}
    if case["kind"] == "norm_train":
        g = s["gy"].float().view_as(x)
        if case["act"] == "silu":
            g = g * _silu_slope(pre)
        elif case["act"] == "gelu":
            g = g * (half + pre * torch.exp(-0.5 * pre * pre) * (1 / math.sqrt(2 * math.pi)))
        out["grad_weight"], out["grad_bias"] = (g * xh).sum((0, 1)).view(C), g.sum((0, 1)).view(C)
        g = g * w
        grad = r * (g - g.mean((1, 3), keepdim=True) - xh * (g * xh).mean((1, 3), keepdim=True))
        out["grad_x"] = grad.reshape(shape).to(s["x"].dtype)
    return out


def _leaf(t):
    return None if t is None else t.detach().requires_grad_()


def _own_conv(s):
    import m2_amd
    case = s["case"]
    act = "silu" if case["silu"] else None
    if case["kind"] == "conv_step":
        # the state before the token is kept, as a program does that may take a token back
        y = m2_amd.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], activation=act, out_state=s["next"])
        return {"y": y, "state": s["next"]}
    if case["kind"] == "conv":
        y, state = m2_amd.causal_conv(s["x"], s["weight"], s["bias"], activation=act, state=s["state"], lengths=s["lengths"], return_state=True)
        return {"y": y, "state": state}
    ins = {"x": _leaf(s["x"]), "weight": _leaf(s["weight"]), "bias": _leaf(s["bias"])}
    if s["state"] is not None:
        ins["state"] = _leaf(s["state"])
    y, state = m2_amd.causal_conv(ins["x"], ins["weight"], ins["bias"], activation=act, state=ins.get("state"), lengths=s["lengths"], return_state=True)
    outs, given = ([y, state], [s["gy"], s["gstate"]]) if case["K"] > 1 else ([y], [s["gy"]])
    grads = torch.autograd.grad(outs, list(ins.values()), given, allow_unused=True)
    found = {"y": y.detach(), "state": state.detach()}
    for (name, t), g in zip(ins.items(), grads):
        found["grad_" + name] = torch.zeros_like(t) if g is None else g
    return found


def _own_scan(s):
    import m2_amd
    case = s["case"]
    if case["kind"] == "scan_step":
        y = m2_amd.selective_scan_step(s["x"], s["dt"], s["state"], s["A"], s["Bm"], s["Cm"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"], dt_softplus=True,
                                       out_state=s["next"])
        return {"y": y, "state": s["next"]}

    def call(i):
        return m2_amd.selective_scan(i["x"], i["dt"], i["A"], i["B"], i["C"], D=i["D"], z=i.get("z"), dt_bias=i["dt_bias"], dt_softplus=True,
                                     state=i.get("state"), lengths=s["lengths"], return_state=True)

    ins = {"x": s["x"], "dt": s["dt"], "A": s["A"], "B": s["Bm"], "C": s["Cm"], "D": s["D"], "dt_bias": s["dt_bias"]}
    for name in ("z", "state"):
        if s[name] is not None:
            ins[name] = s[name]
    if case["kind"] == "scan":
        y, state = call(ins)
        return {"y": y, "state": state}
    ins = {name: _leaf(t) for name, t in ins.items()}
    y, state = call(ins)
    grads = torch.autograd.grad([y, state], list(ins.values()), [s["gy"], s["gstate"]])
    return {"y": y.detach(), "state": state.detach(), **{"grad_" + name: g for name, g in zip(ins, grads)}}


def _own_norm(s):
    import m2_amd
    case = s["case"]
    act = case["act"] or None
    if case["kind"] == "norm":
        return {"y": m2_amd.group_norm(s["x"], case["G"], s["weight"], s["bias"], activation=act)}
    x, w, b = _leaf(s["x"]), _leaf(s["weight"]), _leaf(s["bias"])
    y = m2_amd.group_norm(x, case["G"], w, b, activation=act)
    gx, gw, gb = torch.autograd.grad(y, [x, w, b], s["gy"])
    return {"y": y.detach(), "grad_x": gx, "grad_weight": gw, "grad_bias": gb}


def run(state):
    kind = state["case"]["kind"]
    if kind.startswith("conv"):
        return _own_conv(state) if own else _plain_conv(state)
    if kind.startswith("scan"):
        return _own_scan(state) if own else _plain_scan(state)
    return _own_norm(state) if own else _plain_norm(state)


def work(case):
    kind, B, L, C = case["kind"], case["B"], case["L"], case["C"]
    size, values = 4 if case["f32"] else 2, B * L * C
    train = kind.endswith("train")
    if kind.startswith("norm"):
        # x and y; with gradients gy and the gradient of x
        return {"bytes": size * values * (4 if train else 2) + 4 * C * (4 if train else 2), "flops": (30 if train else 12) * values}
    if kind.startswith("conv"):
        K = case["K"]
        states = B * (K - 1) * C * size * ((2 if case["state"] else 1) + (2 if train and case["state"] else train))
        return {"bytes": size * values * (4 if train else 2) + states + 4 * C * (K + 1) * (2 if train else 1), "flops": (6 * K + 16 if train else 2 * K + 5) * values}
    N, G = case["N"], case["G"]
    wide = 4 if case["gate"] else 3                       # x, dt, y and z
    wide = 2 * wide if train else wide                    # and as many gradients
    states = 4 * B * C * N * ((2 if case["state"] else 1) + (2 if train and case["state"] else train))
    shared = size * B * L * G * N * (4 if train else 2)
    return {"bytes": size * values * wide + shared + states + 4 * C * (N + 2) * (2 if train else 1), "flops": (22 if train else 7) * values * N}


def _exact_conv(s):
    """Every output from its window of inputs; gradients by differentiating that."""
    case, K = s["case"], s["case"]["K"]
    step, train = case["kind"] == "conv_step", case["kind"] == "conv_train"
    x, w, b = (s["x"].unsqueeze(1) if step else s["x"]).double(), s["weight"].double(), s["bias"].double()
    B, L, C = x.shape
    h = s["state"].double() if s["state"] is not None else torch.zeros(B, K - 1, C, dtype=torch.float64, device=x.device)
    if train:
        for t in (x, w, b, h):
            t.requires_grad_()
    with torch.set_grad_enabled(train):
        rows = torch.cat([h, x], dim=1)
        pre = torch.matmul(rows.unfold(1, K, 1).unsqueeze(-2), w.unsqueeze(-1)).squeeze(-1).squeeze(-1) + b
        y = pre * torch.sigmoid(pre) if case["silu"] else pre
        ends = [L] * B if s["lengths"] is None else s["lengths"].tolist()
        y = torch.stack([torch.cat([y[i, :n], torch.zeros_like(y[i, n:])]) for i, n in enumerate(ends)])
        last = torch.stack([rows[i, n:n + K - 1] for i, n in enumerate(ends)])
    out = {"y": y[:, 0] if step else y.detach(), "state": last.detach()}
    if train:
        gx, gw, gb, gh = torch.autograd.grad([y, last], [x, w, b, h], [s["gy"].double(), s["gstate"].double()], allow_unused=True)
        out.update(grad_x=gx, grad_weight=gw, grad_bias=gb)
        if s["state"] is not None:
            out["grad_state"] = torch.zeros_like(h) if gh is None else gh
    return out


def _exact_scan(s):
    """The recurrence, token by token; gradients by differentiating it."""
    case, G, N = s["case"], s["case"]["G"], s["case"]["N"]
    step, train = case["kind"] == "scan_step", case["kind"] == "scan_train"
    names = [n for n in ("x", "dt", "A", "Bm", "Cm", "D", "dt_bias", "z", "state") if s[n] is not None]
    v = {n: s[n].double().clone() for n in names}
    if step:
        v = {n: t.unsqueeze(1) if n in ("x", "dt", "Bm", "Cm", "z") else t for n, t in v.items()}
    B, L, C = v["x"].shape
    if train:
        for t in v.values():
            t.requires_grad_()
    ys = []
    with torch.set_grad_enabled(train):
        h = v["state"] if "state" in v else torch.zeros(B, C, N, dtype=torch.float64, device=s["x"].device)
        d = torch.logaddexp(v["dt"] + v["dt_bias"], torch.zeros_like(v["dt_bias"]))
        if s["lengths"] is not None:
            inside = (torch.arange(L, device=h.device)[None, :] < s["lengths"][:, None])[..., None].double()
            d = d * inside
        for xt, dt, bt, ct in zip(v["x"].unbind(1), d.unbind(1), v["Bm"].unbind(1), v["Cm"].unbind(1)):
            bt, ct = bt.repeat_interleave(C // G, 1), ct.repeat_interleave(C // G, 1)
            h = torch.exp(dt[..., None] * v["A"]) * h + (dt * xt)[..., None] * bt
            ys.append(torch.matmul(h.unsqueeze(-2), ct.unsqueeze(-1))[..., 0, 0])
        y = torch.stack(ys, 1) + v["D"] * v["x"]
        del ys
        if "z" in v:
            y = y * (v["z"] * torch.sigmoid(v["z"]))
        if s["lengths"] is not None:
            y = y * inside
    out = {"y": y[:, 0] if step else y.detach(), "state": h.detach()}
    if train:
        grads = torch.autograd.grad([y, h], list(v.values()), [s["gy"].double(), s["gstate"].double()])
        out.update({"grad_" + n.replace("m", ""): g for n, g in zip(v, grads)})
    return out


def _exact_norm(s):
    """Mean and variance of each group; gradients by differentiating that."""
    case, C, G = s["case"], s["case"]["C"], s["case"]["G"]
    train = case["kind"] == "norm_train"
    x, w, b = s["x"].double(), s["weight"].double(), s["bias"].double()
    if train:
        for t in (x, w, b):
            t.requires_grad_()
    with torch.set_grad_enabled(train):
        rows = x.reshape(case["B"], -1, G, C // G).transpose(1, 2).flatten(2)
        var, mean = torch.var_mean(rows, dim=2, unbiased=False)
        rows = (rows - mean[..., None]) / torch.sqrt(var + 1e-5)[..., None]
        y = rows.view(case["B"], G, -1, C // G).transpose(1, 2).reshape(x.shape) * w + b
        if case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu":
            y = y * torch.special.ndtr(y)
    out = {"y": y.detach()}
    if train:
        out["grad_x"], out["grad_weight"], out["grad_bias"] = torch.autograd.grad(y, [x, w, b], s["gy"].double())
    return out


def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    if case["kind"].startswith("conv"):
        return _exact_conv(state)
    return _exact_scan(state) if case["kind"].startswith("scan") else _exact_norm(state)

"""Workloads of the sequence operators: the gated linear recurrence, the block norms and the
8-bit activation checkpoints, each with its plain form in elementary torch operations."""

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
GROUP = 32      # channels that share a scale in 8 bits
SEGMENT = 16    # steps between the states that an 8-bit checkpoint of the recurrence keeps
EPS = 1e-5


def _package():
    path = os.path.join(os.getcwd(), "snn-delays_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import delrec.block_norm
    import delrec.checkpoint8
    import delrec.gated
    import delrec.linear
    return delrec


# ------------------------------------------------------------------------------- cases


def listed():
    return [
        # one time step of a streaming batch of 256 sensors or users: latency
        {"name": "step", "op": "step", "T": 1, "B": 256, "N": 512, "D": 1, "dtype": "fp32", "decay_input": True},
        # a long recording taken in at once, one sequence: the scan splits over time
        {"name": "prefill_long", "op": "scan", "T": 65536, "B": 1, "N": 512, "D": 1, "dtype": "bf16",
         "decay_input": True, "train": False, "ragged": False, "bits8": False, "gate_mean": 4.0},
        # the event-stream model's hidden layer (250 bins, batch 256, 512 wide) in training
        {"name": "scan_train", "op": "scan", "T": 250, "B": 256, "N": 512, "D": 1, "dtype": "fp32",
         "decay_input": False, "train": True, "ragged": False, "bits8": False, "gate_mean": 2.0},
        # a padded batch of recordings with a gate per head of 65 channels and packed pieces
        {"name": "scan_train_heads", "op": "scan", "T": 1021, "B": 24, "N": 520, "D": 65, "dtype": "bf16",
         "decay_input": True, "train": True, "ragged": True, "bits8": False, "gate_mean": 3.0},
        # the long-horizon task's length (784 steps), its inputs kept in 8 bits for the backward pass
        {"name": "scan_train_8bit", "op": "scan", "T": 784, "B": 256, "N": 512, "D": 1, "dtype": "bf16",
         "decay_input": True, "train": True, "ragged": False, "bits8": True, "gate_mean": 3.0},
        # one time step of 64 streams between two blocks: latency
        {"name": "join_step", "op": "join", "T": 1, "B": 64, "N": 512, "dtype": "bf16", "gate": "sigmoid",
         "next": True, "train": False, "ragged": False},
        # between two blocks of the event-stream model in training
        {"name": "join_train", "op": "join", "T": 250, "B": 256, "N": 512, "dtype": "fp32", "gate": "silu",
         "next": True, "train": True, "ragged": False},
        # the widest hidden size of the long-horizon sweep
        {"name": "join_train_wide", "op": "join", "T": 784, "B": 64, "N": 2048, "dtype": "bf16",
         "gate": "sigmoid", "next": True, "train": True, "ragged": False},
        # after the last block, a padded batch, 700 channels
        {"name": "join_train_last", "op": "join", "T": 333, "B": 37, "N": 700, "dtype": "fp16",
         "gate": "none", "next": False, "train": True, "ragged": True},
        # the event-stream input (700 channels) put away and brought back
        {"name": "checkpoint", "op": "pack", "T": 250, "B": 256, "N": 700, "dtype": "fp32"},
        # a small model's activations: latency
        {"name": "checkpoint_small", "op": "pack", "T": 128, "B": 64, "N": 128, "dtype": "bf16"},
        # the event-stream model's first projection, its input kept in 8 bits: a training pass
        {"name": "linear_8bit", "op": "linear", "T": 250, "B": 256, "K": 700, "N": 512, "dtype": "fp32",
         "spikes": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["step", "scan", "scan", "scan", "join", "join", "pack", "linear"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "step":
        D = rng.choice([1, 1, rng.randint(2, 80)])
        return {"op": op, "T": 1, "B": _log(rng, 1, 1024), "N": D * max(1, _log(rng, 32, 2048) // D), "D": D,
                "dtype": dtype, "decay_input": rng.random() < 0.5}
    if op == "scan":
        D = rng.choice([1, 1, 1, rng.randint(2, 130)])
        N = D * max(1, _log(rng, 48, 2048) // D)
        B = _log(rng, 1, 256)
        T = _log(rng, 2, max(2, min(65536, 32_000_000 // (B * N))))
        return {"op": op, "T": T, "B": B, "N": N, "D": D, "dtype": dtype, "decay_input": rng.random() < 0.5,
                "train": rng.random() < 0.7, "ragged": rng.random() < 0.4, "bits8": rng.random() < 0.3,
                "gate_mean": rng.choice([0.0, 2.0, 4.0])}
    if op == "join":
        N = _log(rng, 32, 8192)
        B = _log(rng, 1, 256)
        T = _log(rng, 1, max(1, min(4096, 32_000_000 // (B * N))))
        return {"op": op, "T": T, "B": B, "N": N, "dtype": dtype, "gate": rng.choice(["none", "sigmoid", "silu"]),
                "next": rng.random() < 0.7, "train": rng.random() < 0.7, "ragged": rng.random() < 0.4}
    if op == "pack":
        N = _log(rng, 1, 4096)
        B = _log(rng, 1, 256)
        return {"op": op, "T": _log(rng, 1, max(1, min(4096, 32_000_000 // (B * N)))), "B": B, "N": N, "dtype": dtype}
    K, N, B = _log(rng, 32, 1024), _log(rng, 32, 1024), _log(rng, 8, 256)
    return {"op": "linear", "T": _log(rng, 16, max(16, min(784, 60_000 // B))), "B": B, "K": K, "N": N,
            "dtype": "fp32", "spikes": rng.random() < 0.5}


# ------------------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    T, B, N = case["T"], case["B"], case["N"]

    def normal(*shape, mean=0.0, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    s = {"case": dict(case)}
    op = case["op"]
    if op == "step":
        s["z"] = normal(B, N)
        s["f"] = normal(B, N // case["D"], mean=2.0, std=1.5)
        s["state"] = normal(B, N, dtype=torch.float32)
        return s
    if op == "linear":
        x = normal(T, B, case["K"])
        s["x"] = (x > 1.5).to(dt) if case["spikes"] else x
        s["w"] = normal(N, case["K"], std=case["K"] ** -0.5)
        s["b"] = normal(N, std=0.1)
        s["g"] = normal(T, B, N, std=0.01)
        for k in ("x", "w", "b"):
            s[k].requires_grad_(True)
        return s
    if op == "pack":
        s["x"] = normal(T, B, N) * torch.exp(normal(T, B, 1, dtype=torch.float32)).to(dt)
        return s
    s["lengths"] = None
    if case["ragged"]:
        n = torch.randint(0, T + 1, (B,), generator=g, device="cuda")
        n[int(seed) % B] = T
        s["lengths"] = n.to(torch.int32)
    if op == "scan":
        s["z"] = normal(T, B, N)
        s["f"] = normal(T, B, N // case["D"], mean=case["gate_mean"], std=1.5)
        s["h0"] = normal(B, N, dtype=torch.float32)
        s["resets"] = torch.rand(T, B, generator=g, device="cuda") < 4.0 / T if case["ragged"] else None
        if case["train"]:
            s["gh"] = normal(T, B, N, std=0.01)
            s["ghT"] = normal(B, N, std=0.01, dtype=torch.float32)
        leaves = ("z", "f", "h0")
    else:
        s["x"] = normal(T, B, N, std=1.5)
        s["y"] = normal(T, B, N, std=0.7)
        s["w"] = normal(N, mean=1.0, std=0.1, dtype=torch.float32)
        s["scale"] = normal(N, mean=0.5, std=0.1, dtype=torch.float32)
        s["u"] = normal(T, B, N) if case["gate"] != "none" else None
        s["nw"] = normal(N, mean=1.0, std=0.1, dtype=torch.float32) if case["next"] else None
        if case["train"]:
            s["gx"] = normal(T, B, N, std=0.01)
            s["gn"] = normal(T, B, N, std=0.01) if case["next"] else None
        leaves = ("x", "y", "u", "w", "scale", "nw")
    if case["train"]:
        for k in leaves:
            if s[k] is not None:
                s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------------- plain forms, 32 bits


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 0 from h = 0, and the running products of a:
    the affine maps of 1, 2, 4, ... steps put together."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], a[d:] * b[:-d] + b[d:]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b, a


def _valid(T, lengths, like):
    if lengths is None:
        return None
    return (torch.arange(T, device=like.device)[:, None] < lengths[None, :]).unsqueeze(-1)


def _spread(f, D):
    return f if D == 1 else f.repeat_interleave(D, -1)


def _plain8(x):
    """What x (float32) stands for after 8 bits."""
    N = x.shape[-1]
    p = torch.nn.functional.pad(x, (0, -N % GROUP)).unflatten(-1, (-1, GROUP))
    m, e = torch.frexp(p.abs().amax(-1, keepdim=True))
    e = torch.where(m > 126.0 / 128.0, e + 1, e) - 7
    e = torch.where(m == 0, torch.full_like(e, -126), e).clamp(min=-126).int()
    up, down = ((127 + e) << 23).view(torch.float32), ((127 - e) << 23).view(torch.float32)
    return (torch.round(p * down) * up).flatten(-2)[..., :N]


def _coefficients(z, f, case, valid, resets):
    """(a as it acts on the state, sigmoid, 1 - sigmoid, factor of z), identities at padded steps."""
    D = case["D"]
    a, om = torch.sigmoid(f), torch.sigmoid(-f)
    a, om = _spread(a, D), _spread(om, D)
    act = a if resets is None else torch.where(resets.unsqueeze(-1), torch.zeros_like(a), a)
    c = om if case["decay_input"] else torch.ones_like(om)
    if valid is not None:
        act = torch.where(valid, act, torch.ones_like(act))
        c = torch.where(valid, c, torch.zeros_like(c))
    return act, a, om, c


def _plain_scan(s):
    case, lengths, resets = s["case"], s["lengths"], s["resets"]
    T, B, N, D = case["T"], case["B"], case["N"], case["D"]
    dt = s["z"].dtype
    z, f, h0 = s["z"].detach().float(), s["f"].detach().float(), s["h0"].detach()
    valid = _valid(T, lengths, z)
    act, a, om, c = _coefficients(z, f, case, valid, resets)
    h, p = _scan(act, c * z)
    h = h + p * h0
    out = h if valid is None else torch.where(valid, h, torch.zeros_like(h))
    res = [out.to(dt), h[-1].clone()]
    if not case["train"]:
        return res
    before = torch.cat([h0[None], h[:-1]])
    if case["bits8"]:
        z, f = _plain8(z), _plain8(f)
        act, a, om, c = _coefficients(z, f, case, valid, resets)
        first = before[::SEGMENT]
        pad = -T % SEGMENT
        cut = lambda v: torch.nn.functional.pad(v, (0, 0, 0, 0, 0, pad)).unflatten(0, (-1, SEGMENT)).transpose(0, 1)  # noqa: E731
        hs, ps = _scan(cut(act), cut(c * z))
        hs = hs + ps * first
        before = torch.cat([first[None], hs[:-1]]).transpose(0, 1).flatten(0, 1)[:T]
    gh = s["gh"].float()
    if valid is not None:
        gh = torch.where(valid, gh, torch.zeros_like(gh))
    nxt = torch.cat([act[1:], torch.ones_like(act[:1])])
    G, q = _scan(nxt.flip(0), gh.flip(0))
    G = (G + q * s["ghT"]).flip(0)
    if resets is not None:
        before = torch.where(resets.unsqueeze(-1), torch.zeros_like(before), before)
    df = a * om * G * (before - z if case["decay_input"] else before)
    if valid is not None:
        df = torch.where(valid, df, torch.zeros_like(df))
    if D > 1:
        df = df.unflatten(-1, (-1, D)).sum(-1)
    return res + [(c * G).to(dt), df.to(dt), act[0] * G[0]]


def _act(u, kind):
    """act(u) and its derivative."""
    if kind == "none":
        return 1.0, None
    sg, so = torch.sigmoid(u), torch.sigmoid(-u)
    return (sg, sg * so) if kind == "sigmoid" else (u * sg, sg * (1.0 + u * so))


def _plain_join(s):
    case = s["case"]
    dt = s["x"].dtype
    valid = _valid(case["T"], s["lengths"], s["x"])
    clean = lambda v: v if valid is None else torch.where(valid, v, torch.zeros_like(v))  # noqa: E731
    load = lambda k: None if s[k] is None else clean(s[k].detach().float())  # noqa: E731
    x, y, u = load("x"), load("y"), load("u")
    w, sc = s["w"].detach(), s["scale"].detach()
    ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + EPS)
    yh = y * ry
    c, dc = _act(u, case["gate"])
    new = x + sc * c * (yh * w)
    res = [new.to(dt)]
    if case["next"]:
        nw = s["nw"].detach()
        rx = torch.rsqrt(new.square().mean(-1, keepdim=True) + EPS)
        xh = new * rx
        res.append((xh * nw).to(dt))
    if not case["train"]:
        return res
    G = clean(s["gx"].float())
    dnw = None
    if case["next"]:
        gn = clean(s["gn"].float())
        v = gn * nw
        G = G + rx * (v - xh * (v * xh).mean(-1, keepdim=True))
        dnw = (gn * xh).sum((0, 1), dtype=torch.float64).float()
    q = (G * c * yh).sum((0, 1), dtype=torch.float64)
    v = G * sc * c * w
    res += [G.to(dt), (ry * (v - yh * (v * yh).mean(-1, keepdim=True))).to(dt)]
    if dc is not None:
        res.append((G * sc * yh * w * dc).to(dt))
    res += [(q * sc).float(), (q * w).float()]
    return res + ([dnw] if case["next"] else [])


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "step":
        a, om = torch.sigmoid(s["f"].float()), torch.sigmoid(-s["f"].float())
        a, om = _spread(a, case["D"]), _spread(om, case["D"])
        z = s["z"].float()
        h = a * s["state"] + (om * z if case["decay_input"] else z)
        return [h.to(s["z"].dtype), h]
    if op == "scan":
        return _plain_scan(s)
    if op == "join":
        return _plain_join(s)
    if op == "pack":
        return _plain8(s["x"].float()).to(s["x"].dtype)
    x, w, g = s["x"].detach().flatten(0, 1), s["w"].detach(), s["g"].flatten(0, 1)
    out = (x @ w.t() + s["b"].detach()).view_as(s["g"])
    return [out, (g @ w).view_as(s["x"]), g.t() @ _plain8(x), g.sum(0)]


# ------------------------------------------------------------------------------- a pass


def run(s):
    if not own:
        with torch.no_grad():
            return _plain(s)
    delrec = _package()
    case = s["case"]
    op = case["op"]
    if op == "step":
        return list(delrec.gated.gated_step(s["z"], s["f"], s["state"], decay_input=case["decay_input"]))
    if op == "scan":
        h, hT = delrec.gated.gated_scan(s["z"], s["f"], s["h0"], lengths=s["lengths"], resets=s["resets"],
                                        decay_input=case["decay_input"], checkpoint8=case["bits8"])
        if not case["train"]:
            return [h, hT]
        grads = torch.autograd.grad((h, hT), (s["z"], s["f"], s["h0"]), (s["gh"], s["ghT"]))
        return [h.detach(), hT.detach(), *grads]
    if op == "join":
        new, n = delrec.block_norm.block_join(s["x"], s["y"], s["w"], gate=s["u"], gate_act=case["gate"],
                                              scale=s["scale"], next_weight=s["nw"], eps=EPS,
                                              lengths=s["lengths"])
        outs = [v for v in (new, n) if v is not None]
        if not case["train"]:
            return outs
        ins = [s[k] for k in ("x", "y", "u", "w", "scale", "nw") if s[k] is not None]
        grads = torch.autograd.grad(outs, ins, [v for v in (s["gx"], s["gn"]) if v is not None])
        return [v.detach() for v in outs] + list(grads)
    if op == "pack":
        return delrec.checkpoint8.unpack8(delrec.checkpoint8.pack8(s["x"]))
    out = delrec.linear.linear(s["x"], s["w"], s["b"], binary_input=case["spikes"], checkpoint8=True)
    return [out.detach(), *torch.autograd.grad(out, (s["x"], s["w"], s["b"]), s["g"])]


def work(case):
    """Every input read once, every output written once; operations counted per element."""
    w, op = BYTES[case["dtype"]], case["op"]
    T, B, N = case["T"], case["B"], case["N"]
    n = T * B * N
    if op == "step":
        return {"bytes": (2 * w + 8) * n + w * n // case["D"], "flops": 12 * n}
    if op == "scan":
        nf = n // case["D"]
        if not case["train"]:
            return {"bytes": w * (2 * n + nf) + 8 * B * N, "flops": 12 * n}
        return {"bytes": w * (4 * n + 2 * nf) + 16 * B * N, "flops": 36 * n}
    if op == "join":
        gate, nxt = case["gate"] != "none", case["next"]
        fwd = 3 + gate + nxt
        if not case["train"]:
            return {"bytes": w * n * fwd + 12 * N, "flops": 20 * n}
        return {"bytes": w * n * (fwd + 3 + gate + nxt) + 24 * N, "flops": 70 * n}
    if op == "pack":
        return {"bytes": 2 * n * w + 2 * n, "flops": 6 * n}
    M, K = T * B, case["K"]
    return {"bytes": 4 * (2 * M * K + 2 * M * N + 2 * N * K + 2 * N), "flops": 6 * M * N * K}


# -------------------------------------------------------------------- definitions in 64 bits


def _exact8(x):
    N = x.shape[-1]
    rows = x.reshape(-1, N)
    groups = -(-N // GROUP)
    buf = torch.zeros(rows.shape[0], groups * GROUP, dtype=torch.float64, device=x.device)
    buf[:, :N] = rows
    buf = buf.view(-1, groups, GROUP)
    top = buf.abs().max(dim=2).values
    # the smallest power of two 2^k, k >= -126, with top <= 126 * 2^k
    k = torch.floor(torch.log2(torch.clamp(top, min=2.0 ** -140))) - 6
    two = lambda k: ((k.long() + 1023) << 52).view(torch.float64)  # noqa: E731  2^k, exactly
    k = torch.where(top > 126 * two(k), k + 1, k)
    k = torch.where(top <= 126 * two(k - 1), k - 1, k)
    step = two(torch.clamp(k, min=-126)).unsqueeze(2)
    return (torch.round(buf / step) * step).view(rows.shape[0], -1)[:, :N].reshape(x.shape)


def _exact_scan(s):
    case = s["case"]
    T, B, N, D = case["T"], case["B"], case["N"], case["D"]
    G_ = N // D
    z, f = s["z"].detach().double(), s["f"].detach().double()
    live = torch.ones(T, B, dtype=torch.bool, device=z.device)
    if s["lengths"] is not None:
        live = torch.arange(T, device=z.device).view(T, 1) < s["lengths"].view(1, B)
    cut = s["resets"] if s["resets"] is not None else torch.zeros_like(live)
    pos = s["lengths"] is not None or s["resets"] is not None

    def gates(v):
        return (1 / (1 + torch.exp(-v))).unsqueeze(-1).expand(T, B, G_, D).reshape(T, B, N)

    def forward(zz, a, start, every):
        """States before each step and after it; `every` > 0: begun anew from `start` at each such step."""
        b = (1 - a) * zz if case["decay_input"] else zz
        pre, post = torch.empty_like(b), torch.empty_like(b)
        h = start[0]
        for t in range(T):
            if every and t % every == 0:
                h = start[t // every]
            pre[t] = h
            if pos:
                new = a[t] * torch.where(cut[t].view(B, 1), 0.0, h) + b[t]
                h = torch.where(live[t].view(B, 1), new, h)
                post[t] = h
            else:
                h = torch.addcmul(b[t], a[t], h, out=post[t])
        return pre, post

    a = gates(f)
    pre, post = forward(z, a, s["h0"].detach().double()[None], 0)
    m = live.view(T, B, 1)
    res = [torch.where(m, post, 0.0), post[-1].clone()]
    if not case["train"]:
        return res
    if case["bits8"]:
        z, a = _exact8(z), gates(_exact8(f))
        pre, _ = forward(z, a, pre[::SEGMENT].clone(), SEGMENT)
    del post
    gh = s["gh"].double()
    carry = s["ghT"].double()
    dz, df = torch.zeros_like(z), torch.zeros(T, B, G_, dtype=torch.float64, device=z.device)
    for t in range(T - 1, -1, -1):
        at, ok, keep = a[t], live[t].view(B, 1), ~cut[t].view(B, 1)
        g = carry + gh[t]
        before = torch.where(keep, pre[t], 0.0)
        if case["decay_input"]:
            dz[t] = torch.where(ok, g * (1 - at), 0.0)
            before = before - z[t]
        else:
            dz[t] = torch.where(ok, g, 0.0)
        df[t] = torch.where(ok, g * at * (1 - at) * before, 0.0).view(B, G_, D).sum(-1)
        carry = torch.where(ok, torch.where(keep, at * g, 0.0), carry)
    return res + [dz, df, carry]


def _exact_join(s):
    case = s["case"]
    T, B = case["T"], case["B"]
    live = torch.ones(T, B, dtype=torch.bool, device=s["x"].device)
    if s["lengths"] is not None:
        live = torch.arange(T, device=live.device).view(T, 1) < s["lengths"].view(1, B)
    idx = live.flatten().nonzero().squeeze(1)
    rows = lambda v: v.detach().double().flatten(0, 1)[idx].requires_grad_(case["train"])  # noqa: E731
    vec = lambda k: s[k].detach().double().requires_grad_(case["train"])  # noqa: E731
    x, y = rows(s["x"]), rows(s["y"])
    u = rows(s["u"]) if s["u"] is not None else None
    w, sc = vec("w"), vec("scale")
    branch = y / (y.pow(2).mean(1, keepdim=True) + EPS).sqrt() * w
    if u is not None:
        gate = 1 / (1 + torch.exp(-u))
        branch = branch * (gate if case["gate"] == "sigmoid" else gate * u)
    new = x + sc * branch
    outs, ins, gs = [new], [x, y], []
    if u is not None:
        ins.append(u)
    ins += [w, sc]
    if case["next"]:
        nw = vec("nw")
        ins.append(nw)
        outs.append(new / (new.pow(2).mean(1, keepdim=True) + EPS).sqrt() * nw)

    def whole(v):
        if v.dim() == 1:
            return v
        full = torch.zeros(T * B, v.shape[1], dtype=torch.float64, device=v.device)
        full[idx] = v
        return full.view(T, B, -1)

    if case["train"]:
        gs = [s[k].double().flatten(0, 1)[idx] for k in (("gx", "gn") if case["next"] else ("gx",))]
        gs = list(torch.autograd.grad(outs, ins, gs))
    return [whole(v.detach()) for v in outs + gs]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "scan":
        with torch.no_grad():
            return _exact_scan(s)
    if op == "join":
        return _exact_join(s)
    with torch.no_grad():
        if op == "step":
            gate = 1 / (1 + torch.exp(-s["f"].double()))
            gate = gate.unsqueeze(-1).expand(*gate.shape, case["D"]).flatten(-2)
            z = s["z"].double()
            h = gate * s["state"].double() + ((1 - gate) * z if case["decay_input"] else z)
            return [h, h.clone()]
        if op == "pack":
            return _exact8(s["x"].double())
        x, w, g = s["x"].double().flatten(0, 1), s["w"].double(), s["g"].double().flatten(0, 1)
        return [(x @ w.t() + s["b"].double()).view_as(s["g"]), (g @ w).view_as(s["x"]),
                g.t() @ _exact8(x), g.sum(0)]

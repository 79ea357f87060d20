"""Workloads of the selective state space layer and the vocabulary losses: the short causal convolution,
the selective scan (both for whole sequences and for single steps), the softmax cross entropy of a
projection onto a large vocabulary and the distillation from a teacher's top logits, each with its plain
form in elementary torch operations."""

import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
IGNORE = -100


def _package():
    path = os.path.join(os.getcwd(), "snn-delays_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import delrec.selective
    import delrec.short_conv
    import delrec.vocab_loss
    return delrec


# ------------------------------------------------------------------------------- cases


def listed():
    return [
        # one time step of a streaming batch of 256 sensors or users: latency
        {"name": "conv_step", "op": "conv_step", "B": 256, "N": 512, "K": 4, "dtype": "fp32", "act": "silu"},
        # the event-stream model's hidden layer (250 bins, batch 256, 512 wide) in training
        {"name": "conv_train", "op": "conv", "T": 250, "B": 256, "N": 512, "K": 4, "dtype": "bf16", "act": "silu",
         "train": True, "ragged": False},
        # a padded batch of recordings with packed pieces, the event-stream input's 700 channels
        {"name": "conv_train_packed", "op": "conv", "T": 1021, "B": 24, "N": 700, "K": 3, "dtype": "fp32",
         "act": "none", "train": True, "ragged": True},
        # one time step of 64 streams: latency
        {"name": "scan_step", "op": "scan_step", "B": 64, "N": 512, "S": 16, "G": 1, "dtype": "bf16"},
        # a long recording taken in at once, one sequence: the scan splits over time
        {"name": "scan_prefill", "op": "scan", "T": 16384, "B": 1, "N": 512, "S": 16, "G": 1, "dtype": "bf16",
         "train": False, "ragged": False},
        # the event-stream model's hidden layer in training
        {"name": "scan_train", "op": "scan", "T": 250, "B": 256, "N": 512, "S": 16, "G": 1, "dtype": "fp32",
         "train": True, "ragged": False},
        # a padded batch of recordings with packed pieces, four groups of 130 channels, 24 states
        {"name": "scan_train_packed", "op": "scan", "T": 1021, "B": 24, "N": 520, "S": 24, "G": 4, "dtype": "bf16",
         "train": True, "ragged": True},
        # the loss of one step of 64 streams, without gradients: latency
        {"name": "entropy_step", "op": "entropy", "T": 1, "B": 64, "D": 512, "V": 32000, "dtype": "bf16",
         "train": False, "ragged": False, "bias": False, "reduction": "none"},
        # a training batch of 8192 positions on the hidden layer's 512 channels
        {"name": "entropy_train", "op": "entropy", "T": 32, "B": 256, "D": 512, "V": 32768, "dtype": "bf16",
         "train": True, "ragged": False, "bias": False, "reduction": "mean"},
        # a padded batch on the framework's default type, an odd vocabulary, with a bias
        {"name": "entropy_train_fp32", "op": "entropy", "T": 250, "B": 16, "D": 700, "V": 5003, "dtype": "fp32",
         "train": True, "ragged": True, "bias": True, "reduction": "mean"},
        # a student of 512 channels learning from 64 kept logits a position
        {"name": "distill_train", "op": "distill", "T": 64, "B": 64, "D": 512, "V": 32768, "K": 64, "dtype": "bf16",
         "train": True, "ragged": False, "bias": False, "temperature": 2.0, "reduction": "mean"},
        # a small student, few kept logits, a padded batch
        {"name": "distill_small", "op": "distill", "T": 16, "B": 32, "D": 128, "V": 8191, "K": 20, "dtype": "fp16",
         "train": True, "ragged": True, "bias": True, "temperature": 1.0, "reduction": "none"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["conv_step", "conv", "conv", "scan_step", "scan", "scan", "scan", "entropy", "entropy",
                     "distill", "distill"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "conv_step":
        return {"op": op, "B": _log(rng, 1, 1024), "N": _log(rng, 16, 4096), "K": rng.randint(2, 8), "dtype": dtype,
                "act": rng.choice(["silu", "none"])}
    if op == "conv":
        N, B = _log(rng, 16, 4096), _log(rng, 1, 256)
        return {"op": op, "T": _log(rng, 1, max(1, min(16384, 32_000_000 // (B * N)))), "B": B, "N": N,
                "K": rng.randint(2, 8), "dtype": dtype, "act": rng.choice(["silu", "none"]),
                "train": rng.random() < 0.7, "ragged": rng.random() < 0.4}
    if op in ("scan_step", "scan"):
        G = rng.choice([1, 1, 1, 2, 4])
        N = G * max(1, _log(rng, 16, 2048) // G)
        S = _log(rng, 1, 128)
        if op == "scan_step":
            return {"op": op, "B": _log(rng, 1, 256), "N": N, "S": S, "G": G, "dtype": dtype}
        B = _log(rng, 1, 256)
        T = _log(rng, 1, max(1, min(16384, 400_000_000 // (B * N * S))))
        return {"op": op, "T": T, "B": B, "N": N, "S": S, "G": G, "dtype": dtype, "train": rng.random() < 0.7,
                "ragged": rng.random() < 0.4}
    D, V = _log(rng, 32, 1024), _log(rng, 100, 65536)
    B = _log(rng, 1, 256)
    T = _log(rng, 1, max(1, min(1024, 130_000_000_000 // (D * V * B), 250_000_000 // (V * B))))
    case = {"op": op, "T": T, "B": B, "D": D, "V": V, "dtype": dtype, "train": rng.random() < 0.7,
            "ragged": rng.random() < 0.4, "bias": rng.random() < 0.3, "reduction": rng.choice(["mean", "sum", "none"])}
    if op == "distill":
        case["K"] = _log(rng, 1, min(128, V))
        case["temperature"] = rng.choice([1.0, 2.0, 3.5])
    return case


# ------------------------------------------------------------------------------ inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = DTYPES[case["dtype"]]
    f32 = torch.float32
    op = case["op"]
    B = case["B"]
    T = case.get("T", 1)

    def normal(*shape, mean=0.0, std=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": dict(case), "lengths": None, "resets": None}
    if case.get("ragged"):
        n = torch.randint(0, T + 1, (B,), generator=g, device="cuda")
        n[int(seed) % B] = T
        s["lengths"] = n.to(torch.int32)
    leaves = ()
    if op in ("conv", "conv_step"):
        N, K = case["N"], case["K"]
        lead = (T, B) if op == "conv" else (B,)
        s["x"] = normal(*lead, N)
        s["w"] = (uniform(N, K) * 2 - 1) * K ** -0.5
        s["b"] = normal(N, std=0.1, dtype=f32)
        s["state"] = normal(K - 1, B, N)
        if op == "conv":
            s["resets"] = uniform(T, B) < 4.0 / T if case["ragged"] else None
            if case["train"]:
                s["gy"] = normal(T, B, N, std=0.01)
                s["gs"] = normal(K - 1, B, N, std=0.01)
                leaves = ("x", "w", "b", "state")
    elif op in ("scan", "scan_step"):
        N, S, G = case["N"], case["S"], case["G"]
        lead = (T, B) if op == "scan" else (B,)
        s["x"] = normal(*lead, N)
        s["dt"] = normal(*lead, N, std=0.5)
        # steps between 0.001 and 0.1 at dt = 0, decay rates 1 .. S
        s["dt_bias"] = torch.log(torch.expm1(torch.exp(uniform(N) * math.log(100.0) + math.log(1e-3))))
        s["A"] = -(torch.arange(1, S + 1, device="cuda", dtype=f32) * (0.9 + 0.2 * uniform(N, S)))
        s["B"] = normal(*lead, G, S)
        s["C"] = normal(*lead, G, S)
        s["D"] = normal(N, mean=1.0, std=0.1, dtype=f32)
        s["gate"] = normal(*lead, N)
        s["h0"] = normal(B, N, S, dtype=f32)
        if op == "scan":
            s["resets"] = uniform(T, B) < 4.0 / T if case["ragged"] else None
            if case["train"]:
                s["gy"] = normal(T, B, N, std=0.01)
                s["ghT"] = normal(B, N, S, std=0.01, dtype=f32)
                leaves = ("x", "dt", "A", "B", "C", "h0", "D", "gate", "dt_bias")
    else:
        D, V = case["D"], case["V"]
        s["x"] = normal(T, B, D)
        s["w"] = normal(V, D, std=2.0 * D ** -0.5)
        s["b"] = normal(V, std=0.5) if case["bias"] else None
        if op == "entropy":
            # frequent tokens are far more frequent; one position in twelve is not counted
            t = torch.exp(uniform(T, B) * math.log(V + 1.0)).long().clamp(1, V) - 1
            s["target"] = torch.where(uniform(T, B) < 1 / 12, torch.full_like(t, IGNORE), t)
        else:
            K = case["K"]
            score = uniform(T * B, V)
            top = score.topk(K, dim=1).indices.view(T, B, K)
            s["indices"] = top.to(torch.int32)
            s["logits"] = normal(T, B, K, std=2.0).sort(-1, descending=True).values
            del score
        if case["train"]:
            s["g"] = normal(T, B, std=0.01, dtype=f32) if case["reduction"] == "none" else None
            leaves = ("x", "w", "b")
    for k in leaves:
        if s[k] is not None:
            s[k].requires_grad_(True)
    return s


# ---------------------------------------------------------------------- plain forms, 32 bits


def _valid(T, lengths, like):
    if lengths is None:
        return None
    return (torch.arange(T, device=like.device)[:, None] < lengths[None, :]).unsqueeze(-1)


def _act(p, kind):
    """act(p) and its derivative."""
    if kind == "none":
        return p, torch.ones_like(p)
    a, b = torch.sigmoid(p), torch.sigmoid(-p)
    return p * a, a * (1.0 + p * b)


def _plain_conv_step(s):
    case = s["case"]
    x, w, st = s["x"].float(), s["w"], s["state"].float()
    K = case["K"]
    p = s["b"] + w[:, K - 1] * x
    for j in range(K - 1):
        p = p + w[:, j] * st[j]
    new = torch.cat([s["state"][1:], s["x"][None]])
    return [_act(p, case["act"])[0].to(s["x"].dtype), new]


def _plain_conv(s):
    case, lengths, resets = s["case"], s["lengths"], s["resets"]
    T, B, N, K = case["T"], case["B"], case["N"], case["K"]
    dt = s["x"].dtype
    valid = _valid(T, lengths, s["x"])
    x = s["x"].detach().float()
    if valid is not None:
        x = torch.where(valid, x, torch.zeros_like(x))
    w, b = s["w"].detach(), s["b"].detach()
    ext = torch.cat([s["state"].detach().float(), x])                 # position t at K-1+t
    part = torch.zeros(T + K - 1, B, dtype=torch.long, device=x.device)
    if resets is not None:
        part[K - 1:] = resets.long().cumsum(0)

    def tap(d):
        """x d steps back, 0 where a reset lies between."""
        v = ext[K - 1 - d:K - 1 - d + T]
        same = (part[K - 1 - d:K - 1 - d + T] == part[K - 1:]).unsqueeze(-1)
        return torch.where(same, v, torch.zeros_like(v)), same

    p = b.expand(T, B, N)
    for d in range(K):
        p = p + w[:, K - 1 - d] * tap(d)[0]
    y, dy = _act(p, case["act"])
    if valid is not None:
        y = torch.where(valid, y, torch.zeros_like(y))
    n = torch.full((B,), T, device=x.device) if lengths is None else lengths.long()
    at = n[None, :] + torch.arange(K - 1, device=x.device)[:, None]   # rows of ext that are the new state
    seen = part[K - 1:]
    last = torch.where(n > 0, seen.gather(0, (n - 1).clamp(min=0)[None])[0], torch.zeros_like(n))
    keep = (part.gather(0, at) == last[None]).unsqueeze(-1)
    idx = at.unsqueeze(-1).expand(K - 1, B, N)
    new = ext.gather(0, idx)
    new = torch.where(keep, new, torch.zeros_like(new))
    res = [y.to(dt), new.to(dt)]
    if not case["train"]:
        return res
    dp = s["gy"].float() * dy
    if valid is not None:
        dp = torch.where(valid, dp, torch.zeros_like(dp))
    de = torch.zeros_like(ext)
    dw = torch.empty_like(w)
    for d in range(K):
        v, same = tap(d)
        de[K - 1 - d:K - 1 - d + T] += torch.where(same, w[:, K - 1 - d] * dp, torch.zeros_like(dp))
        dw[:, K - 1 - d] = (dp * v).sum((0, 1), dtype=torch.float64).float()
    gs = torch.where(keep, s["gs"].float(), torch.zeros_like(new))
    de.scatter_add_(0, idx, gs)
    dx = de[K - 1:]
    if valid is not None:
        dx = torch.where(valid, dx, torch.zeros_like(dx))
    return res + [dx.to(dt), dw, dp.sum((0, 1), dtype=torch.float64).float(), de[:K - 1].to(dt)]


def _pairs(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 0 from h = 0, and the running products of a:
    the affine maps of 1, 2, 4, ... steps put together."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], a[d:] * b[:-d] + b[d:]])
        a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b, a


def _spread(v, N):
    """(.., G, S) -> (.., N, S)"""
    return v.repeat_interleave(N // v.shape[-2], -2)


def _plain_scan_step(s):
    x, N = s["x"].float(), s["case"]["N"]
    delta = torch.nn.functional.softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(delta.unsqueeze(-1) * s["A"]) * s["h0"] \
        + (delta * x).unsqueeze(-1) * _spread(s["B"].float(), N)
    y = (h * _spread(s["C"].float(), N)).sum(-1) + s["D"] * x
    return [(y * _act(s["gate"].float(), "silu")[0]).to(s["x"].dtype), h]


def _plain_scan(s):
    case, lengths, resets = s["case"], s["lengths"], s["resets"]
    T, B, N, S, G = (case[k] for k in ("T", "B", "N", "S", "G"))
    dt = s["x"].dtype
    valid = _valid(T, lengths, s["x"])
    clean = lambda v: v if valid is None else torch.where(valid, v, torch.zeros_like(v))  # noqa: E731
    x, u, z = clean(s["x"].detach().float()), clean(s["gate"].detach().float()), s["dt"].detach().float()
    A, D = s["A"].detach(), s["D"].detach()
    z = clean(z + s["dt_bias"].detach())
    delta = torch.nn.functional.softplus(z)
    wide = None if valid is None else valid.unsqueeze(-1)
    cleans = lambda v: v if wide is None else torch.where(wide, v, torch.zeros_like(v))  # noqa: E731
    Bm, Cm = (cleans(s[k].detach().float()) for k in ("B", "C"))
    a = torch.exp(delta.unsqueeze(-1) * A)
    if resets is not None:
        a = torch.where(resets[:, :, None, None], torch.zeros_like(a), a)
    if wide is not None:
        a = torch.where(wide, a, torch.ones_like(a))
    h0 = s["h0"].detach()
    h, q = _pairs(a, (delta * x).unsqueeze(-1) * _spread(Bm, N))
    h = h + q * h0
    del q
    o = (h * _spread(Cm, N)).sum(-1) + D * x
    act, dact = _act(u, "silu")
    res = [clean(o * act).to(dt), h[-1].clone()]
    if not case["train"]:
        return res
    gy = clean(s["gy"].float())
    go = gy * act
    dgate = gy * o * dact
    dC = (go.unsqueeze(-1) * h).unflatten(2, (G, -1)).sum(3)
    last = torch.ones_like(a[:1])
    gh, q = _pairs(torch.cat([a[1:], last]).flip(0), (go.unsqueeze(-1) * _spread(Cm, N)).flip(0))
    gh = (gh + q * s["ghT"]).flip(0)
    del q
    dB = cleans((gh * (delta * x).unsqueeze(-1)).unflatten(2, (G, -1)).sum(3))
    gb = (gh * _spread(Bm, N)).sum(-1)
    w = gh * a * torch.cat([h0[None], h[:-1]])
    if wide is not None:
        w = torch.where(wide, w, torch.zeros_like(w))
    ddelta = (w * A).sum(-1) + gb * x
    dA = (w * delta.unsqueeze(-1)).sum((0, 1), dtype=torch.float64).float()
    ddt = clean(ddelta * torch.sigmoid(z))
    dx = clean(gb * delta + D * go)
    return res + [dx.to(dt), ddt.to(dt), dA, dB.to(dt), cleans(dC).to(dt), a[0] * gh[0],
                  (go * x).sum((0, 1), dtype=torch.float64).float(), clean(dgate).to(dt),
                  ddt.sum((0, 1), dtype=torch.float64).float()]


def _reduced(loss, counted, reduction):
    if reduction == "none":
        return loss
    total = loss.sum(dtype=torch.float64)
    return (total / counted.sum().clamp(min=1) if reduction == "mean" else total).float()


def _row_scale(s, counted):
    """d (result) / d (a position's loss)."""
    case = s["case"]
    if case["reduction"] == "none":
        c = s["g"].flatten()
    elif case["reduction"] == "sum":
        c = torch.ones(counted.numel(), device=counted.device)
    else:
        c = (1.0 / counted.sum().clamp(min=1)).expand(counted.numel())
    return torch.where(counted, c, torch.zeros_like(c)).unsqueeze(-1)


def _plain_loss(s):
    case = s["case"]
    T, B, V = case["T"], case["B"], case["V"]
    dt = s["x"].dtype
    tau = case.get("temperature", 1.0)
    x, w = s["x"].detach().float().flatten(0, 1), s["w"].detach().float()
    counted = torch.ones(T * B, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        counted = _valid(T, s["lengths"], x).expand(T, B, 1).reshape(-1)
    if case["op"] == "entropy":
        target = s["target"].flatten()
        counted = counted & (target != IGNORE)
    x = torch.where(counted.unsqueeze(-1), x, torch.zeros_like(x))
    z = x @ w.t()
    if s["b"] is not None:
        z += s["b"].detach().float()
    z /= tau
    top = z.amax(-1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(-1, keepdim=True)
    if case["op"] == "entropy":
        idx = target.clamp(min=0).unsqueeze(-1)
        p = torch.ones_like(idx, dtype=torch.float32)
        logp = torch.zeros_like(p)
    else:
        idx = s["indices"].flatten(0, 1).long()
        t = s["logits"].flatten(0, 1).float() / tau
        t = t - t.amax(-1, keepdim=True)
        logp = t - torch.log(torch.exp(t).sum(-1, keepdim=True))
        p = torch.exp(logp)
    loss = tau * tau * (p * (logp - (z.gather(1, idx) - top - torch.log(total)))).sum(-1)
    loss = torch.where(counted, loss, torch.zeros_like(loss))
    res = [_reduced(loss.view(T, B), counted, case["reduction"])]
    if not case["train"]:
        return res
    g = e.div_(total)
    g.scatter_add_(1, idx, -p)
    g *= _row_scale(s, counted) * tau
    res += [(g @ w).view(T, B, -1).to(dt), (g.t() @ x).to(dt)]
    return res + ([g.sum(0).to(dt)] if s["b"] is not None else [])


PLAIN = {"conv_step": _plain_conv_step, "conv": _plain_conv, "scan_step": _plain_scan_step, "scan": _plain_scan,
         "entropy": _plain_loss, "distill": _plain_loss}


# ------------------------------------------------------------------------------- a pass


def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        with torch.no_grad():
            return PLAIN[op](s)
    delrec = _package()
    if op == "conv_step":
        return list(delrec.short_conv.short_conv_step(s["x"], s["w"], s["b"], s["state"], act=case["act"]))
    if op == "conv":
        y, new = delrec.short_conv.short_conv(s["x"], s["w"], s["b"], s["state"], act=case["act"],
                                              lengths=s["lengths"], resets=s["resets"])
        if not case["train"]:
            return [y, new]
        grads = torch.autograd.grad((y, new), (s["x"], s["w"], s["b"], s["state"]), (s["gy"], s["gs"]))
        return [y.detach(), new.detach(), *grads]
    if op == "scan_step":
        return list(delrec.selective.selective_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["h0"], D=s["D"],
                                                    gate=s["gate"], dt_bias=s["dt_bias"]))
    if op == "scan":
        y, hT = delrec.selective.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], s["h0"], D=s["D"],
                                                gate=s["gate"], dt_bias=s["dt_bias"], lengths=s["lengths"],
                                                resets=s["resets"])
        if not case["train"]:
            return [y, hT]
        ins = [s[k] for k in ("x", "dt", "A", "B", "C", "h0", "D", "gate", "dt_bias")]
        return [y.detach(), hT.detach(), *torch.autograd.grad((y, hT), ins, (s["gy"], s["ghT"]))]
    if op == "entropy":
        loss = delrec.vocab_loss.linear_cross_entropy(s["x"], s["w"], s["target"], s["b"], ignore_index=IGNORE,
                                                      reduction=case["reduction"], lengths=s["lengths"])
    else:
        loss = delrec.vocab_loss.linear_distill(s["x"], s["w"], s["indices"], s["logits"], s["b"],
                                                temperature=case["temperature"], reduction=case["reduction"],
                                                lengths=s["lengths"])
    if not case["train"]:
        return [loss]
    return [loss.detach(), *torch.autograd.grad(loss, [s[k] for k in ("x", "w", "b") if s[k] is not None], s["g"])]


def work(case):
    """Every input read once, every output written once; operations counted per element.  A padded batch
    holds half of its positions."""
    w, op, B = BYTES[case["dtype"]], case["op"], case["B"]
    T = case.get("T", 1)
    part = 0.5 if case.get("ragged") else 1.0
    if op == "conv_step":
        N, K = case["N"], case["K"]
        return {"bytes": w * B * N * 2 * K + 4 * N * (K + 1), "flops": B * N * (2 * K + 4)}
    if op == "conv":
        N, K = case["N"], case["K"]
        n = T * B * N
        io = (1 + part if not case["train"] else 2 + 2 * part) * w * n
        return {"bytes": io + (2 if not case["train"] else 4) * w * (K - 1) * B * N + 4 * N * (K + 1),
                "flops": part * n * ((2 * K + 4) if not case["train"] else (6 * K + 12))}
    if op in ("scan_step", "scan"):
        N, S, G = case["N"], case["S"], case["G"]
        n, m = T * B * N, T * B * G * S
        train = case.get("train", False)
        # x, dt, gate in, y out; B and C in; in training gy in, three gradients out, dB and dC out
        io = w * ((3 * part + 1) * n + 2 * part * m)
        if train:
            io += w * ((part + 3) * n + 2 * m)
        io += (4 if train else 2) * 4 * B * N * S + (8 if train else 4) * N * (S + 2)
        return {"bytes": io, "flops": part * n * S * (24 if train else 7)}
    M, D, V = part * T * B, case["D"], case["V"]
    rows = M * D * w + (M * 8 if op == "entropy" else M * case["K"] * (4 + w))
    if not case["train"]:
        return {"bytes": rows + V * D * w, "flops": 2 * M * V * D}
    return {"bytes": rows + T * B * D * w + 2 * V * D * w, "flops": 6 * M * V * D}


# -------------------------------------------------------------------- definitions in 64 bits


def _exact_conv(s):
    """Step by step with a window of the last K - 1 inputs."""
    case = s["case"]
    op, B, N, K = case["op"], case["B"], case["N"], case["K"]
    T = case.get("T", 1)
    train = case.get("train", False)
    leaf = lambda v: v.detach().double().requires_grad_(train)  # noqa: E731
    x, w, b, state = (leaf(s[k]) for k in ("x", "w", "b", "state"))
    window = [state[j] for j in range(K - 1)]
    outs = []
    for t in range(T):
        now = x[t] if op == "conv" else x
        live = None
        if s["lengths"] is not None:
            live = (t < s["lengths"]).view(B, 1)
            now = torch.where(live, now, 0.0)
        before = window
        if s["resets"] is not None:
            cut = s["resets"][t].view(B, 1)
            before = [torch.where(cut, 0.0, v) for v in window]
        p = b + sum(w[:, j] * v for j, v in enumerate(before + [now]))
        y = p / (1 + torch.exp(-p)) if case["act"] == "silu" else p
        after = before[1:] + [now]
        if live is not None:
            y = torch.where(live, y, 0.0)
            after = [torch.where(live, v, o) for v, o in zip(after, window)]
        window = after
        outs.append(y)
    y = torch.stack(outs) if op == "conv" else outs[0]
    new = torch.stack(window)
    if not train:
        return [y, new]
    grads = torch.autograd.grad((y, new), (x, w, b, state), (s["gy"].double(), s["gs"].double()))
    return [y.detach(), new.detach(), *grads]


def _exact_scan(s):
    case = s["case"]
    op, B, N, S, G = (case[k] for k in ("op", "B", "N", "S", "G"))
    T = case.get("T", 1)
    lead = (lambda v: v) if op == "scan" else (lambda v: v[None])
    x, z, u, Bm, Cm = (lead(s[k].detach()).double() for k in ("x", "dt", "gate", "B", "C"))
    A, D = s["A"].detach().double(), s["D"].detach().double()
    z = z + s["dt_bias"].detach().double()
    delta = torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs()))
    sig = 1 / (1 + torch.exp(-u))
    grp = torch.arange(N, device=x.device) // (N // G)
    live = torch.ones(T, B, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        live = torch.arange(T, device=x.device).view(T, 1) < s["lengths"].view(1, B)
    cut = s["resets"] if s["resets"] is not None else torch.zeros_like(live)
    plain = s["lengths"] is None and s["resets"] is None
    h = s["h0"].detach().double()
    train = case.get("train", False)
    pre = torch.empty(T, B, N, S, dtype=torch.float64, device=x.device) if train else None
    o = torch.empty(T, B, N, dtype=torch.float64, device=x.device)
    for t in range(T):
        if not plain:
            kept = h
            h = torch.where(cut[t].view(B, 1, 1), 0.0, h)
        if train:
            pre[t] = h
        new = torch.exp(delta[t].unsqueeze(-1) * A).mul_(h)
        new.addcmul_((delta[t] * x[t]).unsqueeze(-1), Bm[t][:, grp])
        o[t] = torch.einsum("bns,bns->bn", new, Cm[t][:, grp]) + D * x[t]
        h = new if plain else torch.where(live[t].view(B, 1, 1), new, kept)
    m = live.unsqueeze(-1)
    y = torch.where(m, o * u * sig, 0.0)
    if op == "scan_step":
        return [y[0], h]
    if not train:
        return [y, h]
    gy = torch.where(m, s["gy"].double(), 0.0)
    x0 = torch.where(m, x, 0.0)
    go = gy * u * sig
    go = torch.where(m, go, 0.0)
    dgate = torch.where(m, gy * o * sig * (1 + u * (1 - sig)), 0.0)
    dx, dz = torch.zeros_like(x), torch.zeros_like(x)
    dB, dC, dA = torch.zeros_like(Bm), torch.zeros_like(Cm), torch.zeros_like(A)
    carry = s["ghT"].double()
    for t in range(T - 1, -1, -1):
        ok = live[t].view(B, 1, 1)
        a = torch.exp(delta[t].unsqueeze(-1) * A)
        ah = a * pre[t]
        db = (delta[t] * x[t]).unsqueeze(-1)
        g = carry + go[t].unsqueeze(-1) * Cm[t][:, grp]
        now = ah + db * Bm[t][:, grp]
        dC[t] = torch.where(ok, (go[t].unsqueeze(-1) * now).view(B, G, N // G, S).sum(2), 0.0)
        dB[t] = torch.where(ok, (g * db).view(B, G, N // G, S).sum(2), 0.0)
        gb = torch.einsum("bns,bns->bn", g, Bm[t][:, grp])
        w = torch.where(ok, g * ah, 0.0)
        dA += torch.einsum("bns,bn->ns", w, torch.where(m[t], delta[t], 0.0))
        ok1 = ok.squeeze(-1)
        dx[t] = torch.where(ok1, gb * delta[t] + D * go[t], 0.0)
        dz[t] = torch.where(ok1, (torch.einsum("bns,ns->bn", w, A) + gb * x[t]) / (1 + torch.exp(-z[t])), 0.0)
        back = torch.where(cut[t].view(B, 1, 1), 0.0, a * g)
        carry = torch.where(ok, back, carry)
    return [y, h, dx, dz, dA, dB, dC, carry, (go * x0).sum((0, 1)), dgate, dz.sum((0, 1))]


def _exact_loss(s):
    case = s["case"]
    T, B, V, train = case["T"], case["B"], case["V"], case["train"]
    tau = case.get("temperature", 1.0)
    rows = torch.ones(T, B, dtype=torch.bool, device=s["x"].device)
    if s["lengths"] is not None:
        rows = torch.arange(T, device=rows.device).view(T, 1) < s["lengths"].view(1, B)
    if case["op"] == "entropy":
        rows = rows & (s["target"] != IGNORE)
    idx = rows.flatten().nonzero().squeeze(1)
    x = s["x"].detach().flatten(0, 1)[idx].double().requires_grad_(train)
    w = s["w"].detach().double().requires_grad_(train)
    b = s["b"].detach().double().requires_grad_(train) if s["b"] is not None else None
    logq = (x @ w.t() if b is None else torch.addmm(b, x, w.t())).div(tau).log_softmax(-1)
    if case["op"] == "entropy":
        each = -logq.gather(1, s["target"].flatten()[idx].unsqueeze(1)).squeeze(1)
    else:
        p = (s["logits"].flatten(0, 1)[idx].double() / tau).softmax(-1)
        each = tau ** 2 * (p * (p.log() - logq.gather(1, s["indices"].flatten(0, 1)[idx].long()))).sum(-1)
    if case["reduction"] == "none":
        out = torch.zeros(T * B, dtype=torch.float64, device=x.device).index_put((idx,), each).view(T, B)
    else:
        out = each.sum() / (max(1, idx.numel()) if case["reduction"] == "mean" else 1)
    if not train:
        return [out.detach()]
    ins = [x, w] + ([b] if b is not None else [])
    grads = list(torch.autograd.grad(out, ins, None if s["g"] is None else s["g"].double()))
    dx = torch.zeros(T * B, case["D"], dtype=torch.float64, device=x.device)
    dx[idx] = grads[0]
    return [out.detach(), dx.view(T, B, -1), *grads[1:]]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("conv", "conv_step"):
        return _exact_conv(s)
    if case["op"] in ("scan", "scan_step"):
        with torch.no_grad():
            return _exact_scan(s)
    return _exact_loss(s)

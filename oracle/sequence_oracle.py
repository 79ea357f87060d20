"""float64 restatements of the sequence operators on the CPU, from their formulas, each with a
bound on what fp32 arithmetic may add to its outputs (test-only).

u = 2^-24 is the rounding of one fp32 operation.  A gate's sigmoid is good to 8 u (exp 2 ulp,
reciprocal 1 ulp, an addition, a product); with the roundings of a step's products and sums,
each step adds at most 16 u of the magnitudes it handles, and what came before is carried on
with the gate.  Composed maps (segments of time) make the same products in another order."""

import torch

U = 2.0 ** -24
SEGMENT = 16


def sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def restore8(x):
    """What float64 x (..., N) stands for after 8 bits: groups of 32 channels, the smallest
    power of two 2^k, k >= -126, with max |x| <= 126 * 2^k over the finite values."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[-1], 32):
        g = x[..., lo:lo + 32]
        fin = torch.isfinite(g)
        top = torch.where(fin, g.abs(), torch.zeros_like(g)).amax(-1, keepdim=True)
        m, e = torch.frexp(top)                        # top = m 2^e, m in [0.5, 1)
        k = torch.where(m * 128 > 126, e - 6, e - 7)
        k = torch.where(top == 0, torch.full_like(k, -126), k).clamp(min=-126)
        step = ((k.to(torch.int64) + 1023) << 52).view(torch.float64)
        q = torch.round(g / step)
        q = torch.where(k == 122, q.clamp(-63, 63), q)   # 64 * 2^122 is past float32
        out[..., lo:lo + 32] = torch.where(fin, q * step, g)
    return out


def gated_scan(z, f, h0=None, lengths=None, resets=None, decay_input=True):
    """Returns dict(h, hT, pre, err): pre the state before each step, err the bound of h."""
    T, B, N = z.shape
    D = N // f.shape[-1]
    h = torch.zeros(B, N, dtype=torch.float64) if h0 is None else h0.double().clone()
    err = torch.zeros_like(h)
    out = dict(h=torch.zeros(T, B, N, dtype=torch.float64), pre=torch.zeros(T, B, N, dtype=torch.float64),
               err=torch.zeros(T, B, N, dtype=torch.float64))
    for t in range(T):
        out["pre"][t] = h
        a = sigmoid(f[t].double()).repeat_interleave(D, -1)
        c = sigmoid(-f[t].double()).repeat_interleave(D, -1) if decay_input else torch.ones_like(a)
        for b in range(B):
            if lengths is not None and t >= int(lengths[b]):
                continue
            if resets is not None and bool(resets[t, b]):
                new, e = c[b] * z[t, b].double(), torch.zeros(N, dtype=torch.float64)
                mag = new.abs()
            else:
                new = a[b] * h[b] + c[b] * z[t, b].double()
                mag = (a[b] * h[b]).abs() + (c[b] * z[t, b].double()).abs()
                e = a[b] * err[b]
            h[b], err[b] = new, e + 16 * U * mag
            out["h"][t, b], out["err"][t, b] = h[b], err[b]
    out["hT"], out["errT"] = h, err
    return out


def gated_scan_backward(z, f, pre, perr, gh, ghT, lengths=None, resets=None, decay_input=True):
    """dz, df, dh0 by the formula, from the states before each step (pre, known to perr), with
    the bounds of the three."""
    T, B, N = z.shape
    G_ = f.shape[-1]
    D = N // G_
    carry, ce = ghT.double().clone(), torch.zeros(B, N, dtype=torch.float64)
    dz, ez = torch.zeros(T, B, N, dtype=torch.float64), torch.zeros(T, B, N, dtype=torch.float64)
    df, ef = torch.zeros(T, B, G_, dtype=torch.float64), torch.zeros(T, B, G_, dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        a = sigmoid(f[t].double()).repeat_interleave(D, -1)
        om = sigmoid(-f[t].double()).repeat_interleave(D, -1)      # 1 - a, which float64 loses at f > 37
        for b in range(B):
            if lengths is not None and t >= int(lengths[b]):
                continue
            cut = resets is not None and bool(resets[t, b])
            g, ge = carry[b] + gh[t, b].double(), ce[b] + 16 * U * (carry[b].abs() + gh[t, b].double().abs())
            ab, zb = a[b], z[t, b].double()
            hp = torch.zeros_like(ab) if cut else pre[t, b]
            he = torch.zeros_like(ab) if cut else perr[t, b]
            c = om[b] if decay_input else torch.ones_like(ab)
            dz[t, b], ez[t, b] = c * g, c * ge + 16 * U * (c * g).abs()
            x = hp - zb if decay_input else hp
            mag = hp.abs() + zb.abs() if decay_input else hp.abs()
            s = ab * om[b]
            df[t, b] = (s * g * x).view(G_, D).sum(-1)
            ef[t, b] = (s * (ge * mag + g.abs() * he + (32 + D) * U * g.abs() * mag)).view(G_, D).sum(-1)
            carry[b] = torch.zeros_like(ab) if cut else ab * g
            ce[b] = torch.zeros_like(ab) if cut else ab * ge + 16 * U * (ab * g).abs()
    return dict(dz=dz, df=df, dh0=carry, ez=ez, ef=ef, e0=ce)


def recompute(z, f, pre, lengths=None, resets=None, decay_input=True):
    """The states before each step when those before every 16th are pre's and the others come
    from (z, f): what the backward pass of an 8-bit checkpoint sees.  (states, bound)."""
    T = z.shape[0]
    states, err = [], []
    for t0 in range(0, T, SEGMENT):
        t1 = min(T, t0 + SEGMENT)
        r = gated_scan(z[t0:t1], f[t0:t1], pre[t0], None if lengths is None else lengths - t0,
                       None if resets is None else resets[t0:t1], decay_input)
        states.append(r["pre"])
        err.append(torch.cat([torch.zeros_like(r["err"][:1]), r["err"][:-1]]))
    return torch.cat(states), torch.cat(err)


def _gate(u, kind):
    if u is None or kind == "none":
        return None
    s = sigmoid(u)
    return s if kind == "sigmoid" else u * s


def block_join(x, y, w, u, kind, scale, nw, eps, has_next):
    """(x', n) in the dtype given (float64), differentiable; y None: (None, norm of x)."""
    new = x
    if y is not None:
        br = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
        if w is not None:
            br = br * w
        g = _gate(u, kind)
        if g is not None:
            br = br * g
        if scale is not None:
            br = br * scale
        new = x + br
    n = None
    if has_next:
        n = new / torch.sqrt((new * new).mean(-1, keepdim=True) + eps)
        if nw is not None:
            n = n * nw
    return (new if y is not None else None), n

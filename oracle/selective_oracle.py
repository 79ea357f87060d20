"""float64 restatements of the short convolution, the selective scan and the vocabulary losses on the
CPU, from their formulas, each with a bound on what fp32 arithmetic may add to its outputs (test-only).

u = 2^-24 is the rounding of one fp32 operation; a sum of n terms adds at most n u of the sum of
their magnitudes in any order.  A sigmoid of v is good to (10 + 2 |v|) u: ex2 or exp 4 u, the
argument's rounding |v| u and the product's another, reciprocal 2 u, a sum and a product."""

import torch

U = 2.0 ** -24


def sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def silu(p, ep):
    """silu(p), its derivative, and the bounds of both for p good to ep."""
    s, o = sigmoid(p), sigmoid(-p)
    y, d = p * s, s * (1.0 + p * o)
    rel = (10 + 2 * p.abs()) * U
    # |silu'| <= 1.1, |silu''| <= 0.5
    return y, d, 1.1 * ep + y.abs() * (rel + 2 * U), 0.5 * ep + s * (1 + p.abs() * o) * (2 * rel + 4 * U)


def lengths_of(lengths, B, T):
    return [T] * B if lengths is None else [max(0, min(T, int(n))) for n in lengths]


def short_conv(x, w, b=None, state=None, act="silu", lengths=None, resets=None, gy=None, gs=None):
    """dict of values and, under 'e_' names, bounds: y, new; with gy (or gs) dx, dw, db, ds."""
    T, B, N = x.shape
    K = w.shape[1]
    x, w = x.double(), w.double()
    b = torch.zeros(N, dtype=torch.float64) if b is None else b.double()
    state = torch.zeros(K - 1, B, N, dtype=torch.float64) if state is None else state.double()
    n = lengths_of(lengths, B, T)
    y, ey = torch.zeros(T, B, N, dtype=torch.float64), torch.zeros(T, B, N, dtype=torch.float64)
    new = torch.zeros(K - 1, B, N, dtype=torch.float64)
    back = gy is not None or gs is not None
    gy = torch.zeros(T, B, N, dtype=torch.float64) if gy is None else gy.double()
    gs = torch.zeros(K - 1, B, N, dtype=torch.float64) if gs is None else gs.double()
    dext, eext = torch.zeros(T + K - 1, B, N, dtype=torch.float64), torch.zeros(T + K - 1, B, N, dtype=torch.float64)
    dw, ew = torch.zeros(N, K, dtype=torch.float64), torch.zeros(N, K, dtype=torch.float64)
    db, eb = torch.zeros(N, dtype=torch.float64), torch.zeros(N, dtype=torch.float64)
    deep = (T + B + 64) * U        # a weight's sum: rows of a chunk, then chunks and sequences
    for i in range(B):
        first = -(K - 1)           # the first input that is still seen
        ext = torch.cat([state[:, i], x[:, i]])
        for t in range(n[i]):
            if resets is not None and bool(resets[t, i]):
                first = t
            taps = [(d, t - d) for d in range(K) if t - d >= first]
            p, mag = b.clone(), b.abs()
            for d, pos in taps:
                p = p + w[:, K - 1 - d] * ext[K - 1 + pos]
                mag = mag + (w[:, K - 1 - d] * ext[K - 1 + pos]).abs()
            ep = (K + 1) * U * mag
            if act == "silu":
                y[t, i], dact, ey[t, i], ed = silu(p, ep)
            else:
                y[t, i], dact, ey[t, i], ed = p, torch.ones_like(p), ep, torch.zeros_like(p)
            g = gy[t, i] * dact
            eg = gy[t, i].abs() * ed + U * g.abs()
            for d, pos in taps:
                wk, xv = w[:, K - 1 - d], ext[K - 1 + pos]
                dext[K - 1 + pos, i] += wk * g
                eext[K - 1 + pos, i] += wk.abs() * (eg + (K + 1) * U * g.abs())
                dw[:, K - 1 - d] += g * xv
                ew[:, K - 1 - d] += xv.abs() * (eg + deep * g.abs())
            db += g
            eb += eg + deep * g.abs()
        for j in range(K - 1):
            pos = n[i] - (K - 1) + j
            if pos >= first:
                new[j, i] = ext[K - 1 + pos]
                dext[K - 1 + pos, i] += gs[j, i]
                eext[K - 1 + pos, i] += 2 * U * (gs[j, i].abs() + dext[K - 1 + pos, i].abs())
    r = dict(y=y, new=new, e_y=ey, e_new=torch.zeros_like(new))
    if back:
        r.update(dx=dext[K - 1:], ds=dext[:K - 1], dw=dw, db=db, e_dx=eext[K - 1:], e_ds=eext[:K - 1], e_dw=ew, e_db=eb)
    return r


def selective(x, dt, A, Bm, Cm, h0=None, D=None, gate=None, dt_bias=None, softplus=True, lengths=None, resets=None,
              gy=None, ghT=None):
    """dict of values and bounds: y, hT; with gy (or ghT) dx, ddt, dA, dB, dC, dh0, dD, dgate, dbias.
    Bm, Cm (T,B,G,S)."""
    T, B, N = x.shape
    G, S = Bm.shape[2:]
    f = torch.float64
    x, dt, A, Bm, Cm = (v.double() for v in (x, dt, A, Bm, Cm))
    zeros = lambda *s: torch.zeros(*s, dtype=f)   # noqa: E731
    Dv = zeros(N) if D is None else D.double()
    wide = lambda v: v.repeat_interleave(N // G, -2)   # noqa: E731  (.., G, S) -> (.., N, S)
    n = torch.tensor(lengths_of(lengths, B, T))
    live = torch.arange(T)[:, None] < n[None]
    clean = lambda v: torch.where(live.view(T, B, *[1] * (v.dim() - 2)), v, torch.zeros_like(v))   # noqa: E731
    x, dt, Bm, Cm = clean(x), clean(dt), clean(Bm), clean(Cm)
    z = dt if dt_bias is None else dt + dt_bias.double()
    if softplus:
        delta, sig = torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs())), sigmoid(z)
        rd = (10 + z.abs()) * U          # z's rounding moves delta by |z| u sigmoid(z) <= |z| u delta
    else:
        delta, sig, rd = z, torch.ones_like(z), torch.full_like(z, 2 * U)
    ed = delta.abs() * rd if softplus else z.abs() * U
    rd = torch.where(delta == 0, torch.zeros_like(rd), ed / delta.abs().clamp(min=1e-300))
    if gate is not None:
        u = clean(gate.double())
        act, dact, eact, edact = silu(u, torch.zeros_like(u))
    else:
        act, dact, eact, edact = torch.ones_like(x), zeros(T, B, N), zeros(T, B, N), zeros(T, B, N)
    h = zeros(B, N, S) if h0 is None else h0.double().clone()
    eh = torch.zeros_like(h)
    pre, epre = zeros(T, B, N, S), zeros(T, B, N, S)
    post, epost = zeros(T, B, N, S), zeros(T, B, N, S)
    a, ra = zeros(T, B, N, S), zeros(T, B, N, S)
    o, eo = zeros(T, B, N), zeros(T, B, N)
    for t in range(T):
        ok = live[t].view(B, 1, 1)
        cut = torch.zeros(B, 1, 1, dtype=torch.bool) if resets is None else resets[t].view(B, 1, 1)
        pre[t], epre[t] = torch.where(cut, 0.0, h), torch.where(cut, 0.0, eh)
        v = delta[t].unsqueeze(-1) * A
        a[t] = torch.exp(v)
        ra[t] = v.abs() * (rd[t].unsqueeze(-1) + 3 * U) + 5 * U
        b = (delta[t] * x[t]).unsqueeze(-1) * wide(Bm[t])
        new = a[t] * pre[t] + b
        enew = a[t] * epre[t] + (a[t] * pre[t]).abs() * (ra[t] + U) + b.abs() * (rd[t].unsqueeze(-1) + 3 * U) + U * new.abs()
        h, eh = torch.where(ok, new, h), torch.where(ok, enew, eh)
        post[t], epost[t] = h, eh
        C = wide(Cm[t])
        o[t] = (C * h).sum(-1) + Dv * x[t]
        eo[t] = (C.abs() * eh).sum(-1) + (S + 3) * U * ((C * h).abs().sum(-1) + (Dv * x[t]).abs())
    y = clean(o * act)
    ey = clean(eo * act.abs() + o.abs() * eact + 2 * U * y.abs())
    r = dict(y=y, e_y=ey, hT=h, e_hT=eh)
    if gy is None and ghT is None:
        return r
    gy = zeros(T, B, N) if gy is None else clean(gy.double())
    carry = zeros(B, N, S) if ghT is None else ghT.double().clone()
    ecarry = torch.zeros_like(carry)
    go, ego = gy * act, gy.abs() * (eact + U * act.abs())
    r["dgate"], r["e_dgate"] = gy * dact * o, gy.abs() * (dact.abs() * eo + edact * o.abs() + 3 * U * (dact * o).abs())
    names = dict(dx=(T, B, N), ddt=(T, B, N), dA=(N, S), dB=(T, B, G, S), dC=(T, B, G, S))
    for k, shape in names.items():
        r[k], r["e_" + k] = zeros(*shape), zeros(*shape)
    deep = (T + B + 64) * U
    grp = lambda v: v.view(B, G, N // G, S).sum(2)   # noqa: E731
    for t in range(T - 1, -1, -1):
        ok = live[t].view(B, 1, 1)
        ok1 = ok.squeeze(-1)
        cut = torch.zeros(B, 1, 1, dtype=torch.bool) if resets is None else resets[t].view(B, 1, 1)
        C, Bt, d = wide(Cm[t]), wide(Bm[t]), delta[t].unsqueeze(-1)
        gt, egt = go[t].unsqueeze(-1), ego[t].unsqueeze(-1)
        g = carry + C * gt
        eg = ecarry + C.abs() * egt + 2 * U * (carry.abs() + (C * gt).abs())
        dxv = (delta[t] * x[t]).unsqueeze(-1)
        edx = (ed[t] * x[t].abs() + U * dxv.squeeze(-1).abs()).unsqueeze(-1)
        sums = 40 + N // 32        # channels of a sum: in a thread, over lanes, over tiles
        zero = torch.zeros_like
        r["dC"][t] = grp(torch.where(ok, gt * post[t], zero(g)))
        r["e_dC"][t] = grp(torch.where(ok, gt.abs() * epost[t] + egt * post[t].abs() + sums * U * (gt * post[t]).abs(), zero(g)))
        r["dB"][t] = grp(torch.where(ok, g * dxv, zero(g)))
        r["e_dB"][t] = grp(torch.where(ok, eg * dxv.abs() + g.abs() * edx + sums * U * (g * dxv).abs(), zero(g)))
        gb, egb = (g * Bt).sum(-1), ((eg + (S + 1) * U * g.abs()) * Bt.abs()).sum(-1)
        w = torch.where(ok, a[t] * g * pre[t], zero(g))
        ew = torch.where(ok, a[t] * (eg * pre[t].abs() + g.abs() * epre[t]) + w.abs() * (ra[t] + 3 * U), zero(g))
        wa, ewa = (w * A).sum(-1), ((ew + (S + 5) * U * w.abs()) * A.abs()).sum(-1)
        r["dA"] += (w * d).sum(0)
        r["e_dA"] += (ew * d.abs() + w.abs() * (ed[t].unsqueeze(-1) + deep * d.abs())).sum(0)
        r["dx"][t] = torch.where(ok1, gb * delta[t] + Dv * go[t], zero(gb))
        r["e_dx"][t] = torch.where(ok1, egb * delta[t].abs() + gb.abs() * ed[t] + Dv.abs() * ego[t]
                                   + 3 * U * ((gb * delta[t]).abs() + (Dv * go[t]).abs()), zero(gb))
        dd = wa + gb * x[t]
        edd = ewa + egb * x[t].abs() + 3 * U * (wa.abs() + (gb * x[t]).abs())
        r["ddt"][t] = torch.where(ok1, dd * sig[t], zero(dd))
        # sigmoid'(z) <= sigmoid(z), so z's rounding |z| u counts with it
        r["e_ddt"][t] = torch.where(ok1, (edd + dd.abs() * (14 + 3 * z[t].abs()) * U) * sig[t], zero(dd))
        back = torch.where(cut, 0.0, a[t] * g)
        eback = torch.where(cut, 0.0, a[t] * eg + (a[t] * g).abs() * (ra[t] + U))
        carry, ecarry = torch.where(ok, back, carry), torch.where(ok, eback, ecarry)
    r["dh0"], r["e_dh0"] = carry, ecarry
    for k, v, e in (("dD", go * x, ego * x.abs()), ("dbias", r["ddt"], r["e_ddt"])):
        r[k] = v.sum((0, 1))
        r["e_" + k] = (e + deep * v.abs()).sum((0, 1))
    return r


def vocab_loss(x, w, index, bias=None, logits=None, tau=1.0, ignore=-100, lengths=None, reduction="mean", g=None,
               half=U):
    """dict of values and bounds: loss; with g (the gradient of the result) dx, dw, db.  index (T,B) for the
    cross entropy, (T,B,K) with a teacher's logits.  half: the rounding of the stored logits' gradient."""
    T, B, D = x.shape
    V = w.shape[0]
    f = torch.float64
    live = torch.arange(T)[:, None] < torch.tensor(lengths_of(lengths, B, T))[None]
    if logits is None:
        idx, t = index.reshape(T * B, 1).long(), torch.zeros(T * B, 1, dtype=f)
        on = live.flatten() & (idx[:, 0] != ignore)
        kept = torch.ones_like(idx, dtype=torch.bool)
    else:
        idx, t = index.reshape(T * B, -1).long(), logits.double().reshape(T * B, -1) / tau
        kept = (idx >= 0) & (t != -float("inf"))
        on = live.flatten() & kept.any(1)
    rows = on.nonzero()[:, 0]
    idx, t, kept = idx[rows], t[rows], kept[rows]
    x2, w2 = x.double().reshape(T * B, D)[rows], w.double()
    b = torch.zeros(V, dtype=f) if bias is None else bias.double()
    z = (x2 @ w2.t() + b) / tau
    mag = (x2.abs() @ w2.abs().t() + b.abs()) / tau
    # the tensor core's accumulator truncates, 2 u of the running sum per 16 products; a target's logit is one
    # of them and is allowed what a dot product of its own in fp32 would add (D / 32 terms a lane, then 5),
    # the sum below counting the product's error twice as it is
    ez = (D / 16 + 12) * 2 * U * mag
    et = (D / 32 * 8 + 16) * U * mag
    lse = torch.logsumexp(z, 1)
    # the sum of V exponentials: 64 terms one after another, then tiles; the exponents' roundings
    elt = (2 * U * (z.abs() + lse.abs()[:, None]) + 100 * U + V / 2048 * U) + ez
    q = torch.exp(z - lse[:, None])
    elt = elt + (q * elt).sum(1, keepdim=True)         # of log q: its own and the sum's
    tk = torch.where(kept, t, torch.full_like(t, -float("inf")))
    lp = tk - torch.logsumexp(tk, 1, keepdim=True)
    p = torch.exp(lp)
    lp0 = torch.where(kept, lp, torch.zeros_like(lp))
    ii = idx.clamp(0, V - 1)
    zt = torch.where(kept, z.gather(1, ii), torch.zeros_like(lp))
    rp = (30 + 4 * torch.where(kept, t, torch.zeros_like(t)).abs().amax(1, keepdim=True) + 2 * lp0.abs()) * U
    if logits is None:
        rp = torch.zeros_like(rp)
    each = tau * tau * ((p * (lp0 - zt)).sum(1) + lse)
    K = idx.shape[1]
    eeach = tau * tau * ((p * (rp * (1 + lp0.abs() + zt.abs()) + et.gather(1, ii) + (K + 8) * U * (lp0.abs() + zt.abs()))).sum(1)
                         + (q * elt).sum(1) + 8 * U * lse.abs() + 110 * U)
    bad = kept & ((idx >= V) | (idx < 0))
    each = torch.where(bad.any(1), torch.full_like(each, float("nan")), each)
    n = max(1, rows.numel())
    if reduction == "none":
        loss, el = torch.zeros(T * B, dtype=f), torch.zeros(T * B, dtype=f)
        loss[rows], el[rows] = each, eeach
        loss, el = loss.view(T, B), el.view(T, B)
    else:
        s = n if reduction == "mean" else 1
        loss, el = each.sum() / s, eeach.sum() / s + 4 * U * each.abs().sum() / s
    r = dict(loss=loss, e_loss=el)
    if g is None:
        return r
    g = g.double()
    c = (g.reshape(-1)[rows] if reduction == "none" else (g / (n if reduction == "mean" else 1)).expand(rows.numel())) * tau
    P = torch.zeros_like(q).scatter_add_(1, ii, p)
    eP = torch.zeros_like(q).scatter_add_(1, ii, p * (rp + (K + 2) * U))
    G = c[:, None] * (q - P)
    eG = c.abs()[:, None] * (q * (elt + et) + eP + 4 * U * (q + P))
    eG = eG + half * (G.abs() + eG) + c.abs().max().item() * 2.0 ** -38 if rows.numel() else eG

    def spread(v):
        full = torch.zeros(T * B, v.shape[1], dtype=f)
        full[rows] = v
        return full.view(T, B, -1)

    acc = lambda k: (k / 16 + 24) * 2 * U   # noqa: E731
    r["dx"], r["e_dx"] = spread(G @ w2), spread((eG + acc(V) * G.abs()) @ w2.abs())
    r["dw"], r["e_dw"] = G.t() @ x2, (eG + acc(n) * G.abs()).t() @ x2.abs()
    r["db"], r["e_db"] = G.sum(0), (eG + (n + 8) * U * G.abs()).sum(0)
    return r

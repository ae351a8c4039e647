"""Definitions, in 64 bits, of the long-sequence operators (rotary positions, query / key norms, window attention, ring cache),
with error bounds for kernels that compute in fp32 and round operands and results to the tensors' type.

Bounds are worst cases of rounding: an fp32 operation is off by at most E = 2^-24 of its result, a sum of n terms by at
most n E of the sum of their absolute values, a rounding to the type by U = eps / 2 of the value."""
import torch

E = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------------- rotary
def turn(x, table, rows, inter, inverse=False):
    """x float64 [B, N, H, dh], rows int64 [B, N]: (y, sum of the absolute values of each result's terms)."""
    rot = 2 * table.shape[1]
    t = table.double()[rows][:, :, None]                                        # [B, N, 1, pairs, 2]
    c, s = t[..., 0], t[..., 1] * (-1 if inverse else 1)
    r = x[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    y = (a * c - b * s, b * c + a * s)
    m = ((a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs())
    join = (lambda u: torch.stack(u, -1).flatten(-2)) if inter else (lambda u: torch.cat(u, -1))
    return torch.cat((join(y), x[..., rot:]), -1), torch.cat((join(m), x[..., rot:].abs()), -1)


def norm_turn(x, g, eps, table, rows, inter):
    """(y, bound without the result's own rounding): y = R(g x r)."""
    x = x.double()
    dh = x.shape[-1]
    g = torch.ones(dh, dtype=torch.float64, device=x.device) if g is None else g.double()
    n = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * g
    # the mean of dh squares (dh + 3 roundings, half of that after the root), root, quotient, two products: all relative
    rel = (dh / 2 + 8) * E
    if table is None:
        return n, rel * n.abs()
    y, m = turn(n, table, rows, inter)
    return y, (rel + 3 * E) * m


def norm_turn_grad(x, g, eps, table, rows, inter, dy):
    """(dx, its bound, dgamma, its bound); bounds without the results' own roundings."""
    x, dy = x.double(), dy.double()
    dh = x.shape[-1]
    g = torch.ones(dh, dtype=torch.float64, device=x.device) if g is None else g.double()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    u, m = (dy, dy.abs()) if table is None else turn(dy, table, rows, inter, inverse=True)
    t, ta = u * g, m * g.abs()
    mean, mean_a = (t * x).mean(-1, keepdim=True), (ta * x.abs()).mean(-1, keepdim=True)
    dx = r * (t - x * r * r * mean)
    rel = (3 * (dh / 2 + 8) + dh + 12) * E                   # r three times over, the sum of dh products, the rest
    bx = rel * r * (ta + x.abs() * r * r * mean_a)
    terms = (m * x.abs() * r).reshape(-1, dh)
    dg = (u * x * r).reshape(-1, dh).sum(0)
    bg = (terms.shape[0] + dh / 2 + 16) * E * terms.sum(0)   # a chain of at most every row
    return dx, bx, dg, bg


# --------------------------------------------------------------------------------------------------- window attention
def visible(N, window, sinks, causal, n, device):
    i = torch.arange(N, device=device)[:, None]
    j = torch.arange(N, device=device)[None, :]
    ok = torch.ones(N, N, dtype=torch.bool, device=device) if window < 0 else ((i - j).abs() <= window) | (j < sinks)
    if causal:
        ok = ok & (j <= i)
    return ok & (i < n) & (j < n)


def window_attention(q, k, v, window, sinks, causal, scale, lengths, do=None):
    """Every result and its bound, float64: dict of name -> (value, bound with the result's own rounding)."""
    B, N, Hq, dh = q.shape
    Hk = k.shape[2]
    G = Hq // Hk
    U = unit(q.dtype)
    UP = U if q.dtype != torch.float32 else E                # P and dS as operands of their product
    names = ['o'] + (['dq', 'dk', 'dv'] if do is not None else [])
    shapes = {'o': q, 'dq': q, 'dk': k, 'dv': k}
    out = {t: [torch.zeros(shapes[t].shape, dtype=torch.float64, device=q.device) for _ in range(2)] for t in names}
    for b in range(B):
        n = N if lengths is None else max(0, min(N, int(lengths[b])))
        if n == 0:
            continue
        ok = visible(n, window, sinks, causal, n, q.device)
        for h in range(Hq):
            Q, K, V = q[b, :n, h].double(), k[b, :n, h // G].double(), v[b, :n, h // G].double()
            s = (Q @ K.T * scale).masked_fill(~ok, float('-inf'))
            P = torch.softmax(s, -1)
            P = torch.where(ok, P, torch.zeros_like(P))      # rows are never empty here: a query sees itself
            # a score: dh products and their sum, the scale, and the subtraction of the maximum (up to twice the largest)
            sa = (Q.abs() @ K.abs().T * scale).masked_fill(~ok, 0.0)
            ds = ((dh + 3) * E * sa + 4 * E * sa.amax(-1, keepdim=True)).amax(-1, keepdim=True)
            relp = 2 * ds + 8 * E                            # exp2 within 2 E, and the reference point of the row on both sides
            A = P @ V.abs()
            O = P @ V
            bo = A * (UP + relp + (2 * n + 4) * E)
            out['o'][0][b, :n, h] = O
            out['o'][1][b, :n, h] = bo + U * O.abs()
            if do is None:
                continue
            D = do[b, :n, h].double()
            dP, dPa = D @ V.T, D.abs() @ V.abs().T
            delta = (D * O).sum(-1, keepdim=True)
            bdelta = (D.abs() * (bo + U * O.abs())).sum(-1, keepdim=True) + dh * E * (D * O).abs().sum(-1, keepdim=True)
            dS = P * (dP - delta)
            relb = relp + (n + 8) * E                        # P made again from the row's log-sum
            bS = dS.abs() * (UP + relb + 2 * E) + P * (dh * E * dPa + bdelta)
            e = lambda M, bM, X: bM @ X.abs() + n * E * (M.abs() @ X.abs())          # noqa: E731  sum over up to n terms
            dq = dS @ K * scale
            out['dq'][0][b, :n, h] = dq
            out['dq'][1][b, :n, h] = scale * e(dS, bS, K) + (U + 2 * E) * dq.abs()
            out['dk'][0][b, :n, h // G] += dS.T @ Q * scale
            out['dk'][1][b, :n, h // G] += scale * G * e(dS.T, bS.T, Q)
            out['dv'][0][b, :n, h // G] += P.T @ D
            out['dv'][1][b, :n, h // G] += G * e(P.T, P.T * (UP + relb), D)
    for t in ('dk', 'dv'):
        if t in out:
            out[t][1] += (U + 2 * E) * out[t][0].abs()
    return out


def ring_slot(p, C, sinks):
    return p if p < sinks else sinks + (p - sinks) % (C - sinks)


def decode(q, k, v, kc, vc, lengths, window, sinks, scale):
    """(out, bound, k cache, v cache) of one new token a sequence; the caches as their own type, updated."""
    B, Hq, dh = q.shape
    Hk, C = kc.shape[1:3]
    kc, vc = kc.clone(), vc.clone()
    U = unit(q.dtype)
    o = torch.zeros(B, Hq, dh, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(o)
    for b in range(B):
        p = int(lengths[b])
        if p < 0:
            continue
        if window < 0 and p >= C:
            o[b] = float('nan')
            continue
        S = 0 if window < 0 else sinks
        slot = p if window < 0 else ring_slot(p, C, S)
        kc[b, :, slot], vc[b, :, slot] = k[b], v[b]
        at = list(range(p + 1)) if window < 0 else \
            [ring_slot(t, C, S) for t in list(range(min(S, p + 1))) + list(range(max(S, p - window), p + 1))]
        at = torch.tensor(at, device=q.device)
        for h in range(Hq):
            K, V = kc[b, h // (Hq // Hk), at].double(), vc[b, h // (Hq // Hk), at].double()
            s = K @ q[b, h].double() * scale
            sa = K.abs() @ q[b, h].double().abs() * scale
            P = torch.softmax(s, 0)
            o[b, h] = P @ V
            rel = 2 * ((dh + 6) * E * sa).max() + (2 * len(at) + 24) * E
            bound[b, h] = rel * (P @ V.abs()) + U * o[b, h].abs()
    return o, bound, kc, vc


def fill(k, v, C, sinks, lengths, kc, vc):
    kc, vc = kc.clone(), vc.clone()
    for b in range(k.shape[0]):
        n = k.shape[1] if lengths is None else max(0, min(k.shape[1], int(lengths[b])))
        for t in range(n):
            kc[b, :, ring_slot(t, C, sinks)], vc[b, :, ring_slot(t, C, sinks)] = k[b, t], v[b, t]
    return kc, vc


def within(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f'{what}: not finite'
    off = (got - want).abs() - bound
    worst = float(off.max()) if off.numel() else 0.0
    assert worst <= 0, f'{what}: over its bound by {worst:.3e} at {int(off.argmax())} of {tuple(got.shape)}'

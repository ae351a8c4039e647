"""Cases for timing the long-sequence attention operators: rotary positions, query/key norms with the rotation, attention
with a sliding window and sinks (forward, backward), its prefill and its single-token step on a ring cache.

``run`` computes a case either in elementary torch operations (``own`` false) or through the package (``own`` true)."""
import math

import torch

own = False

DEV = 'cuda'
DT = {'bf16': torch.bfloat16, 'f32': torch.float32}


# ------------------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # rotation of one new token's queries and keys in a streaming encoder: latency
        dict(name='rotary one token', op='rotary', B=1, N=1, H=12, dh=64, rot=64, axes=1, inter=False, scaling='none',
             start=577, build=False, dtype='bf16'),
        # a training batch of 384-pixel images, axial (row, column) positions, tables kept by the model
        dict(name='rotary axial train', op='rotary', B=32, N=577, H=12, dh=64, rot=64, axes=2, inter=False, scaling='none',
             start=0, build=False, dtype='bf16'),
        # one long stream far from its start, positions scaled, part of the head, the angles made for this call
        dict(name='rotary far scaled', op='rotary', B=1, N=16411, H=16, dh=80, rot=40, axes=1, inter=True, scaling='yarn',
             start=1000003, build=True, dtype='f32'),
        # norm + rotation of one token for 8 streams: latency
        dict(name='qk norm one token', op='qknorm', B=8, N=1, Hq=16, Hk=4, dh=64, rot=64, inter=False, train=False,
             dtype='bf16'),
        # a training batch of 224-pixel images
        dict(name='qk norm train', op='qknorm', B=128, N=197, Hq=12, Hk=12, dh=64, rot=64, inter=False, train=True,
             dtype='bf16'),
        # a long sequence with grouped heads, part of the head rotated, float32
        dict(name='qk norm long', op='qknorm', B=1, N=32769, Hq=16, Hk=4, dh=80, rot=40, inter=True, train=True,
             dtype='f32'),
        # 384-pixel images, neighbourhood attention with a visible class token
        dict(name='window train image', op='window', B=16, N=577, Hq=12, Hk=12, dh=64, window=64, sinks=1, causal=False,
             ragged=False, train=True, dtype='bf16'),
        # a long causal sequence with grouped heads of 128
        dict(name='window train long', op='window', B=1, N=16384, Hq=16, Hk=4, dh=128, window=1024, sinks=4, causal=True,
             ragged=False, train=True, dtype='bf16'),
        # images of several sizes padded to one length, float32, every key visible, heads of 80
        dict(name='window train ragged f32', op='window', B=3, N=1001, Hq=16, Hk=16, dh=80, window=-1, sinks=0,
             causal=False, ragged=True, train=True, dtype='f32'),
        # prompts of a streaming encoder: attention and the ring cache they leave behind
        dict(name='prefill', op='prefill', B=4, N=4097, Hq=12, Hk=12, dh=64, window=512, sinks=4, ragged=True, dtype='bf16'),
        # one stream, one token: latency
        dict(name='decode one stream', op='decode', B=1, Hq=12, Hk=12, dh=64, window=511, sinks=1, filled='full',
             dtype='bf16'),
        # many streams with long windows and grouped heads: the cache's bandwidth
        dict(name='decode many streams', op='decode', B=64, Hq=16, Hk=4, dh=128, window=4095, sinks=4, filled='mixed',
             dtype='bf16'),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['rotary', 'qknorm', 'window', 'window', 'prefill', 'decode'])
    dtype = rng.choice(['bf16', 'bf16', 'f32'])
    dh = rng.choice([32, 64, 64, 80, 128])
    Hk = rng.choice([1, 2, 3, 4, 8, 12])
    G = min(rng.choice([1, 1, 2, 3, 4]), 16 // Hk)
    sinks = rng.choice([0, 1, 4, rng.randint(2, 70)])
    if op == 'rotary':
        rows = _log(rng, 1, 16000)
        B = rng.choice([1, 2, 5, 16])
        axes = rng.choice([1, 1, 2])
        rot = rng.choice([dh, dh // 2])
        return dict(op=op, B=B, N=max(1, rows // B), H=Hk * G, dh=dh, rot=rot, axes=axes, inter=rng.random() < 0.5,
                    scaling=rng.choice(['none', 'linear', 'ntk', 'yarn']), start=rng.choice([0, _log(rng, 1, 4000000)]),
                    build=rng.random() < 0.5, dtype=dtype)
    if op == 'qknorm':
        rows = _log(rng, 1, 14000)
        B = rng.choice([1, 3, 8, 32])
        return dict(op=op, B=B, N=max(1, rows // B), Hq=Hk * G, Hk=Hk, dh=dh, rot=rng.choice([0, dh // 2, dh]),
                    inter=rng.random() < 0.5, train=rng.random() < 0.7, dtype=dtype)
    if op == 'window':
        N = _log(rng, 1, 6000)
        B = max(1, min(rng.choice([1, 2, 4, 16]), 8000 // N))
        window = rng.choice([-1, _log(rng, 1, 1000), _log(rng, 1, 1000)]) if N <= 1500 else _log(rng, 8, 1000)
        return dict(op=op, B=B, N=N, Hq=Hk * G, Hk=Hk, dh=dh, window=window, sinks=sinks, causal=rng.random() < 0.5,
                    ragged=rng.random() < 0.4, train=rng.random() < 0.8, dtype=dtype)
    if op == 'prefill':
        N = _log(rng, 1, 6000)
        return dict(op=op, B=max(1, min(rng.choice([1, 2, 4]), 8000 // N)), N=N, Hq=Hk * G, Hk=Hk, dh=dh,
                    window=_log(rng, 1, 1024), sinks=sinks, ragged=rng.random() < 0.5, dtype=dtype)
    window = _log(rng, 1, 6000)
    return dict(op=op, B=max(1, min(_log(rng, 1, 64), 60000 // window)), Hq=Hk * G, Hk=Hk, dh=dh, window=window, sinks=sinks,
                filled=rng.choice(['full', 'mixed', 'young']), dtype=dtype)


# ----------------------------------------------------------------------------------------------------------- the inputs
def _scaling(case):
    kind = case['scaling']
    return {'none': None, 'linear': dict(type='linear', factor=4.0), 'ntk': dict(type='ntk', factor=8.0),
            'yarn': dict(type='yarn', factor=16.0, original=4096)}[kind]


def _lengths(case, g):
    """Tokens of each padded sequence: the first fills its row, the others end anywhere."""
    B, N = case['B'], case['N']
    if not case['ragged']:
        return None
    n = torch.randint(1, N + 1, (B,), generator=g, device=DEV)
    n[0] = N
    return n.to(torch.int32)


def _positions(case):
    B, N, start = case['B'], case['N'], case['start']
    i = torch.arange(N, device=DEV, dtype=torch.int64)
    if case['axes'] == 1:
        return i + start
    side = max(1, math.isqrt(N))
    return torch.stack((start + i // side, start + i % side), 1)       # rows and columns of the patch grid


def _ring(case):
    """Slots of a ring cache: the sinks, and the window with the new token, up to a multiple of 64."""
    return case['sinks'] + -(-(case['window'] + 1) // 64) * 64


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(1000003 * (seed + 1) + 17)
    dt = DT[case['dtype']]
    op = case['op']

    def normal(*shape, mul=1.0):
        return (torch.randn(*shape, generator=g, device=DEV) * mul).to(dt)

    s = dict(case=case)
    if op == 'rotary':
        B, N, H, dh = case['B'], case['N'], case['H'], case['dh']
        s['x'] = normal(B, N, 2 * H, dh)[:, :, :H]                     # the queries of a packed projection
        s['dy'] = normal(B, N, H, dh)
        s['positions'] = _positions(case)
        s['table'] = None if case['build'] else _plain_table(s['positions'], case['rot'], _scaling(case))
    elif op == 'qknorm':
        B, N, Hq, Hk, dh = case['B'], case['N'], case['Hq'], case['Hk'], case['dh']
        qkv = normal(B, N, Hq + 2 * Hk, dh, mul=1.7)
        s['q'], s['k'] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk]
        s['gq'] = 1 + 0.2 * torch.randn(dh, generator=g, device=DEV)
        s['gk'] = 1 + 0.2 * torch.randn(dh, generator=g, device=DEV)
        s['table'] = _plain_table(torch.arange(N, device=DEV), case['rot'], None) if case['rot'] else None
        if case['train']:
            s['dq'], s['dk'] = normal(B, N, Hq, dh), normal(B, N, Hk, dh)
    elif op in ('window', 'prefill'):
        B, N, Hq, Hk, dh = case['B'], case['N'], case['Hq'], case['Hk'], case['dh']
        qkv = normal(B, N, Hq + 2 * Hk, dh)
        s['q'], s['k'], s['v'] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]
        s['lengths'] = _lengths(case, g)
        if op == 'prefill':
            C = _ring(case)
            s['kc'], s['vc'] = (torch.zeros(B, Hk, C, dh, device=DEV, dtype=dt) for _ in range(2))
        elif case['train']:
            s['do'] = normal(B, N, Hq, dh)
    else:
        B, Hq, Hk, dh, w = case['B'], case['Hq'], case['Hk'], case['dh'], case['window']
        C = _ring(case)
        s['q'], s['k'], s['v'] = normal(B, Hq, dh), normal(B, Hk, dh), normal(B, Hk, dh)
        s['kc'], s['vc'] = normal(B, Hk, C, dh), normal(B, Hk, C, dh)
        lo, hi = {'full': (C + w, 4 * C), 'mixed': (0, 3 * C), 'young': (0, max(1, w // 2))}[case['filled']]
        s['lengths'] = torch.randint(lo, hi + 1, (B,), generator=g, device=DEV).to(torch.int32)
    return s


# ------------------------------------------------------------------------------------------------------ the plain forms
def _plain_table(positions, dim, scaling, base=10000.0):
    """(cos, sin) of every position and pair, float32 [P, dim / 2, 2]; the axes of 2-D positions share the pairs evenly."""
    pos = positions.double().reshape(positions.shape[0], -1)
    A = pos.shape[1]
    d = dim // A
    i = torch.arange(d // 2, device=pos.device, dtype=torch.float64)
    kind, f = (scaling['type'], scaling['factor']) if scaling else (None, 1.0)
    if kind == 'ntk':
        base = base * f ** (d / (d - 2)) if d > 2 else base
    freq = base ** (-2.0 * i / d)
    m = 1.0
    if kind == 'linear':
        freq = freq / f
    elif kind == 'yarn':
        ramp = ((scaling['original'] * freq / (2 * math.pi) - 1.0) / 31.0).clamp(0, 1)
        freq = freq * ((1 - ramp) / f + ramp)
        m = 0.1 * math.log(f) + 1.0
    a = (pos[:, :, None] * freq).reshape(pos.shape[0], dim // 2)
    return (m * torch.stack((a.cos(), a.sin()), -1)).float()


def _plain_rotate(x, table, inter):
    """x float32 [B, N, H, dh], row n of the table for token n."""
    rot = 2 * table.shape[1]
    c, s = table[None, :, None, :, 0], table[None, :, None, :, 1]
    r = x[..., :rot]
    if inter:
        a, b = r[..., 0::2], r[..., 1::2]
        y = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = r[..., :rot // 2], r[..., rot // 2:]
        y = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _plain_rotary(x, table, inter):
    return _plain_rotate(x.float(), table, inter).to(x.dtype)


def _plain_qk_norm(q, k, gq, gk, table, inter):
    def one(x, g):
        y = x.float()
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * g
        return (y if table is None else _plain_rotate(y, table, inter)).to(x.dtype)
    return one(q, gq), one(k, gk)


BLOCK = 128


def _plain_window(q, k, v, window, sinks, causal, lengths):
    """softmax over the visible keys.  A finite window goes by blocks of queries against the keys that a block can reach
    (and the sinks apart), so nothing of size N x N is made."""
    B, N, Hq, dh = q.shape
    Hk = k.shape[2]
    G = Hq // Hk
    dev = q.device
    n = torch.full((B,), N, device=dev) if lengths is None else lengths
    qf = q.float().view(B, N, Hk, G, dh).permute(0, 2, 1, 3, 4)                       # [B, Hk, N, G, dh]
    kf, vf = (t.float().permute(0, 2, 1, 3) for t in (k, v))                          # [B, Hk, N, dh]
    S = min(sinks, N)
    if window < 0 or 2 * window + BLOCK >= N:
        blk, nb, left, span = N, 1, 0, N
        kw, vw = kf[:, :, None], vf[:, :, None]
    else:
        blk, nb, left = BLOCK, -(-N // BLOCK), window
        right = 0 if causal else window
        span = left + blk + right
        pad = nb * blk - N
        qf = torch.nn.functional.pad(qf, (0, 0, 0, 0, 0, pad))
        kw, vw = (torch.nn.functional.pad(t, (0, 0, left, pad + right)).unfold(2, span, blk).transpose(-1, -2).contiguous()
                  for t in (kf, vf))                                                  # [B, Hk, nb, span, dh]
    qb = qf.reshape(B, Hk, nb, blk * G, dh)
    i = torch.arange(nb, device=dev)[:, None, None] * blk + torch.arange(blk, device=dev)[None, :, None]
    j = torch.arange(nb, device=dev)[:, None, None] * blk - left + torch.arange(span, device=dev)[None, None, :]
    seen = (j >= 0) & (j < N)
    if window >= 0:
        seen = seen & (((i - j).abs() <= window) | (j < S))
    if causal:
        seen = seen & (j <= i)
    nn = n.view(B, 1, 1, 1)
    seen = (seen[None] & (j[None] < nn) & (i[None] < nn))[:, None, :, :, None, :]      # [B, 1, nb, blk, 1, span]
    s = torch.matmul(qb, kw.transpose(-1, -2).contiguous()) * dh ** -0.5
    s = s.view(B, Hk, nb, blk, G, span).masked_fill(~seen, -math.inf)
    if S and nb > 1:                                                                  # sinks that the block does not reach
        js = torch.arange(S, device=dev)
        far = js[None, None, :] < (j[:, :, :1])
        if not causal:
            far = far | (js[None, None, :] > j[:, :, -1:])
        far = (far[None] & (js[None, None, None] < nn) & (i[None] < nn))[:, None, :, :, None, :]
        ks, vs = kf[:, :, None, :S].expand(B, Hk, nb, S, dh), vf[:, :, None, :S].expand(B, Hk, nb, S, dh)
        t = torch.matmul(qb, ks.transpose(-1, -2).contiguous()) * dh ** -0.5
        s = torch.cat((s, t.view(B, Hk, nb, blk, G, S).masked_fill(~far, -math.inf)), -1)
        vw = torch.cat((vw, vs), 3)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    den = p.sum(-1, keepdim=True)
    p = p / torch.where(den == 0, torch.ones_like(den), den)
    o = torch.matmul(p.view(B, Hk, nb, blk * G, -1), vw.contiguous())
    o = o.reshape(B, Hk, nb * blk, G, dh)[:, :, :N].permute(0, 2, 1, 3, 4).reshape(B, N, Hq, dh)
    return o.to(q.dtype)


def _plain_fill(k, v, kc, vc, lengths, sinks):
    """Each slot takes the last token that belongs in it."""
    B, N, Hk, dh = k.shape
    C = kc.shape[2]
    R = C - sinks
    n = (torch.full((B,), N, device=k.device) if lengths is None else lengths.long())[:, None]
    c = torch.arange(C, device=k.device)[None]
    p = torch.where(c < sinks, c, n - 1 - torch.remainder(n - 1 - c, R))
    has = (p < n) & ((c < sinks) | (p >= sinks))
    at = p.clamp(0, N - 1)[:, None, :, None].expand(B, Hk, C, dh)
    has = has[:, None, :, None]
    kc.copy_(torch.where(has, k.permute(0, 2, 1, 3).gather(2, at), kc))
    vc.copy_(torch.where(has, v.permute(0, 2, 1, 3).gather(2, at), vc))


def _plain_decode(q, k, v, kc, vc, lengths, window, sinks):
    B, Hq, dh = q.shape
    Hk, C = kc.shape[1:3]
    R = C - sinks
    p = lengths.long()
    slot = torch.where(p < sinks, p, sinks + torch.remainder(p - sinks, R))
    b = torch.arange(B, device=q.device)
    kc[b, :, slot] = k
    vc[b, :, slot] = v
    c = torch.arange(C, device=q.device)[None]
    pos = torch.where(c < sinks, c, p[:, None] - torch.remainder(p[:, None] - c, R))
    seen = (pos <= p[:, None]) & ((c < sinks) | ((pos >= sinks) & (p[:, None] - pos <= window)))
    s = torch.matmul(q.float().view(B, Hk, Hq // Hk, dh), kc.float().transpose(-1, -2).contiguous()) * dh ** -0.5
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(s - s.amax(-1, keepdim=True))
    return (torch.matmul(e, vc.float()) / e.sum(-1, keepdim=True)).reshape(B, Hq, dh).to(q.dtype)


# -------------------------------------------------------------------------------------------------------------- a pass
def run(s):
    case = s['case']
    op = case['op']
    if own:
        from vit_amd import functional as VF
    if op == 'rotary':
        x = s['x'].detach().requires_grad_(True)
        table = s['table']
        if own:
            if table is None:
                table = VF.rotary_table(s['positions'], case['rot'], scaling=_scaling(case))
            y = VF.rotary(x, table, interleaved=case['inter'])
        else:
            if table is None:
                table = _plain_table(s['positions'], case['rot'], _scaling(case))
            y = _plain_rotary(x, table, case['inter'])
        dx, = torch.autograd.grad(y, x, s['dy'])
        return dict(y=y.detach(), dx=dx, table=table)
    if op == 'qknorm':
        ins = [s['q'], s['k'], s['gq'], s['gk']]
        if case['train']:
            ins = [t.detach().requires_grad_(True) for t in ins]
        if own:
            q, k = VF.qk_norm_rotary(*ins, s['table'], interleaved=case['inter'])
        else:
            q, k = _plain_qk_norm(*ins, s['table'], case['inter'])
        if not case['train']:
            return dict(q=q, k=k)
        grads = torch.autograd.grad((q, k), ins, (s['dq'], s['dk']))
        return dict(q=q.detach(), k=k.detach(), dq=grads[0], dk=grads[1], dgq=grads[2], dgk=grads[3])
    if op == 'window':
        ins = [s['q'], s['k'], s['v']]
        if case['train']:
            ins = [t.detach().requires_grad_(True) for t in ins]
        f = VF.window_attention if own else _plain_window
        o = f(*ins, case['window'], sinks=case['sinks'], causal=case['causal'], lengths=s['lengths'])
        if not case['train']:
            return dict(o=o)
        grads = torch.autograd.grad(o, ins, s['do'])
        return dict(o=o.detach(), dq=grads[0], dk=grads[1], dv=grads[2])
    if op == 'prefill':
        if own:
            o = VF.window_attention(s['q'], s['k'], s['v'], case['window'], sinks=case['sinks'], causal=True,
                                    lengths=s['lengths'])
            VF.window_cache_fill(s['k'], s['v'], s['kc'], s['vc'], sinks=case['sinks'], lengths=s['lengths'])
        else:
            o = _plain_window(s['q'], s['k'], s['v'], case['window'], case['sinks'], True, s['lengths'])
            _plain_fill(s['k'], s['v'], s['kc'], s['vc'], s['lengths'], case['sinks'])
        return dict(o=o, k_cache=s['kc'], v_cache=s['vc'])
    if own:
        o = VF.window_decode(s['q'], s['k'], s['v'], s['kc'], s['vc'], s['lengths'], case['window'], sinks=case['sinks'])
    else:
        o = _plain_decode(s['q'], s['k'], s['v'], s['kc'], s['vc'], s['lengths'], case['window'], case['sinks'])
    return dict(o=o, k_cache=s['kc'], v_cache=s['vc'])


# ------------------------------------------------------------------------------------------------------------- its work
def _pairs(N, window, sinks, causal):
    """Visible (query, key) pairs of one sequence of N tokens."""
    if window < 0:
        return N * (N + 1) // 2 if causal else N * N
    w, S = min(window, N - 1), min(sinks, N)
    one = (w + 1) * N - w * (w + 1) // 2
    m = max(0, N - 1 - w)                                       # queries i > w: their sinks j < S with j < i - w
    e = min(S, m)
    far = e * (e + 1) // 2 + (m - e) * S
    if causal:
        return one + far
    e = max(0, S - 1 - w)                                       # queries i < S - 1 - w: sinks j > i + w
    return 2 * one - N + far + e * (e + 1) // 2


def _sizes(case):
    """Tokens of each sequence; ragged ones as their generator gives them on average."""
    return [case['N']] + [(case['N'] + 1) // 2 if case['ragged'] else case['N']] * (case['B'] - 1)


def work(case):
    e = 2 if case['dtype'] == 'bf16' else 4
    op, dh = case['op'], case['dh']
    if op == 'rotary':
        n = case['B'] * case['N'] * case['H']
        return {'bytes': 4 * n * dh * e + case['N'] * case['rot'] * 4, 'flops': 2 * n * case['rot'] * 3}
    if op == 'qknorm':
        n = case['B'] * case['N'] * (case['Hq'] + case['Hk'])
        return {'bytes': (5 if case['train'] else 2) * n * dh * e, 'flops': (20 if case['train'] else 6) * n * dh}
    if op == 'window' or op == 'prefill':
        sizes = _sizes(case)
        pairs = case['Hq'] * sum(_pairs(m, case['window'], case['sinks'], op == 'prefill' or case['causal']) for m in sizes)
        rows = sum(sizes)
        train = op == 'window' and case['train']
        nbytes = rows * dh * e * ((6 * case['Hq'] + 6 * case['Hk']) if train else (2 * case['Hq'] + 2 * case['Hk']))
        if op == 'prefill':
            nbytes += 2 * sum(min(m, _ring(case)) for m in sizes) * case['Hk'] * dh * e
        return {'bytes': nbytes, 'flops': (14 if train else 4) * dh * pairs}
    w, C = case['window'], _ring(case)
    held = {'full': w + 1 + case['sinks'], 'mixed': int(0.83 * (w + 1 + case['sinks'])) + 1, 'young': w // 4 + 1}[case['filled']]
    n = case['B'] * held
    return {'bytes': 2 * n * case['Hk'] * dh * e + 2 * case['B'] * (case['Hq'] + case['Hk']) * dh * e,
            'flops': 4 * n * case['Hq'] * dh}


# --------------------------------------------------------------------------------------- the definitions, in 64 bits
def _exact_turn(positions, dim, scaling):
    """Unit complex numbers (times the attention factor) by which the pairs are turned, complex128 [P, dim / 2]."""
    pos = positions.double()
    pos = pos[:, None] if pos.dim() == 1 else pos
    d = dim // pos.shape[1]
    cols, m = [], 1.0
    for a in range(pos.shape[1]):
        for i in range(d // 2):
            base = 10000.0
            if scaling and scaling['type'] == 'ntk' and d > 2:
                base *= scaling['factor'] ** (d / (d - 2))
            freq = math.exp(-2.0 * i / d * math.log(base))
            if scaling and scaling['type'] == 'linear':
                freq /= scaling['factor']
            if scaling and scaling['type'] == 'yarn':
                turns = scaling['original'] * freq / (2 * math.pi)
                keep = min(1.0, max(0.0, (turns - 1.0) / 31.0))
                freq = keep * freq + (1 - keep) * freq / scaling['factor']
                m = 0.1 * math.log(scaling['factor']) + 1.0
            cols.append(pos[:, a] * freq)
    angle = torch.stack(cols, 1)
    return torch.polar(torch.full_like(angle, m), angle)


def _exact_rotate(x, turn, inter):
    rot = 2 * turn.shape[1]
    if inter:
        z = torch.view_as_complex(x[..., :rot].unflatten(-1, (rot // 2, 2)).contiguous()) * turn[None, :, None]
        y = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(x[..., :rot // 2].contiguous(), x[..., rot // 2:rot].contiguous()) * turn[None, :, None]
        y = torch.cat((z.real, z.imag), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _exact_attention(q, k, v, do, n, window, sinks, causal):
    """One sequence: q [n, Hq, dh], k / v [n, Hk, dh] in float64, gradients by their formulas; rows in chunks."""
    N, Hq, dh = q.shape
    Hk = k.shape[1]
    G = Hq // Hk
    scale = 1.0 / math.sqrt(dh)
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    j = torch.arange(n, device=q.device)
    step = max(64, (1 << 27) // max(1, n * G))
    for h in range(Hk):
        heads = slice(h * G, (h + 1) * G)
        K, V = k[:n, h], v[:n, h]
        for a in range(0, n, step):
            e = min(n, a + step)
            i = torch.arange(a, e, device=q.device)[:, None]
            hidden = torch.zeros(e - a, n, dtype=torch.bool, device=q.device)
            if window >= 0:
                hidden |= ((i - j) > window) & (j >= sinks)
                hidden |= ((j - i) > window) & (j >= sinks)
            if causal:
                hidden |= j > i
            Q = q[a:e, heads]
            z = (Q.reshape(-1, dh) @ K.T).view(e - a, G, n) * scale
            z[hidden[:, None].expand_as(z)] = -math.inf
            P = torch.softmax(z, -1)
            O = (P.view(-1, n) @ V).view(e - a, G, dh)
            o[a:e, heads] = O
            if do is None:
                continue
            D = do[a:e, heads]
            dP = (D.reshape(-1, dh) @ V.T).view(e - a, G, n)
            dS = P * (dP - (D * O).sum(-1, keepdim=True))
            dq[a:e, heads] = (dS.view(-1, n) @ K).view(e - a, G, dh) * scale
            dk[:n, h] += dS.view(-1, n).T @ Q.reshape(-1, dh) * scale
            dv[:n, h] += P.view(-1, n).T @ D.reshape(-1, dh)
    return o, dq, dk, dv


def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    if op == 'rotary':
        turn = _exact_turn(s['positions'], case['rot'], _scaling(case))
        table = torch.view_as_real(turn)
        if s['table'] is not None:                         # a kept table is an input, with its own rounding
            table, turn = None, torch.view_as_complex(s['table'].double())
        return dict(y=_exact_rotate(s['x'].double(), turn, case['inter']),
                    dx=_exact_rotate(s['dy'].double(), turn.conj(), case['inter']), table=table)
    if op == 'qknorm':
        turn = None if s['table'] is None else torch.view_as_complex(s['table'].double())
        out = {}
        for name, x, g in (('q', s['q'], s['gq']), ('k', s['k'], s['gk'])):
            x, g = x.double(), g.double()
            r = 1.0 / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + 1e-6)
            y = g * x * r
            out[name] = y if turn is None else _exact_rotate(y, turn, case['inter'])
            if case['train']:
                u = s['d' + name].double()
                u = u if turn is None else _exact_rotate(u, turn.conj(), case['inter'])
                out['dg' + name] = (u * x * r).sum((0, 1, 2))
                out['d' + name] = r * (u * g - x * r * r * (u * g * x).mean(-1, keepdim=True))
        return out
    if op == 'window' or op == 'prefill':
        causal = op == 'prefill' or case['causal']
        pairs = case['B'] * case['Hq'] * case['N'] ** 2 * case['dh']
        if pairs > 2e12:
            return None
        n = [case['N']] * case['B'] if s['lengths'] is None else s['lengths'].tolist()
        q, k, v = (s[t].double() for t in 'qkv')
        do = s['do'].double() if 'do' in s else None
        each = [_exact_attention(q[b], k[b], v[b], None if do is None else do[b], n[b], case['window'], case['sinks'],
                                 causal) for b in range(case['B'])]
        o, dq, dk, dv = (torch.stack(t) for t in zip(*each))
        if op == 'window':
            return dict(o=o, dq=dq, dk=dk, dv=dv) if case['train'] else dict(o=o)
        kc, vc = (torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (s['kc'], s['vc']))
        S, R = case['sinks'], kc.shape[2] - case['sinks']
        for b in range(case['B']):
            first, last = torch.arange(min(S, n[b])), torch.arange(max(S, n[b] - R), max(S, n[b]))
            at = torch.cat((first, last))
            slot = torch.cat((first, S + (last - S) % R))
            kc[b, :, slot] = k[b, at].transpose(0, 1)
            vc[b, :, slot] = v[b, at].transpose(0, 1)
        return dict(o=o, k_cache=kc, v_cache=vc)
    S, R, w, G = case['sinks'], s['kc'].shape[2] - case['sinks'], case['window'], case['Hq'] // case['Hk']
    kc, vc, q = s['kc'].double(), s['vc'].double(), s['q'].double()
    o = torch.zeros_like(q)
    for b, p in enumerate(s['lengths'].tolist()):
        slot = p if p < S else S + (p - S) % R
        kc[b, :, slot], vc[b, :, slot] = s['k'][b].double(), s['v'][b].double()
        first = torch.arange(0, min(S, p + 1))
        last = torch.arange(max(S, p - w), max(S, p + 1))
        at = torch.cat((first, S + (last - S) % R)).to(DEV)
        for h in range(case['Hk']):
            z = q[b, h * G:(h + 1) * G] @ kc[b, h, at].T / math.sqrt(case['dh'])
            o[b, h * G:(h + 1) * G] = torch.softmax(z, -1) @ vc[b, h, at]
    return dict(o=o, k_cache=kc, v_cache=vc)

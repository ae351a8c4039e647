"""Window attention at scores whose log-sum has few or no bits left behind the point: forward and gradients.

Queries and keys are rows of a Hadamard matrix times 2^p, so that every score is exact in either type: 2^(2 p) times the width for
a key of the query's own code, 0 for the others.  The softmax of a row is then known whatever p is: equal shares for the keys
of its code, or, where it sees none of them, for all that it sees."""
import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


def _codes(g, width, p, dtype, B, N, H, dh, codes):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < width:
        h = torch.cat((torch.cat((h, h), 1), torch.cat((h, -h), 1)), 0)
    x = torch.zeros(B, N, H, dh, dtype=torch.float64, device='cuda')
    x[..., :width] = h.cuda()[torch.randint(0, codes, (B, N, H), generator=g, device='cuda')] * 2.0 ** p
    y = x.to(DT[dtype])
    assert torch.equal(y.double(), x)
    return y


def _want(q, k, v, do, window, sinks, causal, lengths, far):
    """Values and bounds as in long_ref, but for the scores, which are exact here.  What is left of P's error: two exponentials
    and two sums of up to n terms, and the rounding of the row's log-sum where it is small (at most 2^-15 of 2^9, times ln 2); and
    an exponential under 2^-126, the smallest normal fp32, may come as 0."""
    B, N, Hq, dh = q.shape
    G = Hq // k.shape[2]
    U = R.unit(q.dtype)
    UP = U if q.dtype != torch.float32 else R.E
    out = {t: [torch.zeros(x.shape, dtype=torch.float64, device='cuda') for _ in range(2)] for t, x in
           dict(o=q, dq=q, dk=k, dv=k).items()}
    for b in range(B):
        n = N if lengths is None else int(lengths[b])
        ok = R.visible(n, window, sinks, causal, n, 'cuda')
        for h in range(Hq):
            Q, K, V, D = (t.double() for t in (q[b, :n, h], k[b, :n, h // G], v[b, :n, h // G], do[b, :n, h]))
            P = torch.softmax((Q @ K.T).masked_fill(~ok, float('-inf')), -1)
            rel = (4 * n + 24) * R.E + (0 if far else 0.7 * 2.0 ** -15)
            tiny = 2.0 ** -126 * ok.double()
            O, A = P @ V, P @ V.abs()
            bo = A * (UP + rel) + tiny @ V.abs()
            dP, dPa = D @ V.T, D.abs() @ V.abs().T
            bD = (D.abs() * (bo + U * O.abs())).sum(-1, keepdim=True) + dh * R.E * (D * O).abs().sum(-1, keepdim=True)
            dS = P * (dP - (D * O).sum(-1, keepdim=True))
            bS = dS.abs() * (UP + rel + 2 * R.E) + P * (dh * R.E * dPa + bD) + tiny * (dPa + (D * O).abs().sum(-1, keepdim=True))
            e = lambda M, bM, X: bM @ X.abs() + n * R.E * (M.abs() @ X.abs())          # noqa: E731
            for t, x, bound, at in (('o', O, bo, h), ('dq', dS @ K, e(dS, bS, K), h), ('dk', dS.T @ Q, e(dS.T, bS.T, Q), h // G),
                                    ('dv', P.T @ D, e(P.T, P.T * (UP + rel) + tiny.T, D), h // G)):
                out[t][0][b, :n, at] += x
                out[t][1][b, :n, at] += G * bound if at != h or G > 1 else bound
    for t in out:
        out[t][1] += (U + 2 * R.E) * out[t][0].abs()
    return out


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('p', [1, 3, 6, 9, 12])
@pytest.mark.parametrize('case', [
    # B, N, Hq, Hk, dh, window, sinks, causal, padded: few scores; two waves a row, sinks apart; workgroups of 128 rows
    (1, 50, 2, 1, 64, -1, 0, False, False), (2, 77, 2, 2, 80, 9, 3, True, True), (1, 90, 1, 1, 32, 0, 0, False, False),
    (2, 300, 4, 2, 64, -1, 0, True, True), (1, 700, 2, 1, 64, 20, 5, True, False), (2, 260, 2, 2, 128, 40, 2, False, True),
    (14, 333, 8, 8, 64, 70, 1, False, True), (14, 300, 8, 8, 128, -1, 0, True, False)], ids=str)
def test_known_softmax(case, p, dtype):
    from vit_amd import functional as VF
    B, N, Hq, Hk, dh, window, sinks, causal, padded = case
    g = torch.Generator(device='cuda').manual_seed(71)
    width = 1 << (dh.bit_length() - 1)
    q, k = _codes(g, width, p, dtype, B, N, Hq, dh, 12), _codes(g, width, p, dtype, B, N, Hk, dh, 7)
    v, do = (torch.randn(B, N, h, dh, generator=g, device='cuda').to(DT[dtype]) for h in (Hk, Hq))
    lengths = torch.randint(1, N + 1, (B,), generator=g, device='cuda', dtype=torch.int32) if padded else None
    ins = [t.requires_grad_(True) for t in (q, k, v)]
    o = VF.window_attention(*ins, window, sinks=sinks, causal=causal, scale=1.0, lengths=lengths)
    got = dict(zip(('o', 'dq', 'dk', 'dv'), (o.detach(), *torch.autograd.grad(o, ins, do))))
    want = _want(*(t.detach() for t in ins), do, window, sinks, causal, lengths, width * 4 ** p > 512)
    for t, x in got.items():
        R.within(x, *want[t], t)

"""Window attention with sinks on the GPU: forward and gradients against the definition in 64 bits."""
import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _rand(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device='cuda').to(DT[dtype])


def _qkv(g, dtype, B, N, Hq, Hk, dh):
    qkv = _rand(g, dtype, B, N, Hq + 2 * Hk, dh)
    return qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hk], qkv[:, :, Hq + Hk:]


def _check(q, k, v, do, window, sinks, causal, lengths=None, scale=None):
    from vit_amd import functional as VF
    ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = VF.window_attention(*ins, window, sinks=sinks, causal=causal, lengths=lengths, scale=scale)
    dq, dk, dv = torch.autograd.grad(o, ins, do)
    assert o.dtype == q.dtype and o.is_contiguous()
    want = R.window_attention(q, k, v, window, sinks, causal, scale or q.shape[-1] ** -0.5, lengths, do)
    got = dict(o=o.detach(), dq=dq, dk=dk, dv=dv)
    for t, x in got.items():
        R.within(x, *want[t], t)
    with torch.no_grad():                                                            # the same bits without a backward
        assert torch.equal(VF.window_attention(q, k, v, window, sinks=sinks, causal=causal, lengths=lengths, scale=scale), o)
    return got


@pytest.mark.parametrize('causal', [False, True], ids=['both', 'causal'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('case', [
    # B, N, Hq, Hk, dh, window, sinks
    (1, 1, 1, 1, 8, 0, 0), (2, 1, 2, 1, 64, 3, 5), (1, 2, 1, 1, 32, 0, 1), (1, 31, 2, 2, 32, 4, 0), (2, 33, 4, 2, 64, 7, 1),
    (1, 64, 2, 2, 64, -1, 0), (1, 65, 3, 1, 80, 16, 40), (2, 127, 2, 2, 128, 20, 3), (1, 129, 4, 4, 40, 200, 9),
    (1, 197, 3, 3, 64, 12, 1), (1, 300, 2, 1, 96, 0, 2), (1, 300, 4, 1, 64, 31, 70), (1, 513, 2, 2, 64, 64, 33),
    (1, 577, 1, 1, 120, 100, 4), (1, 400, 2, 2, 24, -1, 3), (1, 700, 1, 1, 64, 40, 650)], ids=str)
def test_against_definition(case, dtype, causal):
    B, N, Hq, Hk, dh, window, sinks = case
    g = _gen(11)
    q, k, v = _qkv(g, dtype, B, N, Hq, Hk, dh)
    _check(q, k, v, _rand(g, dtype, B, N, Hq, dh), window, sinks, causal)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_many_workgroups(dtype):
    """Enough rows that the four-wave workgroups run (queries' and keys')."""
    g = _gen(12)
    q, k, v = _qkv(g, dtype, 8, 1025, 8, 8, 64)
    _check(q, k, v, _rand(g, dtype, 8, 1025, 8, 64), 50, 5, False)
    q, k, v = _qkv(g, dtype, 8, 1030, 8, 8, 128)
    _check(q, k, v, _rand(g, dtype, 8, 1030, 8, 128), 130, 1, True)
    q, k, v = _qkv(g, dtype, 16, 520, 8, 8, 80)
    _check(q, k, v, _rand(g, dtype, 16, 520, 8, 80), 33, 0, True)
    q, k, v = _qkv(g, dtype, 16, 520, 8, 8, 32)
    _check(q, k, v, _rand(g, dtype, 16, 520, 8, 32), 77, 3, False)


@pytest.mark.parametrize('causal', [False, True], ids=['both', 'causal'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('window,sinks', [(-1, 0), (10, 2), (40, 100)])
def test_lengths_and_poison_in_the_padding(window, sinks, dtype, causal):
    g = _gen(13)
    B, N, Hq, Hk, dh = 6, 150, 4, 2, 64
    q, k, v = (t.clone() for t in _qkv(g, dtype, B, N, Hq, Hk, dh))
    do = _rand(g, dtype, B, N, Hq, dh)
    lengths = torch.tensor([150, 0, 1, 64, 65, 97], dtype=torch.int32, device='cuda')
    clean = _check(q, k, v, do, window, sinks, causal, lengths)
    for b, n in enumerate(lengths.tolist()):
        for t, bad in ((q, float('nan')), (k, float('inf')), (v, float('nan')), (do, float('-inf'))):
            t[b, n:] = bad
        for t in clean.values():
            assert (t[b, n:] == 0).all()
    poisoned = _check(q, k, v, do, window, sinks, causal, lengths)
    for t in clean:
        assert torch.equal(clean[t], poisoned[t]), t
    lengths[0], lengths[2] = 1 << 30, -5                                             # past the rows: all of them; below 0: none
    _check(q, k, v, do, window, sinks, causal, lengths)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_layouts(dtype):
    """Heads-first tensors, a misaligned view, heads that are no unit stride, expanded keys, a gradient that is expanded."""
    from vit_amd import functional as VF
    g = _gen(14)
    B, N, H, dh = 2, 70, 4, 64
    heads = [_rand(g, dtype, B, H, N, dh).transpose(1, 2) for _ in range(3)]
    do = _rand(g, dtype, B, H, N, dh).transpose(1, 2)
    _check(*heads, do, 9, 2, True)
    odd = [_rand(g, dtype, B, N, H, dh + 1)[..., 1:] for _ in range(3)]
    _check(*odd, do, 9, 2, False)
    strided = [_rand(g, dtype, B, N, H, 2 * dh)[..., ::2] for _ in range(3)]
    _check(*strided, _rand(g, dtype, B, N, H, dh + 1)[..., 1:], 9, 2, False)
    one = _rand(g, dtype, B, N, 1, dh).requires_grad_(True)
    q = heads[0].detach()
    o = VF.window_attention(q, one.expand(B, N, H, dh), one.expand(B, N, H, dh), 9, sinks=1)
    got, = torch.autograd.grad(o.sum(), one)
    want = R.window_attention(q, one.detach().expand(B, N, H, dh), one.detach().expand(B, N, H, dh), 9, 1, False, dh ** -0.5, None,
                              torch.ones(1, dtype=q.dtype, device='cuda').expand(B, N, H, dh))
    U = R.unit(q.dtype)
    total = (want['dk'][0] + want['dv'][0]).sum(2, keepdim=True)
    size = (want['dk'][0].abs() + want['dv'][0].abs()).sum(2, keepdim=True)
    # each head's gradient within its bound, then the sum over heads and of the two roles in the tensors' type
    R.within(got, total, (want['dk'][1] + want['dv'][1]).sum(2, keepdim=True) + 3 * U * size, 'shared')


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_large_scores_and_scales(dtype):
    """Rows whose scores lie far apart, and a running maximum that keeps moving."""
    g = _gen(15)
    q, k, v = _qkv(g, dtype, 1, 300, 2, 2, 64)
    k = k * torch.linspace(0.1, 6, 300, device='cuda')[None, :, None, None].to(k.dtype)
    do = _rand(g, dtype, 1, 300, 2, 64)
    _check(q, k, v, do, 120, 3, True, scale=0.5)
    _check(q, k, v, do, 120, 3, False, scale=1e-3)


def test_minus_infinity_scores():
    """Keys at the type's lowest value, and queries whose every score is minus infinity but their own."""
    from vit_amd import functional as VF
    g = _gen(16)
    q = torch.rand(1, 40, 1, 32, generator=g, device='cuda') + 0.5
    k, v = (torch.randn(1, 40, 1, 32, generator=g, device='cuda') for _ in range(2))
    k[0, ::3] = torch.finfo(torch.float32).min / 64
    k[0, 1::3] = float('-inf')
    o = VF.window_attention(q, k, v, 8, sinks=2)
    s = (q[0, :, 0].double() @ k[0, :, 0].double().T) * 32 ** -0.5
    P = torch.softmax(s.masked_fill(~R.visible(40, 8, 2, False, 40, 'cuda'), float('-inf')), -1)
    assert torch.allclose(o[0, :, 0].double(), P @ v[0, :, 0].double(), atol=1e-4)


@pytest.mark.parametrize('causal', [False, True], ids=['both', 'causal'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('window', [3, 40, 150])
def test_a_row_depends_on_nothing_that_it_does_not_see(window, dtype, causal):
    """NaN and infinities in some tokens' k and v: the rows that do not see them are the same bits or, where a tile was shared,
    within the bounds; rows that see one are not finite."""
    from vit_amd import functional as VF
    g = _gen(20)
    N, sinks = 400, 2
    q, k, v = (t.clone() for t in _qkv(g, dtype, 1, N, 2, 1, 64))
    want = R.window_attention(q, k, v, window, sinks, causal, 0.125, None)['o']
    for j, t, x in ((100, v, float('nan')), (130, v, float('inf')), (260, k, float('nan')), (261, v, float('-inf'))):
        t[0, j] = x
    o = VF.window_attention(q, k, v, window, sinks=sinks, causal=causal)
    seen = R.visible(N, window, sinks, causal, N, 'cuda')[:, [100, 130, 260, 261]].any(1)
    assert not torch.isfinite(o[0, seen]).any()
    assert torch.isfinite(o[0, ~seen]).all()
    R.within(o[:, ~seen], want[0][:, ~seen], want[1][:, ~seen], 'unseen')


def test_same_bits_again_and_two_streams():
    from vit_amd import functional as VF
    g = _gen(17)
    sets = [(_qkv(g, 'bf16', 2, 600, 4, 2, 64), _rand(g, 'bf16', 2, 600, 4, 64)) for _ in range(2)]

    def step(s):
        ins = [t.detach().requires_grad_(True) for t in s[0]]
        o = VF.window_attention(*ins, 60, sinks=4)
        return (o.detach(), *torch.autograd.grad(o, ins, s[1]))
    alone = [step(s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s, st in zip(sets, streams):
            with torch.cuda.stream(st):
                got.append(step(s))
    torch.cuda.synchronize()
    for i, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, alone[i % 2]))


def test_captured_in_a_graph():
    """Forward and backward in one graph, replayed on new values with eager work between the replays."""
    from vit_amd import functional as VF
    g = _gen(18)
    x = _rand(g, 'bf16', 1, 200, 12, 64)
    do = _rand(g, 'bf16', 1, 200, 4, 64)
    lengths = torch.tensor([200], dtype=torch.int32, device='cuda')
    gam = torch.ones(64, device='cuda')
    table = VF.rotary_table(torch.arange(200, device='cuda'), 64)

    def step(x):
        x = x.detach().requires_grad_(True)
        q, k = VF.qk_norm_rotary(x[:, :, :4], x[:, :, 4:8], gam, gam, table)
        o = VF.window_attention(q, k, x[:, :, 8:], 30, sinks=2, causal=True, lengths=lengths)
        return o.detach(), torch.autograd.grad(o, x, do)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(x)
    for r in range(4):
        x.copy_(_rand(g, 'bf16', 1, 200, 12, 64))
        lengths.fill_(200 - 31 * r)
        want = step(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), r


def test_gradients_against_differences():
    from vit_amd import functional as VF
    g = _gen(19)
    q, k, v = (t.clone() for t in _qkv(g, 'f32', 1, 40, 2, 1, 16))
    w = torch.randn(1, 40, 2, 16, generator=g, device='cuda')
    ins = [t.requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(VF.window_attention(*ins, 6, sinks=2, causal=True), ins, w)
    dirs = [torch.randn(t.shape, generator=g, device='cuda', dtype=torch.float64) for t in ins]
    h = 1e-4

    def loss(s):
        a = [t.detach().double() + s * d for t, d in zip(ins, dirs)]
        return (R.window_attention(*a, 6, 2, True, 0.25, None)['o'][0] * w.double()).sum()
    diff = float((loss(h) - loss(-h)) / (2 * h))
    got = float(sum((u.double() * d).sum() for u, d in zip(grads, dirs)))
    size = float(sum((u.double() * d).abs().sum() for u, d in zip(grads, dirs)))
    # h^2 of a third derivative of order 100 of these values; each fp32 gradient within a few hundred E of its terms
    assert abs(got - diff) <= size * (1000 * h * h + 512 * R.E), (got, diff)


def test_empty():
    from vit_amd import functional as VF
    for B, N in ((0, 5), (2, 0)):
        x = torch.zeros(B, N, 3, 64, device='cuda', requires_grad=True)
        o = VF.window_attention(x, x, x, 4, sinks=1)
        o.sum().backward()
        assert o.shape == x.shape and x.grad.shape == x.shape


def test_refusals():
    from vit_amd import functional as VF
    from vit_amd._lib import VitkError
    x = torch.randn(1, 8, 4, 64, device='cuda')
    y = x[:, :, :3]
    i32 = torch.ones(1, dtype=torch.int32, device='cuda')
    for bad in (lambda: VF.window_attention(x[0], x, x, 2), lambda: VF.window_attention(x, y, y, 2),
                lambda: VF.window_attention(x, x, y, 2), lambda: VF.window_attention(x, x[:, :7], x[:, :7], 2),
                lambda: VF.window_attention(x, x.bfloat16(), x, 2), lambda: VF.window_attention(x, x, x, 2, sinks=-1),
                lambda: VF.window_attention(*[x[..., :60]] * 3, 2), lambda: VF.window_attention(*[torch.zeros(1, 2, 1, 136, device='cuda')] * 3, 2),
                lambda: VF.window_attention(x, x, x, 2, lengths=i32.long()),
                lambda: VF.window_attention(x, x, x, 2, lengths=torch.ones(2, dtype=torch.int32, device='cuda'))):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: VF.window_attention(x, x, x, 2, scale=0.0), lambda: VF.window_attention(x, x, x, 2, scale=-1.0),
                lambda: VF.window_attention(x, x, x, 2, scale=float('inf')), lambda: VF.window_attention(x.cpu(), x, x, 2),
                lambda: VF.window_attention(x, x, x, 2, lengths=i32.cpu())):
        with pytest.raises(VitkError):
            bad()
    with pytest.raises(TypeError):
        VF.window_attention(*[x.half()] * 3, 2)

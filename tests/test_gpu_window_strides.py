"""Window attention on tensors whose tokens share memory (a gradient that is broadcast over the tokens, expanded or overlapping
queries, keys and values), at lengths that end inside a tile: what lies behind the last token is nobody's."""
import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}

CASES = [
    # B, N, Hq, Hk, dh, padded: few scores; two waves a row; workgroups of 128 rows at a narrow and a wide head
    (2, 45, 2, 1, 64, False), (2, 45, 2, 1, 80, True), (2, 197, 4, 2, 64, False), (3, 333, 2, 2, 128, True),
    (14, 577, 8, 8, 64, True), (14, 577, 8, 4, 96, False)]


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _rand(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device='cuda').to(DT[dtype])


def _overlapping(g, dtype, B, N, H, dh):
    """Tokens 8 elements apart, heads behind them."""
    sh = 8 * N + dh
    return torch.as_strided(_rand(g, dtype, B * H * sh), (B, N, H, dh), (H * sh, 8, sh, 1))


def _lengths(g, B, N, padded):
    if not padded:
        return None
    n = torch.randint(1, N + 1, (B,), generator=g, device='cuda', dtype=torch.int32)
    n[0] = N - 5
    return n


def _grads(loss, q, k, v, window, sinks, causal, lengths):
    """Results of a training step whose loss is `loss` of the attention's output."""
    from vit_amd import functional as VF
    ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
    assert all(a.stride() == t.stride() for a, t in zip(ins, (q, k, v)))
    o = VF.window_attention(*ins, window, sinks=sinks, causal=causal, lengths=lengths)
    return dict(zip(('o', 'dq', 'dk', 'dv'), (o.detach(), *torch.autograd.grad(loss(o), ins))))


def _check(got, q, k, v, do, window, sinks, causal, lengths):
    want = R.window_attention(q, k, v, window, sinks, causal, q.shape[-1] ** -0.5, lengths, do)
    for t, x in got.items():
        R.within(x, *want[t], t)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('case', CASES, ids=str)
@pytest.mark.parametrize('window,sinks,causal', [(-1, 0, False), (-1, 0, True), (9, 2, False), (64, 0, True), (64, 40, False)])
def test_gradient_broadcast_over_the_tokens(window, sinks, causal, case, dtype):
    """What autograd hands to the backward of a sum over the tokens has a token stride of 0."""
    B, N, Hq, Hk, dh, padded = case
    g = _gen(61)
    q, k, v = _rand(g, dtype, B, N, Hq, dh), _rand(g, dtype, B, N, Hk, dh), _rand(g, dtype, B, N, Hk, dh)
    w = _rand(g, dtype, B, Hq, dh)
    lengths = _lengths(g, B, N, padded)
    do = w[:, None].expand(B, N, Hq, dh)
    for pool in (lambda o: o.sum(1), lambda o: torch.einsum('bnhd->bhd', o), lambda o: o.flatten(2).sum(1).view(B, Hq, dh)):
        _check(_grads(lambda o: (pool(o) * w).sum(), q, k, v, window, sinks, causal, lengths), q, k, v, do, window, sinks, causal,
               lengths)
        if B > 4:
            break                                        # one of them at the large sizes


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('case', CASES, ids=str)
@pytest.mark.parametrize('what', ['q', 'k', 'v', 'do'])
def test_expanded_and_overlapping_tokens(what, case, dtype):
    B, N, Hq, Hk, dh, padded = case
    g = _gen(62)
    H = dict(q=Hq, k=Hk, v=Hk, do=Hq)
    lengths = _lengths(g, B, N, padded)
    for one in (_rand(g, dtype, B, 1, H[what], dh).expand(B, N, H[what], dh), _overlapping(g, dtype, B, N, H[what], dh)):
        t = {x: _rand(g, dtype, B, N, H[x], dh) for x in H}
        t[what] = one
        for window, sinks, causal in ((-1, 0, False), (20, 3, True)):
            got = _grads(lambda o: _Feed.apply(o, t['do']), t['q'], t['k'], t['v'], window,
                         sinks, causal, lengths)
            _check(got, t['q'], t['k'], t['v'], t['do'], window, sinks, causal, lengths)


class _Feed(torch.autograd.Function):
    """A number whose gradient is `do`, with the strides that it has."""
    @staticmethod
    def forward(ctx, o, do):
        ctx.do = do
        return o.new_zeros(())

    @staticmethod
    def backward(ctx, _):
        return ctx.do, None


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_expanded_values_that_are_infinite(dtype):
    """Infinity in an element of one row that stands for all tokens: that element is infinite everywhere, the others finite."""
    from vit_amd import functional as VF
    g = _gen(63)
    for B, N, H in ((1, 40, 2), (14, 577, 8)):
        q, k = _rand(g, dtype, B, N, H, 64), _rand(g, dtype, B, N, H, 64)
        v = _rand(g, dtype, B, 1, H, 64)
        v[0, 0, 1, 5] = float('inf')
        o = VF.window_attention(q, k, v.expand(B, N, H, 64), -1)
        assert (o[0, :, 1, 5] == float('inf')).all()
        o[0, :, 1, 5] = 0
        assert torch.isfinite(o).all()

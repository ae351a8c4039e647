"""Rotary positions and the query / key norm with the rotation, on the GPU, against their definitions in 64 bits."""
import math

import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _table(P, pairs, g):
    a = torch.rand(P, pairs, generator=g, device='cuda') * 6.3
    return torch.stack((a.cos(), a.sin()), -1).contiguous()


def _view(kind, B, N, H, dh, dtype, g):
    """[B, N, H, dh] views of several layouts."""
    r = lambda *s: torch.randn(*s, generator=g, device='cuda').to(dtype)          # noqa: E731
    if kind == 'packed':
        return r(B, N, 3 * H, dh)[:, :, H:2 * H]
    if kind == 'heads first':
        return r(B, H, N, dh).transpose(1, 2)
    if kind == 'odd stride':
        return r(B, N, H, dh + 3)[..., 1:dh + 1]
    if kind == 'broadcast':
        return r(B, N, 1, dh).expand(B, N, H, dh)
    if kind == 'last strided':
        return r(B, N, H, 2 * dh)[..., ::2]
    return r(B, N, H, dh)


# ------------------------------------------------------------------------------------------------------------- table
@pytest.mark.parametrize('kind', ['int32', 'int64', 'float32', 'float64'])
@pytest.mark.parametrize('scaling', [None, dict(type='linear', factor=4.0), dict(type='ntk', factor=8.0),
                                     dict(type='yarn', factor=16.0, original=2048)], ids=['none', 'linear', 'ntk', 'yarn'])
def test_table(kind, scaling):
    from vit_amd import functional as VF
    dt = getattr(torch, kind)
    pos = torch.tensor([0, 1, 2, 77, 4095, 65537, 3999999, 2 ** 24 - 1], device='cuda')
    pos = pos.to(dt) if dt in (torch.int32, torch.int64) else pos.to(dt) + (0.5 if dt == torch.float64 else 0)
    t = VF.rotary_table(pos, 64, scaling=scaling)
    freqs, mul = VF.rotary_frequencies(64, 10000.0, scaling)
    a = pos.double()[:, None] * torch.tensor(freqs, dtype=torch.float64, device='cuda')
    want = mul * torch.stack((a.cos(), a.sin()), -1)
    # the angle's own rounding in 64 bits, the sines' (a few units of 2^-53), one rounding to fp32
    R.within(t, want, (2.0 ** -52 * a.abs() + 1e-14)[..., None] * mul + R.E * want.abs() + 1e-38, 'table')


def test_table_axes_far_and_empty():
    from vit_amd import functional as VF
    pos = torch.stack((torch.arange(40) // 8, torch.arange(40) % 8), 1).cuda()
    t = VF.rotary_table(pos, 24)
    for a in range(2):
        assert torch.equal(t[:, 6 * a:6 * a + 6], VF.rotary_table(pos[:, a].contiguous(), 12))
    assert torch.equal(VF.rotary_table(pos.t().contiguous().t(), 24), t)          # any strides
    far = torch.tensor([2 ** 40 + 12345], device='cuda')
    want = math.cos(float(far.item()))
    assert abs(VF.rotary_table(far, 2).flatten()[0].item() - want) < 2e-4 * 1 + R.E   # the angle is whole: 2^40 is exact
    assert VF.rotary_table(torch.zeros(0, dtype=torch.int64, device='cuda'), 8).shape == (0, 4, 2)


# ------------------------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize('inter', [False, True], ids=['half', 'inter'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('shape', [(1, 1, 1, 2, 2), (2, 5, 3, 64, 64), (1, 7, 12, 64, 32), (2, 3, 5, 80, 40), (1, 130, 4, 80, 80),
                                   (1, 4, 2, 7, 6), (3, 2, 2, 33, 10), (1, 9, 1, 200, 192), (2, 700, 8, 64, 64)], ids=str)
def test_rotary(shape, dtype, inter):
    from vit_amd import functional as VF
    B, N, H, dh, rot = shape
    g = _gen(1)
    for kind in ('plain', 'packed', 'heads first', 'odd stride', 'broadcast', 'last strided'):
        x = _view(kind, B, N, H, dh, DT[dtype], g)
        table = _table(N + 3, rot // 2, g)
        leaf = x.detach().requires_grad_(True)
        y = VF.rotary(leaf, table, offset=3, interleaved=inter)
        assert y.is_contiguous() and y.dtype == x.dtype
        rows = (torch.arange(N, device='cuda') + 3).expand(B, N)
        U = R.unit(x.dtype)
        want, m = R.turn(x.double(), table, rows, inter)
        R.within(y.detach(), want, 3 * R.E * m + U * want.abs(), f'y {kind}')
        assert torch.equal(y.detach()[..., rot:], x[..., rot:])
        dy = _view(kind, B, N, H, dh, DT[dtype], g)
        dx, = torch.autograd.grad(y, leaf, dy)
        want, m = R.turn(dy.double(), table, rows, inter, inverse=True)
        R.within(dx, want, 3 * R.E * m + U * want.abs(), f'dx {kind}')


@pytest.mark.parametrize('ids', [torch.int32, torch.int64], ids=['i32', 'i64'])
def test_rotary_position_ids(ids):
    from vit_amd import functional as VF
    g = _gen(2)
    x = torch.randn(2, 6, 3, 16, generator=g, device='cuda')
    table = _table(9, 8, g)
    pos = torch.randint(0, 9, (2, 6), generator=g, device='cuda').to(ids)
    want, m = R.turn(x.double(), table, pos.long(), False)
    R.within(VF.rotary(x, table, pos=pos), want, 3 * R.E * m + R.E * want.abs(), 'y')
    pos[0, 1], pos[1, 5] = 9, -1                                                    # outside of the table
    y = VF.rotary(x, table[:, :4].contiguous(), pos=pos)
    assert y[0, 1, :, :8].isnan().all() and y[1, 5, :, :8].isnan().all()
    assert torch.equal(y[0, 1, :, 8:], x[0, 1, :, 8:])
    y[0, 1], y[1, 5] = 0, 0
    assert torch.isfinite(y).all()


# ------------------------------------------------------------------------------------------------------ norm and turn
@pytest.mark.parametrize('inter', [False, True], ids=['half', 'inter'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('shape', [(1, 1, 1, 1, 8, 8), (2, 5, 3, 1, 64, 64), (1, 7, 12, 12, 64, 32), (2, 3, 5, 2, 80, 40),
                                   (1, 9, 4, 4, 128, 0), (1, 4, 2, 1, 7, 6), (3, 2, 2, 2, 127, 10), (2, 6, 3, 3, 20, 20),
                                   (2, 2100, 8, 4, 64, 64)], ids=str)
def test_qk_norm_rotary(shape, dtype, inter):
    from vit_amd import functional as VF
    B, N, Hq, Hk, dh, rot = shape
    g = _gen(3)
    U = R.unit(DT[dtype])
    for kind in ('plain', 'packed', 'heads first', 'odd stride', 'last strided') if N < 1000 else ('packed',):
        q, k = _view(kind, B, N, Hq, dh, DT[dtype], g), _view(kind, B, N, Hk, dh, DT[dtype], g) * 3
        gq = torch.randn(dh, generator=g, device='cuda')
        table = _table(N + 1, rot // 2, g) if rot else None
        rows = (torch.arange(N, device='cuda') + 1).expand(B, N)
        ins = [t.detach().requires_grad_(True) for t in (q, k, gq)]
        yq, yk = VF.qk_norm_rotary(*ins, None, table, offset=1 if rot else 0, interleaved=inter)
        dyq, dyk = _view(kind, B, N, Hq, dh, DT[dtype], g), _view('plain', B, N, Hk, dh, DT[dtype], g)
        dq, dk, dgq = torch.autograd.grad((yq, yk), ins, (dyq, dyk))
        for x, gam, y, dy, dx, what in ((q, gq, yq, dyq, dq, 'q'), (k, None, yk, dyk, dk, 'k')):
            want, b = R.norm_turn(x, gam, 1e-6, table, rows, inter)
            R.within(y.detach(), want, b + U * want.abs(), f'{what} {kind}')
            want, b, wg, bg = R.norm_turn_grad(x, gam, 1e-6, table, rows, inter, dy)
            R.within(dx, want, b + U * want.abs(), f'd{what} {kind}')
            if gam is not None:
                R.within(dgq, wg, bg + R.E * wg.abs(), f'dgamma {kind}')


def test_qk_norm_zero_rows_empty_and_same_bits():
    from vit_amd import functional as VF
    g = _gen(4)
    q = torch.randn(2, 50, 4, 64, generator=g, device='cuda').bfloat16()
    q[0, 3] = 0                                                                     # the norm of nothing is eps's
    k = torch.randn(2, 50, 2, 64, generator=g, device='cuda').bfloat16()
    gq, gk = torch.rand(64, generator=g, device='cuda'), torch.rand(64, generator=g, device='cuda')
    table = VF.rotary_table(torch.arange(50, device='cuda'), 64)

    def step():
        ins = [t.detach().requires_grad_(True) for t in (q, k, gq, gk)]
        y = VF.qk_norm_rotary(*ins, table)
        return (*y, *torch.autograd.grad(y, ins, [torch.ones_like(t) for t in y]))
    a, b = step(), step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert (a[0][0, 3] == 0).all() and torch.isfinite(a[2].float()).all()
    e = torch.zeros(0, 5, 4, 64, device='cuda', requires_grad=True)
    g1 = torch.ones(64, device='cuda', requires_grad=True)
    y, _ = VF.qk_norm_rotary(e, e[:, :, :2], g1, None, table)
    y.sum().backward()
    assert (g1.grad == 0).all() and e.grad.shape == e.shape


def test_gradients_against_differences():
    """Directional derivatives of the fp32 kernels against central differences of the definition."""
    from vit_amd import functional as VF
    g = _gen(5)
    q, k = (torch.randn(1, 4, 2, 16, generator=g, device='cuda') for _ in range(2))
    gq, gk = (torch.randn(16, generator=g, device='cuda') for _ in range(2))
    table = VF.rotary_table(torch.arange(4, device='cuda'), 16)
    rows = torch.arange(4, device='cuda')[None]
    w = torch.randn(2, 1, 4, 2, 16, generator=g, device='cuda')
    ins = [t.requires_grad_(True) for t in (q, k, gq, gk)]
    y = VF.qk_norm_rotary(*ins, table)
    grads = torch.autograd.grad(y, ins, list(w))
    dirs = [torch.randn(t.shape, generator=g, device='cuda', dtype=torch.float64) for t in ins]
    h = 1e-4

    def loss(s):
        a = [t.detach().double() + s * d for t, d in zip(ins, dirs)]
        return sum((R.norm_turn(a[i], a[2 + i], 1e-6, table, rows, False)[0] * w[i].double()).sum() for i in range(2))
    diff = float((loss(h) - loss(-h)) / (2 * h))
    got = float(sum((u.double() * d).sum() for u, d in zip(grads, dirs)))
    size = float(sum((u.double() * d).abs().sum() for u, d in zip(grads, dirs)))
    # differences: h^2 of a third derivative of order 10 of these values; gradients: the norm's bound of about 60 E
    assert abs(got - diff) <= size * (100 * h * h + 128 * R.E), (got, diff)


# ------------------------------------------------------------------------------------------------------------ refusals
def test_refusals():
    from vit_amd import functional as VF
    from vit_amd._lib import VitkError
    x = torch.randn(1, 4, 2, 16, device='cuda')
    table = VF.rotary_table(torch.arange(4, device='cuda'), 16)
    ok = VF.rotary(x, table)
    assert ok.shape == x.shape
    for bad in (lambda: VF.rotary(x[0], table), lambda: VF.rotary(x, None), lambda: VF.rotary(x, table[:, :, 0]),
                lambda: VF.rotary(x, table.double()), lambda: VF.rotary(x[..., :8].contiguous(), table),
                lambda: VF.rotary(x, table, pos=torch.zeros(1, 3, dtype=torch.int64, device='cuda')),
                lambda: VF.rotary(x, table, pos=torch.zeros(1, 4, dtype=torch.int64, device='cuda'), offset=1),
                lambda: VF.rotary_table(torch.arange(4, device='cuda'), 15),
                lambda: VF.rotary_table(torch.zeros(4, 3, device='cuda'), 16),
                lambda: VF.rotary_table(torch.zeros(4, device='cuda', dtype=torch.bool), 16),
                lambda: VF.rotary_table(torch.arange(4, device='cuda'), 16, scaling=dict(type='other', factor=2)),
                lambda: VF.rotary_table(torch.arange(4, device='cuda'), 16, scaling=dict(type='yarn', factor=2)),
                lambda: VF.qk_norm_rotary(x, x[:, :3], None, None), lambda: VF.qk_norm_rotary(x, x.bfloat16(), None, None),
                lambda: VF.qk_norm_rotary(x, x, torch.ones(8, device='cuda'), None),
                lambda: VF.qk_norm_rotary(x, x, None, None, offset=1)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: VF.rotary(x, table, offset=1), lambda: VF.rotary(x, table, offset=-1),
                lambda: VF.qk_norm_rotary(x, x, None, None, eps=0.0), lambda: VF.rotary(x.cpu(), table),
                lambda: VF.qk_norm_rotary(*(torch.zeros(1, 2, 2, 136, device='cuda') for _ in range(2)), None, None)):
        with pytest.raises(VitkError):
            bad()
    with pytest.raises(TypeError):
        VF.rotary(x.half(), table)
    y = VF.rotary(x.requires_grad_(True), table)
    gx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()

"""The long-sequence operators under what a program does around them: saved tensors that were moved to the host and back,
checkpointing, one tensor in several places, values changed between forward and backward, a single far-strided token, sequences
near the largest position."""
import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _block():
    """A call of every differentiable operator on one projection x [2, 70, 8, 64], and its inputs."""
    from vit_amd import functional as VF
    g = _gen(41)
    x = torch.randn(2, 70, 8, 64, generator=g, device='cuda').bfloat16()
    gq, gk = (torch.rand(64, generator=g, device='cuda') + 0.5 for _ in range(2))
    table = VF.rotary_table(torch.arange(70, device='cuda'), 64)
    pos = torch.randint(0, 70, (2, 70), generator=g, device='cuda')
    lengths = torch.tensor([70, 33], dtype=torch.int32, device='cuda')

    def run(x, gq, gk):
        q, k = VF.qk_norm_rotary(x[:, :, :4], x[:, :, 4:6], gq, gk, table, pos=pos)
        o = VF.window_attention(q, k, x[:, :, 6:], 9, sinks=2, causal=True, lengths=lengths)
        return VF.rotary(o, table, pos=pos, interleaved=True)
    do = torch.randn(2, 70, 4, 64, generator=g, device='cuda').bfloat16()
    return run, (x, gq, gk), do


def _grads(run, ins, do):
    ins = [t.detach().requires_grad_(True) for t in ins]
    o = run(*ins)
    junk = [torch.full((2, 70, 8, 64), 9.0, dtype=torch.bfloat16, device='cuda') for _ in range(16)]    # over what was freed
    grads = torch.autograd.grad(o, ins, do)
    del junk
    return (o.detach(), *grads)


def test_saved_tensors_moved_to_the_host():
    run, ins, do = _block()
    want = _grads(run, ins, do)
    with torch.autograd.graph.save_on_cpu():
        got = _grads(run, ins, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_checkpointed():
    from torch.utils.checkpoint import checkpoint
    run, ins, do = _block()
    want = _grads(run, ins, do)
    for reentrant in (False, True):
        ins2 = [t.detach().requires_grad_(True) for t in ins]
        o = checkpoint(run, *ins2, use_reentrant=reentrant)
        o.backward(do)
        assert all(torch.equal(a, b) for a, b in zip((o.detach(), *(t.grad for t in ins2)), want))


def test_one_tensor_as_query_key_and_value():
    from vit_amd import functional as VF
    g = _gen(42)
    x = torch.randn(1, 50, 3, 32, generator=g, device='cuda', requires_grad=True)
    do = torch.randn(1, 50, 3, 32, generator=g, device='cuda')
    got, = torch.autograd.grad(VF.window_attention(x, x, x, 5, sinks=1), x, do)
    parts = [x.detach().clone().requires_grad_(True) for _ in range(3)]
    dq, dk, dv = torch.autograd.grad(VF.window_attention(*parts, 5, sinks=1), parts, do)
    # three fp32 values in any order: two roundings of a partial sum
    assert ((got - (dq + dk + dv)).abs() <= 4 * 2 ** -24 * (dq.abs() + dk.abs() + dv.abs())).all()


def test_changed_between_forward_and_backward():
    from vit_amd import functional as VF
    run, ins, do = _block()
    table = VF.rotary_table(torch.arange(70, device='cuda'), 64)
    lengths = torch.tensor([70, 33], dtype=torch.int32, device='cuda')
    x = ins[0].detach().requires_grad_(True)
    for call, what in ((lambda: VF.rotary(x, table), table), (lambda: VF.qk_norm_rotary(x, x, None, None, table)[0], table),
                       (lambda: VF.window_attention(x, x, x, 4, lengths=lengths), lengths)):
        o = call()
        what.mul_(1)
        with pytest.raises(RuntimeError, match='modified by an inplace operation'):
            o.backward(torch.ones_like(o))


def test_no_second_derivative():
    from vit_amd import functional as VF
    run, ins, do = _block()
    x = ins[0].detach().requires_grad_(True)
    table = VF.rotary_table(torch.arange(70, device='cuda'), 64)
    for call in (lambda: VF.rotary(x, table), lambda: VF.qk_norm_rotary(x, x, None, None, table)[0],
                 lambda: VF.window_attention(x, x, x, 4)):
        o = call()
        dx, = torch.autograd.grad(o, x, torch.ones_like(o), create_graph=True)
        with pytest.raises(RuntimeError):
            dx.float().sum().backward()


def test_one_token_with_a_far_stride():
    """The stride of a dimension of one token is nowhere gone along, whatever it is."""
    from vit_amd import functional as VF
    x = torch.randn(2, 1, 4, 64, generator=_gen(43), device='cuda').bfloat16()
    far = torch.as_strided(x, x.shape, (256, 1 << 24, 64, 1))
    want, got = [], []
    for src, to in ((x, want), (far, got)):
        ins = [src.detach().requires_grad_(True) for _ in range(3)]
        o = VF.window_attention(*ins, 3, causal=True)
        to += [o.detach(), *torch.autograd.grad(o, ins, src.detach())]
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('window,sinks', [(20, 3), (7, 0), (0, 5)])
def test_decode_near_the_largest_position(window, sinks):
    """A sequence of 2^31 - 1 tokens sees what a short one sees whose ring stands at the same slot."""
    from vit_amd import functional as VF
    g = _gen(44)
    slots = sinks + window + 3
    ring = slots - sinks
    far = 2 ** 31 - 1
    near = sinks + 4 * ring + (far - sinks) % ring
    q, k, v = (torch.randn(2, h, 64, generator=g, device='cuda').bfloat16() for h in (4, 2, 2))
    kc, vc = (torch.randn(2, 2, slots, 64, generator=g, device='cuda').bfloat16() for _ in range(2))
    res = []
    for n in (near, far):
        c = kc.clone(), vc.clone()
        o = VF.window_decode(q, k, v, *c, torch.full((2,), n, dtype=torch.int32, device='cuda'), window, sinks=sinks)
        res.append((o, *c))
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_prefill_lengths_beyond_the_prompts():
    """Lengths past the padded width mean the whole width, for the steps after it too."""
    from vit_amd.window import WindowCache
    g = _gen(45)
    x = torch.randn(2, 11, 6, 64, generator=g, device='cuda').bfloat16()
    t = torch.randn(2, 6, 64, generator=g, device='cuda').bfloat16()
    res = []
    for n in ([11, 5], [40, 5]):
        c = WindowCache(2, 2, 64, 6, 1)
        o = c.prefill(x[:, :, :2], x[:, :, 2:4], x[:, :, 4:], torch.tensor(n, dtype=torch.int32, device='cuda'))
        res.append((o, c.step(t[:, :2], t[:, 2:4], t[:, 4:]), c.lengths, c.k, c.v))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize('case', [(1, 87, 2, 1, 128, 2, 1, True), (2, 40, 3, 3, 64, -1, 0, False), (1, 200, 2, 2, 40, 90, 3, True),
                                  (1, 700, 2, 1, 96, 3, 2, True), (1, 5, 1, 1, 64, 1, 0, False)], ids=str)
def test_small_calls_round_once(monkeypatch, case):
    """Where a call has few scores, P, dS and o in D are held as two bf16 each (a rounding's remainder is under 2^-8 of the value,
    and is rounded by 2^-8 of itself): 2^-16 where large calls have 2^-8, and then the result's own rounding."""
    from vit_amd import functional as VF
    B, N, Hq, Hk, dh, window, sinks, causal = case
    g = _gen(46)
    q, k, v, do = (torch.randn(B, N, h, dh, generator=g, device='cuda').bfloat16() for h in (Hq, Hk, Hk, Hq))
    ins = [t.requires_grad_(True) for t in (q, k, v)]
    o = VF.window_attention(*ins, window, sinks=sinks, causal=causal)
    got = dict(zip(('o', 'dq', 'dk', 'dv'), (o.detach(), *torch.autograd.grad(o, ins, do))))
    monkeypatch.setattr(R, 'unit', lambda dtype: 2.0 ** -16)
    want = R.window_attention(*(t.detach() for t in ins), window, sinks, causal, dh ** -0.5, None, do)
    for t, x in got.items():
        R.within(x, want[t][0], want[t][1] + 2.0 ** -8 * want[t][0].abs(), t)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_far_rows(dtype):
    """Tokens just under and over 16 MiB apart (the larger stride is copied, not refused)."""
    from vit_amd import functional as VF
    near = torch.randn(1, 5, 2, 32, generator=_gen(47), device='cuda').to(dtype)
    want = VF.window_attention(near, near, near, 2, causal=True)
    for stride in ((1 << 24) // near.element_size() - 64, (1 << 24) // near.element_size() + 64):
        store = torch.full((4 * stride + 64,), float('nan'), dtype=dtype, device='cuda')
        far = torch.as_strided(store, near.shape, (0, stride, 32, 1))
        far.copy_(near)
        assert torch.equal(VF.window_attention(far, far, far, 2, causal=True), want)
        kc = torch.zeros(1, 2, 5, 32, dtype=dtype, device='cuda')
        vc = torch.zeros_like(kc)
        VF.window_cache_fill(far, far, kc, vc)
        assert torch.equal(kc, near.transpose(1, 2)) and torch.equal(vc, kc)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('case', [(1, 1201, 4, 1, 128, 40, 5), (2, 1001, 6, 2, 80, 100, 33), (1, 2100, 2, 2, 64, 10, 70),
                                  (3, 700, 4, 4, 24, 3, 1)], ids=str)
def test_sinks_of_their_own_launch(case, dtype):
    """Few rows and sinks that every query sees: two waves a row, and the sinks' keys in workgroups that share the queries."""
    from vit_amd import functional as VF
    B, N, Hq, Hk, dh, window, sinks = case
    g = _gen(48)
    q, k, v, do = (torch.randn(B, N, h, dh, generator=g, device='cuda').to(dtype) for h in (Hq, Hk, Hk, Hq))
    lengths = torch.randint(1, N + 1, (B,), generator=g, device='cuda', dtype=torch.int32)
    for causal, n in ((True, None), (False, lengths)):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = VF.window_attention(*ins, window, sinks=sinks, causal=causal, lengths=n)
        got = dict(zip(('o', 'dq', 'dk', 'dv'), (o.detach(), *torch.autograd.grad(o, ins, do))))
        want = R.window_attention(q, k, v, window, sinks, causal, dh ** -0.5, n, do)
        for t, x in got.items():
            R.within(x, *want[t], t)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('case', [
    # B, N, Hq, Hk, dh, window, sinks, causal, padded: workgroups of 128 rows at every width, every order of the work
    (9, 1030, 8, 8, 32, 200, 5, False, False), (9, 1030, 8, 8, 80, 300, 3, True, False), (9, 1030, 7, 7, 80, -1, 0, False, False),
    (9, 1030, 8, 8, 96, 30, 4, True, False), (9, 1030, 8, 8, 48, -1, 0, False, True), (9, 1030, 8, 8, 112, -1, 0, True, True),
    (11, 1030, 7, 7, 64, 260, 40, False, True), (5, 1030, 16, 2, 72, -1, 0, True, False), (5, 1030, 16, 4, 128, 400, 130, True, False),
    (40, 200, 14, 7, 64, 20, 1, False, True), (1, 4100, 18, 18, 64, 70, 3, True, False)], ids=str)
def test_large_calls(case, dtype):
    from vit_amd import functional as VF
    B, N, Hq, Hk, dh, window, sinks, causal, padded = case
    g = _gen(49)
    q, k, v, do = (torch.randn(B, N, h, dh, generator=g, device='cuda').to(dtype) for h in (Hq, Hk, Hk, Hq))
    n = torch.randint(0, N + 1, (B,), generator=g, device='cuda', dtype=torch.int32) if padded else None
    ins = [t.requires_grad_(True) for t in (q, k, v)]
    o = VF.window_attention(*ins, window, sinks=sinks, causal=causal, lengths=n)
    got = dict(zip(('o', 'dq', 'dk', 'dv'), (o.detach(), *torch.autograd.grad(o, ins, do))))
    want = R.window_attention(*(t.detach() for t in ins), window, sinks, causal, dh ** -0.5, n, do)
    for t, x in got.items():
        R.within(x, *want[t], t)
    again = torch.autograd.grad(VF.window_attention(*ins, window, sinks=sinks, causal=causal, lengths=n), ins, do)
    assert all(torch.equal(a, got[t]) for a, t in zip(again, ('dq', 'dk', 'dv')))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('N', [40, 600])
@pytest.mark.parametrize('window', [-1, 9])
def test_infinite_values(N, window, dtype):
    """An infinite value makes the rows that see it infinite in its element, with its sign, and leaves the others alone."""
    from vit_amd import functional as VF
    g = _gen(50)
    q, k, v = (torch.randn(2, N, 2, 64, generator=g, device='cuda').to(dtype) for _ in range(3))
    want, bound = R.window_attention(q, k, v, window, 0, False, 0.125, None)['o']
    v[0, 21, 1, 5], v[1, 30, 0, 63] = float('inf'), float('-inf')
    o = VF.window_attention(q, k, v, window)
    i = torch.arange(N, device='cuda')
    hit = torch.zeros_like(o, dtype=torch.bool)
    for b, j, h, d, sign in ((0, 21, 1, 5, 1.0), (1, 30, 0, 63, -1.0)):
        seen = (i - j).abs() <= (window if window >= 0 else N)
        assert (o[b, seen, h, d] == sign * float('inf')).all()
        hit[b, seen, h, d] = True
    R.within(o[~hit], want[~hit], bound[~hit], 'others')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('B,N,H,dh', [(4, 1, 8, 80), (2, 5, 2, 64), (1, 300, 4, 128), (9, 1030, 8, 32), (16, 1, 3, 24)])
def test_rows_that_see_themselves_alone(B, N, H, dh, dtype):
    """The softmax of one score is 1 whatever the score: dq is exactly 0, and so is dk where every row is like that."""
    from vit_amd import functional as VF
    g = _gen(51)
    q, k, v, do = (torch.randn(B, N, h, dh, generator=g, device='cuda').to(dtype) for h in (2 * H, H, H, 2 * H))
    ins = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, _ = torch.autograd.grad(VF.window_attention(*ins, 0), ins, do)
    assert not dq.any() and not dk.any()
    for window, sinks, lengths in ((-1, 0, None), (3, 2, torch.ones(B, dtype=torch.int32, device='cuda'))):
        dq, dk, _ = torch.autograd.grad(VF.window_attention(*ins, window, sinks=sinks, causal=True, lengths=lengths), ins, do)
        assert not dq[:, 0].any()
        assert lengths is None or not (dq.any() or dk.any())
    dq, _, _ = torch.autograd.grad(VF.window_attention(*ins, 0, sinks=1, causal=True), ins, do)
    assert not dq[:, 0].any() and (N == 1 or dq[:, 1:].any(-1).all())

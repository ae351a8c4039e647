"""The ring cache on the GPU: one new token a sequence, and whole prompts into it."""
import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _rand(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device='cuda').to(DT[dtype])


def _one(g, dtype, B, Hq, Hk, dh, C, window, sinks, lengths, poison=True):
    from vit_amd import functional as VF
    q, k, v = _rand(g, dtype, B, Hq, dh), _rand(g, dtype, B, Hk, dh), _rand(g, dtype, B, Hk, dh)
    kc, vc = _rand(g, dtype, B, Hk, C, dh), _rand(g, dtype, B, Hk, C, dh)
    lengths = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    want, bound, wk, wv = R.decode(q, k, v, kc, vc, lengths, window, sinks, dh ** -0.5)
    if poison:                                       # whatever is not visible may hold anything
        for b, p in enumerate(lengths.tolist()):
            seen = set(range(max(0, p + 1))) if window < 0 else \
                {R.ring_slot(t, C, sinks) for t in [*range(min(sinks, p + 1)), *range(max(sinks, p - window), p + 1)]}
            for c in range(C):
                if c not in seen:
                    for t in (kc, wk):
                        t[b, :, c] = float('nan')
                    for t in (vc, wv):
                        t[b, :, c] = float('inf')
    o = VF.window_decode(q, k, v, kc, vc, lengths, window, sinks=sinks)
    lost = want.isnan()
    assert torch.equal(o.isnan(), lost)
    R.within(torch.where(lost, torch.zeros_like(o), o), want.nan_to_num(0.0), bound, 'out')
    for a, b in ((kc, wk), (vc, wv)):                # whole caches, bit for bit: the new token and nothing else
        assert torch.equal(a.view(torch.int16 if a.element_size() == 2 else torch.int32),
                           b.view(torch.int16 if b.element_size() == 2 else torch.int32))
    again = VF.window_decode(q, k, v, kc, vc, lengths, window, sinks=sinks)
    assert torch.equal(again.nan_to_num(5.0), o.nan_to_num(5.0))
    return o


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('case', [
    # B, Hq, Hk, dh, slots, window, sinks, lengths
    (1, 1, 1, 8, 1, 0, 0, [0]), (2, 2, 1, 64, 8, 4, 3, [0, 7]), (4, 4, 4, 32, 20, 9, 2, [0, 1, 11, 400]),
    (3, 6, 2, 64, 64, 63, 0, [5, 63, 64]), (3, 5, 1, 80, 77, 70, 6, [-1, 76, 100000]), (5, 4, 2, 128, 200, 130, 9, [8, 9, 10, 199, 200]),
    (2, 12, 12, 64, 576, 511, 1, [577, 1 << 30]), (2, 7, 1, 40, 40, 10, 20, [19, 45]), (4, 4, 4, 64, 50, -1, 0, [0, 49, 50, -3]),
    (1, 2, 2, 120, 30, -1, 7, [29]), (2, 16, 2, 64, 33, 32, 0, [31, 97]), (1, 4, 1, 8, 6, 2, 3, [2147483000])], ids=str)
def test_one_token(case, dtype):
    B, Hq, Hk, dh, C, window, sinks, lengths = case
    _one(_gen(21), dtype, B, Hq, Hk, dh, C, window, sinks, lengths)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('Hq,Hk,dh', [(2, 2, 64), (8, 2, 128), (3, 1, 80)])
def test_split_over_the_keys(Hq, Hk, dh, dtype):
    """Few heads and long windows: the keys are dealt to several workgroups."""
    _one(_gen(22), dtype, 2, Hq, Hk, dh, 9000, 8900, 4, [8950, 31], poison=False)
    _one(_gen(23), dtype, 2, Hq, Hk, dh, 5000, -1, 0, [4999, 5000], poison=False)
    _one(_gen(24), dtype, 2, Hq, Hk, dh, 6100, 6000, 2, [40000, -1], poison=False)


def test_many_sequences():
    g = _gen(25)
    _one(g, 'bf16', 150, 4, 4, 64, 70, 60, 3, [int(n) for n in torch.randint(0, 300, (150,), generator=torch.Generator().manual_seed(1))],
         poison=False)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('case', [
    # B, N, Hk, dh, slots, sinks, lengths
    (1, 1, 1, 8, 1, 0, None), (2, 9, 2, 64, 8, 2, None), (3, 50, 1, 40, 20, 3, [0, 50, 17]), (2, 30, 3, 128, 64, 4, [3, 29]),
    (1, 100, 2, 80, 7, 6, None), (2, 12, 1, 64, 12, 0, [12, 99])], ids=str)
def test_fill(case, dtype):
    from vit_amd import functional as VF
    B, N, Hk, dh, C, sinks, lengths = case
    g = _gen(26)
    kv = _rand(g, dtype, B, N, 2 * Hk, dh)
    k, v = kv[:, :, :Hk], kv[:, :, Hk:]
    kc, vc = _rand(g, dtype, B, Hk, C, dh), _rand(g, dtype, B, Hk, C, dh)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device='cuda')
    wk, wv = R.fill(k, v, C, sinks, lengths, kc, vc)
    VF.window_cache_fill(k, v, kc, vc, sinks=sinks, lengths=n)
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_prompt_then_tokens_equal_the_whole_sequence(dtype):
    """The operators as they are used: norms and rotation, prefill of ragged prompts, then token by token; against the
    causal window attention of the whole sequences at once (whose rows are within their bounds of the definition, as are
    these: the two may differ by both)."""
    from vit_amd import functional as VF
    from vit_amd.window import WindowCache
    g = _gen(27)
    B, N, Hq, Hk, dh, window, sinks, start = 2, 90, 4, 2, 64, 20, 3, [40, 7]
    x = _rand(g, dtype, B, N, Hq + 2 * Hk, dh)
    gq, gk = (torch.rand(dh, generator=g, device='cuda') + 0.5 for _ in range(2))
    table = VF.rotary_table(torch.arange(N, device='cuda'), dh)
    q, k = VF.qk_norm_rotary(x[:, :, :Hq], x[:, :, Hq:Hq + Hk], gq, gk, table)
    v = x[:, :, Hq + Hk:]
    want = R.window_attention(q, k, v, window, sinks, True, dh ** -0.5, None)['o']
    cache = WindowCache(B, Hk, dh, window, sinks, dtype=DT[dtype])
    lengths = torch.tensor(start, dtype=torch.int32, device='cuda')
    o = cache.prefill(q, k, v, lengths)
    for b in range(B):
        R.within(o[b, :start[b]], want[0][b, :start[b]], want[1][b, :start[b]], 'prefill')
    rows = torch.arange(B, device='cuda')
    for t in range(N - max(start)):
        at = cache.lengths.long()
        xt = x[rows, at][:, None]
        qt, kt = VF.qk_norm_rotary(xt[:, :, :Hq], xt[:, :, Hq:Hq + Hk], gq, gk, table, pos=at[:, None])
        o = cache.step(qt[:, 0], kt[:, 0], xt[:, 0, Hq + Hk:])
        for b in range(B):
            p = start[b] + t
            R.within(o[b], want[0][b, p], want[1][b, p], f'token {p}')
    assert cache.lengths.tolist() == [s + N - max(start) for s in start]


def test_step_captured_in_a_graph():
    from vit_amd.window import WindowCache
    g = _gen(28)
    B, H, dh = 3, 4, 64
    x = _rand(g, 'bf16', 3, B, H, dh)
    one, two = (WindowCache(B, H, dh, 16, 2, dtype=torch.bfloat16) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one.step(*x)
    torch.cuda.current_stream().wait_stream(side)
    one.reset()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = one.step(*x)
    one.reset()
    for _ in range(40):
        x.copy_(_rand(g, 'bf16', 3, B, H, dh))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, two.step(*x))
    assert torch.equal(one.lengths, two.lengths)


def test_refusals():
    from vit_amd import functional as VF
    from vit_amd._lib import VitkError
    q, k, v = torch.randn(2, 4, 64, device='cuda'), torch.randn(2, 2, 64, device='cuda'), torch.randn(2, 2, 64, device='cuda')
    kc, vc = torch.zeros(2, 2, 10, 64, device='cuda'), torch.zeros(2, 2, 10, 64, device='cuda')
    n = torch.zeros(2, dtype=torch.int32, device='cuda')
    VF.window_decode(q, k, v, kc, vc, n, 7, sinks=2)
    for bad in (lambda: VF.window_decode(q, k, v, kc, vc, n.long(), 7), lambda: VF.window_decode(q, k, v, kc, vc, None, 7),
                lambda: VF.window_decode(q, k, v, kc.bfloat16(), vc, n, 7), lambda: VF.window_decode(q, k, v, kc[:, :1], vc[:, :1], n, 7),
                lambda: VF.window_decode(q, k, v, kc.transpose(1, 2), vc.transpose(1, 2), n, 7),
                lambda: VF.window_decode(q[0], k, v, kc, vc, n, 7), lambda: VF.window_decode(q, k[:, :1], v, kc, vc, n, 7),
                lambda: VF.window_cache_fill(k[:, None], v, kc, vc)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: VF.window_decode(q, k, v, kc, vc, n, 8, sinks=2), lambda: VF.window_decode(q, k, v, kc, vc, n, 7, sinks=-1),
                lambda: VF.window_decode(q[:, :3], k, v, kc, vc, n, 7), lambda: VF.window_decode(q, k, v, kc, vc, n, 7, scale=0.0),
                lambda: VF.window_decode(q.cpu(), k, v, kc, vc, n, 7),
                lambda: VF.window_cache_fill(k[:, None], v[:, None], kc, vc, sinks=10)):
        with pytest.raises(VitkError):
            bad()
    with pytest.raises(RuntimeError):
        VF.window_decode(q.clone().requires_grad_(True), k, v, kc, vc, n, 7)

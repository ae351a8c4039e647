"""An infinite value is a step's end, not a hang: window attention with one takes a small multiple of its ordinary time."""
import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('N,Hq,Hk,dh,window,sinks,causal', [(4096, 16, 4, 128, -1, 0, True), (8192, 8, 8, 64, 300, 2, False)], ids=str)
def test_time(N, Hq, Hk, dh, window, sinks, causal, dtype):
    """Four walks over the same tiles at most, and their first and last tile: 20 times leaves room for a busy machine (taken key by
    key it was 140 to 200 times, and grew with the sequence)."""
    from vit_amd import functional as VF
    g = torch.Generator(device='cuda').manual_seed(84)
    q, k, v = (torch.randn(1, N, h, dh, generator=g, device='cuda').to(dtype) for h in (Hq, Hk, Hk))

    def best():
        t = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            VF.window_attention(q, k, v, window, sinks=sinks, causal=causal)
            b.record()
            torch.cuda.synchronize()
            t.append(a.elapsed_time(b))
        return min(t)
    plain = best()
    v[:, 0, :, 3] = float('inf')
    v[:, N // 2, :, 4] = float('-inf')
    assert best() < 20 * plain


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('B,N,H,window,sinks,causal', [
    (1, 90, 2, 7, 1, True), (2, 300, 4, 30, 3, False), (9, 1030, 8, 70, 2, True), (9, 1030, 8, 300, 0, False), (9, 520, 8, -1, 0, True)], ids=str)
def test_every_kind(B, N, H, window, sinks, causal, dtype):
    """+inf, -inf, both and NaN in elements of v, each for itself: the rows that see them have what the sum gives, the other rows
    and the other elements are within their bounds."""
    from vit_amd import functional as VF
    g = torch.Generator(device='cuda').manual_seed(85)
    q, k, v = (torch.randn(B, N, H, 64, generator=g, device='cuda').to(dtype) for _ in range(3))
    want, bound = R.window_attention(q, k, v, window, sinks, causal, 0.125, None)['o']
    inf, nan = float('inf'), float('nan')
    special = [(40, 3, inf), (41, 5, -inf), (44, 7, inf), (47, 7, -inf), (50, 9, nan), (0, 11, inf), (N - 1, 13, -inf)]
    for j, d, x in special:
        v[:, j, :, d] = x
    o = VF.window_attention(q, k, v, window, sinks=sinks, causal=causal)
    seen = R.visible(N, window, sinks, causal, N, 'cuda')
    for j, d, x in special:
        want[:, seen[:, j], :, d] += x                   # inf + -inf: NaN
    bad = ~torch.isfinite(want)
    assert torch.equal(o.isnan(), want.isnan()) and torch.equal(torch.isfinite(o), ~bad)
    assert torch.equal(o.double()[bad].nan_to_num(0.0), want[bad].nan_to_num(0.0))
    R.within(o[~bad], want[~bad], bound[~bad], 'finite')

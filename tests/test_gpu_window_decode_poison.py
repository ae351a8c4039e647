"""The ring cache's step where its keys are dealt to several workgroups, and with many short sequences: what is not visible is not
read, whatever it holds (tests of one workgroup a row stand in test_gpu_window_decode.py)."""
import pytest
import torch

import long_ref as R

pytestmark = pytest.mark.gpu
DT = {'f32': torch.float32, 'bf16': torch.bfloat16}


def _hidden(C, window, sinks, lengths):
    """bool [B, C]: slots whose token the new one does not see (its own slot is written by the call)."""
    c = torch.arange(C, device='cuda')[None]
    p = lengths.long()[:, None]
    if window < 0:
        seen = (c <= p) & (p < C)
    else:
        at = torch.where(c < sinks, c, p - torch.remainder(p - c, C - sinks))        # the last token up to p that has the slot
        seen = (at <= p) & ((c < sinks) | ((at >= sinks) & (p - at <= window)))
    return ~seen


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('case', [
    # B, Hq, Hk, dh, slots, window, sinks, lengths
    (2, 2, 2, 64, 9000, 8900, 4, [8950, 31]), (2, 8, 2, 128, 9000, 8900, 4, [12345, 31]), (2, 3, 1, 80, 9000, 8900, 4, [8904, 8905]),
    (2, 2, 2, 64, 5000, -1, 0, [4999, 5000]), (2, 8, 2, 128, 5000, -1, 0, [17, 4000]), (2, 3, 1, 80, 5000, -1, 3, [0, 4999]),
    (2, 2, 2, 64, 6100, 6000, 2, [40000, -1]), (2, 8, 2, 128, 6100, 6000, 2, [6003, 2]), (1, 5, 1, 40, 9000, 7000, 70, [1 << 30]),
    (2, 12, 4, 32, 30000, 20000, 9, [29999, 20010]), (150, 4, 4, 64, 70, 60, 3, None), (150, 6, 2, 128, 90, 60, 3, None)], ids=str)
def test_hidden_slots_hold_anything(case, dtype):
    from vit_amd import functional as VF
    B, Hq, Hk, dh, C, window, sinks, lengths = case
    g = torch.Generator(device='cuda').manual_seed(83)
    q, k, v = (torch.randn(B, h, dh, generator=g, device='cuda').to(DT[dtype]) for h in (Hq, Hk, Hk))
    kc, vc = (torch.randn(B, Hk, C, dh, generator=g, device='cuda').to(DT[dtype]) for _ in range(2))
    n = torch.randint(0, 300, (B,), generator=g, device='cuda', dtype=torch.int32) if lengths is None else \
        torch.tensor(lengths, dtype=torch.int32, device='cuda')
    want, bound, wk, wv = R.decode(q, k, v, kc, vc, n, window, sinks, dh ** -0.5)
    hidden = _hidden(C, window, sinks, n)[:, None, :, None]
    for t, w, bad in ((kc, wk, float('nan')), (vc, wv, float('inf'))):
        t.masked_fill_(hidden, bad)
        w.masked_fill_(hidden, bad)
    o = VF.window_decode(q, k, v, kc, vc, n, window, sinks=sinks)
    lost = want.isnan()
    assert torch.equal(o.isnan(), lost)
    R.within(torch.where(lost, torch.zeros_like(o), o), want.nan_to_num(0.0), bound, 'out')
    bits = torch.int16 if dtype == 'bf16' else torch.int32
    assert torch.equal(kc.view(bits), wk.view(bits)) and torch.equal(vc.view(bits), wv.view(bits))

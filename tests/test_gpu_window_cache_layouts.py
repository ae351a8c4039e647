"""Prompts into the ring cache from tensors of any strides, as the attention beside it takes them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('layout', ['every other element', 'heads first', 'misaligned', 'one head for all', 'one token for all'])
def test_prefill(layout, dtype):
    from vit_amd import functional as VF
    from vit_amd.window import WindowCache
    B, N, H, dh = 2, 13, 3, 40
    g = torch.Generator(device='cuda').manual_seed(86)

    def make():
        r = lambda *s: torch.randn(*s, generator=g, device='cuda').to(dtype)          # noqa: E731
        return {'every other element': lambda: r(B, N, H, 2 * dh)[..., ::2], 'heads first': lambda: r(B, H, N, dh).transpose(1, 2),
                'misaligned': lambda: r(B, N, H, dh + 1)[..., 1:], 'one head for all': lambda: r(B, N, 1, dh).expand(B, N, H, dh),
                'one token for all': lambda: r(B, 1, H, dh).expand(B, N, H, dh)}[layout]()
    q, k, v = make(), make(), make()
    res = []
    for ins in ((q, k, v), [t.contiguous() for t in (q, k, v)]):
        cache = WindowCache(B, H, dh, 6, 2, dtype=dtype)
        o = cache.prefill(*ins)
        kc, vc = torch.zeros_like(cache.k), torch.zeros_like(cache.v)
        VF.window_cache_fill(ins[1], ins[2], kc, vc, sinks=2)
        res.append((o, cache.k, cache.v, kc, vc))
    assert all(torch.equal(a, b) for a, b in zip(*res))

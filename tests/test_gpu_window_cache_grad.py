"""The ring cache keeps no graph: what would cut one is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_fill_refuses_what_needs_a_gradient():
    from vit_amd import functional as VF
    from vit_amd._lib import VitkError
    from vit_amd.window import WindowCache
    g = torch.Generator(device='cuda').manual_seed(82)
    k, v = (torch.randn(1, 6, 2, 32, generator=g, device='cuda') for _ in range(2))
    kc, vc = (torch.zeros(1, 2, 8, 32, device='cuda') for _ in range(2))
    for a, b in ((k.clone().requires_grad_(True), v), (k, v.clone().requires_grad_(True))):
        with pytest.raises(RuntimeError, match='no_grad') as e:
            VF.window_cache_fill(a, b, kc, vc)
        assert not isinstance(e.value, VitkError)
        assert not kc.any() and not vc.any()
        with torch.no_grad():
            VF.window_cache_fill(a, b, kc, vc)
        assert torch.equal(kc[:, :, :6], k.transpose(1, 2)) and torch.equal(vc[:, :, :6], v.transpose(1, 2))
        kc.zero_(), vc.zero_()
    cache = WindowCache(1, 2, 32, 5, dtype=torch.float32)
    q = k.clone().requires_grad_(True)
    assert not cache.prefill(q, q, v).requires_grad                                  # a cache's own calls are under no_grad

"""torch.ops.vit_amd.window_attention: which of its outputs carry a gradient."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_statistics_are_not_differentiable(dtype):
    """lse and out_lo are for the backward: asking for their gradient is an error, not a gradient that lacks a term."""
    import vit_amd.torch_ops  # noqa: F401
    O = torch.ops.vit_amd
    g = torch.Generator(device='cuda').manual_seed(81)
    x = torch.randn(1, 40, 2, 32, generator=g, device='cuda').to(dtype).requires_grad_(True)
    out, lse, lo = O.window_attention(x, x, x, 5, 1, False, 0.2, None)
    assert out.requires_grad and not lse.requires_grad and not lo.requires_grad
    with pytest.raises(RuntimeError, match='does not require grad'):
        lse.sum().backward()
    want, = torch.autograd.grad(out.float().sum(), x)

    def f(x):
        o, s, _ = O.window_attention(x, x, x, 5, 1, False, 0.2, None)
        return o.float().sum(), s
    for call in (f, torch.compile(f, backend='aot_eager', fullgraph=True)):
        total, s = call(x)
        assert not s.requires_grad and torch.equal(s, lse)
        assert torch.equal(torch.autograd.grad(total, x)[0], want)

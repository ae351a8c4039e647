"""torch.library registration of the long-sequence operators: schemas and fake functions on the CPU; on the GPU the same numbers as
vit_amd.functional, opcheck, and a traced step."""
import pytest
import torch


def test_registered_with_fake_functions():
    import vit_amd.torch_ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    O = torch.ops.vit_amd
    assert 'Tensor(a3!) k_cache' in str(O.window_decode.default._schema)
    with FakeTensorMode():
        x = torch.empty(2, 9, 8, 64, device='cuda', dtype=torch.bfloat16)
        table = torch.empty(9, 32, 2, device='cuda')
        assert O.rotary(x[:, :, :4], table, None, 0, False).shape == (2, 9, 4, 64)
        q, k = O.qk_norm_rotary(x[:, :, :4], x[:, :, 4:6], None, None, table, None, 0, 1e-6, False)
        o, lse, lo = O.window_attention(q, k, x[:, :, 6:], 4, 1, True, 0.125, None)
        assert o.shape == lo.shape == (2, 9, 4, 64) and lse.shape == (2, 4, 9) and lse.dtype == torch.float32
        grads = O.window_attention_backward(o, q, k, x[:, :, 6:], o, lse, lo, 4, 1, True, 0.125, None)
        assert [g.shape[2] for g in grads] == [4, 2, 2]
        c = torch.empty(2, 2, 16, 64, device='cuda', dtype=torch.bfloat16)
        assert O.window_decode(q[:, 0], k[:, 0], k[:, 0], c, c.clone(), torch.empty(2, device='cuda', dtype=torch.int32), 4, 1,
                               0.125).shape == (2, 4, 64)


def _step(x, gq, gk, table, O):
    q, k = O.qk_norm_rotary(x[:, :, :4], x[:, :, 4:6], gq, gk, None, None, 0, 1e-6, False)
    q, k = O.rotary(q, table, None, 0, True), O.rotary(k, table, None, 0, True)
    return O.window_attention(q, k, x[:, :, 6:], 12, 2, True, 0.125, None)[0]


@pytest.mark.gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
def test_same_as_functional_and_traced(dtype):
    import vit_amd.torch_ops  # noqa: F401
    from vit_amd import functional as VF
    O = torch.ops.vit_amd
    g = torch.Generator(device='cuda').manual_seed(31)
    x = torch.randn(2, 50, 8, 64, generator=g, device='cuda').to(dtype)
    gq, gk = (torch.rand(64, generator=g, device='cuda') + 0.5 for _ in range(2))
    table = VF.rotary_table(torch.arange(50, device='cuda'), 32)
    do = torch.randn(2, 50, 4, 64, generator=g, device='cuda').to(dtype)

    def grads(f, *a):
        ins = [t.clone().requires_grad_(True) for t in (x, gq, gk)]
        o = f(*ins, table, *a)
        return (o.detach(), *torch.autograd.grad(o, ins, do))

    def plain(x, gq, gk, table):
        q, k = VF.qk_norm_rotary(x[:, :, :4], x[:, :, 4:6], gq, gk)
        q, k = VF.rotary(q, table, interleaved=True), VF.rotary(k, table, interleaved=True)
        return VF.window_attention(q, k, x[:, :, 6:], 12, sinks=2, causal=True)
    want = grads(plain)
    for got in (grads(_step, O), grads(torch.compile(lambda *a: _step(*a, O), backend='aot_eager', fullgraph=True))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_opcheck():
    import vit_amd.torch_ops  # noqa: F401
    from vit_amd import functional as VF
    O = torch.ops.vit_amd
    x = torch.randn(1, 20, 4, 32, device='cuda')
    table = VF.rotary_table(torch.arange(20, device='cuda'), 32)
    gam = torch.ones(32, device='cuda', requires_grad=True)
    k = torch.randn(1, 20, 2, 32, device='cuda', requires_grad=True)
    x.requires_grad_(True)
    torch.library.opcheck(O.rotary.default, (x, table, None, 0, False))
    torch.library.opcheck(O.qk_norm_rotary.default, (x, k, gam, None, table, None, 0, 1e-6, True))
    torch.library.opcheck(O.window_attention.default, (x, k, k, 5, 1, False, 0.2, None))
    c = torch.zeros(1, 2, 8, 32, device='cuda')
    n = torch.tensor([3], dtype=torch.int32, device='cuda')
    d = [t.detach()[:, 0] for t in (x, k, k)]
    torch.library.opcheck(O.window_decode.default, (*d, c, c.clone(), n, 5, 1, 0.2))

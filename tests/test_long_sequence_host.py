"""CPU part of the long-sequence operators: the C entry points' checks (they return before any launch), the frequencies of the
rotary positions, and the wrappers' refusal of tensors that are not on the GPU."""
import ctypes
import math

import pytest
import torch

P = 1 << 20                 # a pointer that no check dereferences: 16-byte aligned
F32, BF16 = 0, 1


@pytest.fixture(scope='module')
def L():
    from vit_amd._lib import lib
    return lib()


def _bad(L, status, words):
    assert status == 1, status
    assert words in L.vitk_last_error().decode(), L.vitk_last_error()


def rotary(L, dtype=BF16, B=1, N=4, H=2, dh=64, x=P, st=(512, 128, 64), table=P, rows=4, rot=64, pos=0, offset=0, y=P):
    return L.vitk_rotary(dtype, 0, 0, B, N, H, dh, x, *st, table, rows, rot, pos, 0, offset, y, 0)


@pytest.mark.parametrize('kw,words', [
    (dict(dtype=2), 'bad dtype'), (dict(H=0), 'bad shape'), (dict(N=-1), 'bad shape'), (dict(rot=63), 'rotated width'),
    (dict(rot=66), 'rotated width'), (dict(table=0), 'table'), (dict(table=P + 8), 'table'), (dict(offset=1), 'outside the table'),
    (dict(offset=-1), 'outside the table'), (dict(x=0), 'null'), (dict(y=0), 'null'),
    (dict(B=1 << 20, N=1 << 12, rows=1 << 12), 'too many')])
def test_rotary_refusals(L, kw, words):
    _bad(L, rotary(L, **kw), words)


def norm(L, dtype=BF16, B=1, N=4, Hq=2, Hk=1, dh=64, q=P, eps=1e-6, table=P, rows=4, rot=64):
    return L.vitk_qk_norm_rotary_fwd(dtype, 0, B, N, Hq, Hk, dh, q, 512, 128, 64, P, 512, 128, 64, 0, 0, eps, table, rows, rot, 0, 0, 0,
                                     P, P, 0)


@pytest.mark.parametrize('kw,words', [(dict(dtype=5), 'bad dtype'), (dict(Hk=0), 'bad shape'), (dict(dh=129), 'head width'),
                                      (dict(eps=0.0), 'eps'), (dict(rows=3), 'outside the table'), (dict(q=0), 'null'),
                                      (dict(B=1 << 16, N=1 << 15, rows=1 << 15), 'too many')])
def test_norm_refusals(L, kw, words):
    _bad(L, norm(L, **kw), words)


def window(L, dtype=BF16, B=1, N=16, Hq=4, Hk=2, dh=64, q=P, st=(8192, 512, 64), scale=0.125, w=4, sinks=1, out=P):
    return L.vitk_window_attn_fwd(dtype, B, N, Hq, Hk, dh, q, *st, P, 8192, 512, 64, P, 8192, 512, 64, scale, w, sinks, 0, 0, out, 0, 0, 0)


@pytest.mark.parametrize('kw,words', [
    (dict(dtype=3), 'bad dtype'), (dict(N=1 << 28), 'bad shape'), (dict(Hk=3), 'no multiple'), (dict(dh=60), 'head width'),
    (dict(dh=136), 'head width'), (dict(dh=0), 'head width'), (dict(scale=0.0), 'scale'), (dict(scale=-1.0), 'scale'),
    (dict(scale=math.inf), 'scale'), (dict(scale=math.nan), 'scale'), (dict(sinks=-1), 'sinks'), (dict(q=0), 'q must be'),
    (dict(q=P + 8), 'q must be'), (dict(st=(8192, 500, 64)), 'q must be'), (dict(dtype=F32, st=(8192, 510, 64)), 'q must be'),
    (dict(out=P + 4), 'out must be'), (dict(B=1 << 20, N=1 << 18), 'too many')])
def test_window_refusals(L, kw, words):
    _bad(L, window(L, **kw), words)


def test_window_backward_refusals(L):
    def call(lse=P, ws=P, dq=P, on=512):
        return L.vitk_window_attn_bwd(BF16, 1, 16, 4, 2, 64, P, 8192, 512, 64, P, 8192, 512, 64, P, 8192, 512, 64, 0.125, 4, 1, 0, 0,
                                      P, 0, lse, P, 8192, on, 64, dq, P, P, ws, 0)
    _bad(L, call(lse=0), 'null')
    _bad(L, call(ws=0), 'null')
    _bad(L, call(ws=P + 8), 'aligned')
    _bad(L, call(on=508), 'dout must be')
    assert L.vitk_window_attn_bwd_workspace_bytes(BF16, 2, 1000, 8, 2, 64, 10, 4) >= 2 * 1000 * 8 * 4
    assert L.vitk_window_attn_bwd_workspace_bytes(BF16, 0, 1000, 8, 2, 64, 10, 4) == 0


def decode(L, dtype=BF16, B=1, Hq=4, Hk=2, dh=64, q=P, C=16, n=P, scale=0.1, w=10, sinks=2, kc=P, qh=64):
    return L.vitk_window_decode(dtype, B, Hq, Hk, dh, q, 256, qh, P, 128, 64, P, 128, 64, kc, P, C, n, scale, w, sinks, P, 0, 0)


@pytest.mark.parametrize('kw,words', [
    (dict(dtype=9), 'bad dtype'), (dict(Hq=3), 'bad shape'), (dict(dh=4), 'head width'), (dict(C=0), 'bad cache'),
    (dict(C=12), 'cannot hold'), (dict(w=2 ** 31 - 1), 'cannot hold'), (dict(sinks=-2), 'bad cache'), (dict(scale=0.0), 'scale'),
    (dict(q=P + 2), 'aligned'), (dict(kc=0), 'aligned'), (dict(n=0), 'aligned'), (dict(qh=60), 'aligned')])
def test_decode_refusals(L, kw, words):
    _bad(L, decode(L, **kw), words)


def test_fill_and_table_refusals(L):
    def fill(C=16, sinks=2, N=4, k=P):
        return L.vitk_window_cache_fill(BF16, 1, N, 2, 64, k, 512, 128, 64, P, 512, 128, 64, 0, P, P, C, sinks, 0)
    _bad(L, fill(C=2), 'bad sizes')
    _bad(L, fill(N=-1), 'bad sizes')
    _bad(L, fill(k=P + 1), 'aligned')
    f = (ctypes.c_double * 200)()
    fp = ctypes.cast(f, ctypes.c_void_p)
    _bad(L, L.vitk_rotary_table(4, 1, 8, P, 8, fp, 1.0, P, 0), 'position type')
    _bad(L, L.vitk_rotary_table(0, 3, 8, P, 8, fp, 1.0, P, 0), 'pairs')
    _bad(L, L.vitk_rotary_table(0, 1, 8, P, 129, fp, 1.0, P, 0), 'pairs')
    _bad(L, L.vitk_rotary_table(0, 1, 8, 0, 8, fp, 1.0, P, 0), 'null')


def test_nothing_to_do_is_no_error(L):
    assert rotary(L, B=0) == 0 and rotary(L, N=0) == 0 and norm(L, B=0) == 0 and window(L, N=0) == 0 and decode(L, B=0) == 0


def test_wrappers_refuse_cpu_tensors():
    from vit_amd import functional as VF
    from vit_amd._lib import VitkError
    from vit_amd.window import WindowCache
    x = torch.zeros(1, 4, 2, 64)
    n = torch.zeros(1, dtype=torch.int32)
    c = torch.zeros(1, 2, 8, 64)
    for f in (lambda: VF.rotary(x, torch.zeros(4, 32, 2)), lambda: VF.qk_norm_rotary(x, x, None, None),
              lambda: VF.window_attention(x, x, x, 2), lambda: VF.window_decode(x[:, 0], x[:, 0], x[:, 0], c, c, n, 2),
              lambda: VF.window_cache_fill(x, x, c, c), lambda: VF.rotary_table(torch.arange(4), 64)):
        with pytest.raises(VitkError):
            f()
    for kw in (dict(window=-1), dict(window=4, slots=4), dict(window=4, sinks=2, slots=6), dict(window=2, sinks=-1)):
        with pytest.raises(ValueError):
            WindowCache(1, 2, 64, device='cpu', **kw)


def test_frequencies():
    from vit_amd.functional import rotary_frequencies as rf
    plain, m = rf(64)
    assert m == 1.0 and plain[0] == 1.0 and abs(plain[31] - 10000 ** (-62 / 64)) < 1e-18
    assert rf(64, scaling=dict(type='linear', factor=4))[0] == [w / 4 for w in plain]
    ntk, _ = rf(64, scaling=dict(type='ntk', factor=8))
    assert ntk[0] == 1.0 and abs(ntk[31] * 8 / plain[31] - 1) < 1e-12        # the slowest pair is interpolated by the factor
    yarn, m = rf(64, scaling=dict(type='yarn', factor=16, original=4096))
    assert abs(m - (0.1 * math.log(16) + 1)) < 1e-15
    for w, y in zip(plain, yarn):
        turns = 4096 * w / (2 * math.pi)
        if turns >= 32:
            assert y == w
        elif turns <= 1:
            assert abs(y - w / 16) < 1e-18
        else:
            assert w / 16 < y < w
    for bad in (dict(type='ntk'), dict(factor=2), dict(type='linear', factor=-1), dict(type='yarn', factor=2), dict(type='linear', factor=2, x=1),
                dict(type='yarn', factor=2, original=10, beta_fast=1, beta_slow=1)):
        with pytest.raises(ValueError):
            rf(64, scaling=bad)
    for bad in ((63,), (0,), (64, 0.0)):
        with pytest.raises(ValueError):
            rf(*bad)


def test_more_work_than_a_launch_holds(L):
    """Refused by its size, not by a failed launch: workgroups times threads past 2^32."""
    _bad(L, norm(L, B=1 << 12, N=1 << 16, Hq=1, Hk=1, dh=127, rot=2, rows=1 << 16), 'too many')
    _bad(L, window(L, B=1 << 24, N=16, Hq=4), 'too many')
    _bad(L, window(L, B=1 << 14, N=1 << 17, Hk=1, Hq=1), 'too many')
    _bad(L, decode(L, B=1 << 26), 'too many')

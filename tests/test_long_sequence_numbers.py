"""Numbers past the C entry points' types: ctypes cuts them to the type's bits without a word, so they have to be refused, or
held to the type's range, before they get there."""
import ctypes

import pytest
import torch

BIG = 2 ** 32 + 5                     # 5 in 32 bits
P = 1 << 20


@pytest.fixture
def calls(monkeypatch):
    """The wrappers on tensors without memory, and a library that takes down what it is given."""
    from vit_amd import _lib, ops
    seen = []

    class Fake:
        def __getattr__(self, name):
            def f(*args):
                types = _lib._SIGNATURES[name][0]
                assert len(args) == len(types), name
                seen.append((name, args, types))
                return 0
            return f
    monkeypatch.setattr(ops, 'lib', lambda: Fake())
    monkeypatch.setattr(ops, '_req_here', lambda *ts: 0)
    monkeypatch.setattr(ops, '_stream', lambda: 0)
    monkeypatch.setattr(ops, '_stream_on', lambda dev: 0)
    return seen


def _rows(B, N, H, dh=16):
    return torch.empty(1, 1, 1, dh, device='meta').expand(B, N, H, dh)


def _i32(*shape):
    return torch.empty(*shape, dtype=torch.int32, device='meta')


def _cases():
    from vit_amd import ops
    x, t = _rows(1, 4, 2), torch.empty(4, 8, 2, device='meta')
    c = torch.empty(1, 2, 16, 16, device='meta')
    one = x[:, 0]
    yield 'decode sinks', lambda n: ops.window_decode(one, one, one, c, c, _i32(1), 4, n, 0.25)
    yield 'decode window', lambda n: ops.window_decode(one, one, one, c, c, _i32(1), n, 2, 0.25)
    yield 'fill sinks', lambda n: ops.window_cache_fill(x, x, c, c, n)
    yield 'attention sinks', lambda n: ops.window_attn_fwd(ops.window_attn_plan(x, x, x, 4, n, True, 0.25, None), x, x, x, None)
    yield 'attention window', lambda n: ops.window_attn_fwd(ops.window_attn_plan(x, x, x, n, 1, True, 0.25, None), x, x, x, None)
    yield 'rotary offset', lambda n: ops.rotary(x, t, offset=n)
    yield 'norm offset', lambda n: ops.qk_norm_rotary_fwd(ops.qk_norm_rotary_plan(x, x, None, None, t, None, n, 1e-6, False), x, x, None,
                                                          None, t, None)


@pytest.mark.parametrize('n', [BIG, -2 ** 32, 2 ** 31, 2 ** 63, 2 ** 64 + 1, -2 ** 64])
@pytest.mark.parametrize('case', [0, 1, 2, 3, 4, 5, 6])
def test_numbers_arrive_as_they_are_or_not_at_all(calls, case, n):
    name, call = list(_cases())[case]
    try:
        call(n)
    except (ValueError, RuntimeError):
        return
    assert calls
    for what, args, types in calls:
        for a, t in zip(args, types):
            if t in (ctypes.c_int, ctypes.c_long):
                assert t(a).value == a, (name, what, a)


@pytest.mark.parametrize('shape', [(BIG, 4, 2), (1, BIG, 2), (1, 4, BIG), (2 ** 31, 1, 1)], ids=str)
def test_sizes_past_32_bits_are_refused(calls, shape):
    from vit_amd import ops
    B, N, H = shape
    x, t = _rows(B, N, H), torch.empty(4, 8, 2, device='meta')
    c = torch.empty(1, 1, 16, 16, device='meta').expand(B, H, 16, 16)
    one = _rows(B, 1, H)[:, 0]
    yes = [lambda: ops.rotary(x, t), lambda: ops.qk_norm_rotary_plan(x, x, None, None, None, None, 0, 1e-6, False),
           lambda: ops.window_attn_plan(x, x, x, 4, 0, False, 0.25, None),
           lambda: ops.window_cache_fill(x, x, c, c, 0)]
    if N != BIG:
        yes.append(lambda: ops.window_decode(one, one, one, c, c, _i32(B), 4, 0, 0.25))
    for f in yes:
        with pytest.raises(ValueError):
            f()
    assert not calls


def test_a_cache_of_more_slots_than_32_bits_count_is_refused(calls):
    from vit_amd import ops
    one, x = _rows(1, 1, 1)[:, 0], _rows(1, 4, 1)
    c = torch.empty(1, 1, BIG, 16, device='meta')
    for f in (lambda: ops.window_decode(one, one, one, c, c, _i32(1), 4, 0, 0.25), lambda: ops.window_cache_fill(x, x, c, c, 0)):
        with pytest.raises(ValueError):
            f()
    assert not calls


def test_an_offset_whose_sum_with_the_tokens_overflows():
    from vit_amd._lib import lib
    L = lib()
    far = 2 ** 63 - 1
    assert L.vitk_rotary(1, 0, 0, 1, 4, 2, 64, P, 512, 128, 64, P, 4, 64, 0, 0, far, P, 0) == 1
    assert 'outside the table' in L.vitk_last_error().decode()
    assert L.vitk_qk_norm_rotary_fwd(1, 0, 1, 4, 2, 1, 64, P, 512, 128, 64, P, 512, 128, 64, 0, 0, 1e-6, P, 4, 64, 0, 0, far, P, P, 0) == 1
    assert 'outside the table' in L.vitk_last_error().decode()

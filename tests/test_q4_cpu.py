"""Host-side checks of the 4-bit decode step: the restatement agrees with itself, and calls that cannot run are refused before anything
is launched (no device is needed for that: what is wrong with the arguments is said first)."""
import ctypes as C
import importlib
import math

import numpy as np
import pytest
import torch

from oracle import q4

P = 1 << 20  # an aligned address that no refused call reads
_CTX = C.create_string_buffer(4096)  # stands for a context: a call refused for its arguments does not look into it
CTX = C.addressof(_CTX)
BAD, UNSUPPORTED = 1, 2


def test_every_place_of_a_page_is_used_once():
    for g in (32, 64, 128):
        k, v, ks, vs = q4.page_places(g)
        assert sorted(np.concatenate([k.ravel(), v.ravel()])) == list(range(4096))
        places = np.unique(np.concatenate([ks.ravel(), vs.ravel()]))
        assert list(places) == list(range(1024, q4.page_bytes(g) // 2))


@pytest.mark.parametrize("g", [32, 64, 128])
def test_pages_hold_what_the_groups_stand_for(g):
    rng = np.random.default_rng(g)
    K, V = (rng.standard_normal((3, 2, 16, 128)).astype(np.float16) for _ in range(2))
    k, v = q4.open_pages(q4.fill_pages(K, V, g), g)
    assert np.array_equal(k, q4.values(*q4.quantize(K, g), g)) and np.array_equal(v, q4.values(*q4.quantize(V, g), g))


def test_a_groups_extreme_is_exact_and_ties_go_to_the_even_code():
    x = np.zeros((1, 32), np.float16)
    x[0, :8] = [-8, 0.5, 1.5, 2.5, -0.5, -1.5, 7.75, 8.0]
    codes, s = q4.quantize(x, 32)
    assert s[0, 0] == -1.0  # of -8 and 8 the positive one
    assert list(codes[0, :8]) == [7, 0, -2, -2, 0, 2, -8, -8]
    assert q4.values(codes, s, 32)[0, 7] == 8.0


def test_groups_with_something_that_is_no_number_read_as_nan():
    x = np.ones((3, 64), np.float16)
    x[0, 3], x[1, 40], x[2, 5] = np.inf, np.nan, -np.inf
    v = q4.values(*q4.quantize(x, 32), 32)
    nan = np.isnan(v).reshape(3, 2, 32).all(-1)
    assert nan.tolist() == [[True, False], [False, True], [True, False]] and np.isnan(v).sum() == 96


def _plan_args(**change):
    a = dict(ctx=CTX, cached=P, new=P, batch=4, table=P, width=8, free=P, capacity=64, count=P, count_out=P, slots=P, positions=P, lens=P, first=P,
             tokens=16, info=P, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), BAD), (dict(batch=-1), BAD), (dict(width=0), BAD), (dict(capacity=-1), BAD), (dict(tokens=-1), BAD), (dict(batch=4097), UNSUPPORTED),
    (dict(cached=None), BAD), (dict(new=None), BAD), (dict(table=None), BAD), (dict(free=None), BAD), (dict(count=None), BAD), (dict(count_out=None), BAD),
    (dict(slots=None), BAD), (dict(positions=None), BAD), (dict(lens=None), BAD), (dict(first=None), BAD), (dict(info=None), BAD)])
def test_plan_blocks_refuses(pkg, change, status):
    lib = pkg.load_library()
    assert lib.w8a8_plan_blocks(*_plan_args(**change)) == status and lib.w8a8_last_error()


def _write_args(**change):
    a = dict(ctx=CTX, qkv=P, q_norm=P, k_norm=P, eps=1e-6, freqs=P, positions=P, slots=P, cache=P, blocks=9, layer=0, layers=2, tokens=3, n_q=8, n_kv=2,
             dim=128, group=32, q_out=P, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), BAD), (dict(tokens=-1), BAD), (dict(blocks=0), BAD), (dict(blocks=-1), BAD), (dict(layer=2), BAD), (dict(layer=-1), BAD),
    (dict(layers=0), BAD), (dict(n_kv=0), BAD), (dict(n_q=-1), BAD), (dict(dim=64), UNSUPPORTED), (dict(group=16), UNSUPPORTED), (dict(group=96), UNSUPPORTED),
    (dict(qkv=None), BAD), (dict(slots=None), BAD), (dict(cache=None), BAD), (dict(cache=P + 8), BAD), (dict(q_norm=None), BAD), (dict(k_norm=None), BAD),
    (dict(freqs=None), BAD), (dict(positions=None), BAD), (dict(qkv=P + 2), BAD), (dict(q_out=P + 4), BAD)])
def test_kv4_write_refuses(pkg, change, status):
    lib = pkg.load_library()
    assert lib.w8a8_kv4_write(*_write_args(**change)) == status and lib.w8a8_last_error()


def _read_args(**change):
    a = dict(ctx=CTX, cache=P, blocks=9, slots=P, layer=0, layers=2, tokens=3, n_kv=2, dim=128, group=32, k=P, v=P, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), BAD), (dict(tokens=-1), BAD), (dict(blocks=0), BAD), (dict(layer=2), BAD), (dict(n_kv=0), BAD), (dict(dim=256), UNSUPPORTED),
    (dict(group=0), UNSUPPORTED), (dict(slots=None), BAD), (dict(k=None, v=None), BAD), (dict(k=P + 2), BAD), (dict(v=P + 4), BAD), (dict(cache=None), BAD)])
def test_kv4_read_refuses(pkg, change, status):
    lib = pkg.load_library()
    assert lib.w8a8_kv4_read(*_read_args(**change)) == status and lib.w8a8_last_error()


def _attention_args(**change):
    a = dict(ctx=CTX, q=P, cache=P, blocks=9, table=P, lens=P, out=P, batch=2, heads=8, dim=128, width=4, scale=0.1, layer=0, layers=2, n_kv=2, group=32,
             quant=0, xq=None, xs=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), BAD), (dict(batch=-1), BAD), (dict(batch=4097), UNSUPPORTED), (dict(blocks=0), BAD), (dict(width=0), BAD), (dict(width=1 << 28), BAD),
    (dict(layer=2), BAD), (dict(heads=0), UNSUPPORTED), (dict(heads=7), UNSUPPORTED), (dict(heads=18), UNSUPPORTED), (dict(dim=64), UNSUPPORTED),
    (dict(group=256), UNSUPPORTED), (dict(q=None), BAD), (dict(table=None), BAD), (dict(lens=None), BAD), (dict(out=None), BAD), (dict(q=P + 8), BAD),
    (dict(out=P + 4), BAD), (dict(xq=P), BAD), (dict(xq=P, xs=P, quant=0), UNSUPPORTED), (dict(xq=P, xs=P, quant=2), UNSUPPORTED),
    (dict(xq=P, xs=P, quant=96), UNSUPPORTED), (dict(xq=P, xs=P, quant=1024), UNSUPPORTED), (dict(xq=P + 1, xs=P, quant=64), BAD)])
def test_kv4_attention_refuses(pkg, change, status):
    lib = pkg.load_library()
    for call in (lib.w8a8_kv4_attention_decode, lib.w8a8_kv4_attention_decode_ahead):
        assert call(*_attention_args(**change)) == status and lib.w8a8_last_error()


def _linear_args(**change):
    a = dict(ctx=CTX, w=P, s=P, g=64, xq=P, xs=P, y=P, M=2, N=32, K=128, epilogue=0, residual=None, stream=None)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,status", [
    (dict(ctx=None), BAD), (dict(M=-1), BAD), (dict(N=0), BAD), (dict(K=0), BAD), (dict(K=127), UNSUPPORTED), (dict(g=63), UNSUPPORTED),
    (dict(K=(1 << 20) + 2), UNSUPPORTED), (dict(w=None), BAD), (dict(s=None), BAD), (dict(xq=None), BAD), (dict(xs=None), BAD), (dict(y=None), BAD),
    (dict(epilogue=3), BAD), (dict(epilogue=1), BAD), (dict(residual=P), BAD), (dict(epilogue=2, N=24), BAD)])
def test_linear4_refuses(pkg, change, status):
    lib = pkg.load_library()
    assert lib.w8a8_linear4_q(*_linear_args(**change)) == status and lib.w8a8_last_error()


def test_weight4_calls_refuse(pkg):
    lib = pkg.load_library()
    for args, status in (((None, P, 4, 64, 32, P, P, None), BAD), ((CTX, None, 4, 64, 32, P, P, None), BAD), ((CTX, P, 0, 64, 32, P, P, None), BAD),
                         ((CTX, P, 4, 63, 32, P, P, None), UNSUPPORTED), ((CTX, P, 4, 64, 31, P, P, None), UNSUPPORTED), ((CTX, P, 4, 64, 32, None, P, None), BAD)):
        assert lib.w8a8_quantize_weight4(*args) == status
    for args, status in (((None, P, 4, 64, P, None), BAD), ((CTX, None, 4, 64, P, None), BAD), ((CTX, P, 4, 65, P, None), UNSUPPORTED), ((CTX, P, 4, 64, P + 1, None), BAD)):
        assert lib.w8a8_unpack_weight4(*args) == status


def test_sizes_of_caches_and_scratch(pkg):
    assert pkg.kv4_cache_bytes(10, 3, 2, 128, 32) == 10 * 3 * 2 * 2304 and pkg.kv4_cache_bytes(1, 1, 1, 128, 64) == 2176 and pkg.kv4_cache_bytes(1, 1, 1, 128, 128) == 2112
    assert pkg.kv4_cache_bytes(1 << 20, 36, 8, 128, 32) == (1 << 20) * 36 * 8 * 2304  # past 32 bits
    assert not any(pkg.kv4_cache_bytes(*a) for a in ((0, 1, 1, 128, 32), (1, 0, 1, 128, 32), (1, 1, 0, 128, 32), (1, 1, 1, 64, 32), (1, 1, 1, 128, 48)))
    assert pkg.kv4_attention_workspace_bytes(32, 8) > 0 and pkg.kv4_attention_workspace_bytes(8, 1) > pkg.kv4_attention_workspace_bytes(4, 1)
    assert not any(pkg.kv4_attention_workspace_bytes(*a) for a in ((0, 1), (9, 1), (5, 2), (4, 0)))
    assert math.gcd(q4.page_bytes(32), q4.page_bytes(64), q4.page_bytes(128)) % 16 == 0


def _both_call_modules(pkg):
    capi, lib = importlib.import_module(pkg.__name__ + ".capi"), pkg.load_library()
    made = capi._load_calls(lib)
    return [made] if isinstance(made, capi._CtypesCalls) else [made, capi._CtypesCalls(lib)]


def test_calls_refuse_alike_from_python(pkg):
    for calls in _both_call_modules(pkg):
        for name, args, changes in (("w8a8_plan_blocks", _plan_args, (dict(ctx=None), dict(batch=4097), dict(info=None))),
                                    ("w8a8_kv4_write", _write_args, (dict(tokens=-1), dict(dim=64), dict(qkv=P + 2))),
                                    ("w8a8_kv4_read", _read_args, (dict(k=None, v=None), dict(group=0))),
                                    ("w8a8_kv4_attention_decode", _attention_args, (dict(heads=7), dict(out=P + 4))),
                                    ("w8a8_kv4_attention_decode_ahead", _attention_args, (dict(heads=7), dict(out=P + 4))),
                                    ("w8a8_linear4_q", _linear_args, (dict(K=127), dict(w=None), dict(epilogue=2, N=24)))):
            call, plain = getattr(calls, name), getattr(pkg.load_library(), name)
            for change in changes:
                assert call(*args(**change)) == plain(*args(**change)) != 0
            with pytest.raises((TypeError, C.ArgumentError)):
                call(*args()[:-1])
            with pytest.raises((AttributeError, TypeError, C.ArgumentError)):
                call(*["no address" if a == P else a for a in args()])


def test_calls_hand_over_what_they_are_given(pkg):
    """Bound to functions that note their arguments: tensors arrive as their addresses, None as null, numbers as they are."""
    calls, lib = _both_call_modules(pkg)[0], pkg.load_library()
    if type(calls).__name__ == "_CtypesCalls":
        pytest.skip("w8a8_calls is not built")
    names, seen, kept = [n for n in dir(calls) if n.startswith("w8a8_")], [], []
    try:
        for n in names:
            plain = getattr(lib, n)
            kept.append(C.CFUNCTYPE(C.c_int, *plain.argtypes)(lambda *a: seen.append(a) or 7))
        calls.bind({n: C.cast(f, C.c_void_p).value for n, f in zip(names, kept)})
        for n in names:
            types = getattr(lib, n).argtypes
            tensors = [torch.empty(4) for _ in types]
            args = [t if ty is C.c_void_p and i % 3 else None if ty is C.c_void_p else 0.375 if ty is C.c_float else 1000 + i
                    for i, (ty, t) in enumerate(zip(types, tensors))]
            args[0] = (1 << 47) - 8
            assert getattr(calls, n)(*args) == 7
            assert list(seen.pop()) == [a.data_ptr() if isinstance(a, torch.Tensor) else a for a in args]
            whole = next(i for i, ty in enumerate(types) if ty is C.c_int)
            for wrong, error in ((1 << 31, OverflowError), (1 << 70, OverflowError), (1.5, TypeError), (None, TypeError)):
                with pytest.raises(error):
                    getattr(calls, n)(*args[:whole], wrong, *args[whole + 1:])
            assert not seen
    finally:
        calls.bind({n: C.cast(getattr(lib, n), C.c_void_p).value for n in names})

"""Refusals of the speculative-decoding entry points at the C ABI (CPU only: no
kernel is launched, the pointers are never followed)."""
import ctypes

import pytest

from torchplusplus_amd import _native

E_INVALID, E_UNSUPPORTED, E_WORKSPACE = -1, -2, -4
I64, I32, F32 = ctypes.c_int64, ctypes.c_int, ctypes.c_float


def p(v=1024):
    return ctypes.c_void_p(v)


def s(*v):
    return (I64 * len(v))(*v)


def rope(q=p(), freq=p(4096), b=2, t=3, hq=4, hk=2, d=64, r=64, dtype=1, strides=s(768, 256, 64)):
    return _native.lib().tpp_rope_at(q, p(), p(), p(), strides, strides, strides, strides, p(), I64(3), I32(0), freq,
                                     F32(1.0), I64(b), I64(t), I64(hq), I64(hk), I64(d), I64(r), I32(0), I32(dtype), None)


def append(k=p(), codes=p(), b=2, t=3, h=2, d=64, room=32, code=1, dtype=1, strides=s(384, 128, 64),
           code_strides=s(4096, 2048)):
    return _native.lib().tpp_kv_quant_append(k, p(), strides, strides, codes, p(), p(), p(), code_strides, s(64, 32),
                                             None, I64(0), None, I64(b), I64(t), I64(h), I64(d), I64(room), I32(code),
                                             I32(dtype), None)


def read(out=p(), b=2, h=2, n=5, d=64, room=32, code=2, dtype=0):
    return _native.lib().tpp_kv_quant_read(p(), p(), p(), p(), s(4096, 2048), s(64, 32), out, p(), I64(b), I64(h), I64(n),
                                           I64(d), I64(room), I32(code), I32(dtype), None)


def attn(q=p(), b=2, t=3, hq=4, hkv=2, d=64, room=4096, code=0, dtype=1, exps=p(), ws=None, bytes_=0, lens=p()):
    st = s(768, 256, 64)
    return _native.lib().tpp_tree_attn(q, p(), p(), p(), exps, exps, st, s(524288, 262144, 64), s(524288, 262144, 64),
                                       s(8192, 4096), st, lens, None, I64(b), I64(t), I64(hq), I64(hkv), I64(d),
                                       I64(room), F32(0.0), I32(code), I32(dtype), ws, ctypes.c_size_t(bytes_), None)


def verify(tok=p(), par=None, q=None, b=2, t=3, v=1000, dtype=2, ws=p(), bytes_=1 << 20):
    return _native.lib().tpp_verify_draft(tok, par, p(), s(4000, 1000), q, s(3000, 1000), p(), p(), p(), p(), I64(b),
                                          I64(t), I64(v), I32(dtype), ws, ctypes.c_size_t(bytes_), None)


@pytest.mark.parametrize("call,want", [
    (lambda: rope(q=None), E_INVALID), (lambda: rope(freq=None), E_INVALID), (lambda: rope(strides=None), E_INVALID),
    (lambda: rope(r=66), E_INVALID), (lambda: rope(r=3), E_INVALID), (lambda: rope(d=63, r=2), E_INVALID),
    (lambda: rope(hq=0), E_INVALID), (lambda: rope(dtype=2), E_UNSUPPORTED), (lambda: rope(b=1 << 40), E_UNSUPPORTED),
    (lambda: append(k=None), E_INVALID), (lambda: append(d=80), E_UNSUPPORTED), (lambda: append(code=3), E_UNSUPPORTED),
    (lambda: append(dtype=2), E_UNSUPPORTED), (lambda: append(k=p(1026)), E_INVALID),
    (lambda: append(strides=s(384, 128, 63)), E_INVALID), (lambda: append(codes=p(1028)), E_INVALID),
    (lambda: append(code_strides=s(4096, 2049)), E_INVALID), (lambda: append(t=-1), E_INVALID),
    (lambda: read(n=33), E_INVALID), (lambda: read(n=-1), E_INVALID), (lambda: read(out=p(1032)), E_INVALID),
    (lambda: read(code=0), E_UNSUPPORTED), (lambda: read(d=96), E_UNSUPPORTED),
    (lambda: attn(q=None), E_INVALID), (lambda: attn(lens=None), E_INVALID), (lambda: attn(t=0), E_UNSUPPORTED),
    (lambda: attn(t=65), E_UNSUPPORTED), (lambda: attn(hq=5), E_INVALID), (lambda: attn(d=257), E_UNSUPPORTED),
    (lambda: attn(code=1, exps=None), E_INVALID), (lambda: attn(code=5), E_UNSUPPORTED), (lambda: attn(dtype=2), E_UNSUPPORTED),
    (lambda: attn(room=0), E_INVALID), (lambda: attn(b=65536), E_UNSUPPORTED), (lambda: attn(), E_WORKSPACE),
    (lambda: attn(ws=p(64), bytes_=1 << 30), E_WORKSPACE), (lambda: attn(ws=p(), bytes_=64), E_WORKSPACE),
    (lambda: verify(tok=None), E_INVALID), (lambda: verify(par=p(), q=p()), E_UNSUPPORTED), (lambda: verify(t=65), E_UNSUPPORTED),
    (lambda: verify(t=0), E_UNSUPPORTED), (lambda: verify(v=0), E_INVALID), (lambda: verify(v=1 << 31), E_INVALID),
    (lambda: verify(dtype=3), E_UNSUPPORTED), (lambda: verify(ws=None), E_WORKSPACE),
    (lambda: verify(bytes_=8), E_WORKSPACE), (lambda: verify(b=65536), E_UNSUPPORTED)])
def test_refused_before_any_launch(call, want):
    lib = _native.lib()
    assert call() == want
    assert len(lib.tpp_last_error_string()) > 0


def test_empty_calls_do_nothing():
    assert rope(b=0) == 0 and rope(t=0) == 0 and append(b=0) == 0 and append(t=0) == 0 and read(n=0) == 0
    assert attn(b=0) == 0 and verify(b=0) == 0


def test_workspace_sizes():
    lib = _native.lib()
    f, g = lib.tpp_tree_attn_workspace_size, lib.tpp_verify_draft_workspace_size
    f.restype = g.restype = ctypes.c_size_t
    attn_bytes = lambda *a: f(*[I64(x) for x in a[:6]], I32(a[6]))  # noqa: E731
    assert attn_bytes(1, 1, 2, 1, 128, 100, 0) == 0 and attn_bytes(0, 1, 2, 1, 128, 4096, 0) == 0
    assert attn_bytes(1, 1, 2, 1, 96, 1 << 20, 0) == 0
    assert attn_bytes(2, 3, 4, 2, 64, 4096, 0) % (2 * 3 * 4 * 66 * 4) == 0 < attn_bytes(2, 3, 4, 2, 64, 4096, 0)
    assert g(I64(3), I64(4097)) == 3 * 2 * 16 + 3 * 16 and g(I64(0), I64(5)) == 0

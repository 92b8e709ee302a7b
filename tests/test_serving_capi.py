"""Refusals of the entry points of a mixed batch at the C ABI (CPU only: no kernel is
launched, the pointers are never followed)."""
import ctypes

import pytest

from torchplusplus_amd import _native

E_INVALID, E_UNSUPPORTED, E_WORKSPACE = -1, -2, -4
I64, I32, F32 = ctypes.c_int64, ctypes.c_int, ctypes.c_float


def p(v=1024):
    return ctypes.c_void_p(v)


def s(*v):
    return (I64 * len(v))(*v)


def packed(q=p(), k=p(), cu=p(), cu_k=None, strides=s(256, 64), b=2, n=10, nk=10, hq=4, hk=2, d=64, fill=0, dtype=1):
    return _native.lib().tpp_attn_packed(q, k, p(), p(), strides, strides, strides, strides, cu, cu_k, I64(b), I64(n), I64(nk),
                                         I64(hq), I64(hk), I64(d), F32(0.0), I32(1), I32(-1), I32(-1), I32(fill), I32(dtype),
                                         None, ctypes.c_size_t(0), None)


def paged(q=p(), k=p(), table=p(), lens=p(), strides=s(4096, 2048, 64), b=2, hq=4, hk=2, d=64, pages=9, page=32, width=5,
          t_stride=5, dtype=1, ws=None, bytes_=0):
    return _native.lib().tpp_attn_paged(q, k, p(), p(), s(256, 64), strides, strides, s(256, 64), table, I64(t_stride),
                                        I64(width), lens, I64(b), I64(hq), I64(hk), I64(d), I64(pages), I64(page), F32(0.0),
                                        I32(-1), I32(dtype), ws, ctypes.c_size_t(bytes_), None)


def rope(qkv=p(), q=p(), kp=p(), strides=s(4096, 2048, 64), stride=512, n=3, hq=4, hk=2, d=64, pages=9, page=32, ctx=100,
         pos=p(), slots=p(), cos=p(), dtype=1, cs=0):
    return _native.lib().tpp_qkv_rope_paged(qkv, I64(stride), q, None, kp, p(), strides, strides, None, None, cos, p(),
                                            I64(ctx), pos, slots, I64(n), I64(hq), I64(hk), I64(d), I64(pages), I64(page),
                                            F32(1e-6), I32(dtype), I32(cs), None)


def logprobs(x=p(), tok=p(), n=2, v=1000, top=0, top_ptr=p(), dtype=1, stride=1000, ws=None, bytes_=0):
    return _native.lib().tpp_token_logprobs(x, I64(stride), tok, p(), p(), top_ptr, top_ptr, I64(n), I64(v), I64(top),
                                            I32(dtype), ws, ctypes.c_size_t(bytes_), None)


@pytest.mark.parametrize("call,want", [
    (lambda: packed(q=None), E_INVALID), (lambda: packed(k=None), E_INVALID), (lambda: packed(cu=None), E_INVALID),
    (lambda: packed(strides=None), E_INVALID), (lambda: packed(nk=9), E_INVALID), (lambda: packed(hq=5), E_INVALID),
    (lambda: packed(hk=0), E_INVALID), (lambda: packed(b=-1), E_INVALID), (lambda: packed(n=-1, nk=-1), E_INVALID),
    (lambda: packed(d=0), E_INVALID), (lambda: packed(d=257), E_UNSUPPORTED), (lambda: packed(dtype=2), E_UNSUPPORTED),
    (lambda: packed(hq=1 << 16, hk=1 << 16), E_UNSUPPORTED), (lambda: packed(b=(1 << 20) + 1), E_UNSUPPORTED),
    (lambda: packed(n=(1 << 30) + 1, nk=(1 << 30) + 1), E_UNSUPPORTED),
    (lambda: paged(q=None), E_INVALID), (lambda: paged(k=None), E_INVALID), (lambda: paged(table=None), E_INVALID),
    (lambda: paged(lens=None), E_INVALID), (lambda: paged(strides=None), E_INVALID), (lambda: paged(hq=3), E_INVALID),
    (lambda: paged(pages=-1), E_INVALID), (lambda: paged(width=-1), E_INVALID), (lambda: paged(t_stride=-1), E_INVALID),
    (lambda: paged(page=24), E_UNSUPPORTED), (lambda: paged(page=8), E_UNSUPPORTED), (lambda: paged(page=2048), E_UNSUPPORTED),
    (lambda: paged(page=0), E_UNSUPPORTED), (lambda: paged(d=300), E_UNSUPPORTED), (lambda: paged(dtype=2), E_UNSUPPORTED),
    (lambda: paged(b=65536), E_UNSUPPORTED), (lambda: paged(width=1 << 27), E_UNSUPPORTED),
    (lambda: rope(qkv=None), E_INVALID), (lambda: rope(q=None), E_INVALID), (lambda: rope(kp=None), E_INVALID),
    (lambda: rope(pos=None), E_INVALID), (lambda: rope(slots=None), E_INVALID), (lambda: rope(cos=None), E_INVALID),
    (lambda: rope(strides=None), E_INVALID), (lambda: rope(stride=511), E_INVALID), (lambda: rope(qkv=p(1026)), E_INVALID),
    (lambda: rope(strides=s(4096, 2048, 68)), E_INVALID), (lambda: rope(stride=516), E_INVALID), (lambda: rope(ctx=0), E_INVALID),
    (lambda: rope(n=-1), E_INVALID), (lambda: rope(d=96, stride=1000), E_UNSUPPORTED), (lambda: rope(page=24), E_UNSUPPORTED),
    (lambda: rope(dtype=2), E_UNSUPPORTED), (lambda: rope(cs=3), E_UNSUPPORTED), (lambda: rope(n=1 << 32), E_UNSUPPORTED),
    (lambda: logprobs(x=None), E_INVALID), (lambda: logprobs(tok=None), E_INVALID), (lambda: logprobs(n=-1), E_INVALID),
    (lambda: logprobs(v=0), E_INVALID), (lambda: logprobs(stride=-1), E_INVALID), (lambda: logprobs(top=33), E_UNSUPPORTED),
    (lambda: logprobs(top=-1), E_UNSUPPORTED), (lambda: logprobs(v=4, top=5), E_UNSUPPORTED),
    (lambda: logprobs(dtype=3), E_UNSUPPORTED), (lambda: logprobs(v=1 << 31), E_UNSUPPORTED),
    (lambda: logprobs(top=4, top_ptr=None, n=600), E_INVALID)])
def test_refused_before_any_launch(call, want):
    lib = _native.lib()
    assert call() == want
    assert len(lib.tpp_last_error_string()) > 0


def test_empty_calls_do_nothing():
    assert packed(n=0, nk=0) == 0 and packed(b=0) == 0 and paged(b=0) == 0 and rope(n=0) == 0 and logprobs(n=0) == 0

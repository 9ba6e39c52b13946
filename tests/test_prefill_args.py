"""What the calls over packed query tokens and build_tables refuse, on the host and before any
launch; and the plans' workspace."""

from __future__ import annotations

import ctypes

import pytest

from vllm_fastdecoder_amd import _lib

P = 4096  # a pointer that is never followed


def _paged(**over):
    a = dict(q=P, qst=512, qsh=64, k=P, v=P, sb=4096, sh=128, st=256, B=9, bt=P, bts=8, W=8, cu=P,
             lens=P, n=2, T=7, mq=5, causal=1, H=8, KVH=2, D=64, BS=16, scale=0.1, dt=0, out=P,
             ost=512, osh=64, odt=0, lse=P, lsh=7, ws=None, wsb=0, stream=None,
             counters=None)
    a.update(over)
    return _lib.load_lib().fd_paged_prefill(*a.values())


def _varlen(**over):
    a = dict(q=P, qst=512, qsh=64, k=P, kst=128, ksh=64, v=P, vst=128, vsh=64, cuq=P, cuk=P, n=2,
             T=7, Tk=30, mq=5, mk=20, causal=0, H=8, KVH=2, D=64, scale=0.1, dt=0, out=P, ost=512,
             osh=64, odt=0, lse=P, lsh=7, ws=None, wsb=0, stream=None, counters=None)
    a.update(over)
    return _lib.load_lib().fd_varlen_attention(*a.values())


def _tables(**over):
    a = dict(qsl=P, ctx=P, n=2, T=7, BS=16, bt=P, bts=8, W=8, nb=9, free=P, nf=3, tin=P, tout=P + 4,
             slots=P, pos=P, lens=P, err=None, stream=None)
    a.update(over)
    return _lib.load_lib().fd_build_tables(*a.values())


COMMON = [dict(n=-1), dict(T=-1), dict(mq=-1), dict(H=7), dict(KVH=0), dict(D=0), dict(D=513),
          dict(dt=3), dict(dt=-1), dict(odt=1), dict(scale=float("nan")), dict(scale=float("inf")),
          dict(q=None), dict(k=None), dict(v=None), dict(out=None), dict(lse=None)]


@pytest.mark.parametrize("over", COMMON + [dict(BS=0), dict(W=-1), dict(B=-1), dict(bts=7),
                                           dict(bt=None), dict(cu=None), dict(lens=None)], ids=str)
def test_paged_prefill_refuses(over):
    assert _paged(**over) in (_lib.FD_ERR_INVALID, _lib.FD_ERR_UNSUPPORTED)
    assert b"paged_prefill" in _lib.load_lib().fd_last_error()


@pytest.mark.parametrize("over", COMMON + [dict(Tk=-1), dict(mk=-1), dict(cuq=None),
                                           dict(cuk=None)], ids=str)
def test_varlen_attention_refuses(over):
    assert _varlen(**over) in (_lib.FD_ERR_INVALID, _lib.FD_ERR_UNSUPPORTED)
    assert b"varlen_attention" in _lib.load_lib().fd_last_error()


@pytest.mark.parametrize("over", [dict(n=-1), dict(T=-1), dict(BS=0), dict(W=-1), dict(bts=7),
                                  dict(nb=-1), dict(nf=-1), dict(qsl=None), dict(ctx=None),
                                  dict(bt=None), dict(slots=None), dict(pos=None), dict(lens=None),
                                  dict(free=None), dict(tin=None), dict(tout=None),
                                  dict(tout=P)], ids=str)
def test_build_tables_refuses(over):
    assert _tables(**over) == _lib.FD_ERR_INVALID
    assert b"build_tables" in _lib.load_lib().fd_last_error()


def test_calls_of_no_tokens_launch_nothing():
    assert _paged(n=0) == _lib.FD_OK and _paged(T=0, q=None) == _lib.FD_OK
    assert _varlen(n=0, cuk=None) == _lib.FD_OK and _varlen(T=0) == _lib.FD_OK


@pytest.mark.parametrize("over", [dict(n=-1), dict(T=-1), dict(H=0), dict(KVH=3), dict(D=0),
                                  dict(mq=-1), dict(mk=-1), dict(BS=-1), dict(dt=5)], ids=str)
def test_workspace_size_refuses(over):
    a = dict(n=2, T=7, H=8, KVH=2, D=64, mq=5, mk=20, BS=16, dt=0)
    size = ctypes.c_size_t()
    assert _lib.load_lib().fd_prefill_workspace_size(*a.values(), ctypes.byref(size)) == 0
    a.update(over)
    assert _lib.load_lib().fd_prefill_workspace_size(*a.values(), ctypes.byref(size)) \
        == _lib.FD_ERR_INVALID
    a = dict(n=2, T=7, H=8, KVH=2, D=64, mq=5, mk=20, BS=16, dt=0)
    assert _lib.load_lib().fd_prefill_workspace_size(*a.values(), None) == _lib.FD_ERR_INVALID

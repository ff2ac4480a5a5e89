"""Refusals of the prompt and shared-prefix attention: arguments are checked
before the GPU is touched (no GPU here)."""
import ctypes as C

import pytest

import specdec as S

L = S.lib()
PTR = 4096  # never read: every call here is refused


def prompt(**kw):
    a = dict(q=PTR, ldq=512, kv=PTR, num_blocks=4, Hkv=2, hd=64, tables=PTR, max_blocks=4, ctx=PTR, off=PTR, B=2, T=8,
             Hq=8, out=PTR, ldo=512, ws=PTR, ws_bytes=1 << 40)
    a.update(kw)
    return L.specdec_attention_prompt(a["q"], a["ldq"], a["kv"], a["num_blocks"], a["Hkv"], a["hd"], a["tables"],
                                      a["max_blocks"], a["ctx"], a["off"], a["B"], a["T"], a["Hq"], a["out"], a["ldo"],
                                      a["ws"], a["ws_bytes"], None)


def shared(**kw):
    a = dict(q=PTR, kv=PTR, num_blocks=4, Hkv=2, hd=64, tables=PTR, max_blocks=4, ctx=PTR, mask=PTR, off=PTR, pages=PTR,
             ng=1, B=2, R=3, Hq=8, out=PTR, ws=PTR, ws_bytes=1 << 40)
    a.update(kw)
    return L.specdec_attention_shared_prefix(a["q"], a["kv"], a["num_blocks"], a["Hkv"], a["hd"], a["tables"],
                                             a["max_blocks"], a["ctx"], a["mask"], a["off"], a["pages"], a["ng"],
                                             a["B"], a["R"], a["Hq"], a["out"], a["ws"], a["ws_bytes"], None)


COMMON = [dict(q=None), dict(kv=None), dict(tables=None), dict(ctx=None), dict(out=None), dict(hd=96), dict(hd=256),
          dict(Hkv=3), dict(Hkv=0), dict(Hkv=-2), dict(Hq=0), dict(num_blocks=0), dict(max_blocks=0),
          dict(max_blocks=(1 << 26) + 1), dict(B=-1), dict(B=1025), dict(q=PTR + 2), dict(kv=PTR + 8),
          dict(out=PTR + 4), dict(Hq=2048, Hkv=16)]


@pytest.mark.parametrize("bad", COMMON + [dict(off=None), dict(T=-1), dict(T=(1 << 24) + 1), dict(ldq=504),
                                          dict(ldo=504), dict(ldq=516), dict(ldo=516), dict(Hq=129, Hkv=1, ldq=1 << 14,
                                                                                            ldo=1 << 14)])
def test_prompt_refuses(bad):
    assert prompt(**bad) == S.EINVAL
    assert "attention_prompt" in S.last_error()


@pytest.mark.parametrize("bad", COMMON + [dict(mask=None), dict(off=None), dict(pages=None), dict(R=0), dict(R=65),
                                          dict(ng=-1), dict(ng=3)])
def test_shared_prefix_refuses(bad):
    assert shared(**bad) == S.EINVAL
    assert "attention_shared_prefix" in S.last_error()


def test_empty_calls_do_nothing():
    assert prompt(B=0) == S.OK and prompt(T=0) == S.OK
    assert shared(B=0, ng=0) == S.OK


def test_errors_of_the_binding():
    with pytest.raises(S.SpecdecError):
        S.check(prompt(hd=32))
    assert isinstance(C.c_size_t(L.specdec_attention_prompt_workspace_bytes(0, 0, 0, 0, 0, 0)).value, int)

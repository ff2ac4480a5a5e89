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


def fork(**kw):
    a = dict(tables=PTR, nblk=PTR, lens=PTR, ref=PTR, num_blocks=8, max_reqs=4, max_blocks=3, src=PTR, dst=PTR, n=2,
             kv=PTR, layers=2, stride=8 * 2 * 2 * 16 * 64, Hkv=2, hd=64, status=PTR, ws=PTR, ws_bytes=1 << 30)
    a.update(kw)
    return L.specdec_kv_fork_pages(a["tables"], a["nblk"], a["lens"], a["ref"], a["num_blocks"], a["max_reqs"],
                                   a["max_blocks"], a["src"], a["dst"], a["n"], a["kv"], a["layers"], a["stride"],
                                   a["Hkv"], a["hd"], a["status"], a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("bad", [
    dict(tables=None), dict(nblk=None), dict(lens=None), dict(ref=None), dict(src=None), dict(dst=None),
    dict(status=None), dict(ws=None), dict(kv=None), dict(num_blocks=0), dict(max_reqs=0), dict(max_blocks=0),
    dict(n=-1), dict(n=5), dict(layers=-1), dict(layers=65536), dict(stride=8 * 2 * 2 * 16 * 64 - 8),
    dict(stride=8 * 2 * 2 * 16 * 64 + 4), dict(Hkv=0), dict(hd=0), dict(hd=60), dict(kv=PTR + 8), dict(ws=PTR + 2),
    dict(ws_bytes=100)])
def test_fork_refuses(bad):
    assert fork(**bad) == S.EINVAL
    assert "kv_fork_pages" in S.last_error()


def test_null_handles_are_refused():
    assert L.specdec_kv_fork(None, None, None, 0, None, 0, 0, 0, 0, None) == S.EINVAL
    assert L.specdec_engine_fork(None, 0, None, None, 0, None) == S.EINVAL


@pytest.mark.parametrize("ws", [dict(ws=None), dict(ws_bytes=64), dict(ws=PTR + 4)])
def test_workspaces_are_checked(ws):
    assert prompt(**ws) == S.EINVAL and "workspace" in S.last_error()
    assert shared(**ws) == S.EINVAL and "workspace" in S.last_error()

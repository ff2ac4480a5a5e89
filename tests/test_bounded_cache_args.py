"""Refusals of the operators of a bounded cache: arguments are checked before
the GPU is touched (no GPU here)."""
import pytest

import specdec as S

L = S.lib()
PTR = 4096  # never read: every call here is refused


def attend(adds, **kw):
    a = dict(q=PTR, ldq=512, kv=PTR, num_blocks=4, Hkv=2, hd=64, tables=PTR, max_blocks=4, ctx=PTR, off=PTR, B=2, T=8,
             Hq=8, window=9, sinks=2, weights=PTR, ldw=64, out=PTR, ldo=512, ws=PTR, ws_bytes=1 << 40)
    a.update(kw)
    head = [a[k] for k in ("q", "ldq", "kv", "num_blocks", "Hkv", "hd", "tables", "max_blocks", "ctx", "off", "B", "T", "Hq")]
    tail = [a[k] for k in ("out", "ldo", "ws", "ws_bytes")] + [None]
    if adds:
        return L.specdec_attention_accumulate(*head, a["weights"], a["ldw"], *tail)
    return L.specdec_attention_window(*head, a["window"], a["sinks"], *tail)


COMMON = [dict(q=None), dict(kv=None), dict(tables=None), dict(ctx=None), dict(off=None), dict(out=None), dict(hd=96),
          dict(hd=256), dict(Hkv=3), dict(Hkv=0), dict(Hkv=-2), dict(Hq=0), dict(num_blocks=0), dict(max_blocks=0),
          dict(max_blocks=(1 << 26) + 1), dict(B=-1), dict(B=1025), dict(q=PTR + 2), dict(kv=PTR + 8),
          dict(out=PTR + 4), dict(T=-1), dict(ldq=504), dict(ldo=504), dict(ldq=516), dict(ldo=516),
          dict(Hq=2048, Hkv=16, ldq=1 << 17, ldo=1 << 17), dict(ws=None), dict(ws_bytes=64), dict(ws=PTR + 4)]


@pytest.mark.parametrize("bad", COMMON + [dict(T=(1 << 24) + 1), dict(window=0), dict(window=-5), dict(sinks=-1),
                                          dict(Hq=129, Hkv=1, ldq=1 << 14, ldo=1 << 14)])
def test_window_refuses(bad):
    assert attend(False, **bad) == S.EINVAL
    assert "attention_window" in S.last_error()


@pytest.mark.parametrize("bad", COMMON + [dict(T=65537), dict(weights=None), dict(weights=PTR + 4), dict(ldw=60),
                                          dict(ldw=66), dict(Hq=33, Hkv=1, ldq=1 << 14, ldo=1 << 14)])
def test_accumulate_refuses(bad):
    assert attend(True, **bad) == S.EINVAL
    assert "attention_accumulate" in S.last_error()


def test_accumulate_refuses_its_queries_as_its_output():
    assert attend(True, ws_bytes=1 << 50) == S.EINVAL
    assert "out must not be q" in S.last_error()


def write(**kw):
    a = dict(qkv=PTR, half=0, ld=768, qn=PTR, kn=PTR, eps=1e-5, cos=PTR, sin=PTR, max_pos=9, rot=64, pos=PTR, kv=PTR,
             num_blocks=4, Hkv=2, hd=64, tables=PTR, max_blocks=4, ctx=PTR, off=PTR, B=2, T=8, Hq=8, q=PTR, ldq=512)
    a.update(kw)
    return L.specdec_qk_norm_rope_kv(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(qkv=None), dict(kv=None), dict(tables=None), dict(ctx=None), dict(off=None), dict(q=None), dict(cos=None),
    dict(sin=None), dict(half=2), dict(half=-1), dict(hd=96), dict(hd=32), dict(Hkv=0), dict(Hkv=3), dict(Hq=0),
    dict(Hq=2048, ld=1 << 20, ldq=1 << 20), dict(num_blocks=0), dict(max_blocks=0), dict(max_blocks=(1 << 26) + 1),
    dict(B=-1), dict(B=1025), dict(T=-1), dict(T=(1 << 24) + 1), dict(rot=8), dict(rot=72), dict(rot=-16),
    dict(rot=80), dict(max_pos=0), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(ld=764),
    dict(ld=770), dict(half=1, ld=772), dict(ldq=504), dict(ldq=516), dict(qkv=PTR + 8), dict(q=PTR + 8),
    dict(kv=PTR + 2), dict(qn=PTR + 4), dict(kn=PTR + 4), dict(cos=PTR + 4), dict(sin=PTR + 8)])
def test_write_refuses(bad):
    assert write(**bad) == S.EINVAL
    assert "qk_norm_rope_kv" in S.last_error()


def evict(**kw):
    a = dict(tables=PTR, nblk=PTR, lens=PTR, ref=PTR, num_blocks=8, max_reqs=4, max_blocks=3, reqs=PTR, n=2, keep=20,
             first=4, last=8, weights=PTR, heads=2, ldw=48, kv=PTR, layers=2, stride=8 * 2 * 2 * 16 * 64, Hkv=2, hd=64,
             kept=PTR, status=PTR, ws=PTR, ws_bytes=1 << 30)
    a.update(kw)
    return L.specdec_kv_evict_pages(*a.values(), None)


@pytest.mark.parametrize("bad", [
    dict(tables=None), dict(nblk=None), dict(lens=None), dict(ref=None), dict(reqs=None), dict(weights=None),
    dict(status=None), dict(ws=None), dict(kv=None), dict(num_blocks=0), dict(max_reqs=0), dict(max_blocks=0),
    dict(max_blocks=(1 << 26) + 1), dict(n=-1), dict(n=5), dict(keep=0), dict(keep=-3), dict(first=-1), dict(last=-1),
    dict(first=21), dict(last=21), dict(first=13, last=8), dict(heads=0), dict(heads=1025), dict(ldw=0),
    dict(layers=-1), dict(layers=65536), dict(stride=8 * 2 * 2 * 16 * 64 - 8), dict(stride=8 * 2 * 2 * 16 * 64 + 4),
    dict(Hkv=0), dict(hd=0), dict(hd=60), dict(kv=PTR + 8), dict(ws=PTR + 8), dict(ws_bytes=100)])
def test_evict_refuses(bad):
    assert evict(**bad) == S.EINVAL
    assert "kv_evict_pages" in S.last_error()


def test_null_manager():
    assert L.specdec_kv_evict(None, None, 0, 1, 0, 0, None, 1, 16, None, 0, 0, 0, 0, None, None) == S.EINVAL


def test_empty_calls_do_nothing():
    for w in (False, True):
        assert attend(w, B=0) == S.OK and attend(w, T=0) == S.OK
        none = dict(q=None, kv=None, tables=None, ctx=None, off=None, out=None, ws=None, ws_bytes=0)
        assert attend(w, T=0, **none) == S.OK and attend(w, B=0, **none) == S.OK
    assert write(B=0) == S.OK and write(T=0) == S.OK
    assert write(T=0, qkv=None, kv=None, tables=None, ctx=None, off=None, q=None, cos=None, sin=None) == S.OK


@pytest.mark.parametrize("size", [L.specdec_attention_window_workspace_bytes, L.specdec_attention_accumulate_workspace_bytes])
def test_workspaces_of_larger_calls_do_for_smaller_ones(size):
    most = size(64, 300, 32, 8, 128, 600)
    for B in (1, 7, 64):
        for T in (1, 5, 64, 65, 300):
            for wide in (1, 16, 17, 300, 600):
                assert size(B, T, 32, 8, 128, wide) <= most, (B, T, wide)
    assert size(0, 1, 8, 2, 64, 4) == 0 and size(1, 0, 8, 2, 64, 4) == 0
    assert size(-1, -1, -1, -1, -1, -1) == 0


def test_evict_workspace():
    size = L.specdec_kv_evict_pages_workspace_bytes
    assert size(64, 8, 20, 4, 100) > 0 and size(64, 8, 20, 3, 100) <= size(64, 8, 20, 4, 100)
    assert size(0, 8, 20, 4, 100) == 0 and size(64, 8, 20, -1, 100) == 0 and size(64, 8, 20, 4, 0) == 0
    # a keep that no table reaches takes no more than the table does
    assert size(64, 8, 20, 4, 1 << 30) == size(64, 8, 20, 4, 320)

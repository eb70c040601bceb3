"""Host-side refusals of the step tables, the 8-bit pool and draft verification (no GPU: every call returns before any
device work; the pointers are never dereferenced)."""
import pytest

import msgl

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 7
P = 256  # an address that is never used


def tables(**k):
    a = dict(kept=P, new=2 * P, pt=P, mp=4, held=P, free=P, cap=8, top=P, B=2, T=4, page=16, sl=3 * P, ip=P, pos=P, slots=P, last=P)
    a.update(k)
    return msgl.lib().msgl_step_tables(*a.values(), None)


@pytest.mark.parametrize("bad,rc", [
    (dict(B=-1), INVALID), (dict(T=-1), INVALID), (dict(mp=0), INVALID), (dict(page=0), INVALID), (dict(cap=-1), INVALID),
    (dict(T=(1 << 20) + 1), UNSUPPORTED), (dict(mp=1 << 30, B=3), UNSUPPORTED), (dict(mp=1 << 28), UNSUPPORTED), (dict(kept=None), INVALID), (dict(new=None), INVALID),
    (dict(pt=None), INVALID), (dict(held=None), INVALID), (dict(free=None), INVALID), (dict(top=None), INVALID),
    (dict(sl=None), INVALID), (dict(ip=None), INVALID), (dict(pos=None), INVALID), (dict(slots=None), INVALID),
    (dict(last=None), INVALID), (dict(sl=P), INVALID), (dict(sl=2 * P), INVALID)])
def test_tables(bad, rc):
    assert tables(**bad) == rc and msgl.lib().msgl_last_error()


def test_tables_empty():
    assert tables(B=0) == 0 and tables(B=0, kept=None) == 0


def store(parts=None, **k):
    a = dict(x=P, q=P, kv=P, sc=P, pages=8, pos=P, pt=P, mp=4, sl=P, ip=None, B=4, mq=1, tab=P, maxp=64, qn=P, kn=P, T=4,
             hq=8, hkv=2, d=128, page=16)
    a.update(k)
    L = msgl.lib()
    if parts is None:
        return L.msgl_qknorm_rope_store_kv8(*a.values(), 1e-6, None)
    v = list(a.values())
    return L.msgl_qknorm_rope_store_kv8_partials(v[0], parts, *v[1:], 1e-6, None)


@pytest.mark.parametrize("parts", [None, 3])
@pytest.mark.parametrize("bad,rc", [
    (dict(d=64), UNSUPPORTED), (dict(page=32), UNSUPPORTED), (dict(T=-1), INVALID), (dict(B=-1), INVALID), (dict(hq=0), INVALID),
    (dict(hkv=0), INVALID), (dict(pages=0), INVALID), (dict(mp=0), INVALID), (dict(mp=1 << 28), INVALID), (dict(maxp=0), INVALID), (dict(mq=2), INVALID),
    (dict(B=3), INVALID), (dict(x=None), INVALID), (dict(q=None), INVALID), (dict(kv=None), INVALID), (dict(sc=None), INVALID),
    (dict(pos=None), INVALID), (dict(pt=None), INVALID), (dict(sl=None), INVALID), (dict(tab=None), INVALID),
    (dict(qn=None), INVALID), (dict(kn=P + 8), INVALID), (dict(x=P + 8), INVALID), (dict(q=P + 4), INVALID),
    (dict(kv=P + 8), INVALID), (dict(tab=P + 4), INVALID), (dict(ip=P, B=65535, mq=1 << 20, T=1 << 20, hkv=64), UNSUPPORTED)])
def test_store(parts, bad, rc):
    assert store(parts, **bad) == rc and msgl.lib().msgl_last_error()


def test_store_empty_and_parts():
    assert store(T=0, B=0) == 0 and store(ip=P, mq=0) == 0 and store(ip=P, T=0) == 0
    assert store(0) == INVALID and store(65) == INVALID and store(2, x=None) == INVALID


def attend(**k):
    a = dict(q=P, kv=P, sc=P, pages=8, pt=P, mp=64, sl=P, ip=None, B=2, T=2, mq=1, L=1000, hq=8, hkv=2, d=128, page=16)
    b = dict(out=P, ws=P, n=1 << 30)
    a.update({x: y for x, y in k.items() if x in a})
    b.update({x: y for x, y in k.items() if x in b})
    return msgl.lib().msgl_paged_attention_kv8(*a.values(), 0.1, *b.values(), None)


@pytest.mark.parametrize("bad,rc", [
    (dict(d=64), UNSUPPORTED), (dict(page=32), UNSUPPORTED), (dict(hq=6), UNSUPPORTED), (dict(hq=7), INVALID),
    (dict(hq=32), UNSUPPORTED), (dict(hkv=0), INVALID), (dict(B=-1), INVALID), (dict(T=-1), INVALID), (dict(mq=-1), INVALID),
    (dict(L=-1), INVALID), (dict(L=1025), INVALID), (dict(pages=0), INVALID), (dict(mp=0), INVALID), (dict(mq=2), INVALID),
    (dict(T=3), INVALID), (dict(ip=P, B=65536), UNSUPPORTED), (dict(q=None), INVALID), (dict(kv=None), INVALID),
    (dict(sc=None), INVALID), (dict(sc=P + 1), INVALID), (dict(pt=None), INVALID), (dict(sl=None), INVALID), (dict(out=None), INVALID), (dict(q=P + 8), INVALID),
    (dict(kv=P + 8), INVALID), (dict(out=P + 2), INVALID), (dict(ws=None), WORKSPACE), (dict(ws=P + 8), WORKSPACE),
    (dict(n=100), WORKSPACE)])
def test_attend(bad, rc):
    assert attend(**bad) == rc and msgl.lib().msgl_last_error()


def test_attend_empty_and_workspace():
    size = msgl.lib().msgl_paged_attention_kv8_workspace_size
    assert attend(B=0, T=0) == 0 and attend(ip=P, T=0) == 0 and attend(ip=P, mq=0) == 0
    assert size(0, 8, 2) == 0 and size(1, 0, 2) == 0 and size(1, 7, 2) == 0
    for hq, hkv in ((8, 1), (8, 8), (16, 8), (32, 4)):
        for n in (1, 2, 3, 5, 8, 9, 16, 17, 33, 64, 100, 129, 4096):
            most = size(n, hq, hkv)
            assert all(size(m, hq, hkv) <= most for m in (1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 64, 65, 100, 4000) if m <= n), (hq, n)


def probs(**k):
    a = dict(x=P, ldx=64, n=2, V=64, t=P, p=2 * P, ldp=64)
    a.update(k)
    return msgl.lib().msgl_token_probs(*a.values(), None)


@pytest.mark.parametrize("bad,rc", [
    (dict(n=-1), INVALID), (dict(V=0), INVALID), (dict(ldx=63), INVALID), (dict(ldp=60), INVALID), (dict(x=None), INVALID),
    (dict(p=None), INVALID), (dict(V=327681, ldx=400000, ldp=400000), UNSUPPORTED), (dict(p=P, ldp=68), INVALID),
    (dict(n=1 << 28), UNSUPPORTED)])
def test_probs(bad, rc):
    assert probs(**bad) == rc and msgl.lib().msgl_last_error()


def test_probs_empty():
    assert probs(n=0) == 0 and probs(n=0, x=None) == 0


def verify(**k):
    a = dict(p=P, ldp=64, q=P, ldq=64, tok=P, ip=P, u=P, last=P, B=2, n=3, most=4, V=64, acc=P, out=P)
    a.update(k)
    return msgl.lib().msgl_verify_drafts(*a.values(), None)


@pytest.mark.parametrize("bad,rc", [
    (dict(B=-1), INVALID), (dict(n=-1), INVALID), (dict(most=-1), INVALID), (dict(V=0), INVALID), (dict(ldp=63), INVALID),
    (dict(ldq=63), INVALID), (dict(p=None), INVALID), (dict(tok=None), INVALID), (dict(ip=None), INVALID), (dict(u=None), INVALID),
    (dict(last=None), INVALID), (dict(acc=None), INVALID), (dict(out=None), INVALID), (dict(B=1 << 28), UNSUPPORTED),
    (dict(most=(1 << 20) + 1), UNSUPPORTED)])
def test_verify(bad, rc):
    assert verify(**bad) == rc and msgl.lib().msgl_last_error()


def test_verify_empty():
    assert verify(B=0) == 0 and verify(B=0, q=None, ldq=0) == 0

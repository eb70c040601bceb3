"""Host-side refusals of the adapter, three-axis rotary and page-sparse entry points (no GPU: every
call returns before any device work; the pointers are never dereferenced)."""
import ctypes as C

import pytest

import msgl

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 7
P = 256  # an address that is never used
SEC = (C.c_int * 3)(24, 20, 20)


def mrope(**k):
    a = dict(qkv=P, q=P, kp=P, vp=P, slots=64, pos=P, stride=4, sec=SEC, layout=1, map=P, tab=P, maxp=64,
             qn=P, kn=P, T=4, hq=8, hkv=2, d=128)
    a.update(k)
    return msgl.lib().msgl_qknorm_mrope_store_kv(
        a["qkv"], a["q"], a["kp"], a["vp"], a["slots"], a["pos"], a["stride"], a["sec"], a["layout"], a["map"],
        a["tab"], a["maxp"], a["qn"], a["kn"], a["T"], a["hq"], a["hkv"], a["d"], 1e-6, None)


@pytest.mark.parametrize("bad,rc", [
    (dict(d=64), UNSUPPORTED), (dict(T=-1), INVALID), (dict(hq=0), INVALID), (dict(hkv=0), INVALID),
    (dict(maxp=0), INVALID), (dict(stride=3), INVALID), (dict(sec=None), INVALID), (dict(layout=2), INVALID),
    (dict(sec=(C.c_int * 3)(24, 20, 21)), INVALID), (dict(sec=(C.c_int * 3)(-1, 45, 20)), INVALID),
    (dict(sec=(C.c_int * 3)(20, 22, 22)), INVALID), (dict(qkv=None), INVALID), (dict(pos=None), INVALID),
    (dict(q=P + 8), INVALID), (dict(kp=P + 2), INVALID), (dict(qn=P + 4), INVALID), (dict(map=None), INVALID)])
def test_mrope(bad, rc):
    assert mrope(**bad) == rc and msgl.lib().msgl_last_error()


def test_mrope_partials_and_empty():
    f = msgl.lib().msgl_qknorm_mrope_store_kv_partials
    tail = (P, P, P, 64, P, 4, SEC, 1, P, P, 64, P, P, 4, 8, 2, 128, 1e-6, None)
    assert f(None, 1, *tail) == INVALID and f(P, 0, *tail) == INVALID and f(P, 65, *tail) == INVALID
    assert mrope(T=0) == 0 and mrope(T=0, qkv=None) == 0


def bounds(**k):
    a = dict(k=P, slots=64, pt=P, mp=4, sl=P, ip=None, B=2, mq=1, hkv=2, d=128, page=16, b=P)
    a.update(k)
    return msgl.lib().msgl_kv_page_bounds(a["k"], a["slots"], a["pt"], a["mp"], a["sl"], a["ip"], a["B"], a["mq"],
                                          a["hkv"], a["d"], a["page"], a["b"], None)


@pytest.mark.parametrize("bad,rc", [
    (dict(d=64), UNSUPPORTED), (dict(page=8), UNSUPPORTED), (dict(hkv=0), INVALID), (dict(slots=0), INVALID),
    (dict(slots=63), INVALID), (dict(mp=0), INVALID), (dict(mq=2), INVALID), (dict(mq=-1), INVALID),
    (dict(B=-1), INVALID), (dict(k=None), INVALID), (dict(b=P + 8), INVALID), (dict(sl=None), INVALID),
    (dict(mp=1 << 28), INVALID)])
def test_bounds(bad, rc):
    assert bounds(**bad) == rc and msgl.lib().msgl_last_error()


def test_bounds_empty():
    assert bounds(B=0) == 0 and bounds(ip=P, mq=0) == 0


def select(**k):
    a = dict(q=P, b=P, pages=64, pt=P, mp=64, sl=P, ip=None, B=2, T=2, mq=1, L=1000, hq=8, hkv=2, d=128, page=16,
             top=8, sink=1, recent=1, ids=P, ws=P, n=1 << 30)
    a.update(k)
    return msgl.lib().msgl_select_pages(a["q"], a["b"], a["pages"], a["pt"], a["mp"], a["sl"], a["ip"], a["B"],
                                        a["T"], a["mq"], a["L"], a["hq"], a["hkv"], a["d"], a["page"], a["top"],
                                        a["sink"], a["recent"], a["ids"], a["ws"], a["n"], None)


@pytest.mark.parametrize("bad,rc", [
    (dict(d=64), UNSUPPORTED), (dict(page=32), UNSUPPORTED), (dict(hq=6, hkv=4), INVALID),
    (dict(hq=6, hkv=2), UNSUPPORTED), (dict(hq=32, hkv=2), UNSUPPORTED), (dict(top=0), INVALID),
    (dict(recent=0), INVALID), (dict(sink=-1), INVALID), (dict(sink=5, recent=4), INVALID),
    (dict(sink=2 ** 31 - 1, recent=2 ** 31 - 1), INVALID), (dict(top=1025), UNSUPPORTED),
    (dict(L=1025), INVALID), (dict(L=524289, mp=1 << 20), UNSUPPORTED), (dict(L=-1), INVALID),
    (dict(T=3), INVALID), (dict(mq=2), INVALID), (dict(pages=0), INVALID), (dict(q=None), INVALID),
    (dict(b=P + 8), INVALID), (dict(ids=None), INVALID), (dict(ws=None), WORKSPACE), (dict(ws=P + 4), WORKSPACE),
    (dict(n=100), WORKSPACE)])
def test_select(bad, rc):
    assert select(**bad) == rc and msgl.lib().msgl_last_error()


def test_select_empty_and_workspace():
    L = msgl.lib()
    assert select(B=0, T=0) == 0 and select(ip=P, T=0) == 0 and select(ip=P, mq=0) == 0
    assert L.msgl_select_pages_workspace_size(0, 1000, 8) == 0
    assert L.msgl_select_pages_workspace_size(1, 524289, 8) == 0
    # 16 bytes for each of 64 rows x 8 heads x 2048 pages
    assert L.msgl_select_pages_workspace_size(64, 32768, 8) == 16 * 64 * 8 * 2048
    # bounded for long batches
    assert L.msgl_select_pages_workspace_size(100000, 32768, 8) == 256 * 2 ** 20


def test_select_workspace_serves_smaller_calls():
    size = msgl.lib().msgl_select_pages_workspace_size
    rows, contexts, heads = (1, 15, 16, 17, 300, 4096, 100000), (1, 300, 32768, 50000, 131072, 131088, 200000, 524288), (1, 3, 8, 64)
    for T in rows:
        for L in contexts:
            for h in heads:
                n = size(T, L, h)
                assert all(size(t, l, g) <= n for t in rows if t <= T for l in contexts if l <= L for g in heads if g <= h), (T, L, h)
                # 16 bytes per row of a pass, head and page of the context; 16 rows a pass or more
                pages = max(16, -(-L // 256) * 16)
                assert n >= 16 * min(T, max(16, 2 ** 28 // (16 * pages * h))) * h * pages


def attend(**k):
    a = dict(q=P, k=P, v=P, slots=64, pt=P, mp=64, sl=P, ip=None, B=2, T=2, mq=1, L=1000, ids=P, top=8, hq=8, hkv=2,
             d=128, page=16, out=P)
    a.update(k)
    return msgl.lib().msgl_paged_attention_pages(a["q"], a["k"], a["v"], a["slots"], a["pt"], a["mp"], a["sl"],
                                                 a["ip"], a["B"], a["T"], a["mq"], a["L"], a["ids"], a["top"],
                                                 a["hq"], a["hkv"], a["d"], a["page"], 0.1, a["out"], None)


@pytest.mark.parametrize("bad,rc", [
    (dict(d=64), UNSUPPORTED), (dict(page=32), UNSUPPORTED), (dict(hq=6, hkv=2), UNSUPPORTED),
    (dict(hq=7, hkv=2), INVALID), (dict(top=0), INVALID), (dict(top=1025), UNSUPPORTED), (dict(L=1025), INVALID),
    (dict(L=524289, mp=1 << 20), UNSUPPORTED), (dict(slots=65), INVALID), (dict(T=1), INVALID),
    (dict(mq=0, ip=None), INVALID), (dict(v=None), INVALID), (dict(out=P + 8), INVALID), (dict(ids=None), INVALID)])
def test_attend(bad, rc):
    assert attend(**bad) == rc and msgl.lib().msgl_last_error()


def test_attend_empty():
    assert attend(B=0, T=0) == 0 and attend(ip=P, T=0) == 0 and attend(ip=P, mq=0) == 0


def lora(partial=False, **k):
    a = dict(x=P, ldx=64, a=P, b=P, sc=P, n=2, ids=P, ip=None, B=4, mq=1, y=P, ldy=128, out=P, ldo=128, T=4, N=128,
             K=64, R=16, ws=P, bytes=1 << 30)
    a.update(k)
    head = (a["x"], a["ldx"], a["a"], a["b"], a["sc"], a["n"], a["ids"], a["ip"], a["B"], a["mq"])
    tail = (a["out"], a["ldo"], a["T"], a["N"], a["K"], a["R"], a["ws"], a["bytes"], None)
    L = msgl.lib()
    return L.msgl_lora_partial(*head, *tail) if partial else L.msgl_lora_add(*head, a["y"], a["ldy"], *tail)


@pytest.mark.parametrize("partial", [False, True])
@pytest.mark.parametrize("bad,rc", [
    (dict(K=60, ldx=64), UNSUPPORTED), (dict(N=124), UNSUPPORTED), (dict(R=12), UNSUPPORTED),
    (dict(R=136), UNSUPPORTED), (dict(K=0), INVALID), (dict(R=0), INVALID), (dict(n=-1), INVALID),
    (dict(ldx=56), INVALID), (dict(ldx=65), INVALID), (dict(ldo=120), INVALID), (dict(ldo=130), INVALID),
    (dict(B=3), INVALID), (dict(mq=2), INVALID), (dict(x=None), INVALID), (dict(ids=None), INVALID),
    (dict(a=None), INVALID), (dict(sc=None), INVALID), (dict(out=None), INVALID), (dict(b=P + 8), INVALID),
    (dict(out=P + 4), INVALID), (dict(ws=None), WORKSPACE), (dict(ws=P + 8), WORKSPACE), (dict(bytes=64), WORKSPACE)])
def test_lora(partial, bad, rc):
    assert lora(partial, **bad) == rc and msgl.lib().msgl_last_error()


def test_lora_y_and_empty():
    assert lora(ldo=136) == INVALID  # in place with another stride
    assert lora(y=None, out=P) == INVALID and lora(ldy=120) == INVALID and lora(ldy=129) == INVALID and lora(y=P + 2) == INVALID
    for partial in (False, True):
        assert lora(partial, T=0, B=0) == 0 and lora(partial, ip=P, mq=0) == 0 and lora(partial, ip=P, B=0) == 0
    assert msgl.lib().msgl_lora_workspace_size(0, 64, 16) == 0
    assert msgl.lib().msgl_lora_workspace_size(4, 64, 24) == 4 * 32 * 6  # three bf16 terms, ranks padded to 32

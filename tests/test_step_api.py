"""CPU tests of the entry points around the serving attention (no launches):
the C ABI's refusals and workspaces."""
import ctypes

import pytest
import torch

import htree_amd
from htree_amd import _native as N
from tests.test_cache_api import BAD_CACHES, cache

at = lambda x: ctypes.c_void_p(x << 20)  # never read: the calls are refused or empty
FAKE = at(1)


def size(f, *args):
    n = ctypes.c_int64(-1)
    return getattr(N.lib(), f)(*args, n), n.value


def verify(dtype=0, B=2, rows=6, V=100, p=at(1), p_row=100, q=None, q_row=0, tokens=at(2), starts=at(3), parents=None,
           u=at(4), d=at(5), kept=at(6), path=at(7), nxt=at(8), ws=None, n=0):
    return N.lib().htree_verify_drafts(dtype, B, rows, V, p, p_row, q, q_row, tokens, starts, parents, u, d, kept, path,
                                       nxt, ws, n, None)


def test_verify_refusals():
    assert verify(dtype=3) == N.HTREE_ESHAPE
    assert verify(B=-1) == N.HTREE_ESHAPE
    assert verify(rows=-1) == N.HTREE_ESHAPE
    assert verify(V=0) == N.HTREE_ESHAPE
    assert verify(p_row=-1) == N.HTREE_ESHAPE
    assert verify(B=4097) == N.HTREE_EUNSUPPORTED
    for name in ("p", "tokens", "starts", "u", "d", "kept", "path", "nxt"):
        assert verify(**{name: None}) == N.HTREE_ENULL, name
    for name in ("kept", "path", "nxt"):
        for x in range(1, 6):
            assert verify(**{name: at(x)}) == N.HTREE_EOVERLAP, (name, x)
        assert verify(q=at(20), q_row=100, **{name: at(20)}) == N.HTREE_EOVERLAP
        assert verify(parents=at(20), **{name: at(20)}) == N.HTREE_EOVERLAP
    assert verify(kept=at(7)) == N.HTREE_EOVERLAP and verify(path=at(8)) == N.HTREE_EOVERLAP
    assert verify(B=0, p=None) == N.HTREE_OK
    # few requests over a large vocabulary need a workspace
    need = lambda B, V, drawn, greedy=0, rows=6, dtype=0: \
        size("htree_verify_drafts_workspace_bytes", dtype, B, rows, V, drawn, greedy)
    assert need(2, 100, 1) == (N.HTREE_OK, 0) and need(129, 1 << 20, 1) == (N.HTREE_OK, 0)
    rc, n = need(2, 1 << 17, 0)
    assert rc == N.HTREE_OK and 0 < n < 4096 and need(2, 1 << 16, 1) == (N.HTREE_OK, n)
    big = dict(V=1 << 17, p=at(4000), p_row=1 << 17, n=n)
    assert verify(**big) == N.HTREE_ENULL
    assert verify(**dict(big, n=n - 1), ws=at(9)) == N.HTREE_EWORKSPACE
    assert verify(**big, ws=ctypes.c_void_p((9 << 20) + 8)) == N.HTREE_EUNSUPPORTED
    for x in (2, 3, 4, 5, 6, 7, 8, 4000):
        assert verify(**big, ws=at(x)) == N.HTREE_EOVERLAP
    assert need(4, 0, 0)[0] == N.HTREE_ESHAPE and need(-1, 5, 0)[0] == N.HTREE_ESHAPE
    assert need(4, 5, 0, rows=-1)[0] == N.HTREE_ESHAPE and need(4, 5, 0, dtype=3)[0] == N.HTREE_ESHAPE
    assert need(4097, 5, 0)[0] == N.HTREE_EUNSUPPORTED
    assert N.lib().htree_verify_drafts_workspace_bytes(0, 1, 1, 1, 0, 0, None) == N.HTREE_ENULL
    # greedily: no numbers at all, nor a drafter's probabilities
    greedy = dict(u=None, d=None)
    assert need(2, 100, 0, 1) == (N.HTREE_OK, 24) and need(2, 1 << 20, 0, 1, rows=65) == (N.HTREE_OK, 0)
    assert need(2, 1 << 20, 0, 1, rows=128, dtype=1) == (N.HTREE_OK, 512)
    assert need(2, 8, 0, 1, rows=1 << 21) == (N.HTREE_OK, 0)  # more blocks than a grid holds, at once
    assert verify(**greedy, q=at(20), q_row=100) == N.HTREE_ESHAPE and need(2, 100, 1, 1)[0] == N.HTREE_ESHAPE
    assert verify(**greedy, p=None, ws=at(9), n=24) == N.HTREE_ENULL
    assert verify(**greedy) == N.HTREE_ENULL and verify(**greedy, ws=at(9), n=23) == N.HTREE_EWORKSPACE
    assert verify(**greedy, ws=at(9), n=24, kept=at(2)) == N.HTREE_EOVERLAP
    assert verify(**greedy, ws=at(1), n=24) == N.HTREE_EOVERLAP


def pointers(n, first=4096):
    return (ctypes.c_void_p * n)(*(first + 65536 * i for i in range(n)))


def keep(c=None, layers=2, k=pointers(2), v=pointers(2, 1 << 20), B=2, rows=4, slots=FAKE, starts=FAKE, path=FAKE,
         kept=FAKE):
    return N.lib().htree_keep_drafts(c or cache(), layers, k, v, B, rows, slots, starts, path, kept, None)


def copy(c=None, layers=2, k=pointers(2), v=pointers(2, 1 << 20), n=2, frm=FAKE, to=FAKE, tokens=None):
    return N.lib().htree_copy_pages(c or cache(), layers, k, v, n, frm, to, tokens, None)


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_caches_are_refused(kw, code):
    assert keep(cache(**kw)) == code
    assert copy(cache(**kw)) == code


def test_moving_refusals():
    for f in (keep, copy):
        assert f(layers=-1) == N.HTREE_ESHAPE
        assert f(layers=65536) == N.HTREE_EUNSUPPORTED
        assert f(k=None) == N.HTREE_ENULL and f(v=None) == N.HTREE_ENULL
        assert f(k=pointers(2, 4104)) == N.HTREE_EUNSUPPORTED
        assert f(v=(ctypes.c_void_p * 2)(4096, None)) == N.HTREE_ENULL
        assert f(cache(H_kv=1 << 20)) == N.HTREE_EUNSUPPORTED  # more pieces of a token than blocks
        assert f(layers=0, k=None) == N.HTREE_OK
    assert keep(B=-1) == N.HTREE_ESHAPE and keep(rows=-1) == N.HTREE_ESHAPE
    assert keep(B=4097) == N.HTREE_EUNSUPPORTED
    for name in ("slots", "starts", "path", "kept"):
        assert keep(**{name: None}) == N.HTREE_ENULL
    assert keep(B=0, slots=None) == N.HTREE_OK and keep(rows=0, slots=None) == N.HTREE_OK
    assert copy(n=-1) == N.HTREE_ESHAPE
    assert copy(n=1 << 24) == N.HTREE_EUNSUPPORTED  # more blocks than a grid holds
    assert copy(frm=None) == N.HTREE_ENULL and copy(to=None) == N.HTREE_ENULL
    assert copy(n=0, frm=None) == N.HTREE_OK


def fork(B=2, n=3, page=16, pages=9, width=4, stride=4, ostride=4, n_free=5, table=at(1), lens=at(2), source=at(3),
         free=at(4), out=at(5), olens=at(6), frm=at(7), to=at(8), count=at(9), used=at(10)):
    return N.lib().htree_fork_requests(B, n, page, pages, width, stride, ostride, n_free, table, lens, source, free, out,
                                       olens, frm, to, count, used, None)


def test_fork_refusals():
    for kw in (dict(B=-1), dict(n=-1), dict(pages=-1), dict(width=-1), dict(n_free=-1), dict(stride=3), dict(ostride=3)):
        assert fork(**kw) == N.HTREE_ESHAPE, kw
    for kw in (dict(page=0), dict(page=24), dict(B=4097), dict(n=4097)):
        assert fork(**kw) == N.HTREE_EUNSUPPORTED, kw
    for name in ("table", "lens", "source", "free", "out", "olens", "frm", "to", "count", "used"):
        assert fork(**{name: None}) == N.HTREE_ENULL, name
    for name in ("out", "olens", "frm", "to", "count", "used"):
        for x in range(1, 11):
            if fork.__defaults__[list(fork.__code__.co_varnames).index(name)].value != x << 20:
                assert fork(**{name: at(x)}) == N.HTREE_EOVERLAP, (name, x)
    assert fork(n=0, source=None) == N.HTREE_OK


def unused(B=2, page=16, pages=9, width=4, stride=4, table=at(1), lens=at(2), n_held=3, held=at(3), out=at(4),
           count=at(5), ws=at(6), n=1 << 19):
    return N.lib().htree_unused_pages(B, page, pages, width, stride, table, lens, n_held, held, out, count, ws, n, None)


def test_unused_refusals():
    for kw in (dict(B=-1), dict(pages=-1), dict(width=-1), dict(n_held=-1), dict(stride=3)):
        assert unused(**kw) == N.HTREE_ESHAPE, kw
    for kw in (dict(page=0), dict(page=24), dict(B=4097), dict(ws=ctypes.c_void_p((6 << 20) + 4))):
        assert unused(**kw) == N.HTREE_EUNSUPPORTED, kw
    for name in ("table", "lens", "held", "out", "count"):
        assert unused(**{name: None}) == N.HTREE_ENULL, name
    # small calls need no workspace
    need = lambda *a: size("htree_unused_pages_workspace_bytes", *a)
    assert need(64, 1 << 18, 1024, 4096) == (N.HTREE_OK, 0)
    for many in ((64, (1 << 18) + 1, 1024, 0), (65, 100, 1024, 0), (257, 100, 1, 0), (257, 100, 0, 0), (1, 100, 1, 4097)):
        rc, n = need(*many)
        assert rc == N.HTREE_OK and n > 0
        big = dict(B=many[0], pages=many[1], width=many[2], stride=many[2], n_held=many[3], out=at(400), count=at(500))
        assert unused(ws=at(600), n=n - 1, **big) == N.HTREE_EWORKSPACE
        assert unused(ws=None, n=n, **big) == N.HTREE_ENULL
        assert unused(ws=at(2), n=n, **big) == N.HTREE_EOVERLAP and unused(ws=at(500), n=n, **big) == N.HTREE_EOVERLAP
    for name in ("out", "count"):
        for x in (1, 2, 3):
            assert unused(**{name: at(x)}) == N.HTREE_EOVERLAP
    assert unused(out=at(5)) == N.HTREE_EOVERLAP
    assert unused(pages=0, table=None) == N.HTREE_OK
    assert need(1, -1, 1, 1)[0] == N.HTREE_ESHAPE
    assert need(1, 2 ** 31 - 1, 1, 1)[1] > 2 ** 31
    assert N.lib().htree_unused_pages_workspace_bytes(1, 1, 1, 1, None) == N.HTREE_ENULL


def norm(dtype=1, w=0, rows=4, H=8, Hkv=2, D=64, eps=1e-6, q=FAKE, qr=512, k=FAKE, pos=None, cos=None, sin=None, rope=0,
         qo=FAKE, ko=FAKE):
    return N.lib().htree_head_norm(dtype, w, rows, H, Hkv, D, eps, q, qr, 64, k, 128, 64, None, None, pos, cos, sin, rope,
                                   qo, ko, None)


def norm_bwd(dtype=1, w=0, rows=4, H=8, Hkv=2, D=64, eps=1e-6, q=FAKE, qr=512, k=FAKE, pos=None, cos=None, sin=None,
             rope=0, qo=FAKE, ko=FAKE, dy=FAKE, dw=FAKE, ws=FAKE, n=1 << 30):
    return N.lib().htree_head_norm_backward(dtype, w, rows, H, Hkv, D, eps, q, qr, 64, k, 128, 64, dy, 512, 64, dy, 128,
                                            64, None, None, pos, cos, sin, rope, qo, ko, dw, dw, ws, n, None)


@pytest.mark.parametrize("f", [norm, norm_bwd])
def test_norm_refusals(f):
    for kw in (dict(dtype=3), dict(w=2), dict(rows=-1), dict(H=-1), dict(Hkv=-1), dict(D=0), dict(eps=-1.0),
               dict(eps=float("nan")), dict(pos=FAKE, cos=FAKE, sin=FAKE, rope=0)):
        assert f(**kw) == N.HTREE_ESHAPE, kw
    for kw in (dict(D=264), dict(D=60), dict(dtype=0, D=2), dict(qr=510), dict(q=ctypes.c_void_p(4100)), dict(qr=-64),
               dict(qo=ctypes.c_void_p(4100)), dict(rows=2 ** 31 - 1)):
        assert f(**kw) == N.HTREE_EUNSUPPORTED, kw
    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(cos=FAKE), dict(pos=FAKE),
               dict(cos=FAKE, sin=FAKE, rope=9)):
        assert f(**kw) == N.HTREE_ENULL, kw
    assert f(rows=0, q=None) == N.HTREE_OK
    assert f(H=0, Hkv=0, q=None) == N.HTREE_OK


def test_norm_backward_refusals():
    assert norm(dtype=0, rows=1 << 22, H=32, D=256, qr=8192) == N.HTREE_EUNSUPPORTED  # more threads than a grid holds
    assert norm_bwd(dy=None) == N.HTREE_ENULL
    assert norm_bwd(ws=None) == N.HTREE_ENULL
    need = size("htree_head_norm_backward_workspace_bytes", 64)[1]
    assert norm_bwd(n=need - 1) == N.HTREE_EWORKSPACE
    assert size("htree_head_norm_backward_workspace_bytes", 0)[0] == N.HTREE_ESHAPE


def test_python_needs_the_gpu():
    f = lambda *n, t=torch.int32: torch.zeros(n, dtype=t)
    kc, vc = torch.zeros(2, 16, 1, 32), torch.zeros(2, 16, 1, 32)
    x = torch.zeros(3, 2, 64)
    for call in (lambda: htree_amd.verify_drafts(torch.zeros(2, 5), f(2, t=torch.int64), f(2), torch.zeros(2), torch.zeros(1)),
                 lambda: htree_amd.keep_drafts(kc, vc, f(2, t=torch.int64), f(2), f(2), f(1)),
                 lambda: htree_amd.copy_pages(kc, vc, f(2), f(2)),
                 lambda: htree_amd.fork_requests(f(1, 2), f(1), f(2), f(2), 16, 2),
                 lambda: htree_amd.unused_pages(f(1, 2), f(1), 16, 2), lambda: htree_amd.head_norm(x, x)):
        with pytest.raises(AssertionError, match="GPU"):
            call()

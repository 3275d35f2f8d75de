"""CPU tests of the paged cache's entry points (no launches): the C ABI's
refusals, its workspace, and the Python arguments' checks."""
import ctypes

import pytest
import torch

import htree_amd
from htree_amd import _native as N

FAKE = ctypes.c_void_p(4096)  # never read: the calls are refused or empty


def cache(**kw):
    d = dict(dtype=1, H_kv=2, Dk=128, Dv=128, page_size=16, num_pages=8, k_page=16 * 256, k_token=256,
             k_head=128, v_page=16 * 256, v_token=256, v_head=128)
    d.update(kw)
    return N.HtreeCache(*[d[n] for n, _ in N.HtreeCache._fields_])


def ws_bytes(c, B=4, rows=4, H=32, width=100):
    n = ctypes.c_int64()
    return N.lib().htree_draft_attention_workspace_bytes(c, B, rows, H, width, n), n.value


BAD_CACHES = [
    (dict(dtype=3), N.HTREE_ESHAPE), (dict(dtype=-1), N.HTREE_ESHAPE),
    (dict(H_kv=0), N.HTREE_ESHAPE), (dict(num_pages=0), N.HTREE_ESHAPE), (dict(Dk=0), N.HTREE_ESHAPE),
    (dict(page_size=8), N.HTREE_EUNSUPPORTED), (dict(page_size=48), N.HTREE_EUNSUPPORTED),
    (dict(page_size=8192), N.HTREE_EUNSUPPORTED),
    (dict(Dk=264), N.HTREE_EUNSUPPORTED), (dict(Dv=264), N.HTREE_EUNSUPPORTED),
    (dict(Dk=60), N.HTREE_EUNSUPPORTED), (dict(dtype=0, Dv=42), N.HTREE_EUNSUPPORTED),
    (dict(k_token=250), N.HTREE_EUNSUPPORTED), (dict(k_token=1 << 26), N.HTREE_EUNSUPPORTED), (dict(v_page=-256), N.HTREE_EUNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_bad_caches_are_refused(kw, code):
    c = cache(**kw)
    assert ws_bytes(c)[0] == code
    L = N.lib()
    assert L.htree_draft_attention(c, 4, 4, 32, 100, 100, 1.0, FAKE, 4096, 128, FAKE, FAKE, FAKE, FAKE, FAKE, None,
                                   FAKE, 4096, 128, FAKE, 1 << 40, None) == code
    assert L.htree_cache_append(c, 4, 0, FAKE, 256, 128, FAKE, 256, 128, None, 0, 0, FAKE, None, None, None, 0,
                                None, FAKE, FAKE, None) == code


def attention(c=None, B=4, rows=4, H=32, width=100, stride=100, q=FAKE, row=4096, head=128, kc=FAKE, table=FAKE,
              out=FAKE, ws=FAKE, ws_n=1 << 40):
    c = c or cache()
    return N.lib().htree_draft_attention(c, B, rows, H, width, stride, 1.0, q, row, head, kc, FAKE, table, FAKE,
                                         FAKE, None, out, 4096, 128, ws, ws_n, None)


def test_attention_refusals():
    assert attention(H=31) == N.HTREE_ESHAPE            # not a multiple of H_kv
    assert attention(B=-1) == N.HTREE_ESHAPE
    assert attention(stride=99) == N.HTREE_ESHAPE
    assert attention(width=(1 << 26) + 1, stride=1 << 27) == N.HTREE_EUNSUPPORTED  # 2^30 tokens
    assert attention(q=None) == N.HTREE_ENULL
    assert attention(kc=None) == N.HTREE_ENULL
    assert attention(table=None) == N.HTREE_ENULL
    assert attention(out=ctypes.c_void_p(4100)) == N.HTREE_EUNSUPPORTED
    assert attention(row=4097) == N.HTREE_EUNSUPPORTED
    assert attention(ws=None) == N.HTREE_ENULL
    assert attention(ws_n=ws_bytes(cache())[1] - 1) == N.HTREE_EWORKSPACE
    assert attention(rows=2 ** 31 - 1, H=2048) == N.HTREE_EUNSUPPORTED  # more blocks than a grid holds
    # nothing to do: no launch
    assert attention(rows=0, q=None) == N.HTREE_OK
    assert attention(B=0, q=None) == N.HTREE_OK


def test_attention_workspace():
    # short tables are not split and need none; it does not grow with the rows
    assert ws_bytes(cache(), width=64) == (N.HTREE_OK, 0)
    one = ws_bytes(cache(), width=65)[1]
    assert one > 0
    assert ws_bytes(cache(), B=4000, rows=4000, width=8192)[1] == one
    assert ws_bytes(cache(), B=1, rows=100000, width=8192)[1] == ws_bytes(cache(), B=1, rows=64, width=8192)[1]
    for d in (32, 64, 128, 256):
        assert ws_bytes(cache(Dk=d, Dv=d), B=1, rows=1000, width=8192)[1] <= 160 << 20
    assert N.lib().htree_draft_attention_workspace_bytes(cache(), 1, 1, 32, 1, None) == N.HTREE_ENULL


def tables(B=4, rows=4, page=16, pages=8, width=10, stride=10, n_free=3, ctx=FAKE, slots=FAKE, free=FAKE):
    return N.lib().htree_page_tables(B, rows, page, pages, width, stride, n_free, ctx, FAKE, None, FAKE, free,
                                     FAKE, slots, FAKE, FAKE, FAKE, None)


def test_page_tables_refusals():
    assert tables(B=-1) == N.HTREE_ESHAPE
    assert tables(rows=-1) == N.HTREE_ESHAPE
    assert tables(pages=-1) == N.HTREE_ESHAPE
    assert tables(stride=9) == N.HTREE_ESHAPE
    assert tables(B=0, rows=4) == N.HTREE_ESHAPE
    assert tables(page=0) == N.HTREE_EUNSUPPORTED
    assert tables(page=24) == N.HTREE_EUNSUPPORTED
    assert tables(B=4097) == N.HTREE_EUNSUPPORTED
    assert tables(ctx=None) == N.HTREE_ENULL
    assert tables(slots=None) == N.HTREE_ENULL
    assert tables(free=None) == N.HTREE_ENULL
    assert tables(B=0, rows=0, ctx=None) == N.HTREE_OK


def append(c=None, rows=4, H=0, k=FAKE, k_row=256, q=None, slots=FAKE, pos=None, cos=None, sin=None, rope=0, qo=None):
    return N.lib().htree_cache_append(c or cache(), rows, H, k, k_row, 128, FAKE, 256, 128, q, 4096, 128, slots, pos,
                                      cos, sin, rope, qo, FAKE, FAKE, None)


def test_append_refusals():
    assert append(rows=-1) == N.HTREE_ESHAPE
    assert append(k=None) == N.HTREE_ENULL
    assert append(slots=None) == N.HTREE_ENULL
    assert append(k=ctypes.c_void_p(4098)) == N.HTREE_EUNSUPPORTED
    assert append(k_row=257) == N.HTREE_EUNSUPPORTED
    assert append(cos=FAKE, sin=FAKE, rope=10) == N.HTREE_ENULL          # no positions
    assert append(cos=FAKE, pos=FAKE, rope=10) == N.HTREE_ENULL          # no sin
    assert append(cos=FAKE, sin=FAKE, pos=FAKE, rope=0) == N.HTREE_ESHAPE
    assert append(q=FAKE, H=32, qo=FAKE) == N.HTREE_ENULL                # queries are rotated
    assert append(q=FAKE, H=32, cos=FAKE, sin=FAKE, pos=FAKE, rope=10) == N.HTREE_ENULL  # no q_out
    assert append(q=FAKE, H=0, qo=FAKE, cos=FAKE, sin=FAKE, pos=FAKE, rope=10) == N.HTREE_ESHAPE
    assert append(rows=0, k=None) == N.HTREE_OK


def test_python_needs_the_gpu():
    i32 = lambda *n: torch.zeros(n, dtype=torch.int32)
    kc = torch.zeros(2, 16, 1, 32)
    with pytest.raises(AssertionError, match="GPU"):
        htree_amd.page_tables(i32(1), i32(1), i32(1, 2), i32(2), 16, 2, 1)
    with pytest.raises(AssertionError, match="GPU"):
        htree_amd.cache_append(torch.zeros(1, 1, 32), torch.zeros(1, 1, 32), kc, kc, torch.zeros(1, dtype=torch.int64))
    with pytest.raises(AssertionError, match="GPU"):
        htree_amd.draft_attention(torch.zeros(1, 2, 32), kc, kc, i32(1, 2), i32(1), i32(2))

"""CPU tests of the paged cache's boundary: exported symbols, and every refused call (the checks run on the host, before
anything is enqueued, so they need no GPU)."""
import ctypes as C
import math
import os
import re

import pytest

import cactus_amd.hip as H
import cactus_amd.paged as P

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20      # an aligned address that nobody reads


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(ROOT, "include", "cactus_hip_paged.h")).read()
    names = sorted(set(re.findall(r"\b(cactus_hip_\w+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S))))
    assert names == sorted(P.PAGED_SIGNATURES)
    for n in names:
        assert hasattr(H.lib, n)


def cache(**kw):
    d = dict(k=A, v=A, k_scales=A, v_scales=A, num_pages=10, page_size=16, kv_heads=2, head_dim=64)
    d.update(kw)
    return P._PagedKv(*[d[n] for n, _ in P._PagedKv._fields_])


def append(c=None, **kw):
    d = dict(tables=A, width=4, positions=A, cu=None, batch=3, tokens=3, k=A, ks=128, v=A, vs=128, q=A, qs=256, out=A,
             heads=4, qw=None, kw=None, eps=1e-6, theta=1e4, stream=None)
    d.update(kw)
    return H.lib.cactus_hip_kv_append_paged_f16_dev(C.byref(c or cache()), *d.values())


def read(c=None, **kw):
    d = dict(tables=A, width=4, starts=A, cu=A, batch=3, rows=5, k=A, v=A, stream=None)
    d.update(kw)
    return H.lib.cactus_hip_kv_read_paged_f16_dev(C.byref(c or cache()), *d.values())


def attend(c=None, **kw):
    d = dict(tables=A, width=4, contexts=A, cu=None, batch=3, tokens=3, max_context=64, q=A, qs=256, out=A, heads=4, scale=0.0,
             window=0, sink=0, work=A, bytes=1 << 30, stream=None)
    d.update(kw)
    return H.lib.cactus_hip_attention_paged_f16_dev(C.byref(c or cache()), *d.values())


def ragged(**kw):
    d = dict(q=A, qs=256, k=A, ks=128, v=A, vs=128, out=A, cu=A, batch=3, tokens=7, heads=4, kv_heads=2, dim=64, scale=0.0,
             window=0, sink=0, stream=None)
    d.update(kw)
    return H.lib.cactus_hip_attention_ragged_f16_dev(*d.values())


def refused(rc, words):
    text = H.lib.cactus_hip_last_error().decode()
    H.lib.cactus_hip_clear_error()
    return rc == -1 and words in text


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("bad,words", [(dict(k=None), "null cache"), (dict(v_scales=None), "null cache"),
                                       (dict(head_dim=80), "head_dim"), (dict(head_dim=0), "head_dim"),
                                       (dict(page_size=8), "page_size"), (dict(page_size=48), "page_size"),
                                       (dict(page_size=256), "page_size"), (dict(kv_heads=0), "kv_heads"),
                                       (dict(num_pages=0), "pages"), (dict(num_pages=1 << 31), "pages"),
                                       (dict(k=A + 8), "aligned"), (dict(v=A + 1), "aligned")])
def test_refuses_a_bad_cache(call, bad, words):
    assert refused(call(cache(**bad)), words)


@pytest.mark.parametrize("call", [append, read, attend])
@pytest.mark.parametrize("bad,words", [(dict(tables=None), "block table"), (dict(width=0), "block table"),
                                       (dict(width=1 << 31), "pages"), (dict(batch=(1 << 20) + 1), "sequences")])
def test_refuses_a_bad_batch(call, bad, words):
    assert refused(call(cu=A, **bad), words)


@pytest.mark.parametrize("call", [append, attend])
@pytest.mark.parametrize("bad,words", [(dict(tokens=4), "one row per sequence"), (dict(tokens=(1 << 26) + 1, cu=A), "rows"),
                                       (dict(q=A + 2), "aligned"), (dict(qs=252), "multiple of 8"), (dict(qs=248), "stride below"),
                                       (dict(heads=5), "multiple of the kv heads"), (dict(heads=0), "multiple of the kv heads"),
                                       (dict(heads=1 << 14, qs=1 << 20), "4096"), (dict(out=None), "null rows"),
                                       (dict(out=A + 4), "aligned")])
def test_refuses_bad_query_rows(call, bad, words):
    assert refused(call(**bad), words)


@pytest.mark.parametrize("bad,words", [(dict(positions=None), "positions"), (dict(k=None), "null rows"), (dict(v=None), "null rows"),
                                       (dict(ks=120), "stride below"), (dict(ks=1 << 24), "2^24"), (dict(vs=127), "multiple of 8"), (dict(kw=A + 2), "norm"),
                                       (dict(qw=A + 8), "norm"), (dict(theta=-1.0), "theta"), (dict(theta=math.inf), "theta"),
                                       (dict(theta=math.nan), "theta"), (dict(eps=-1e-6), "eps"), (dict(eps=math.nan), "eps")])
def test_append_refuses(bad, words):
    assert refused(append(**bad), words)


@pytest.mark.parametrize("bad,words", [(dict(cu=None), "cu_seqlens"), (dict(starts=None), "starts"), (dict(k=None), "aligned"),
                                       (dict(v=A + 8), "aligned"), (dict(rows=(1 << 26) + 1), "rows")])
def test_read_refuses(bad, words):
    assert refused(read(**bad), words)


@pytest.mark.parametrize("bad,words", [(dict(contexts=None), "context_lens"), (dict(q=None), "null rows"),
                                       (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
                                       (dict(window=1 << 31), "window"), (dict(sink=1 << 31), "window")])
def test_attention_refuses(bad, words):
    assert refused(attend(**bad), words)


@pytest.mark.parametrize("bad,words", [(dict(dim=96), "head_dim"), (dict(cu=None), "cu_seqlens"), (dict(heads=3), "multiple"),
                                       (dict(kv_heads=0), "multiple"), (dict(k=A + 6), "aligned"), (dict(ks=136 - 4), "multiple of 8"),
                                       (dict(vs=64), "stride below"), (dict(vs=1 << 30), "2^24"), (dict(out=None), "null rows"), (dict(scale=-math.inf), "scale"),
                                       (dict(window=1 << 40), "window"), (dict(batch=1 << 21), "sequences")])
def test_ragged_refuses(bad, words):
    assert refused(ragged(**bad), words)


def test_empty_calls_do_nothing():
    for call in (append, read, attend):
        assert call(batch=0, tokens=0) == 0 if call is not read else call(batch=0, rows=0) == 0
    assert ragged(tokens=0) == 0


def test_refuses_more_rows_than_a_launch_holds():
    many = 1 << 26
    assert refused(attend(cache(kv_heads=2), cu=A, tokens=many, heads=4096, qs=4096 * 64), "too many rows")
    assert refused(attend(cache(kv_heads=4096, head_dim=64), batch=1 << 20, tokens=1 << 20, heads=4096, qs=4096 * 64), "too many rows")
    assert refused(ragged(tokens=many, heads=4096, qs=4096 * 64), "too many rows")
    assert refused(ragged(tokens=many, heads=64, qs=4096, kv_heads=64, ks=4096, vs=4096), "too many rows")
    assert refused(read(cache(kv_heads=64), rows=many), "too many rows")


def test_python_names_what_is_wrong():
    torch = pytest.importorskip("torch")
    kv = P.empty_pages(4, 2, 64, 16, device="cpu")
    with pytest.raises(ValueError, match="on a GPU"):
        P.kv_read(kv, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                  torch.zeros(2, dtype=torch.int32), 1)
    q = torch.zeros((1, 2, 64), dtype=torch.float16)
    with pytest.raises(ValueError, match="on a GPU"):
        P.attention_ragged(q, q, q, torch.zeros(2, dtype=torch.int32))

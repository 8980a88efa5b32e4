"""What the operators for several continuations of a sequence refuse before any CUDA call, and the sizes they ask for: no GPU."""
import ctypes as C

import pytest

from blackwell_b200 import _lib

INVALID = 1


class Cache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p), ("v_scale", C.c_void_p), ("kv_heads", C.c_int),
                ("max_seq", C.c_int), ("batch_elems", C.c_size_t), ("layer_elems", C.c_size_t)]


P = 4096   # an aligned address that is never followed: every call below is refused


def cache(**kw):
    return Cache(**{**dict(k=P, v=P, k_scale=None, v_scale=None, kv_heads=8, max_seq=64, batch_elems=8 * 64 * 128, layer_elems=0), **kw})


BAD_CACHES = [dict(k=None), dict(v=None), dict(k_scale=P), dict(v_scale=P), dict(kv_heads=0), dict(max_seq=0), dict(batch_elems=8 * 64 * 128 + 8),
              dict(layer_elems=64), dict(k=P + 8), dict(v=P + 4), dict(k_scale=P, v_scale=P + 2)]


@pytest.fixture(scope="module")
def lib():
    lib = _lib.load()
    for n in ("bw_attention_tree_scratch_bytes", "bw_beam_select_scratch_bytes"):
        getattr(lib, n).restype = C.c_size_t
    return lib


def write(lib, c=None, **kw):
    a = {**dict(q=P, qkv=P, qw=P, kw=P, first=P, nq=32, M=2, T=3, eps=1e-6, base=1e6), **kw}
    return lib.bw_qk_norm_rope_kv_rows(C.c_void_p(a["q"]), C.byref(c or cache()), C.c_void_p(a["qkv"]), C.c_void_p(a["qw"]), C.c_void_p(a["kw"]),
                                       C.c_void_p(a["first"]), None, None, a["nq"], a["M"], a["T"], C.c_float(a["eps"]), C.c_float(a["base"]), 0, None)


def attend(lib, c=None, **kw):
    a = {**dict(out=P, q=P, first=P, mask=P, hint=0, nq=32, M=2, T=3, scratch=P, n=1 << 30), **kw}
    return lib.bw_attention_tree(C.c_void_p(a["out"]), C.c_void_p(a["q"]), C.byref(c or cache()), C.c_void_p(a["first"]), C.c_void_p(a["mask"]), None,
                                 a["hint"], a["nq"], a["M"], a["T"], 0, C.c_void_p(a["scratch"]), C.c_size_t(a["n"]), None)


def select(lib, **kw):
    a = {**dict(parent=P, token=P, out=2 * P, logits=P, stride=100, vocab=100, score=P, ended=P, eos=2, beams=4, keep=4, M=2, scratch=P, n=1 << 30), **kw}
    return lib.bw_beam_select(C.c_void_p(a["parent"]), C.c_void_p(a["token"]), C.c_void_p(a["out"]), None, C.c_void_p(a["logits"]), C.c_long(a["stride"]),
                              a["vocab"], C.c_void_p(a["score"]), C.c_void_p(a["ended"]), a["eos"], a["beams"], a["keep"], a["M"], C.c_void_p(a["scratch"]),
                              C.c_size_t(a["n"]), None)


def reorder(lib, c=None, **kw):
    a = {**dict(parent=P, to=P, beams=2, M=2, layers=2, stride=8 * 64 * 128), **kw}
    return lib.bw_kv_reorder(C.byref(c or cache(batch_elems=2 * 8 * 64 * 128)), C.c_void_p(a["parent"]), None, C.c_void_p(a["to"]), a["beams"], a["M"],
                             a["layers"], C.c_size_t(a["stride"]), None)


def keep(lib, c=None, **kw):
    a = {**dict(first=P, path=P, count=P, M=2, T=8, layers=2, stride=8 * 64 * 128), **kw}
    return lib.bw_kv_keep_rows(C.byref(c or cache(batch_elems=2 * 8 * 64 * 128)), C.c_void_p(a["first"]), C.c_void_p(a["path"]), C.c_void_p(a["count"]),
                               a["M"], a["T"], a["layers"], C.c_size_t(a["stride"]), None)


@pytest.mark.parametrize("bad", BAD_CACHES, ids=str)
@pytest.mark.parametrize("call", [write, attend, reorder, keep])
def test_bad_caches(lib, call, bad):
    assert call(lib, cache(**bad)) == INVALID


@pytest.mark.parametrize("call, bad", [
    (write, dict(q=None)), (write, dict(qkv=None)), (write, dict(first=None)), (write, dict(nq=0)), (write, dict(M=0)), (write, dict(T=0)),
    (write, dict(base=0.0)), (write, dict(eps=-1.0)), (write, dict(q=P + 4)), (write, dict(qkv=P + 8)), (write, dict(qw=P + 4)), (write, dict(base=float("nan"))),
    (attend, dict(out=None)), (attend, dict(q=None)), (attend, dict(first=None)), (attend, dict(nq=12)), (attend, dict(nq=0)), (attend, dict(M=0)),
    (attend, dict(M=65536)), (attend, dict(T=0)), (attend, dict(T=65)), (attend, dict(hint=-1)), (attend, dict(out=P + 8)), (attend, dict(mask=P + 4)),
    (attend, dict(scratch=P + 8)),
    (select, dict(parent=None)), (select, dict(token=None)), (select, dict(out=None)), (select, dict(logits=None)), (select, dict(score=None)),
    (select, dict(vocab=0)), (select, dict(stride=99)), (select, dict(eos=100)), (select, dict(eos=-1)), (select, dict(beams=0)), (select, dict(beams=65)),
    (select, dict(keep=0)), (select, dict(keep=65)), (select, dict(M=0)), (select, dict(scratch=None)), (select, dict(scratch=P + 4)), (select, dict(n=8)),
    (select, dict(beams=64, vocab=1 << 30, stride=1 << 30)), (select, dict(beams=1, keep=1, vocab=(1 << 31) - 2, stride=1 << 31)),
    (select, dict(out=P, score=P, keep=3)),
    (reorder, dict(parent=None)), (reorder, dict(to=None)), (reorder, dict(beams=0)), (reorder, dict(beams=33)), (reorder, dict(M=0)), (reorder, dict(layers=0)),
    (reorder, dict(stride=8 * 64 * 128 - 128)), (reorder, dict(stride=8 * 64 * 128 + 64)), (reorder, dict(M=70000)),
    (keep, dict(first=None)), (keep, dict(path=None)), (keep, dict(count=None)), (keep, dict(M=0)), (keep, dict(T=0)), (keep, dict(T=65)), (keep, dict(layers=0)),
    (keep, dict(stride=128)),
], ids=lambda v: getattr(v, "__name__", str(v)))
def test_refusals(lib, call, bad):
    assert call(lib, **bad) == INVALID


@pytest.mark.parametrize("call", [write, reorder, keep])
def test_sequences_that_are_written_do_not_overlap(lib, call):
    assert call(lib, cache(batch_elems=8 * 64 * 128 - 128)) == INVALID
    assert call(lib, cache(batch_elems=0)) == INVALID


@pytest.mark.parametrize("call", [reorder, keep])
def test_layers_and_sequences_that_share_rows(lib, call):
    plane = 8 * 64 * 128
    for batch, stride in ((plane, plane), (2 * plane, 3 * plane), (3 * plane - 128, 2 * plane)):
        assert call(lib, cache(batch_elems=batch), layers=2, stride=stride, M=4) == INVALID
    assert call(lib, layers=1 << 28) == INVALID


def test_no_cache_at_all(lib):
    assert lib.bw_attention_tree(C.c_void_p(P), C.c_void_p(P), None, C.c_void_p(P), None, None, 0, 32, 1, 1, 0, None, C.c_size_t(0), None) == INVALID


def test_a_split_context_wants_its_scratch(lib):
    long = cache(max_seq=100000, batch_elems=8 * 100000 * 128)
    assert attend(lib, long, M=1, T=1, scratch=None, n=0) == INVALID
    assert attend(lib, long, M=1, T=1, n=64) == INVALID


def test_scratch_sizes(lib):
    a, b = lib.bw_attention_tree_scratch_bytes, lib.bw_beam_select_scratch_bytes
    assert a(1, 65, 32, 8, 100) == a(0, 1, 32, 8, 100) == a(1, 1, 12, 8, 100) == b(0, 4, 4, 1) == b(100, 65, 4, 1) == 0
    assert 0 < a(1, 1, 32, 8, 64) <= a(64, 64, 64, 8, 1 << 20)
    assert 0 < b(100, 1, 1, 1) < b(151643, 8, 8, 16) < 1 << 28

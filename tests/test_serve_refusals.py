"""Refusals of the paged serving step's entry points: every bad argument is
turned down before any work is enqueued, so these run without a GPU."""
import ctypes as C

import numpy as np
import pytest

import serve_rule as SR
from inferox_b200 import _lib, synth
from inferox_b200._lib import lib

P = C.c_void_p(0x10000)  # never dereferenced: the calls below are refused
Q = C.c_void_p(0x20000)
ODD = C.c_void_p(0x10008)


def name(code):
    return _lib.STATUS[code]


def test_page_bytes():
    assert lib.ifx_kv4_page_bytes(8, 128) == 8 * 4 * 576 * 4
    assert lib.ifx_kv4_page_bytes(1, 32) == 4 * 576
    # 4.5 bits a value
    assert lib.ifx_kv4_page_bytes(3, 96) * 8 == 64 * 2 * 3 * 96 * 4.5
    for g, d in ((0, 128), (8, 0), (8, 48), (8, 288), (2000, 128)):
        assert lib.ifx_kv4_page_bytes(g, d) == 0


def store(ty=0, k=P, ks=1024, v=P, vs=1024, slots=P, n=4, pages=P, np_=4, g=8, d=128):
    return name(lib.ifx_op_kv4_store(ty, k, ks, v, vs, slots, n, pages, np_, g, d, None))


@pytest.mark.parametrize("kw,want", [
    (dict(ty=2), "Unsupported"), (dict(d=48), "Unsupported"), (dict(d=512), "Unsupported"), (dict(d=0), "Unsupported"),
    (dict(g=0), "Shape"), (dict(ks=1023), "Shape"), (dict(vs=8), "Shape"),
    (dict(k=None), "InvalidArgument"), (dict(slots=None), "InvalidArgument"), (dict(pages=None), "InvalidArgument"),
    (dict(k=ODD), "InvalidArgument"), (dict(pages=ODD), "InvalidArgument"), (dict(ks=1025), "InvalidArgument"),
    (dict(ty=1, ks=1028), "InvalidArgument"), (dict(np_=1 << 26), "InvalidArgument"), (dict(n=1 << 31), "InvalidArgument"),
    (dict(n=0, k=None), "Ok"),
])
def test_store(kw, want):
    assert store(**kw) == want


def load(ty=0, pages=P, np_=4, g=8, d=128, slots=P, n=4, k=P, v=P):
    return name(lib.ifx_op_kv4_load(ty, pages, np_, g, d, slots, n, k, v, None))


@pytest.mark.parametrize("kw,want", [
    (dict(ty=7), "Unsupported"), (dict(d=100), "Unsupported"), (dict(g=0), "Shape"), (dict(k=None), "InvalidArgument"),
    (dict(v=ODD), "InvalidArgument"), (dict(n=0), "Ok"),
])
def test_load(kw, want):
    assert load(**kw) == want


def attn(ty=0, q=P, qs=4096, rows=2, pages=P, np_=4, table=P, mp=4, kl=P, qstart=None, n=2, h=32, g=8, d=128, scale=0.1,
         window=0, out=Q, os=4096, ws=P, wsb=1 << 40):
    return name(lib.ifx_op_kv4_attention(ty, q, qs, rows, pages, np_, table, mp, kl, qstart, n, h, g, d, scale, window,
                                         out, os, 0, ws, wsb, None))


@pytest.mark.parametrize("kw,want", [
    (dict(ty=14), "Unsupported"), (dict(d=80), "Unsupported"), (dict(h=31), "Shape"), (dict(h=0), "Shape"),
    (dict(rows=3), "Shape"), (dict(qs=4095), "Shape"), (dict(os=4), "Shape"),
    (dict(q=None), "InvalidArgument"), (dict(out=None), "InvalidArgument"), (dict(kl=None), "InvalidArgument"),
    (dict(table=None), "InvalidArgument"), (dict(pages=None), "InvalidArgument"), (dict(q=ODD), "InvalidArgument"),
    (dict(qs=4097), "InvalidArgument"), (dict(scale=float("nan")), "InvalidArgument"),
    (dict(scale=float("inf")), "InvalidArgument"), (dict(n=9000, rows=9000), "InvalidArgument"),
    (dict(rows=0, n=0), "Ok"), (dict(rows=0, qstart=P), "Ok"),
])
def test_attention(kw, want):
    assert attn(**kw) == want


def extend(lens=P, add=P, n=4, table=P, mp=8, free=P, np_=9, n_free=P, mt=8, lo=Q, nfo=Q, qs=P, slots=P, st=P):
    return name(lib.ifx_op_pages_extend(lens, add, n, table, mp, free, np_, n_free, mt, lo, nfo, qs, slots, None, None,
                                        st, None))


@pytest.mark.parametrize("kw", [
    dict(lens=None), dict(add=None), dict(table=None), dict(free=None), dict(n_free=None), dict(lo=None), dict(nfo=None),
    dict(qs=None), dict(slots=None), dict(st=None), dict(lo=P), dict(nfo=P), dict(n=8193), dict(mp=1 << 26),
    dict(np_=1 << 26), dict(mt=1 << 31),
])
def test_extend(kw):
    assert extend(**kw) == "InvalidArgument"


@pytest.mark.parametrize("at", [0, 1, 3, 5, 7, 8, 9])
def test_release(at):
    a = [P, P, 4, P, 8, P, 9, P, Q, Q, None]
    a[at] = None
    assert name(lib.ifx_op_pages_release(*a)) == "InvalidArgument"
    a = [P, P, 4, P, 8, P, 9, P, P, Q, None]
    assert name(lib.ifx_op_pages_release(*a)) == "InvalidArgument"  # lens_out is lens


def rows(z=P, stride=100, r=2, n=100, u=P, tok=P):
    return name(lib.ifx_op_sample_rows(z, stride, r, n, u, None, None, None, None, tok, None, None))


@pytest.mark.parametrize("kw,want", [
    (dict(n=0), "Shape"), (dict(stride=99), "Shape"), (dict(z=None), "InvalidArgument"), (dict(u=None), "InvalidArgument"),
    (dict(tok=None), "InvalidArgument"), (dict(n=(1 << 24) + 1, stride=1 << 25), "InvalidArgument"),
    (dict(r=1 << 31), "InvalidArgument"), (dict(r=0), "Ok"),
])
def test_sample_rows(kw, want):
    assert rows(**kw) == want


def test_workspace_refuses():
    for h, g, d in ((32, 0, 128), (31, 8, 128), (32, 8, 48), (1 << 17, 8, 128)):
        assert lib.ifx_kv4_attention_workspace(h, g, d) == 0


def test_rule_is_the_weights_q4_0():
    """The restated rule gives the very blocks the library's Q4_0 quantiser writes."""
    x = synth.normal(3, 1, 0.7, 32 * 400).reshape(400, 32)
    x[7] = 0
    x[8] *= 1e-7  # scales in f16's subnormals
    raw = np.frombuffer(synth.quantize(2, x.reshape(-1)), np.uint8).reshape(400, 18)
    q, d = SR.quantise(x)
    assert np.array_equal(raw[:, :2].copy().view(np.float16)[:, 0].view(np.uint16), d[:, 0].view(np.uint16))
    assert np.array_equal(raw[:, 2:] & 15, q[:, 0, :16]) and np.array_equal(raw[:, 2:] >> 4, q[:, 0, 16:])


def test_rule_layout_round_trip():
    rng = np.random.default_rng(0)
    pages = rng.integers(0, 256, (2, lib.ifx_kv4_page_bytes(2, 96))).astype(np.uint8)
    k, v = rng.standard_normal((2, 2, 96)), rng.standard_normal((2, 2, 96))
    (kq, kd), (vq, vd) = SR.quantise(k), SR.quantise(v)
    before = pages.copy()
    for i, slot in enumerate((83, 82)):
        SR.put(pages, slot, kq[i], kd[i], vq[i], vd[i])
    # two rows of two heads: 4.5 bits of 2 * 96 values each, nothing else
    assert 0 < (pages != before).sum() <= 2 * 2 * 2 * 96 * 4.5 / 8
    assert not (pages[0] != before[0]).any()

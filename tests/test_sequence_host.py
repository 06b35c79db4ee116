"""Operators for token sequences, what needs no GPU: refusals of the C ABI and of the Python surface, the oracle's own gradients, modules."""
import ctypes as C
import os
import re

import pytest
import torch

import sequence_oracle as orc
from conftest import ROOT

import dl_templates_b200 as swa
from dl_templates_b200 import _lib

LIB = _lib.lib
BF = torch.bfloat16


def test_library_exports_every_declared_symbol():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "swa_sequence.h")).read(), flags=re.S)
    assert set(re.findall(r"\b(\w+)\s*\(", text)) == set(_lib.SEQUENCE_EXPORTS)
    for n in _lib.SEQUENCE_EXPORTS:
        assert hasattr(LIB, n), n


def geom(**kw):
    d = dict(dtype=_lib.SWA_BF16, B=2, Hq=4, Hkv=2, N=100, d_qk=64, d_v=64, window=16, n_sink=4, sm_scale=0.125, impl=0, lens=None)
    d.update(kw)
    return _lib.SinkGeom(*d.values())


def tensor4(ptr=1 << 20, st=(1 << 16, 1 << 12, 64, 1)):
    t = _lib.Tensor4()
    t.ptr = ptr
    for i in range(4):
        t.stride[i] = st[i]
    return t


@pytest.mark.parametrize("kw, msg", [
    (dict(dtype=7), "dtype"), (dict(B=0), "positive"), (dict(Hq=5), "multiple"), (dict(N=0), "tokens"), (dict(N=(1 << 30) + 1), "tokens"),
    (dict(d_qk=0), "head dims"), (dict(d_v=257), "head dims"), (dict(window=0), "window"), (dict(window=-3), "window"),
    (dict(n_sink=-1), "n_sink"), (dict(n_sink=1025), "n_sink"), (dict(impl=3), "impl"), (dict(B=70000), "65535")])
def test_sink_geometry_is_refused(kw, msg):
    g = geom(**kw)
    assert LIB.sink_swa_select(C.byref(g)) < 0 and msg in LIB.swa_last_error().decode()
    assert LIB.sink_swa_bwd_scratch(C.byref(g)) < 0
    t = tensor4()
    assert LIB.sink_swa_fwd(C.byref(g), *(C.byref(t),) * 4, 1 << 20, None, None) < 0 and msg in LIB.swa_last_error().decode()


def test_sink_entries_refuse_missing_tensors_and_small_scratch():
    g, t, none = geom(), tensor4(), _lib.Tensor4()
    r = C.byref
    assert LIB.sink_swa_fwd(None, r(t), r(t), r(t), r(t), 1 << 20, None, None) < 0
    assert LIB.sink_swa_fwd(r(g), r(t), r(none), r(t), r(t), 1 << 20, None, None) < 0 and b"k is NULL" in LIB.swa_last_error()
    assert LIB.sink_swa_fwd(r(g), r(t), r(t), r(t), r(t), None, None, None) < 0 and b"lse" in LIB.swa_last_error()
    need = LIB.sink_swa_bwd_scratch(r(g))
    assert need >= 4 * 2 * 4 * 100
    assert LIB.sink_swa_bwd(r(g), *(r(t),) * 5, 1 << 20, r(t), r(t), r(t), None, need, None, None) < 0
    for scratch, n in ((1 << 20, need - 1), ((1 << 20) + 4, need)):
        assert LIB.sink_swa_bwd(r(g), *(r(t),) * 5, 1 << 20, r(t), r(t), r(t), scratch, n, None, None) < 0
        assert b"scratch" in LIB.swa_last_error()


@pytest.mark.parametrize("dtype", [0, 2])
def test_scratch_stays_small(dtype):
    """Partial sums of the blocks with sinks: below 200 MB beside the softmax delta for any window, sinks and length."""
    for B, Hq, Hkv in ((1, 1, 1), (1, 16, 4), (8, 64, 8), (64, 32, 32), (3, 8, 1)):
        for N in (1, 100, 1 << 14, 1 << 17, 1 << 20):
            for W in (1, 128, 5000):
                for ns in (0, 1, 4, 130, 1024):
                    g = geom(dtype=dtype, B=B, Hq=Hq, Hkv=Hkv, N=N, window=W, n_sink=ns, d_qk=128, d_v=128)
                    extra = LIB.sink_swa_bwd_scratch(C.byref(g)) - 4 * B * Hq * N
                    assert 0 <= extra < 200 << 20, (B, Hq, Hkv, N, W, ns, extra)
                    assert ns or extra < 256


def test_rope_axes_are_refused():
    t = tensor4()
    ok = dict(pos=1 << 20, stride=(0, 100), n_axes=2, pairs=(8, 8, 0, 0), rows=(10, 10, 0, 0), cs=(1 << 20, 1 << 20, 0, 0))

    def call(B=1, N=100, Cc=64, H=2, dtype=2, **kw):
        d = {**ok, **kw}
        r = _lib.RopeAxes(d["pos"], d["stride"], d["n_axes"], d["pairs"], d["rows"], d["cs"])
        return LIB.rope_axes_apply(dtype, C.byref(r), B, N, Cc, C.byref(t), C.byref(t), H, None, None, 0, 0, None)
    for kw in (dict(n_axes=0), dict(n_axes=5), dict(pairs=(8, 0, 0, 0)), dict(rows=(0, 10, 0, 0)), dict(cs=(1 << 20, 0, 0, 0)),
               dict(pairs=(30, 8, 0, 0)), dict(pos=None), dict(B=0), dict(N=0), dict(Cc=0), dict(H=0), dict(dtype=9), dict(N=1 << 40),
               dict(pairs=(2 ** 31 - 1, 2 ** 31 - 1, 0, 0))):
        assert call(**kw) < 0, kw


def test_cache_entries_are_refused():
    t, none = tensor4(), _lib.Tensor4()

    def cache(**kw):
        d = dict(k=t, v=t, page_table=1 << 20, seq_lens=1 << 20, n_pages=8, page_size=16, max_pages=4)
        d.update(kw)
        return _lib.SinkCache(*d.values())

    def decode(c, Hq=4, Hkv=2, dqk=64, dv=64, W=8, ns=0, impl=0, dtype=2):
        return LIB.sink_swa_decode(dtype, 1, Hq, Hkv, dqk, dv, W, ns, 1.0, impl, C.byref(t), C.byref(c), C.byref(t), None)

    def append(c, q=t, q_out=t, T=1, d=64):
        return LIB.kv_append_rope(2, None, 1, 4, 2, T, d, d, q and C.byref(q), q_out and C.byref(q_out), C.byref(t), C.byref(t), C.byref(c), None, None)
    for kw in (dict(k=none), dict(v=none), dict(page_table=None), dict(seq_lens=None), dict(n_pages=0), dict(page_size=0), dict(max_pages=0),
               dict(max_pages=1 << 20, page_size=1 << 20)):
        assert decode(cache(**kw)) < 0 and append(cache(**kw)) < 0, kw
    c = cache()
    for kw in (dict(Hq=3), dict(dqk=0), dict(dv=300), dict(W=0), dict(ns=-1), dict(ns=5000), dict(impl=9), dict(dtype=5), dict(Hkv=0)):
        assert decode(c, **kw) < 0, kw
    assert append(c, q=t, q_out=None) < 0 and append(c, T=0) < 0 and append(c, d=0) < 0


def test_cpu_tensors_raise():
    q = torch.zeros(1, 2, 4, 16)
    pos, tab = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(4, 8, 2)
    pt, n = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: swa.sink_swa_fwd(q, q, q, 2, 0), lambda: swa.SinkSwa.apply(q, q, q, None, 2, 0, 1.0),
                 lambda: swa.RotaryPEAxes.apply(q, q, pos, tab), lambda: swa.rope_axes_apply_to(q, pos, (tab,)),
                 lambda: swa.kv_append_rope(q, q, q, None, None, q, q, pt, n), lambda: swa.sink_swa_decode(q[:, :, :1], q, q, pt, n, 4, 0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_surface_takes_what_it_documents():
    with pytest.raises(TypeError):
        swa.SinkSwa.apply(torch.zeros(1), torch.zeros(1))
    with pytest.raises(TypeError):
        swa.sink_swa_fwd(torch.zeros(1), None, None, 2, 0)
    with pytest.raises(TypeError):
        swa.kv_append_rope(None, torch.zeros(1), torch.zeros(1), None, (1,), *(torch.zeros(1),) * 4)


def test_selection_rule():
    q = torch.zeros(1, 4, 8, 64, dtype=BF)
    assert swa.sink_selected_impl(q, q, q, 4, 1) == "tc"
    for kw, impl in ((dict(d_qk=72, d_v=8), 2), (dict(d_qk=20), 1), (dict(d_qk=136), 1), (dict(dtype=0), 1), (dict(sm_scale=0.0), 1), (dict(sm_scale=-1.0), 1),
                     (dict(impl=1), 1), (dict(Hq=64, Hkv=1, N=1 << 20, window=1 << 20), 1), (dict(Hq=32, Hkv=1, N=1 << 20, window=1 << 20), 2)):
        g = geom(**kw)
        assert LIB.sink_swa_select(C.byref(g)) == impl, kw
    g = geom(dtype=0, impl=2)
    assert LIB.sink_swa_select(C.byref(g)) < 0 and b"fp32" in LIB.swa_last_error()
    assert swa.sink_selected_impl(q.float(), q.float(), q.float(), 4, 1) == "simt"
    with pytest.raises(RuntimeError, match="window"):
        swa.sink_selected_impl(q, q, q, 0, 1)


def test_module_and_grid_positions():
    m = swa.RotaryPositionEncodingAxes((4, 6, 6), (10, 20, 30))
    assert [tuple(t.shape) for t in m.tables] == [(10, 4, 2), (20, 6, 2), (30, 6, 2)]
    p = m.grid_positions(2, 3, 4)
    assert p.shape == (3, 24) and p.dtype == torch.int32 and p[:, 23].tolist() == [1, 2, 3] and p[:, 5].tolist() == [0, 1, 1]
    with pytest.raises(ValueError):
        swa.RotaryPositionEncodingAxes((4,), (10, 20))


@pytest.mark.parametrize("W, ns, lens", [(3, 2, None), (1, 0, [5, 0]), (20, 0, [9, 4]), (2, 4, [7, 9])])
def test_oracle_against_differences(W, ns, lens):
    """The gradients of the oracle against central differences of its own forward pass, and the rotation's inverse."""
    g = torch.Generator().manual_seed(1)
    q, k, v, do = (torch.randn(2, h, 9, d, generator=g, dtype=torch.float64) for h, d in ((4, 5), (2, 5), (2, 3), (4, 3)))
    val, _ = orc.attention(q, k, v, lens, W, ns, 0.7, do, dtype=torch.float32)
    e = 1e-5
    for x, name in ((q, "dq"), (k, "dk"), (v, "dv")):
        for _ in range(12):
            at = tuple(int(torch.randint(0, n, (1,), generator=g)) for n in x.shape)
            old = float(x[at])
            f = []
            for s in (e, -e):
                x[at] = old + s
                f.append(float((orc.attention(q, k, v, lens, W, ns, 0.7, dtype=torch.float32)[0]["o"] * do).sum()))
            x[at] = old
            assert abs((f[0] - f[1]) / (2 * e) - float(val[name][at])) < 1e-7
    pos = torch.randint(-1, 6, (2, 9), generator=g, dtype=torch.int32)
    tabs = (swa.make_cs_table(1, 6), swa.make_cs_table(1, 6))
    assert torch.allclose(orc.rotate(orc.rotate(q, pos, tabs), pos, tabs, True), q, atol=1e-7)

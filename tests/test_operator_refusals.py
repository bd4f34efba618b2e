"""CPU: what orthogonalize, DeviceMuon, DeviceAdamW, layer_norm and their C entry points refuse before anything is launched."""
import ctypes

import numpy as np
import pytest
import torch

from margipose_amd import _lib, build
from margipose_amd._lib import MposeError

EINVAL = -22
ABC = (3.4445, -4.7750, 2.0315)


@pytest.fixture(scope='module')
def lib():
    build.build()
    return _lib.lib()


def _job(rows, cols, src=256, buf=256, dst=256):
    from margipose_amd.train_helpers import _ORTH_JOB_DT
    j = np.zeros(1, dtype=np.dtype(_ORTH_JOB_DT))
    j[0] = (src, buf, dst, rows, cols, 1.0, 0)
    return j


def _options(**kw):
    o = dict(steps=5, dtype=0, nesterov=0, reserved=0, a=ABC[0], b=ABC[1], c=ABC[2], eps=1e-7)
    o.update(kw)
    return _lib.OrthOptions(*[o[f] for f, _ in _lib.OrthOptions._fields_])


def test_struct_sizes(lib):
    from margipose_amd.train_helpers import _ADAMW_JOB_DT, _ORTH_JOB_DT
    assert lib.mpose_sizeof(13) == np.dtype(_ORTH_JOB_DT).itemsize and lib.mpose_sizeof(14) == ctypes.sizeof(_lib.OrthOptions)
    assert lib.mpose_sizeof(15) == np.dtype(_ADAMW_JOB_DT).itemsize


@pytest.mark.parametrize('rows,cols', [(0, 4), (4, 0), (-1, 4), ((1 << 21) + 1, 1), (1, (1 << 21) + 1), (1 << 15, 1 << 14), (1 << 30, 1 << 30)])
def test_orthogonalisation_refuses_shapes(lib, rows, cols):
    j, o = _job(rows, cols), _options()
    assert lib.mpose_orth_ws_bytes(j.ctypes.data, 1, ctypes.addressof(o)) == EINVAL
    assert lib.mpose_orthogonalize(j.ctypes.data, 1, ctypes.addressof(o), 256, 1 << 40, None) == EINVAL


@pytest.mark.parametrize('bad', [dict(steps=0), dict(steps=25), dict(steps=-3), dict(dtype=3), dict(dtype=-1), dict(eps=-1.0), dict(eps=float('nan')),
                                 dict(eps=float('inf')), dict(a=float('nan')), dict(b=float('inf')), dict(a=5.0, b=5.0, c=5.0), dict(a=2000.0, b=0.0, c=0.0)])
def test_orthogonalisation_refuses_options(lib, bad):
    j, o = _job(8, 8), _options(**bad)
    assert lib.mpose_orth_ws_bytes(j.ctypes.data, 1, ctypes.addressof(o)) == EINVAL
    assert lib.mpose_orthogonalize(j.ctypes.data, 1, ctypes.addressof(o), 256, 1 << 40, None) == EINVAL


def test_orthogonalisation_refuses_pointers_and_workspaces(lib):
    o = _options()
    j = _job(8, 8)
    need = lib.mpose_orth_ws_bytes(j.ctypes.data, 1, ctypes.addressof(o))
    assert need > 0
    run = lambda j, ws, n, o=o: lib.mpose_orthogonalize(j.ctypes.data, 1, ctypes.addressof(o), ws, n, None)      # noqa: E731
    assert run(j, None, need) == EINVAL and run(j, 256, need - 1) == EINVAL and run(j, 257, need) == EINVAL
    assert run(_job(8, 8, src=0), 256, need) == EINVAL and run(_job(8, 8, dst=0), 256, need) == EINVAL
    assert run(_job(8, 8, src=258), 256, need) == EINVAL and run(_job(8, 8, src=257), 256, need, _options(dtype=1)) == EINVAL
    assert lib.mpose_orthogonalize(None, 1, ctypes.addressof(o), 256, need, None) == EINVAL
    assert lib.mpose_orthogonalize(j.ctypes.data, -1, ctypes.addressof(o), 256, need, None) == EINVAL
    assert lib.mpose_orthogonalize(j.ctypes.data, 65536, ctypes.addressof(o), 256, need, None) == EINVAL
    assert lib.mpose_orthogonalize(None, 0, ctypes.addressof(o), None, 0, None) == 0                             # nothing to do
    assert lib.mpose_orthogonalize(j.ctypes.data, 1, None, 256, need, None) == EINVAL
    h = np.zeros(4, dtype=np.float32)
    muon = lambda j, h, dev=None, o=o: lib.mpose_muon_step(j.ctypes.data, 1, ctypes.addressof(o), h, dev, 256, 1 << 40, None)      # noqa: E731
    assert muon(j, None) == EINVAL and muon(_job(8, 8, buf=0), h.ctypes.data) == EINVAL and muon(_job(8, 8, buf=258), h.ctypes.data) == EINVAL
    assert muon(j, h.ctypes.data, None, _options(dtype=1)) == EINVAL


def test_adamw_refuses(lib):
    from margipose_amd.train_helpers import _ADAMW_JOB_DT
    h = np.zeros(8, dtype=np.float32)

    def run(p, g, m, v, n, hyper=h.ctypes.data, dev=None, count=1):
        j = np.zeros(1, dtype=np.dtype(_ADAMW_JOB_DT))
        j[0] = (p, g, m, v, n)
        return lib.mpose_adamw_step(j.ctypes.data, count, hyper, dev, None)
    assert run(0, 4, 4, 4, 1) == EINVAL and run(4, 4, 4, 0, 1) == EINVAL and run(4, 6, 4, 4, 1) == EINVAL and run(4, 4, 4, 4, -1) == EINVAL
    assert run(4, 4, 4, 4, 1, None) == EINVAL and run(4, 4, 4, 4, 1, count=-1) == EINVAL
    assert lib.mpose_adamw_step(None, 1, h.ctypes.data, None, None) == EINVAL
    assert run(0, 0, 0, 0, 0) == 0 and lib.mpose_adamw_step(None, 0, h.ctypes.data, None, None) == 0
    assert lib.mpose_set8(None, h.ctypes.data, None) == EINVAL and lib.mpose_set8(4, None, None) == EINVAL


def test_layer_norm_entries_refuse(lib):
    f = lambda x=16, ld=8, w=16, b=16, y=16, mean=16, rstd=16, rows=1, cols=8, eps=1e-5, io=0, wd=0: lib.mpose_layer_norm_fwd(      # noqa: E731
        x, ld, w, b, y, mean, rstd, rows, cols, eps, io, wd, None)
    for bad in (dict(x=None), dict(y=None), dict(ld=-1), dict(rows=-1), dict(cols=0), dict(cols=-5), dict(eps=-1.0), dict(eps=float('nan')), dict(io=3), dict(wd=-1),
                dict(mean=None), dict(rstd=None), dict(x=18), dict(y=17), dict(w=18), dict(b=17), dict(x=17, io=1), dict(w=17, wd=2)):
        assert f(**bad) == EINVAL, bad
    assert f(rows=0) == 0
    need = lib.mpose_layer_norm_bwd_ws_bytes(5, 8)
    assert need > 0 and lib.mpose_layer_norm_bwd_ws_bytes(0, 8) == 0 and lib.mpose_layer_norm_bwd_ws_bytes(-1, 8) == EINVAL and lib.mpose_layer_norm_bwd_ws_bytes(4, 0) == EINVAL
    g = lambda dy=16, dld=8, x=16, ld=8, w=16, mean=16, rstd=16, dx=16, dw=16, db=16, rows=5, cols=8, io=0, wd=0, ws=16, n=need: lib.mpose_layer_norm_bwd(      # noqa: E731
        dy, dld, x, ld, w, mean, rstd, dx, dw, db, rows, cols, io, wd, ws, n, None)
    for bad in (dict(dy=None), dict(x=None), dict(mean=None), dict(rstd=None), dict(ws=None), dict(n=need - 1), dict(ws=17), dict(dld=-1), dict(ld=-2), dict(rows=-1),
                dict(cols=0), dict(io=9), dict(wd=3), dict(dy=17), dict(dx=18), dict(dw=17), dict(db=18)):
        assert g(**bad) == EINVAL, bad
    assert g(dx=None, dw=None, db=None) == 0 and g(rows=0, dw=None, db=None) == 0


def test_no_cpu_path():
    from margipose_amd.nn_helpers import LayerNorm, layer_norm
    from margipose_amd.train_helpers import DeviceAdamW, DeviceMuon, orthogonalize
    with pytest.raises(MposeError, match='no CPU path'):
        orthogonalize(torch.zeros(3, 4))
    with pytest.raises(MposeError, match='no CPU path'):
        layer_norm(torch.zeros(3, 4), (4,))
    with pytest.raises(MposeError, match='no CPU path'):
        LayerNorm(4)(torch.zeros(3, 4))
    with pytest.raises(MposeError, match='ROCm device'):
        DeviceMuon([torch.zeros(3, 4)])
    with pytest.raises(MposeError, match='ROCm device'):
        DeviceAdamW([torch.zeros(3, 4)])
    with pytest.raises(MposeError, match='at least one'):
        DeviceAdamW([])
    with pytest.raises(MposeError, match='two dimensions'):
        orthogonalize([torch.zeros(3)])


def test_capture_guard_sees_a_live_graph(monkeypatch):
    """The mark on a leaf's accumulation node survives exactly while a graph holds it."""
    from margipose_amd import nn_helpers
    monkeypatch.setattr(_lib, 'stream_ptr', lambda: ctypes.c_void_p(8))
    w = torch.randn(3, requires_grad=True)
    assert nn_helpers._capture_leaves([w]) == (8,)
    y = w * 2
    for _ in range(2):
        with pytest.raises(MposeError, match='outside this capture'):
            nn_helpers._capture_leaves([w])
    del y
    assert nn_helpers._capture_leaves([w]) == (8,)
    y = w * 2
    torch.autograd.graph.get_gradient_edge(w).node.metadata['mpose_captured'] = (8,)      # held by this capture's own call
    assert nn_helpers._capture_leaves([w]) == (8,)
    monkeypatch.setattr(_lib, 'stream_ptr', lambda: ctypes.c_void_p(16))                   # ... and by another stream's
    with pytest.raises(MposeError, match='outside this capture'):
        nn_helpers._capture_leaves([w])

"""The mixture layer's operators without a GPU: argument errors of the C entries are statuses before anything is enqueued,
workspace queries are host only, and the Python wrappers refuse what they document."""

import ctypes
from ctypes import c_void_p

import pytest
import torch

from triturus_amd import _lib
from triturus_amd.gmm import gmm, gmm_grad
from triturus_amd.mx4 import MX4, mm_mx4, mx4_dequantize, mx4_quantize
from triturus_amd.route import Routes, route, route_grad

one, null = c_void_p(16), c_void_p(None)  # never dereferenced: every call below is rejected first
BF16, F32 = _lib.TRT_BF16, _lib.TRT_F32


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_gmm_statuses():
    lib = _lib.load()
    sb = i64(64, 8, 1)

    def rows(a=one, b=one, s=one, c=one, T=4, E=2, K=8, N=8, lda=8, st=sb, dtype=BF16, tile=0, ws=null):
        return lib.trt_gmm(a, b, s, c, T, E, K, N, lda, st, dtype, 0, tile, ws, 0, null)

    for bad in (dict(a=null), dict(b=null), dict(s=null), dict(c=null), dict(T=0), dict(E=0), dict(K=0), dict(N=-1), dict(dtype=_lib.TRT_F64),
                dict(dtype=9), dict(tile=-1), dict(tile=6)):
        assert rows(**bad) == -1, bad
    for bad in (dict(lda=-8), dict(st=i64(-64, 8, 1)), dict(st=i64(64, 8, 2)), dict(st=i64(64, 2, 8)), dict(ws=c_void_p(8))):
        assert rows(**bad) == -2, bad
    for bad in (dict(T=1 << 31), dict(E=1 << 31), dict(lda=1 << 22), dict(st=i64(64, 1 << 22, 1)), dict(N=1 << 22, K=1)):
        assert rows(**bad) == -4, bad
    assert rows(T=(1 << 31) - 1, N=(1 << 22) - 1) == -4  # more workgroups than a grid holds

    def weights(a=one, g=one, s=one, d=one, T=4, E=2, K=8, N=8, lda=8, ldg=8, dtype=F32, tile=0, ws=null):
        return lib.trt_gmm_weights(a, g, s, d, T, E, K, N, lda, ldg, dtype, 0, tile, ws, 0, null)

    for bad in (dict(a=null), dict(g=null), dict(s=null), dict(d=null), dict(T=0), dict(E=-1), dict(K=0), dict(N=0), dict(dtype=1), dict(tile=6)):
        assert weights(**bad) == -1, bad
    for bad in (dict(lda=-1), dict(ldg=-1), dict(ws=c_void_p(4))):
        assert weights(**bad) == -2, bad
    for bad in (dict(T=1 << 31), dict(ldg=1 << 21), dict(K=1 << 21)):
        assert weights(**bad) == -4, bad


def test_gmm_grad_statuses():
    lib = _lib.load()

    def call(g=one, a=one, b=one, s=one, da=one, db=one, T=4, E=2, K=8, N=16, ldg=16, lda=8, st=i64(128, 16, 1), dtype=BF16, ws=null):
        return lib.trt_gmm_grad(g, a, b, s, da, db, T, E, K, N, ldg, lda, st, dtype, 0, ws, 0, null)

    for bad in (dict(g=null), dict(a=null), dict(b=null), dict(s=null), dict(da=null), dict(db=null), dict(T=0), dict(N=0), dict(dtype=1), dict(st=None)):
        assert call(**bad) == -1, bad
    for bad in (dict(ldg=-1), dict(lda=-1), dict(st=i64(128, 16, 3)), dict(ws=c_void_p(8))):
        assert call(**bad) == -2, bad
    for bad in (dict(T=1 << 31), dict(lda=1 << 22), dict(st=i64(128, 1 << 22, 1))):
        assert call(**bad) == -4, bad
    at = c_void_p(1 << 20)
    assert lib.trt_gmm_grad_workspace_bytes(at, at, at, 16384, 8, 2048, 2048, 2048, 2048, i64(1 << 22, 2048, 1), BF16) == 0
    assert lib.trt_gmm_grad_workspace_bytes(at, at, at, 16384, 8, 2049, 2048, 2048, 2049, i64(2049 * 2048, 2048, 1), BF16) == 16384 * 2056 * 2


def test_capture_is_refused_by_name(monkeypatch):
    from triturus_amd import gmm as module

    monkeypatch.setattr(module, "_is_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="gmm_grad"):
        module.refuse_capture("gmm")
    monkeypatch.setattr(module, "_is_capturing", lambda: False)
    module.refuse_capture("gmm")


def test_gmm_workspace_is_for_operands_off_the_boundaries():
    lib = _lib.load()
    at = c_void_p(1 << 20)

    def rows(T, E, K, N, a=at):
        return lib.trt_gmm_workspace_bytes(a, at, T, E, K, N, K, i64(K * N, N, 1), BF16, 0)

    assert rows(16384, 8, 2048, 2048) == 0
    assert rows(16384, 8, 2049, 2048) == 16384 * 2056 * 2  # the rows alone
    assert rows(16384, 8, 2048, 2047) == 8 * 2048 * 2048 * 2  # the matrices alone
    assert rows(16384, 8, 2048, 2048, c_void_p((1 << 20) + 2)) == 16384 * 2048 * 2
    assert rows(2, 8, 2049, 2047) == 0  # few rows: bound by reading the matrices, a copy would not pay
    assert rows(16384, 0, 2049, 2048) == 0 and rows(16384, 8, 0, 2048) == 0  # an invalid call wants none
    w = lib.trt_gmm_weights_workspace_bytes
    assert w(at, at, 16384, 8, 2048, 2048, 2048, 2048, BF16, 0) == 0
    assert w(at, at, 16384, 8, 2049, 2047, 2049, 2047, BF16, 0) == 16384 * (2056 + 2048) * 2
    # few tiles under many rows: sums of pieces of the rows, 64 KiB a tile of 128 x 128
    pieces, rest = divmod(w(at, at, 16384, 1, 512, 512, 512, 512, BF16, 0), 16 * 65536)
    assert 2 <= pieces <= 33 and rest == 0
    assert w(at, at, 16384, 1, 512, 512, 512, 512, BF16, 1) == w(at, at, 200, 1, 512, 512, 512, 512, BF16, 0) == 0


def test_mx4_statuses():
    lib = _lib.load()
    q = lib.trt_mx4_quantize
    assert q(null, one, one, 4, 64, 64, BF16, null) == q(one, null, one, 4, 64, 64, BF16, null) == q(one, one, null, 4, 64, 64, BF16, null) == -1
    assert q(one, one, one, 0, 64, 64, BF16, null) == q(one, one, one, 4, 0, 64, BF16, null) == q(one, one, one, 4, 64, 64, 7, null) == -1
    assert q(one, one, one, 4, 64, -1, BF16, null) == q(one, c_void_p(18), one, 4, 64, 64, BF16, null) == -2
    assert q(one, one, one, 4, (1 << 30) + 1, 1 << 31, BF16, null) == -4
    d = lib.trt_mx4_dequantize
    assert d(null, one, one, 4, 64, 32, 2, F32, null) == d(one, one, one, 4, 64, 32, 2, 1, null) == d(one, one, one, -4, 64, 32, 2, F32, null) == -1
    assert d(one, one, one, 4, 64, -32, 2, F32, null) == -2

    def mm(a=one, sa_=one, b=one, sb_=one, s=null, c=one, T=4, E=1, K=64, N=8, sa=i64(32, 2), sb=i64(0, 32, 0, 2), a_type=-1, dtype=BF16, tile=0, ws=null, n=0):
        return lib.trt_mx4_mm(a, sa_, b, sb_, s, c, T, E, K, N, sa, sb, a_type, dtype, 0, tile, ws, n, null)

    for bad in (dict(a=null), dict(sa_=null), dict(b=null), dict(sb_=null), dict(c=null), dict(T=0), dict(E=0), dict(K=0), dict(N=0), dict(E=2),
                dict(dtype=1), dict(dtype=8), dict(a_type=1), dict(a_type=4), dict(tile=5), dict(tile=-1)):
        assert mm(**bad) == -1, bad
    for bad in (dict(sa=i64(-32, 2)), dict(sb=i64(0, 32, -1, 2)), dict(ws=c_void_p(8))):
        assert mm(**bad) == -2, bad
    for bad in (dict(sa=i64(1 << 23, 2)), dict(sb=i64(0, 1 << 23, 0, 2)), dict(T=1 << 31), dict(N=1 << 23)):
        assert mm(**bad) == -4, bad
    assert mm(a_type=BF16, tile=1) == -3  # values for a kernel that wants codes: a workspace for them
    need = lib.trt_mx4_mm_workspace_bytes
    assert need(4, 1, 64, 8, BF16, BF16, 1) == 4 * 2 * 17
    assert need(4, 1, 64, 8, -1, BF16, 1) == 0
    assert need(1, 1, 4096, 8192, BF16, BF16, 0) == 0  # one row: quantised on the way
    assert need(4096, 1, 4096, 8192, BF16, BF16, 0) == 4096 * 128 * 17


def test_route_statuses():
    lib = _lib.load()

    def call(x=one, w=one, T=4, E=8, k=2, ld=8, dtype=F32, ws=null, n=0):
        return lib.trt_route(x, w, one, one, one, one, T, E, k, ld, dtype, 1, ws, n, null)

    for bad in (dict(x=null), dict(w=null), dict(T=0), dict(E=0), dict(k=0), dict(k=9), dict(dtype=1)):
        assert call(**bad) == -1, bad
    assert call(ld=-1) == -2 and call(T=65, ws=c_void_p(4), n=1 << 20) == -2
    for bad in (dict(E=1025), dict(k=17, E=20), dict(T=1 << 30, k=2)):
        assert call(**bad) == -4, bad
    assert call(T=65) == -3
    ws = lib.trt_route_workspace_bytes
    assert ws(64, 100) == 0 and ws(65, 100) == 100 * 64 and ws(64 * 64, 100) == 100 * 64 and ws(64 * 64 + 1, 100) == 100 * 128 * 5
    g = lib.trt_route_grad
    assert g(null, one, one, one, one, 4, 8, 2, 8, F32, 1, null) == g(one, one, one, one, one, 4, 8, 9, 8, F32, 1, null) == -1
    assert g(one, one, one, one, one, 4, 8, 2, -8, F32, 1, null) == -2
    assert g(one, one, one, one, one, 4, 1025, 2, 8, F32, 1, null) == -4
    assert g(one, one, one, one, one, 4, 8, 2, 8, 1, 1, null) == -1


def test_wrappers_refuse_before_any_launch():
    a, b, s = torch.randn(4, 8), torch.randn(2, 8, 6), torch.tensor([1, 3])
    for call in (lambda: gmm(a, b, s), lambda: gmm_grad(torch.randn(4, 6), a, b, s), lambda: mx4_quantize(a),
                 lambda: mx4_dequantize(MX4(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 8)),
                 lambda: mm_mx4(a, MX4(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 8)), lambda: route(a, 2),
                 lambda: route_grad(torch.randn(4, 2), a, Routes(torch.randn(4, 2), torch.zeros(4, 2, dtype=torch.int32), s, s, s))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    for call in (lambda: gmm(a[0], b, s), lambda: gmm(a, b, s[:1]), lambda: gmm(a, b.half(), s), lambda: gmm(a, b, s.float()), lambda: gmm(a[:, 1:], b, s),
                 lambda: route(a, 9), lambda: route(a, 0), lambda: route(a[0], 1)):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: gmm(a.double(), b.double(), s), lambda: route(a.double(), 2), lambda: mx4_quantize(a.int())):
        with pytest.raises(NotImplementedError):
            call()


def test_import_paths():
    import triturus.gmm
    import triturus.mx4
    import triturus.route

    assert triturus.gmm.gmm is gmm and triturus.gmm.gmm_grad is gmm_grad
    assert triturus.mx4.mm_mx4 is mm_mx4 and triturus.mx4.MX4 is MX4
    assert triturus.route.route is route and triturus.route.Routes is Routes

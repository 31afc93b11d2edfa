"""Workspaces of the grouped products' gradients, without a GPU: the queries are host only."""

import ctypes
import math
import random

import pytest

from triturus_amd import _lib

F32, F16, BF16 = _lib.TRT_F32, _lib.TRT_F16, _lib.TRT_BF16
SIZE = {F32: 4, F16: 2, BF16: 2}
AT = 1 << 20  # an address on the boundaries; never dereferenced


def copies(T, K, N, dtype):
    """Bytes of both operands in rows of whole 16-byte chunks."""
    values = 16 // SIZE[dtype]
    return 16 * T * (-(-K // values) + -(-N // values))


def weights(T, E, K, N, dtype, a=AT):
    return _lib.load().trt_gmm_weights_workspace_bytes(a, AT, T, E, K, N, K, N, dtype, 0)


def grad(T, E, K, N, dtype):
    sb = (ctypes.c_int64 * 3)(K * N, N, 1)
    return _lib.load().trt_gmm_grad_workspace_bytes(AT, AT, AT, T, E, K, N, N, K, sb, dtype)


def held(T, E, K, N, dtype):
    return (T * (K + N) + E * K * N) * SIZE[dtype]


def shapes(count, seed):
    rng = random.Random(seed)

    def between(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    for _ in range(count):
        E = between(1, 600)
        yield between(1, 1 << 22), E, between(1, 9000), between(1, 9000), rng.choice([F32, F16, BF16])


@pytest.mark.parametrize("T,E,K,N,dtype", [(16384, 8, 4097, 4096, F32), (104869, 8, 7911, 8161, F32), (16384, 8, 4104, 4096, F32), (16384, 8, 2056, 2048, F32),
                                           (16384, 8, 4097, 4095, BF16), (26870, 18, 849, 2096, BF16), (6067, 9, 616, 3000, BF16)])
def test_many_tiles_are_not_cut(T, E, K, N, dtype):
    """Where the tiles take several rounds of all CUs, long and short groups average out and a cut gains nothing."""
    aligned = K % 8 == 0 and N % 8 == 0
    assert weights(T, E, K, N, dtype) <= (0 if aligned else copies(T, K, N, dtype))


def test_pieces_take_a_bounded_workspace():
    """The sums of pieces: at most 256 MiB, or half of what the call's operands and result take."""
    for T, E, K, N, dtype in shapes(20000, 5):
        most = max(256 << 20, held(T, E, K, N, dtype) // 2)
        assert weights(T, E, K, N, dtype) <= most + copies(T, K, N, dtype), (T, E, K, N, dtype)
        b = 16 * max(E * K * -(-N * SIZE[dtype] // 16), E * N * -(-K * SIZE[dtype] // 16))  # b may be copied too
        assert grad(T, E, K, N, dtype) <= most + copies(T, K, N, dtype) + b, (T, E, K, N, dtype)


def test_few_tiles_under_many_rows_are_still_cut():
    for T, E, K, N, dtype in ((16384, 1, 512, 512, BF16), (16384, 1, 512, 512, F32), (32768, 1, 2048, 1024, BF16), (1500000, 200, 80, 632, BF16),
                              (500000, 460, 16, 336, BF16), (350000, 500, 240, 128, F32)):
        assert weights(T, E, K, N, dtype) > 0


def test_the_library_alone_decides_on_pieces():
    """gmm.py asks for no workspace only where the library would want none: groups of 32 rows or fewer on average, operands on the boundaries."""
    from triturus_amd.gmm import _few_rows

    rng = random.Random(9)
    wanted = 0
    for T, E, K, N, dtype in shapes(40000, 8):
        K, N = -(-K // 8) * 8, -(-N // 8) * 8
        if rng.random() < 0.3:  # next to the border
            T = max(1, min((1 << 31) - 1, 32 * E + rng.randint(-3, 40 * E)))
        if weights(T, E, K, N, dtype):
            wanted += 1
            assert not _few_rows(T, E), (T, E, K, N, dtype)
    assert wanted > 5000 and _few_rows(64, 2) and not _few_rows(65, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,K,N,dtype", [(3784, 3, 1640, 1760, BF16), (7302, 16, 720, 888, F32)])
def test_the_cut_does_not_depend_on_alignment(dev, T, E, K, N, dtype):
    """The same operands on and off the 16-byte boundaries: the same pieces, so the same sums bit for bit."""
    import torch

    from triturus_amd.gmm import gmm_grad

    dtype = {code: t for t, code in _lib.DTYPE_CODES.items()}[dtype]
    a, g, b = (torch.randn(*shape, device=dev).to(dtype) for shape in ((T, K), (T, N), (E, K, N)))
    sizes = torch.full((E,), T // E, dtype=torch.int32, device=dev)
    off = torch.empty(T * K + 1, device=dev, dtype=dtype)[1:].view(T, K).copy_(a)
    assert a.data_ptr() % 16 == 0 and off.data_ptr() % 16 != 0
    want = torch.stack([a[e * (T // E):(e + 1) * (T // E)].double().T @ g[e * (T // E):(e + 1) * (T // E)].double() for e in range(E)])
    d = gmm_grad(g, a, b, sizes)[1]
    assert torch.equal(gmm_grad(g, off, b, sizes)[1], d)
    # fp32 sums of T / E products, each addition within 2^-23 of the running magnitudes, and the result's own rounding
    size = torch.stack([a[e * (T // E):(e + 1) * (T // E)].double().abs().T @ g[e * (T // E):(e + 1) * (T // E)].double().abs() for e in range(E)])
    bound = (T // E + 1) * 2.0 ** -23 * size + torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2 ** -8)
    assert ((d.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pieces_follow_the_rows(dtype):
    """Few tiles under millions of rows are cut for all CUs, not into as many pieces as under thousands."""
    for T in (1 << 20, 1 << 22):
        assert weights(T, 1, 128, 128, dtype) // 65536 >= 192
        assert weights(T, 2, 128, 256, dtype) // 65536 >= 192
    assert 2 <= weights(16384, 1, 128, 128, dtype) // 65536 <= 33


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("sizes", [[250000, 49990], [0, 1, 400001], [370003]], ids=str)
def test_sums_of_many_pieces(dev, sizes, dtype):
    import torch

    from triturus_amd.gmm import gmm_grad

    K, N, T = 72, 136, sum(sizes) + 10
    assert weights(T, len(sizes), K, N, dtype) // (2 * 65536) > 95
    dtype = {code: t for t, code in _lib.DTYPE_CODES.items()}[dtype]
    a, g, b = torch.randn(T, K, device=dev).to(dtype), (torch.randn(T, N, device=dev) / 64).to(dtype), torch.zeros(len(sizes), K, N, device=dev, dtype=dtype)
    a[-10:], g[-10:] = math.nan, math.inf
    s = torch.tensor(sizes, dtype=torch.int32, device=dev)
    d, r = gmm_grad(g, a, b, s)[1], 0
    for e, n in enumerate(sizes):
        x, y = a[r:r + n].double().T, g[r:r + n].double()
        want, size = x @ y, x.abs() @ y.abs()
        # every addition within 2^-23 of the running magnitudes, however the rows are cut, and the result's own rounding
        info = torch.finfo(dtype)
        bound = (n + 1) * 2.0 ** -23 * size + info.eps / 2 * want.abs() * (1 + 2 ** -8) + info.smallest_normal * info.eps / 2
        assert ((d[e].double() - want).abs() <= bound).all()
        r += n
    assert torch.equal(gmm_grad(g, a, b, s)[1], d)


def test_aligned_operands_need_the_pieces_alone():
    """What gmm.py keeps by shape: on the boundaries both queries say the same, wherever the operands lie."""
    for T, E, K, N, dtype in shapes(5000, 12):
        K, N = -(-K // 8) * 8, -(-N // 8) * 8
        w = weights(T, E, K, N, dtype)
        assert w == grad(T, E, K, N, dtype)
        assert w == _lib.load().trt_gmm_weights_workspace_bytes(AT + 4096, AT + 16, T, E, K, N, K + 8, N + 64, dtype, 0)

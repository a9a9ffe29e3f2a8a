"""Which kernel and tile the block-scaled product takes (decided on the host: nq_diag_fp8_block_form needs no GPU), and the
product on the GPU where that choice matters."""
import ctypes as C

import pytest
import torch

import fp8_block_ref as R
from noeira_amd import _lib as L
from noeira_amd.qlinear import FP8BlockLinear

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def form(M, K, N, dtype):
    """(0 few rows / 1 GEMM, tile rows, tile channels, wavefronts or groups over K, tiles left to a second launch)"""
    got = (C.c_int32 * 5)()
    L.check(L.lib().nq_diag_fp8_block_form(M, N, K, {"f32": L.DT_F32, "bf16": L.DT_BF16}[dtype], got))
    return tuple(got)


def threads(f, M, N):
    """work-items of the launch: a few-rows workgroup is 64 threads per wavefront over K, a GEMM's at most 512"""
    return -(-M // f[1]) * -(-N // f[2]) * (64 * f[3] if f[0] == 0 else 512)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [
    (150_000_000, 128, 16), (2 ** 27 + 100, 16, 1), (2 ** 27 + 100, 4096, 1), (100_000_000, 16, 40), (300_000_000, 64, 17),
    (5, 16, 2 ** 27 + 5), (60, 128, 2 ** 27), (200_000, 4096, 70_000)])
def test_a_kernel_whose_launch_fits_is_taken(M, K, N, dtype):
    """A launch holds fewer than 2^32 work-items; where the shape of lowest estimate would need more, another takes the
    call, as long as one fits."""
    assert threads(form(M, K, N, dtype), M, N) <= 2 ** 32 - 1


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N", [(2 ** 31 - 1, 1), (2 ** 31 - 16, 1000), (2 ** 31 - 300, 16), (1, 2 ** 31 - 1), (64, 2 ** 31 - 20), (1, 2 ** 28)])
def test_what_fits_no_launch_is_refused(M, N, dtype):
    """(One row into 2^28 channels: the widest shape for one row has 32 channels to 512 work-items, 2^32 of them.)"""
    for K in (16, 4096):
        with pytest.raises(L.NQError, match="are too many for one launch"):
            form(M, K, N, dtype)


# every kernel and tile there is, as form() names them; the last: with tiles left to the second launch
FEW = [(0, 16, 16, 8), (0, 16, 16, 16), (0, 16, 32, 8), (0, 32, 32, 8), (0, 32, 64, 8), (0, 64, 64, 8)]
FORMS = {"f32": FEW + [(1, 64, 128, 1), (1, 64, 128, 2), (1, 128, 128, 1), (1, 256, 128, 1)],
         "bf16": FEW + [(1, 64, 128, 2), (1, 128, 128, 1), (1, 128, 256, 1), (1, 256, 256, 1), (1, 256, 256, 1, "and rest")]}
# 65 blocks of K, 16 values in the last, into an odd number of channels; 32 whole blocks into whole tiles.  The GEMM's stage
# buffers (two to four) and its three buffers of four stages' scales are taken in turn: from 13 stages of a group on
# (26 blocks, where two groups share them) a buffer of scales is filled a second time.  A few-rows wavefront of eight
# walks beyond its first four blocks from 33 on.
DEEP = [(17, 8208, 1001), (3, 8208, 1001), (17, 8208, 4001), (300, 8208, 513), (40, 8208, 8101), (500, 8208, 1301), (777, 8208, 2567),
        (321, 8208, 3001), (2045, 8208, 2567), (1300, 8208, 8101), (2304, 8208, 8101), (1030, 8208, 3333),
        (400, 4096, 2560), (512, 4096, 2048), (1024, 4096, 4096), (2048, 4096, 2560), (2304, 4096, 4096), (4096, 4096, 4352)]


def kinds(K, dtype):
    got = set()
    for M, k, N in DEEP:
        if k == K:
            f = form(M, K, N, dtype)
            got.add(f[:4] + ("and rest",) if f[4] else f[:4])
    return got


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_deep_cases_run_every_form(dtype):
    """A retuned choice must not leave a form without a deep case."""
    assert kinds(8208, dtype) == set(FORMS[dtype])
    assert kinds(4096, dtype) >= {f for f in FORMS[dtype] if f[0] == 1}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", DEEP)
def test_deep_products(M, K, N, dtype):
    gen = torch.Generator().manual_seed(M + K + N)
    xq, xs = R.random_rows(gen, M, K)
    wq, ws = R.random_weight(gen, N, K)
    lin = FP8BlockLinear(K, N)
    lin.set_weight(wq, ws)
    bias = torch.randn(N, generator=gen).cuda()
    store = torch.full((M * N + 64,), 77.0, dtype=DTYPES[dtype], device="cuda")
    got = lin.forward_a8(xq, xs, bias=bias, out=store[: M * N].view(M, N), out_dtype=DTYPES[dtype])
    x, w = R.rows(xq, xs), R.matrix(wq, ws)
    y = x @ w.t() + bias.double()
    R.assert_within(got, y, R.product_bound(x, w, y, bias.double(), DTYPES[dtype]), "y")
    assert (store[M * N:] == 77.0).all()
    for _ in range(3):
        assert torch.equal(lin.forward_a8(xq, xs, bias=bias, out_dtype=DTYPES[dtype]), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K,N", [(3, 1008, 8208), (300, 528, 8208), (321, 3008, 8208), (2045, 2576, 8208)])
def test_deep_gradients(M, K, N, dtype):
    """gx[M, K] from gy[M, N]: blocks of N, the kernels of the product."""
    gen = torch.Generator().manual_seed(M + K)
    wq, ws = R.random_weight(gen, N, K)
    lin = FP8BlockLinear(K, N, grad=True)
    lin.set_weight(wq, ws)
    gq, gs = R.random_rows(gen, M, N)
    g, w = R.rows(gq, gs), R.matrix(wq, ws)
    want = g @ w
    got = lin.vjp_a8(gq, gs, out_dtype=DTYPES[dtype])
    R.assert_within(got, want, R.product_bound(g, w.t(), want, None, DTYPES[dtype]), "gx")


def test_arguments():
    got = (C.c_int32 * 5)()
    for args in ((0, 16, 16, 0, got), (1, 0, 16, 0, got), (1, 16, 24, 0, got), (1, 16, 16, 0, None), (1, 16, 16, L.DT_I8, got)):
        assert L.lib().nq_diag_fp8_block_form(*args) == L.NQ_ERR_INVALID and "nq_diag_fp8_block_form" in L.last_error()


@pytest.mark.gpu
def test_more_rows_than_the_smallest_tile_launches():
    """2^27 + 100 rows of one block into one channel: 16 rows to a workgroup would be more than 2^32 work-items."""
    M, K, N = 2 ** 27 + 100, 16, 1
    gen = torch.Generator().manual_seed(3)
    wq, ws = R.random_weight(gen, N, K)
    lin = FP8BlockLinear(K, N)
    lin.set_weight(wq, ws)
    xq = torch.zeros((M, K), dtype=torch.uint8, device="cuda")
    xs = torch.ones((M, 1), device="cuda")
    tail = R.random_rows(gen, 150, K)
    xq[-150:], xs[-150:] = tail
    xq[:150], xs[:150] = tail
    x, w = R.rows(*tail), R.matrix(wq, ws)
    y = lin.forward_a8(xq, xs, out_dtype=torch.float32)
    bound = R.product_bound(x, w, x @ w.t(), None, torch.float32)
    R.assert_within(y[-150:], x @ w.t(), bound, "last rows")
    R.assert_within(y[:150], x @ w.t(), bound, "first rows")
    assert not y[150:-150].any()

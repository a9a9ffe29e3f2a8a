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

"""What the block-scaled fp8 linear and the layer norm refuse, answered on the host before anything is launched (no GPU
needed), and the host-side quantisation of a weight into blocks against its definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from noeira_amd import _lib as L
from noeira_amd import formats as F
from oracle import oracle as O

P = C.c_void_p


def create(IN, OUT, flags=0, fmt=L.FMT_FP8_BLOCK):
    h = P()
    return L.lib().nq_create(C.byref(h), fmt, IN, OUT, 0, flags), h


def refuses(rc, code, words):
    assert rc == code and words in L.last_error(), (rc, L.last_error())


def test_create():
    refuses(create(100, 64)[0], L.NQ_ERR_INVALID, "FP8_BLOCK needs IN to be a multiple of 16")
    refuses(create(0, 64)[0], L.NQ_ERR_INVALID, "IN and OUT must be positive")
    refuses(create(128, 100, L.FLAG_GRAD)[0], L.NQ_ERR_INVALID, "NQ_FLAG_GRAD needs OUT to be a multiple of 16")
    refuses(create(128, 64, L.FLAG_GRAD, L.FMT_FP8_E4M3)[0], L.NQ_ERR_INVALID, "NQ_FLAG_GRAD is for FP8_BLOCK layers")
    refuses(create(128, 64, 8)[0], L.NQ_ERR_INVALID, "unknown flags")
    rc, h = create(960, 101)
    assert rc == L.NQ_OK and L.lib().nq_blocks_bytes(h) == 960 * 101 and L.lib().nq_device_bytes(h) == 0
    assert L.lib().nq_destroy(h) == L.NQ_OK


def test_before_a_weight_is_set():
    lib = L.lib()
    rc, h = create(128, 64, L.FLAG_GRAD)
    assert rc == L.NQ_OK
    one = P(64)
    refuses(lib.nq_forward(h, one, L.DT_FP8_E4M3, one, one, L.DT_F32, 1, None, 0, 0, None), L.NQ_ERR_NOT_LOADED, "no weights")
    refuses(lib.nq_grad_input_fp8_block(h, one, one, one, L.DT_F32, 1, None), L.NQ_ERR_NOT_LOADED, "no weights")
    refuses(lib.nq_grad_input_fp8_block(None, one, one, one, L.DT_F32, 1, None), L.NQ_ERR_INVALID, "null layer handle")
    refuses(lib.nq_set_weight_fp8_block(h, None, None, None), L.NQ_ERR_INVALID, "null codes or scales")
    refuses(lib.nq_set_weight_fp8_block_dev(h, None, one, None), L.NQ_ERR_INVALID, "null codes or scales")
    refuses(lib.nq_set_weight_fp8_block_dev(h, one, P(66), None), L.NQ_ERR_INVALID, "4-byte aligned")
    refuses(lib.nq_set_weight_fp8(h, one, 1.0, None), L.NQ_ERR_INVALID, "not FP8_E4M3")
    rc, other = create(128, 64, fmt=L.FMT_FP8_E4M3)
    refuses(lib.nq_set_weight_fp8_block(other, one, one, None), L.NQ_ERR_INVALID, "not FP8_BLOCK")
    out = P()
    refuses(lib.nq_fuse_glu(C.byref(out), h, h, None), L.NQ_ERR_NOT_LOADED, "no weights")
    for x in (h, other):
        lib.nq_destroy(x)


@pytest.mark.parametrize("args,words", [
    ((64, L.DT_I8, 64, 64, 1, 128), "x must be fp32 or bf16"),
    ((64, L.DT_F32, 64, 64, -1, 128), "M >= 0 and K > 0"),
    ((64, L.DT_F32, 64, 64, 1, 0), "M >= 0 and K > 0"),
    ((None, L.DT_F32, 64, 64, 1, 128), "null pointer"),
    ((64, L.DT_F32, 64, None, 1, 128), "null pointer"),
    ((72, L.DT_F32, 64, 64, 1, 128), "16-byte"),
    ((64, L.DT_F32, 72, 64, 1, 128), "16-byte"),
    ((64, L.DT_F32, 64, 66, 1, 128), "4-byte"),
    ((64, L.DT_F32, 64, 64, 2 ** 31 - 1, 2 ** 31 - 1), "more than 2^31 - 1 blocks"),
])
def test_quantize_rows(args, words):
    refuses(L.lib().nq_quantize_rows_fp8_block(*args, None), L.NQ_ERR_INVALID, words)


def test_quantize_rows_of_nothing():
    assert L.lib().nq_quantize_rows_fp8_block(None, L.DT_F32, None, None, 0, 128, None) == L.NQ_OK


NORM = dict(x=64, xdt=L.DT_F32, gamma=64, beta=64, eps=1e-5, y=128, ydt=L.DT_F32, mean=64, rstd=64, M=2, D=64)


@pytest.mark.parametrize("change,words", [
    (dict(D=0), "M >= 0 and D > 0"), (dict(M=-1), "M >= 0 and D > 0"), (dict(xdt=L.DT_I8), "x must be fp32 or bf16"),
    (dict(ydt=L.DT_I32), "y must be fp32 or bf16"), (dict(eps=-1.0), "eps must be"), (dict(eps=float("nan")), "eps must be"),
    (dict(eps=float("inf")), "eps must be"), (dict(mean=None), "together"), (dict(x=None), "null x"), (dict(x=68), "16-byte"),
    (dict(mean=66), "4-byte"), (dict(rstd=65), "4-byte"), (dict(gamma=68), "16-byte"), (dict(beta=68), "16-byte"), (dict(y=None), "16-byte"), (dict(y=132), "16-byte"),
    (dict(y=64, ydt=L.DT_BF16), "where the types agree"),
])
def test_layer_norm(change, words):
    a = {**NORM, **change}
    refuses(L.lib().nq_layer_norm(a["x"], a["xdt"], a["gamma"], a["beta"], a["eps"], a["y"], a["ydt"], a["mean"], a["rstd"],
                                  a["M"], a["D"], None), L.NQ_ERR_INVALID, words)
    if "y" not in change and "ydt" not in change:
        refuses(L.lib().nq_layer_norm_fp8_block(a["x"], a["xdt"], a["gamma"], a["beta"], a["eps"], 64, 64, a["mean"], a["rstd"],
                                                a["M"], a["D"], None), L.NQ_ERR_INVALID, words)


@pytest.mark.parametrize("codes,scales", [(None, 64), (64, None), (68, 64), (64, 66)])
def test_layer_norm_codes(codes, scales):
    refuses(L.lib().nq_layer_norm_fp8_block(64, L.DT_F32, 64, 64, 1e-5, codes, scales, None, None, 1, 64, None), L.NQ_ERR_INVALID,
            "codes (16-byte aligned) and scales (4-byte) are needed")


GRAD = dict(x=64, xdt=L.DT_F32, mean=64, rstd=64, gamma=64, gy=128, gydt=L.DT_F32, gx=192, gxdt=L.DT_F32, dg=64, db=64, M=4096,
            D=64, ws=None, n=0)


@pytest.mark.parametrize("change,code,words", [
    (dict(D=0), L.NQ_ERR_INVALID, "M >= 0 and D > 0"), (dict(D=2 ** 26 + 1), L.NQ_ERR_INVALID, "2^26"), (dict(gydt=L.DT_I8), L.NQ_ERR_INVALID, "must be fp32 or bf16"),
    (dict(gxdt=7), L.NQ_ERR_INVALID, "must be fp32 or bf16"), (dict(dg=None), L.NQ_ERR_INVALID, "together"),
    (dict(dg=66), L.NQ_ERR_INVALID, "4-byte"), (dict(gy=None), L.NQ_ERR_INVALID, "null pointer"),
    (dict(mean=None), L.NQ_ERR_INVALID, "null pointer"), (dict(rstd=66), L.NQ_ERR_INVALID, "4-byte"), (dict(gx=196), L.NQ_ERR_INVALID, "16-byte"),
    (dict(gx=128, gxdt=L.DT_BF16), L.NQ_ERR_INVALID, "types agree"), (dict(gx=64, gxdt=L.DT_BF16), L.NQ_ERR_INVALID, "types agree"),
])
def test_layer_norm_grad(change, code, words):
    a = {**GRAD, **change}
    refuses(L.lib().nq_layer_norm_grad(a["x"], a["xdt"], a["mean"], a["rstd"], a["gamma"], a["gy"], a["gydt"], a["gx"], a["gxdt"],
                                       a["dg"], a["db"], a["M"], a["D"], a["ws"], a["n"], None), code, words)


def test_nothing_to_do():
    lib = L.lib()
    assert lib.nq_layer_norm(None, 0, None, None, 1e-5, None, 0, None, None, 0, 64, None) == L.NQ_OK
    assert lib.nq_layer_norm_fp8_block(None, 0, None, None, 1e-5, None, None, None, None, 0, 64, None) == L.NQ_OK
    assert lib.nq_layer_norm_grad(None, 0, None, None, None, None, 0, None, 0, None, None, 0, 64, None, 0, None) == L.NQ_OK
    assert lib.nq_layer_norm_grad_workspace_bytes(0, 64) == 0


@pytest.mark.parametrize("N,K", [(1, 16), (128, 128), (129, 144), (300, 960)])
def test_weight_quantisation(N, K):
    rng = np.random.default_rng(N + K)
    w = rng.standard_normal((N, K)).astype(np.float32)
    if N > 128:
        w[128:, :128] = 0.0
    q, s = F.quantize_fp8_block(w)
    assert q.shape == (N, K) and s.shape == (-(-N // 128), -(-K // 128)) and s.dtype == np.float32
    n, k = np.arange(N) // 128, np.arange(K) // 128
    full = s.astype(np.float64)[n][:, k]
    got = O.e4m3_decode(q).reshape(N, K).astype(np.float64) * full
    # half a step: 2^-4 of the value, or half of the smallest subnormal step under the scale; the fp32 quotient's own 2^-24
    assert (np.abs(got - w) <= np.maximum(2.0 ** -4 * np.abs(w), 2.0 ** -10 * full) * (1 + 2.0 ** -20)).all()
    if N > 128:
        assert s[1, 0] == 1.0 and not got[128:, :128].any()
    # the largest magnitude of each block meets the largest code
    assert (np.abs(O.e4m3_decode(q).reshape(N, K)).max() == 448.0)

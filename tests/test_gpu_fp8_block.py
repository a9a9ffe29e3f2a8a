"""The block-scaled fp8 linear on the GPU: the row quantiser bit for bit against IEEE divisions and the oracle's encoder,
the product and its input gradient against 64-bit products of the values that codes and scales stand for, with bounds
counted from the roundings (tests/fp8_block_ref.py)."""
import numpy as np
import pytest
import torch

import fp8_block_ref as R
from noeira_amd import NQError
from noeira_amd import _lib as L
from noeira_amd import formats as F
from noeira_amd.qlinear import FP8BlockLinear, FP8Linear, FusedRows, quantize_rows_fp8_block

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]


def layer(wq, ws, **kw):
    lin = FP8BlockLinear(wq.shape[1], wq.shape[0], **kw)
    lin.set_weight(wq, ws)
    return lin


def bits(t):
    return t.contiguous().view(torch.uint8).cpu()


# ---- the row quantiser ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,K", [(1, 1), (1, 7), (3, 127), (2, 128), (5, 129), (4, 136), (7, 960), (3, 1001), (65, 2560), (2, 4104)])
def test_quantize_rows(M, K, dtype):
    rng = np.random.default_rng(M * 10007 + K)
    x = rng.standard_normal((M, K)) * np.exp(rng.normal(0, 3, (M, 1)))
    x[rng.random((M, K)) < 0.1] = 0.0
    if M > 2:
        x[1] = 0.0
    xt = torch.from_numpy(x.astype(np.float32)).to(dtype).cuda()
    want_q, want_s = R.quantize(xt.float().cpu().numpy())
    store = torch.full((M * K + 64,), 0x55, dtype=torch.uint8, device="cuda")
    sstore = torch.full((want_s.size + 16,), -7.0, device="cuda")
    codes, scales = quantize_rows_fp8_block(xt, store[: M * K].view(M, K), sstore[: want_s.size].view(want_s.shape))
    assert np.array_equal(scales.cpu().numpy().view(np.uint32), want_s.view(np.uint32))
    assert np.array_equal(codes.cpu().numpy(), want_q)
    assert (store[M * K:] == 0x55).all() and (sstore[want_s.size:] == -7.0).all()
    again = quantize_rows_fp8_block(xt)
    assert again[0].dtype == torch.float8_e4m3fn and torch.equal(bits(again[0]), bits(codes)) and torch.equal(again[1], scales)


def test_quantize_ties_go_to_even_and_quotients_are_ieee():
    """A block whose scale is a power of two meets every tie exactly; random fp32 significands meet every remainder."""
    step = np.concatenate([np.arange(0, 449, 0.5), np.arange(0, 36, 1 / 64)]).astype(np.float32)
    x = np.zeros((8, -(-step.size // 127) * 128), np.float32)
    for i, part in enumerate(np.array_split(step, x.shape[1] // 128)):
        x[:, i * 128] = 448.0
        x[:, i * 128 + 1: i * 128 + 1 + part.size] = part
    x *= (2.0 ** np.array([0, -8, 8, -100, 100, -60, -118, 118]))[:, None].astype(np.float32)
    x[1::2] *= -1
    rng = np.random.default_rng(4)
    y = (rng.integers(1 << 23, 1 << 24, (64, 4096)).astype(np.float64) * 2.0 ** rng.integers(-33, -23, (64, 4096))).astype(np.float32)
    y *= (2.0 ** rng.integers(-110, 110, (64, 1))).astype(np.float32)
    for v in (x, y):
        want_q, want_s = R.quantize(v)
        codes, scales = quantize_rows_fp8_block(torch.from_numpy(v).cuda())
        assert np.array_equal(scales.cpu().numpy().view(np.uint32), want_s.view(np.uint32))
        assert np.array_equal(codes.view(torch.uint8).cpu().numpy(), want_q)


def test_quantize_against_device_divisions():
    """Half a million blocks against the device's own divisions and casts: every scale's significand a random one, among
    them all ones (the largest magnitudes 448 (2 - 2^-23) 2^e)."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(16384, 4096, generator=gen, device="cuda") * torch.exp2(torch.randint(-40, 40, (16384, 1), generator=gen, device="cuda").float())
    ones = 448 * (2 - 2.0 ** -23)  # 27 significant bits: the nearest fp32 values on both sides have quotients around it
    x[:64, 0] = torch.tensor([np.nextafter(np.float32(ones), np.float32(s)) for s in (0, 1e9)] * 32, device="cuda") * 8
    x[:64, 1:128].clamp_(-3000, 3000)
    t = x.view(16384, 32, 128)
    top = t.abs().amax(2)
    s = top / torch.full_like(top, 448)
    want = (t / s[:, :, None]).to(torch.float8_e4m3fn)
    codes, scales = quantize_rows_fp8_block(x)
    assert torch.equal(scales, s)
    assert torch.equal(codes.view(torch.uint8), want.view(16384, 4096).view(torch.uint8))


def test_quantize_extremes():
    tiny, huge, inf, nan = 2.0 ** -149, 3.4028235e38, np.inf, np.nan
    x = np.zeros((9, 384), np.float32)
    x[0, :128] = tiny
    x[1, 5], x[1, 6] = huge, -1.0
    x[2, 130] = nan
    x[3, 260], x[3, 261] = inf, 2.0
    x[4, :] = -huge
    x[5, 0], x[5, 1] = 2.0 ** -126, 3 * tiny
    x[6, :] = -0.0
    x[7, 0], x[7, 128] = 448 * 2.0 ** -126, 447 * 2.0 ** -126
    x[8, 383] = -nan
    want_q, want_s = R.quantize(x)
    codes, scales = quantize_rows_fp8_block(torch.from_numpy(x).cuda())
    got_q, got_s = codes.view(torch.uint8).cpu().numpy(), scales.cpu().numpy()
    assert np.array_equal(np.isnan(got_s), np.isnan(want_s))
    assert np.array_equal(got_s[~np.isnan(got_s)], want_s[~np.isnan(want_s)]) and (got_s[~np.isnan(got_s)] >= 2.0 ** -126).all()
    # (the sign of a zero code is the quotient's own)
    assert np.array_equal(got_q, want_q)


# ---- the product ----------------------------------------------------------------------------------------------------

SHAPES = [(1, 16, 1), (1, 128, 16), (1, 960, 2560), (1, 4096, 1040), (2, 272, 129), (3, 144, 33), (5, 4096, 513), (16, 512, 3200),
          (17, 960, 320), (33, 1024, 100), (64, 2560, 960), (65, 2064, 700), (100, 3200, 512), (135, 960, 2567), (256, 960, 2560),
          (257, 512, 384), (300, 4096, 1040), (513, 1040, 257), (700, 640, 1300), (1024, 1024, 2048),
          # a hundred tiles of 256 x 256 and more: one block of K, part of one, two, an odd and an even number of them
          (2100, 128, 4100), (3000, 16, 2832), (2049, 256, 4104), (2304, 656, 4001), (4096, 1024, 2048),
          # the other tiles of the GEMM, and tiles left over after the last full round
          (500, 496, 4001), (1000, 512, 4000), (2045, 528, 4090), (4093, 272, 4345),
          # the blocks of K dealt over two groups of wavefronts: one block, an odd and an even number, part of a last one
          (220, 16, 5000), (313, 128, 4001), (190, 256, 3000), (282, 272, 5000), (282, 400, 5000), (500, 1408, 3001), (700, 1040, 2050),
          (4000, 784, 500), (512, 3200, 2100)]


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_product(M, K, N, dtype):
    gen = torch.Generator().manual_seed(M * 31 + K * 7 + N)
    xq, xs = R.random_rows(gen, M, K)
    wq, ws = R.random_weight(gen, N, K)
    lin = layer(wq, ws)
    x, w = R.rows(xq, xs), R.matrix(wq, ws)
    y = x @ w.t()
    store = torch.full((M * N + 64,), 77.0, dtype=dtype, device="cuda")
    got = lin.forward_a8(xq, xs, out=store[: M * N].view(M, N), out_dtype=dtype)
    R.assert_within(got, y, R.product_bound(x, w, y, None, dtype), "plain")
    assert (store[M * N:] == 77.0).all()
    assert torch.equal(bits(lin.forward_a8(xq, xs, out_dtype=dtype)), bits(got))
    for bdt in DTYPES:
        bias = torch.randn(N, generator=gen).to(bdt).cuda()
        z = y + bias.double()
        got = lin.forward_a8(xq, xs, bias=bias, epilogue="relu", out_dtype=dtype)
        R.assert_within(got, z.clamp(min=0), R.product_bound(x, w, z, bias.double(), dtype), "bias and ReLU")


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(3, 272, 132), (40, 960, 129), (300, 512, 260), (700, 144, 1001), (1100, 256, 2560), (2100, 128, 4100)])
def test_output_that_begins_on_four_bytes(M, K, N, dtype):
    """An output 4 but not 16 bytes aligned gets the aligned one's bits, and nothing beside it is written."""
    gen = torch.Generator().manual_seed(M + N)
    xq, xs = R.random_rows(gen, M, K)
    lin = layer(*R.random_weight(gen, N, K))
    want = lin.forward_a8(xq, xs, out_dtype=dtype)
    first = 4 // want.element_size()
    store = torch.full((M * N + 64,), 77.0, dtype=dtype, device="cuda")
    lin.forward_a8(xq, xs, out=store[first: first + M * N].view(M, N), out_dtype=dtype)
    assert torch.equal(bits(store[first: first + M * N].view(M, N)), bits(want))
    assert (store[:first] == 77.0).all() and (store[first + M * N:] == 77.0).all()


def test_weights_set_again():
    """A second set of weights, from the device or the host, replaces the first, W^T with it; dropping the logical bytes
    leaves the layer running."""
    gen = torch.Generator().manual_seed(8)
    xq, xs = R.random_rows(gen, 70, 272)
    gq, gs = R.random_rows(gen, 70, 144)
    lin = FP8BlockLinear(272, 144, grad=True)
    for turn in range(4):
        wq, ws = R.random_weight(gen, 144, 272)
        if turn % 2:
            lin.set_weight(wq.cpu().numpy(), ws.cpu().numpy())
            L.check(L.lib().nq_keep_only_repacked(lin._h))
        else:
            lin.set_weight(wq, ws)
        x, g, w = R.rows(xq, xs), R.rows(gq, gs), R.matrix(wq, ws)
        R.assert_within(lin.forward_a8(xq, xs, out_dtype=torch.float32), x @ w.t(), R.product_bound(x, w, x @ w.t(), None, torch.float32), "y")
        R.assert_within(lin.vjp_a8(gq, gs), g @ w, R.product_bound(g, w.t(), g @ w, None, torch.float32), "gx")
    buf = np.empty(144 * 272, np.uint8)
    with pytest.raises(NQError, match="no blocks are kept"):
        L.check(L.lib().nq_get_blocks(lin._h, buf.ctypes.data, buf.size))


def test_dequantize_and_device_bytes():
    gen = torch.Generator().manual_seed(3)
    for N, K in ((1, 16), (129, 272), (300, 960)):
        wq, ws = R.random_weight(gen, N, K)
        lin = layer(wq, ws)
        want = (R.decode(wq).float() * ws[torch.arange(N) // 128][:, torch.arange(K) // 128])
        assert torch.equal(lin.dequantized_dev(), want)
        tiles = -(-N // 16) * -(-K // 128) * 2048
        assert lin.device_bytes() == tiles + 4 * ws.numel()
        host = FP8BlockLinear(K, N)
        host.set_weight(wq.cpu().numpy(), ws.cpu().numpy())
        assert torch.equal(host.dequantized_dev(), want)
        buf = np.empty(N * K, np.uint8)
        L.check(L.lib().nq_get_blocks(host._h, buf.ctypes.data, buf.size))
        assert np.array_equal(buf.reshape(N, K), wq.cpu().numpy())
        with pytest.raises(NQError, match="no blocks are kept"):
            L.check(L.lib().nq_get_blocks(lin._h, buf.ctypes.data, buf.size))


@pytest.mark.parametrize("M", [1, 3, 40, 300])
def test_a_nan_stays_in_its_row_or_column(M):
    """K ends inside a block: what lies behind a row's end is the next row's beginning, and must count as zero."""
    K, N = 144, 160
    gen = torch.Generator().manual_seed(M)
    xq, xs = R.random_rows(gen, M, K)
    wq, ws = R.random_weight(gen, N, K)
    clean = layer(wq, ws).forward_a8(xq, xs, out_dtype=torch.float32)
    bad = xq.clone()
    bad[M // 2, :16] = 0x7F
    got = layer(wq, ws).forward_a8(bad, xs, out_dtype=torch.float32)
    keep = torch.arange(M, device="cuda") != M // 2
    assert torch.isnan(got[M // 2]).all() and torch.equal(got[keep], clean[keep])
    sc = xs.clone()
    sc[M // 2, 1] = float("nan")
    got = layer(wq, ws).forward_a8(xq, sc, out_dtype=torch.float32)
    assert torch.isnan(got[M // 2]).all() and torch.equal(got[keep], clean[keep])
    wbad = wq.clone()
    wbad[130, 143] = 0xFF
    got = layer(wbad, ws).forward_a8(xq, xs, out_dtype=torch.float32)
    cols = torch.arange(N, device="cuda") != 130
    assert torch.isnan(got[:, 130]).all() and torch.equal(got[:, cols], clean[:, cols])
    # ReLU's rule: a NaN becomes 0
    assert (layer(wq, ws).forward_a8(bad, xs, epilogue="relu", out_dtype=torch.float32)[M // 2] == 0).all()


def test_infinite_scales_follow_ieee():
    xq = torch.full((3, 256), 0x38, dtype=torch.uint8, device="cuda")  # ones
    xs = torch.ones((3, 2), device="cuda")
    xs[1, 0] = float("inf")
    wq = torch.full((32, 256), 0x38, dtype=torch.uint8, device="cuda")
    wq[1] = 0xB8  # minus ones
    wq[2] = 0
    got = layer(wq, torch.ones((1, 2), device="cuda")).forward_a8(xq, xs, out_dtype=torch.float32)
    assert got[0, 0] == 256 and got[0, 1] == -256 and got[0, 2] == 0
    assert got[1, 0] == float("inf") and got[1, 1] == -float("inf") and torch.isnan(got[1, 2])


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(220, 384, 3000), (500, 1408, 3001), (700, 1040, 2050)])
def test_an_odd_number_of_blocks_over_two_groups(M, K, N, dtype):
    """The second group of wavefronts has a block less: what it does instead adds nothing, also where the last block's
    scales are infinite or its codes NaN."""
    G = -(-K // 128)
    xq = torch.full((M, K), 0x38, dtype=torch.uint8, device="cuda")  # ones
    xs = torch.ones((M, G), device="cuda")
    xs[1, G - 1] = float("inf")
    xq[2, K - 1] = 0x7F
    xs[M - 1, G - 1] = 0.0
    wq = torch.full((N, K), 0x38, dtype=torch.uint8, device="cuda")
    wq[1] = 0xB8  # minus ones
    wq[2] = 0
    wq[N - 1, K - 2] = 0xFF
    ws = torch.ones((-(-N // 128), G), device="cuda")
    ws[1, G - 1] = float("inf")  # channels 128 .. 255
    got = layer(wq, ws).forward_a8(xq, xs, out_dtype=dtype).float()
    assert got[0, 0] == K and got[0, 1] == -K and got[0, 2] == 0 and got[0, 300] == K  # (below 2^11 and whole 16s: exact in bf16)
    assert got[1, 0] == float("inf") and got[1, 1] == -float("inf") and torch.isnan(got[1, 2])
    assert torch.isnan(got[2]).all() and torch.isnan(got[:, N - 1]).all()
    assert (got[3:M - 1, 128:256] == float("inf")).all() and (got[3:M - 1, 256:N - 1] == K).all()
    rest = (G - 1) * 128
    assert got[M - 1, 0] == rest and torch.isnan(got[M - 1, 128:256]).all() and (got[M - 1, 256:N - 1] == rest).all()


def test_nothing_and_refusals():
    gen = torch.Generator().manual_seed(1)
    wq, ws = R.random_weight(gen, 48, 256)
    lin = layer(wq, ws)
    assert lin.forward_a8(torch.empty((0, 256), dtype=torch.uint8, device="cuda"), torch.empty((0, 2), device="cuda")).shape == (0, 48)
    xq, xs = R.random_rows(gen, 4, 256)
    with pytest.raises(NQError, match="scales has 6 values, expected 8"):
        lin.forward_a8(xq, xs.view(-1)[:6])
    with pytest.raises(NQError, match="codes must be"):
        lin.forward_a8(xq.float(), xs)
    with pytest.raises(NQError, match="contiguous"):
        lin.forward_a8(xq, xs.t())
    with pytest.raises(NQError, match="expected 192"):
        lin.forward_a8(xq, xs, out=torch.empty((3, 48), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(NQError, match="are needed"):
        lin.forward_a8(xq, None)
    with pytest.raises(NQError, match="epilogue"):
        lin.forward_a8(xq, xs, epilogue="swiglu")
    with pytest.raises(NQError, match="bias has 47 values"):
        lin.forward_a8(xq, xs, bias=torch.zeros(47, device="cuda"))
    with pytest.raises(NQError, match="not a multiple of 256"):
        lin.forward_a8(xq.view(-1)[:1000], xs)
    with pytest.raises(NQError, match="made with|NQ_FLAG_GRAD"):
        lin.vjp_a8(*R.random_rows(gen, 4, 48))
    x = torch.randn(4, 256, device="cuda")
    y = torch.empty((4, 48), device="cuda")
    rc = L.lib().nq_forward(lin._h, x.data_ptr(), L.DT_F32, None, y.data_ptr(), L.DT_F32, 4, None, 0, 0, None)
    assert rc == L.NQ_ERR_INVALID and "takes e4m3 codes" in L.last_error()
    rc = L.lib().nq_diag_forward_a16(lin._h, x.data_ptr(), L.DT_F32, y.data_ptr(), L.DT_F32, 4, 1, 1, None)
    assert rc == L.NQ_ERR_UNSUPPORTED
    other = FP8Linear(256, 48)
    other.set_weight(wq.cpu().numpy(), 0.5)
    with pytest.raises(NQError, match="share format"):
        FusedRows([other, lin])
    with pytest.raises(NQError, match="multiple of 128 rows"):
        FusedRows([lin, lin])
    with pytest.raises(NQError, match="Q4_0, W4_GROUP"):
        from noeira_amd.qlinear import FusedGLU
        FusedGLU(lin, lin)


@pytest.mark.parametrize("M", [1, 7, 40, 300])
def test_fused_rows(M):
    """q | k | v as one layer: every part's output has the values of its own layer."""
    gen = torch.Generator().manual_seed(M)
    parts = [R.random_weight(gen, n, 960) for n in (384, 128, 200)]
    layers = [layer(*p) for p in parts]
    fused = FusedRows(layers)
    xq, xs = R.random_rows(gen, M, 960)
    x = R.rows(xq, xs)
    bias = torch.randn(712, generator=gen).cuda()
    outs = fused.forward(xq, xs, bias=bias, out_dtype=torch.float32)
    at = 0
    for p, o in zip(parts, outs):
        w, b = R.matrix(*p), bias[at: at + p[0].shape[0]].double()
        y = x @ w.t() + b
        R.assert_within(o, y, R.product_bound(x, w, y, b, torch.float32), "part")
        at += p[0].shape[0]
    whole = torch.cat([R.matrix(*p) for p in parts])
    assert torch.equal(fused_dequantized(fused, 712, 960), whole.float())
    with pytest.raises(NQError):
        fused.forward(xq, xs[:, :7].contiguous())


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M", [1100, 2200])
def test_fused_rows_of_a_batch(M, dtype):
    """Rows enough for the GEMM, whose tiles then lie across the parts' boundaries: values of the parts, with a bias
    across all of them (the blocks may be added in another order than in a part's own call)."""
    gen = torch.Generator().manual_seed(2)
    parts = [R.random_weight(gen, n, 1040) for n in (2048, 1024, 1030)]
    fused = FusedRows([layer(*p) for p in parts])
    xq, xs = R.random_rows(gen, M, 1040)
    x = R.rows(xq, xs)
    for bias in (None, torch.randn(4102, generator=gen).to(dtype).cuda()):
        outs = fused.forward(xq, xs, bias=bias, epilogue="relu", out_dtype=dtype)
        at = 0
        for p, o in zip(parts, outs):
            n, w = p[0].shape[0], R.matrix(*p)
            own = None if bias is None else bias[at: at + n].double()
            z = x @ w.t() if own is None else x @ w.t() + own
            R.assert_within(o, z.clamp(min=0), R.product_bound(x, w, z, own, dtype), "part")
            at += n


def test_fused_rows_refusals():
    gen = torch.Generator().manual_seed(4)
    fused = FusedRows([layer(*R.random_weight(gen, 128, 256)), layer(*R.random_weight(gen, 40, 256))])
    xq, xs = R.random_rows(gen, 4, 256)
    with pytest.raises(NQError, match="are needed"):
        fused.forward(xq)
    with pytest.raises(NQError, match="codes must be"):
        fused.forward(torch.zeros((4, 256), device="cuda"), xs)
    with pytest.raises(NQError, match="output has 159 values, expected 160"):
        fused.forward(xq, xs, outs=[torch.empty((4, 128), device="cuda"), torch.empty(159, device="cuda")])
    with pytest.raises(NQError, match="output must be torch.float32"):
        fused.forward(xq, xs, outs=[torch.empty((4, n), device="cuda", dtype=torch.bfloat16) for n in (128, 40)])
    with pytest.raises(NQError, match="outputs for a layer of"):
        fused.forward(xq, xs, outs=[torch.empty((4, 128), device="cuda")])
    with pytest.raises(NQError, match="bias has 167 values"):
        fused.forward(xq, xs, bias=torch.zeros(167, device="cuda"))


def fused_dequantized(fused, N, K):
    out = torch.empty((N, K), device="cuda")
    L.check(L.lib().nq_dequantize(fused._h, out.data_ptr(), out.numel(), torch.cuda.current_stream().cuda_stream))
    return out


# ---- the input gradient ---------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(1, 16, 16), (1, 960, 2560), (3, 144, 48), (33, 272, 144), (65, 2560, 960), (256, 960, 2576), (515, 1040, 512)])
def test_grad_input(M, K, N, dtype):
    gen = torch.Generator().manual_seed(M + K + N)
    wq, ws = R.random_weight(gen, N, K)
    lin = layer(wq, ws, grad=True)
    gq, gs = R.random_rows(gen, M, N)
    g, w = R.rows(gq, gs), R.matrix(wq, ws)
    want = g @ w
    store = torch.full((M * K + 64,), 5.0, dtype=dtype, device="cuda")
    got = lin.vjp_a8(gq, gs, grad_input=store[: M * K].view(M, K), out_dtype=dtype)
    R.assert_within(got, want, R.product_bound(g, w.t(), want, None, dtype), "gx")
    assert (store[M * K:] == 5.0).all()
    tiles, tiles_t = -(-N // 16) * -(-K // 128) * 2048, -(-K // 16) * -(-N // 128) * 2048
    assert lin.device_bytes() == tiles + tiles_t + 8 * ws.numel()


def test_gradient_against_differences():
    """The layer is linear in the values its codes stand for, so a difference of two forwards along a direction of codes
    is the derivative itself: sum gy (y(x + v) - y(x)) = sum gx v, up to the outputs' own error bounds."""
    gen = torch.Generator().manual_seed(8)
    M, K, N = 24, 272, 144
    wq, ws = R.random_weight(gen, N, K)
    lin = layer(wq, ws, grad=True)
    aq, s = R.random_rows(gen, M, K)
    bq = R.random_rows(gen, M, K)[0]
    gq, gs = R.random_rows(gen, M, N)
    a, b, g, w = R.rows(aq, s), R.rows(bq, s), R.rows(gq, gs), R.matrix(wq, ws)
    ya, yb = (lin.forward_a8(q, s, out_dtype=torch.float32).double() for q in (aq, bq))
    gx = lin.vjp_a8(gq, gs).double()
    lhs, rhs = (g * (yb - ya)).sum(), (gx * (b - a)).sum()
    bound = (g.abs() * (R.product_bound(a, w, a @ w.t(), None, torch.float32) + R.product_bound(b, w, b @ w.t(), None, torch.float32))).sum() \
        + ((b - a).abs() * R.product_bound(g, w.t(), g @ w, None, torch.float32)).sum()
    assert (lhs - rhs).abs() <= bound and lhs.abs() > 100 * bound


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
def test_forward_and_vjp_quantise_their_rows(dtype):
    """`forward` and `vjp` of fp32 / bf16 rows are the quantiser followed by the product, bit for bit."""
    gen = torch.Generator().manual_seed(2)
    wq, ws = R.random_weight(gen, 208, 960)
    lin = layer(wq, ws, grad=True)
    x = torch.randn(37, 960, generator=gen).to(dtype).cuda()
    gy = torch.randn(37, 208, generator=gen).to(dtype).cuda()
    bias = torch.randn(208, generator=gen).cuda()
    assert torch.equal(lin.forward(x, bias=bias), lin.forward_a8(*quantize_rows_fp8_block(x), bias=bias))
    assert torch.equal(lin.vjp(x, gy), lin.vjp_a8(*quantize_rows_fp8_block(gy)))


def test_from_linear():
    rng = np.random.default_rng(6)
    w, b = rng.standard_normal((256, 200)).astype(np.float32), rng.standard_normal(200).astype(np.float32)
    lin = FP8BlockLinear.from_linear(w, b)
    x = torch.from_numpy(rng.standard_normal((19, 256)).astype(np.float32)).cuda()
    xq, xs = quantize_rows_fp8_block(x)
    q, s = (torch.from_numpy(t).cuda() for t in F.quantize_fp8_block(np.ascontiguousarray(w.T)))
    xv, wv, bv = R.rows(xq, xs), R.matrix(q, s), torch.from_numpy(b).cuda().double()
    y = xv @ wv.t() + bv
    R.assert_within(lin.forward(x, out_dtype=torch.float32), y, R.product_bound(xv, wv, y, bv, torch.float32), "from_linear")


# ---- offsets beyond 32 bits -----------------------------------------------------------------------------------------


def test_rows_and_outputs_beyond_four_gigabytes():
    """The last rows of calls whose codes, or whose outputs, end beyond 2^32 bytes."""
    gen = torch.Generator().manual_seed(12)
    for M, K, N, dtype in ((1048583, 4112, 24, torch.bfloat16), (140009, 144, 8200, torch.float32)):
        wq, ws = R.random_weight(gen, N, K)
        lin = layer(wq, ws)
        xq = torch.zeros((M, K), dtype=torch.uint8, device="cuda")
        xs = torch.ones((M, -(-K // 128)), device="cuda")
        tail = R.random_rows(gen, 70, K)
        xq[-70:], xs[-70:] = tail
        assert max(xq.numel(), M * N * torch.finfo(dtype).bits // 8) > 2 ** 32
        y = lin.forward_a8(xq, xs, out_dtype=dtype)
        assert not y[:-70].any()
        x, w = R.rows(*tail), R.matrix(wq, ws)
        R.assert_within(y[-70:], x @ w.t(), R.product_bound(x, w, x @ w.t(), None, dtype), "last rows")
        del y, xq
    x = torch.zeros((2097169, 1040), dtype=torch.bfloat16, device="cuda")
    x[-9:] = torch.randn(9, 1040, generator=gen).to(torch.bfloat16).cuda()
    codes, scales = quantize_rows_fp8_block(x)
    want = quantize_rows_fp8_block(x[-9:].contiguous())
    assert torch.equal(bits(codes[-9:]), bits(want[0])) and torch.equal(scales[-9:], want[1])
    assert not codes[:-9].view(torch.uint8).any() and (scales[:-9] == 1).all()


# ---- streams, graphs ------------------------------------------------------------------------------------------------


def test_recorded_into_graphs_and_on_two_streams():
    """Two captured graphs of one layer, replayed in turn and at once on two streams with eager work between, return the
    eager bits; the quantiser and the gradient are recorded along."""
    gen = torch.Generator().manual_seed(5)
    wq, ws = R.random_weight(gen, 528, 960)
    lin = layer(wq, ws, grad=True)
    xs = [torch.randn(m, 960, generator=gen).cuda() for m in (1, 150)]
    gys = [torch.randn(m, 528, generator=gen).cuda() for m in (1, 150)]

    def step(x, gy):
        return lin.forward(x), lin.vjp(x, gy)

    graphs, outs, ins = [], [], []
    for x, gy in zip(xs, gys):
        step(x, gy)
        torch.cuda.synchronize()
        ins.append((x.clone(), gy.clone()))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*ins[-1]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        for k in (0, 1):
            ins[k][0].copy_(xs[k] * (turn + 1.5))
            ins[k][1].copy_(gys[k] * (turn - 0.5))
        torch.cuda.synchronize()
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            for got, want in zip(outs[k], step(*ins[k])):
                assert torch.equal(got, want), (turn, k)
    a, b = (torch.cuda.Stream(), torch.cuda.Stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        ya = [lin.forward(xs[1]) for _ in range(4)]
    with torch.cuda.stream(b):
        yb = [lin.forward(xs[0]) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, lin.forward(xs[1])) for t in ya) and all(torch.equal(t, lin.forward(xs[0])) for t in yb)


def test_output_types():
    """y and gx are of `out_dtype`, of the given output's type without one, and bf16 / fp32 where neither is given."""
    gen = torch.Generator().manual_seed(9)
    wq, ws = R.random_weight(gen, 144, 272)
    lin = layer(wq, ws, grad=True)
    x, gy = torch.randn(5, 272, generator=gen).cuda(), torch.randn(5, 144, generator=gen).cuda()
    codes, grads = quantize_rows_fp8_block(x), quantize_rows_fp8_block(gy)
    for dtype in DTYPES:
        y, gx = torch.empty((5, 144), dtype=dtype, device="cuda"), torch.empty((5, 272), dtype=dtype, device="cuda")
        want, wantx = lin.forward_a8(*codes, out_dtype=dtype), lin.vjp_a8(*grads, out_dtype=dtype)
        assert want.dtype == wantx.dtype == dtype
        for call in (lambda: lin.forward_a8(*codes, out=y), lambda: lin.forward(x, out=y), lambda: lin.forward(x, out=y, out_dtype=dtype)):
            y.fill_(7.0)
            assert call() is y and torch.equal(y, want)
        for call in (lambda: lin.vjp_a8(*grads, grad_input=gx), lambda: lin.vjp(None, gy, grad_input=gx),
                     lambda: lin.vjp(None, gy, gx, out_dtype=dtype)):
            gx.fill_(7.0)
            assert call() is gx and torch.equal(gx, wantx)
    assert lin.forward(x).dtype == torch.bfloat16 and lin.vjp(None, gy).dtype == torch.float32
    with pytest.raises(NQError, match="out must be torch.float32"):
        lin.forward_a8(*codes, out=y, out_dtype=torch.float32)
    with pytest.raises(NQError, match="grad_input must be torch.float32"):
        lin.vjp_a8(*grads, grad_input=gx, out_dtype=torch.float32)
    with pytest.raises(NQError, match="fp32 or bf16"):
        lin.forward_a8(*codes, out=y.half())

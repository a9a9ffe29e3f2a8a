"""Layer norm and its gradient on the GPU against 64 bits, with bounds counted from the roundings, and the chain it is
made for: norm -> codes -> block-scaled projection, and the gradients back through both."""
import numpy as np
import pytest
import torch

import fp8_block_ref as R
from noeira_amd import NQError
from noeira_amd.norm import LayerNorm
from noeira_amd.qlinear import FP8BlockLinear, quantize_rows_fp8_block

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16]
SHAPES = [(1, 1), (1, 7), (2, 64), (1, 960), (3, 127), (5, 129), (135, 960), (7, 1001), (33, 1024), (4, 2048), (3, 2567), (9, 4096),
          (2, 8192), (2, 11008), (3, 16391), (1030, 512)]
EPS = 1e-5


def inputs(M, D, dtype, seed=0):
    gen = torch.Generator().manual_seed(M * 13 + D + seed)
    x = torch.randn(M, D, generator=gen) * torch.exp(torch.randn(M, 1, generator=gen)) + 3 * torch.randn(M, 1, generator=gen)
    norm = LayerNorm(D, eps=EPS)
    norm.set_params(1 + 0.2 * torch.randn(D, generator=gen), 0.1 * torch.randn(D, generator=gen))
    return norm, x.to(dtype).cuda(), gen


def test_parameters_start_as_ones_and_zeros():
    norm = LayerNorm.make(5)
    assert (norm.gamma == 1).all() and (norm.beta == 0).all()
    with pytest.raises(NQError, match="expected \\[5\\]"):
        norm.set_params(np.ones(4, np.float32), np.zeros(5, np.float32))
    norm.set_params(np.arange(5, dtype=np.float32), np.ones(5, np.float32))
    assert norm.gamma[3] == 3


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,D", SHAPES)
def test_forward(M, D, dtype):
    norm, x, _ = inputs(M, D, dtype)
    y, mean, rstd, e_y, e_mean, r_rstd = R.norm(x, norm.gamma, norm.beta, EPS)
    for out_dtype in DTYPES:
        store = torch.full((M * D + 64,), 9.0, dtype=out_dtype, device="cuda")
        got, gm, gr = norm.forward_train(x, out=store[: M * D].view(M, D))
        R.assert_within(got, y, e_y + R.HALF_STEP[out_dtype] * (y.abs() + e_y), "y")
        R.assert_within(gm, mean, e_mean, "mean")
        R.assert_within(gr, rstd, rstd * r_rstd, "rstd")
        assert (store[M * D:] == 9.0).all()
        assert torch.equal(norm.forward(x, out_dtype=out_dtype), got)
    z = x.clone()
    norm.forward(z, out=z)
    assert torch.equal(z, norm.forward(x))


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,D", SHAPES)
def test_forward_into_codes(M, D, dtype):
    """The codes and scales are the quantiser's of the fp32 result, and lie within half a step of the 64-bit one."""
    norm, x, _ = inputs(M, D, dtype)
    codes, scales, mean, rstd = norm.forward_fp8_train(x)
    y32, m32, r32 = norm.forward_train(x, out_dtype=torch.float32)
    want_q, want_s = quantize_rows_fp8_block(y32)
    assert torch.equal(scales, want_s) and torch.equal(codes.view(torch.uint8), want_q.view(torch.uint8))
    assert torch.equal(mean, m32) and torch.equal(rstd, r32)
    y, _, _, e_y, _, _ = R.norm(x, norm.gamma, norm.beta, EPS)
    step = torch.maximum(2.0 ** -4 * (y.abs() + e_y), 2.0 ** -10 * scales.double()[:, torch.arange(D, device="cuda") // 128])
    R.assert_within(R.rows(codes, scales), y, step * (1 + 2.0 ** -20) + e_y, "values")
    again = norm.forward_fp8(x)
    assert torch.equal(again[0].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(again[1], scales)


@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,D", [(8193, 7), (20000, 64), (9001, 1001), (2100, 1032), (2050, 2567), (2100, 4096), (1500, 4104), (1030, 8191),
                                 (700, 8200), (530, 11007), (600, 16384)])
def test_more_rows_than_teams(M, D, dtype):
    """More rows than the chip holds teams of 64, 256, 512 and 1024 threads (8192, 2048, 1024 and 512): a team walks several,
    the next one requested before the current one is done; y as values and as codes, in place too."""
    norm, x, _ = inputs(M, D, dtype, 7)
    y, mean, rstd, e_y, e_mean, r_rstd = R.norm(x, norm.gamma, norm.beta, EPS)
    got, gm, gr = norm.forward_train(x)
    R.assert_within(got, y, e_y + R.HALF_STEP[dtype] * (y.abs() + e_y), "y")
    R.assert_within(gm, mean, e_mean, "mean")
    R.assert_within(gr, rstd, rstd * r_rstd, "rstd")
    codes, scales, cm, cr = norm.forward_fp8_train(x)
    want = quantize_rows_fp8_block(norm.forward(x, out_dtype=torch.float32))
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])
    assert torch.equal(cm, gm) and torch.equal(cr, gr)
    z = x.clone()
    norm.forward(z, out=z)
    assert torch.equal(z, got)


@pytest.mark.parametrize("D", [20, 960, 1001, 16391])
def test_rows_at_the_ends_of_fp32(D):
    """Statistics are fp32: a row whose squares overflow has rstd 0 and y = beta, one whose squares vanish has
    rstd = 1 / sqrt(eps); without eps a row of one value has rstd infinite and y NaN, as the formula says, and its
    neighbours keep their bits."""
    norm, x, gen = inputs(4, D, torch.float32, 8)
    sign = torch.where(torch.rand(D, generator=gen) < 0.5, -1.0, 1.0).cuda()
    sign[:2] = torch.tensor([1.0, -1.0])
    clean = norm.forward(x)
    x[1], x[2] = 1e25 * sign, 1e-30 * sign
    y, mean, rstd = norm.forward_train(x)
    assert rstd[1] == 0 and torch.equal(y[1], norm.beta)
    assert (rstd[2].double() * EPS ** 0.5 - 1).abs() <= 4 * R.U and (y[2] - norm.beta).abs().max() < 1e-24
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])
    codes, scales = norm.forward_fp8(x)
    assert torch.isfinite(scales).all() and torch.equal(scales[1], quantize_rows_fp8_block(norm.beta.view(1, D))[1][0])
    bare = LayerNorm(D, eps=0.0)
    x[1] = 0.5
    y, mean, rstd = bare.forward_train(x)
    assert rstd[1] == float("inf") and torch.isnan(y[1]).all() and torch.isfinite(y[[0, 3]]).all()
    assert torch.isnan(bare.forward_fp8(x)[1][1]).all() and torch.isfinite(bare.forward_fp8(x)[1][[0, 3]]).all()


@pytest.mark.parametrize("D", [1, 129, 960, 4096, 16391])
def test_constant_rows_and_far_means(D):
    """A row of one value has variance 0: y is beta exactly; a row far from zero loses what its mean's rounding costs, and
    no more (the variance is summed from centred values)."""
    norm, _, gen = inputs(3, D, torch.float32)
    x = torch.full((3, D), 0.75).cuda()
    x[1] = -8192.0
    x[2] = 0.0
    y, mean, rstd = norm.forward_train(x)
    assert torch.equal(y, norm.beta.expand(3, D)) and torch.equal(mean, x[:, 0])
    far = torch.randn(4, D, generator=gen).cuda() + 1e4
    want, _, _, e_y, _, _ = R.norm(far, norm.gamma, norm.beta, EPS)
    R.assert_within(norm.forward(far), want, e_y, "far mean")


@pytest.mark.parametrize("M", [65, 4097])
@pytest.mark.parametrize("D", [16, 20, 960, 1001])
def test_huge_constant_rows(D, M):
    """Rows of one huge power of two: xh is 0, and what lies behind the row in its block, or behind the last row, adds
    nothing, although mean x rstd is beyond fp32 there.  (2^116 sums exactly over the rows' powers of two; rstd is 2^20.)"""
    norm = LayerNorm(D, eps=2.0 ** -40)
    gen = torch.Generator().manual_seed(D)
    norm.set_params(1 + 0.2 * torch.randn(D, generator=gen), 0.1 * torch.randn(D, generator=gen))
    x = torch.full((M, D), 2.0 ** 116).cuda()
    codes, scales, mean, rstd = norm.forward_fp8_train(x)
    assert torch.equal(mean, x[:, 0]) and (rstd == 2.0 ** 20).all()
    want = quantize_rows_fp8_block(norm.beta.expand(M, D).contiguous())
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])
    assert torch.equal(norm.forward(x), norm.beta.expand(M, D))
    gy = torch.ones((M, D)).cuda()
    gx, dg, db = norm.vjp(x, mean, rstd, gy)
    assert (db == M).all() and not dg.any()
    a = norm.gamma.double()
    # the mean's additions and division, each within half a step of sums of at most sum |a|; the difference; x 2^20 is exact
    bound = 2.0 ** 20 * R.U * (2 * (D + 1) * a.abs().mean() + (a - a.mean()).abs())
    R.assert_within(gx, (2.0 ** 20 * (a - a.mean())).expand(M, D), bound.expand(M, D), "gx")


@pytest.mark.parametrize("D", [1040, 16400])
def test_rows_beyond_four_gigabytes(D):
    """The last rows of a call whose rows end beyond 2^32 bytes have the bits of a call of their own."""
    M = 2 ** 31 // D + 100
    norm, _, gen = inputs(1, D, torch.bfloat16)
    x = torch.ones((M, D), dtype=torch.bfloat16, device="cuda")
    x[-9:] = torch.randn(9, D, generator=gen).to(torch.bfloat16).cuda()
    own = x[-9:].clone()
    y, mean, rstd = norm.forward_train(x)
    want = norm.forward_train(own)
    assert torch.equal(y[-9:], want[0]) and torch.equal(mean[-9:], want[1]) and torch.equal(rstd[-9:], want[2])
    assert torch.equal(y[0], norm.beta.to(torch.bfloat16))
    codes, scales = norm.forward_fp8(x)
    wq, wsc = norm.forward_fp8(own)
    assert torch.equal(codes[-9:].view(torch.uint8), wq.view(torch.uint8)) and torch.equal(scales[-9:], wsc)
    gy = torch.zeros_like(x)
    gy[-9:] = 1.0
    gx, dg, db = norm.vjp(x, mean, rstd, gy)
    wx, wg, wb = norm.vjp(own, want[1], want[2], torch.ones_like(own))
    assert torch.equal(gx[-9:], wx) and not gx[:-9].any()
    assert torch.equal(db, wb) and torch.allclose(dg, wg, rtol=0, atol=20 * 9 * R.U * 8)  # nine terms below 8 in another order


def test_non_finite_rows_stay_alone():
    norm, x, _ = inputs(6, 960, torch.float32)
    clean = norm.forward(x)
    bad = x.clone()
    bad[1, 5], bad[4, 959] = float("nan"), float("inf")
    keep = torch.tensor([0, 2, 3, 5], device="cuda")
    got = norm.forward(bad)
    assert torch.isnan(got[1]).all() and torch.isnan(got[4]).all() and torch.equal(got[keep], clean[keep])
    codes, scales = norm.forward_fp8(bad)
    want = norm.forward_fp8(x)
    assert torch.isnan(scales[1]).all() and torch.isnan(scales[4]).all()
    assert torch.equal(scales[keep], want[1][keep]) and torch.equal(codes.view(torch.uint8)[keep], want[0].view(torch.uint8)[keep])


@pytest.mark.parametrize("gdtype", DTYPES, ids=["gy f32", "gy bf16"])
@pytest.mark.parametrize("dtype", DTYPES, ids=["f32", "bf16"])
@pytest.mark.parametrize("M,D", SHAPES + [(1024, 65), (1025, 64), (4200, 129), (1900, 960), (700, 4095), (90, 8191), (300, 8191),
                                         (1100, 8192), (70, 11007), (800, 11007), (65, 16384)])
def test_gradients(M, D, dtype, gdtype):
    norm, x, gen = inputs(M, D, dtype, 1)
    gy = torch.randn(M, D, generator=gen).to(gdtype).cuda()
    _, mean, rstd = norm.forward_train(x)
    gx, dg, db, e_gx, e_dg, e_db = R.norm_grad(x, mean, rstd, norm.gamma, gy)
    for out_dtype in DTYPES:
        store = torch.full((M * D + 64,), 9.0, dtype=out_dtype, device="cuda")
        got = norm.vjp(x, mean, rstd, gy, grad_input=store[: M * D].view(M, D))
        R.assert_within(got[0], gx, e_gx + R.HALF_STEP[out_dtype] * (gx.abs() + e_gx), "gx")
        R.assert_within(got[1], dg, e_dg, "dgamma")
        R.assert_within(got[2], db, e_db, "dbeta")
        assert (store[M * D:] == 9.0).all()
    again = norm.vjp(x, mean, rstd, gy)
    assert again[0].dtype == dtype and torch.equal(again[1], got[1]) and torch.equal(again[2], got[2])
    frozen = norm.vjp(x, mean, rstd, gy, params=False)
    assert frozen[1] is None and frozen[2] is None and torch.equal(frozen[0], again[0])
    # gx over gy's own memory, and over x's
    if dtype == gdtype:
        over = gy.clone()
        res = norm.vjp(x, mean, rstd, over, grad_input=over)
        assert torch.equal(over, again[0]) and torch.equal(res[1], again[1])
    over = x.clone()
    res = norm.vjp(over, mean, rstd, gy, grad_input=over)
    assert torch.equal(over, again[0]) and torch.equal(res[1], again[1])


def test_gradients_against_differences():
    """Central differences of the 64-bit formula along random directions: (L(x + h v) - L(x - h v)) / 2 h with
    L = sum gy y.  The third-order term of L along v is below 1e2 |v|^3 here, so at h = 1e-4 the difference is off by
    1e-6 of it; 1e-4 of the sum of magnitudes leaves room for both and is far below any missing term."""
    norm, x, gen = inputs(6, 200, torch.float32, 2)
    x = x / x.std(dim=1, keepdim=True)
    gy = torch.randn(6, 200, generator=gen).cuda()
    _, mean, rstd = norm.forward_train(x)
    gx, dg, db = norm.vjp(x, mean, rstd, gy)

    def loss(x, g, b):
        return (gy.double() * R.norm(x, g, b, EPS)[0]).sum()

    p = (x.double(), norm.gamma.double(), norm.beta.double())
    for k, grad in enumerate((gx, dg, db)):
        v = torch.randn(p[k].shape, generator=gen).cuda().double()
        h = 1e-4
        hi, lo = (loss(*[t + s * h * v if i == k else t for i, t in enumerate(p)]) for s in (1, -1))
        want, got = (hi - lo) / (2 * h), (grad.double() * v).sum()
        assert (want - got).abs() <= 1e-4 * (grad.double() * v).abs().sum(), k


def test_nothing_and_refusals():
    norm = LayerNorm(64)
    x = torch.empty((0, 64), device="cuda")
    assert norm.forward(x).shape == (0, 64)
    codes, scales, mean, rstd = norm.forward_fp8_train(x)
    assert codes.shape == (0, 64) and scales.shape == (0, 1) and mean.shape == (0,)
    gx, dg, db = norm.vjp(x, mean, rstd, x)
    assert gx.shape == (0, 64) and (dg == 0).all() and (db == 0).all()
    y = torch.randn(4, 64, device="cuda")
    with pytest.raises(NQError, match="not a multiple of DIM"):
        norm.forward(torch.randn(3, 65, device="cuda"))
    with pytest.raises(NQError, match="contiguous"):
        norm.forward(y.t())
    with pytest.raises(NQError, match="must be"):
        norm.forward(y.half())
    with pytest.raises(NQError, match="expected 256"):
        norm.forward(y, out=torch.empty((3, 64), device="cuda"))
    with pytest.raises(NQError, match="mean has 3 values"):
        norm.vjp(y, y[0, :3].contiguous(), y[0, :4].contiguous(), y)
    with pytest.raises(NQError, match="current device"):
        norm.forward(y.cpu())


def test_projection_with_a_norm_and_an_adapter():
    """`proj_fwd` with a norm: over a block-scaled layer the norm hands over codes, beside an adapter it hands over its
    values; every other layer reads the values too."""
    from noeira_amd.lora import LoRAAdapter, proj_fwd
    from noeira_amd.qlinear import QLinear

    norm, x, gen = inputs(21, 960, torch.float32, 4)
    lin = FP8BlockLinear(960, 320)
    wq, ws = R.random_weight(gen, 320, 960)
    lin.set_weight(wq, ws)
    w, bias = R.matrix(wq, ws), torch.randn(320, generator=gen).cuda()
    codes, scales = norm.forward_fp8(x)
    got = proj_fwd(lin, x, bias=bias, norm=norm)
    assert got.dtype == torch.float32 and torch.equal(got, lin.forward_a8(codes, scales, bias=bias, out_dtype=torch.float32))
    assert torch.equal(proj_fwd(lin, x), lin.forward(x, out_dtype=torch.float32))

    ad = LoRAAdapter(960, 320, 8, alpha=4.0)
    a, b = torch.randn(960, 8, generator=gen) * 0.05, torch.randn(8, 320, generator=gen) * 0.05
    ad.set_params(a.numpy(), b.numpy())
    xn = norm.forward(x)
    base = lin.forward(xn, bias=bias, out_dtype=torch.float32)
    got = proj_fwd(lin, x, adapter=ad, bias=bias, norm=norm)
    share = 0.5 * (xn.double() @ a.cuda().double()) @ b.cuda().double()
    mag = 0.5 * (xn.double().abs() @ a.cuda().double().abs()) @ b.cuda().double().abs()
    R.assert_within(got, base.double() + share, 1.01 * (960 + 8 + 8) * 2 * R.U * mag + R.U * (got.double().abs() + 1e-30), "adapter")
    with pytest.raises(NQError, match="fp32"):
        ad.forward_with(lin, xn, out_dtype=torch.bfloat16)
    with pytest.raises(NQError, match="differ in shape"):
        LoRAAdapter(960, 336, 8).forward_with(lin, xn)
    ad.merged = True
    assert torch.equal(ad.forward_with(lin, xn, out_dtype=torch.bfloat16), lin.forward(xn))
    assert torch.equal(proj_fwd(lin, x, adapter=ad, norm=norm), proj_fwd(lin, x, norm=norm))

    q = QLinear(960, 320)
    q.set_weight((torch.randn(320, 960, generator=gen) * 0.05).numpy())
    assert torch.equal(proj_fwd(q, x, norm=norm), q.forward(xn))


@pytest.mark.parametrize("M", [1, 21, 200])
def test_projection_codes_do_not_depend_on_who_else_reads_the_norm(M):
    """Over a block-scaled layer the rows' codes are the norm's fp32 result's, also for bf16 activations: an adapter of
    zeros beside the layer, or a Hessian that is being filled, leaves the projection's bits as they are."""
    from noeira_amd.gptq import HessianAccumulator
    from noeira_amd.lora import LoRAAdapter, proj_fwd

    norm, x, gen = inputs(M, 960, torch.bfloat16, 6)
    lin = FP8BlockLinear(960, 320)
    lin.set_weight(*R.random_weight(gen, 320, 960))
    bias = torch.randn(320, generator=gen).cuda()
    want = proj_fwd(lin, x, bias=bias, norm=norm)
    assert torch.equal(want, lin.forward_a8(*norm.forward_fp8(x), bias=bias, out_dtype=torch.float32))
    hessian = HessianAccumulator(960)
    assert torch.equal(proj_fwd(lin, x, bias=bias, norm=norm, hessian=hessian), want)
    assert hessian.rows == M
    assert torch.equal(proj_fwd(lin, x, bias=bias, norm=norm, adapter=LoRAAdapter(960, 320, 8)), want)
    assert torch.equal(proj_fwd(lin, x, bias=bias, norm=norm, adapter=LoRAAdapter(960, 320, 8), hessian=hessian), want)


def test_two_graphs_at_once():
    """Two recorded backward steps of one norm keep their partial sums apart: replayed together on two streams, each
    returns the eager bits."""
    norm, x, gen = inputs(1500, 1024, torch.bfloat16, 5)
    ins = [(x[:m].clone(), torch.randn(m, 1024, generator=gen).to(torch.bfloat16).cuda()) for m in (1500, 1490)]

    def step(x, gy):
        y, mean, rstd = norm.forward_train(x)
        return (y, mean, rstd) + norm.vjp(x, mean, rstd, gy)

    graphs, outs = [], []
    for a in ins:
        step(*a)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(3):
        for a in ins:
            a[0].mul_(0.5), a[1].add_(0.25)
        want = [step(*a) for a in ins]
        torch.cuda.synchronize()
        for _ in range(4):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            for got, w in zip(outs[k], want[k]):
                assert torch.equal(got, w), (turn, k)


def test_chain_forward_and_back():
    """Norm into codes, a fused q | k | v style projection, an output gradient back through the projection and the norm:
    each step against 64 bits on the step's own inputs, all of it recorded into a graph and replayed."""
    M, D, N = 135, 960, 1280
    norm, x, gen = inputs(M, D, torch.bfloat16, 3)
    wq, ws = R.random_weight(gen, N, D)
    lin = FP8BlockLinear(D, N, grad=True)
    lin.set_weight(wq, ws)
    gy = torch.randn(M, N, generator=gen).to(torch.bfloat16).cuda()

    def step(x, gy):
        codes, scales, mean, rstd = norm.forward_fp8_train(x)
        y = lin.forward_a8(codes, scales)
        gq, gs = quantize_rows_fp8_block(gy)
        gn = lin.vjp_a8(gq, gs, out_dtype=torch.float32)
        return (codes, scales, mean, rstd, y, gq, gs, gn) + norm.vjp(x, mean, rstd, gn)

    codes, scales, mean, rstd, y, gq, gs, gn, gx, dg, db = step(x, gy)
    xv, w, g = R.rows(codes, scales), R.matrix(wq, ws), R.rows(gq, gs)
    want = xv @ w.t()
    R.assert_within(y, want, R.product_bound(xv, w, want, None, torch.bfloat16), "y")
    want = g @ w
    R.assert_within(gn, want, R.product_bound(g, w.t(), want, None, torch.float32), "gn")
    wx, wg, wb, e_gx, e_dg, e_db = R.norm_grad(x, mean, rstd, norm.gamma, gn)
    R.assert_within(gx, wx, e_gx + 2.0 ** -8 * (wx.abs() + e_gx), "gx")
    R.assert_within(dg, wg, e_dg, "dgamma")
    R.assert_within(db, wb, e_db, "dbeta")

    xi, gi = x.clone(), gy.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(xi, gi)
    for k in range(3):
        xi.copy_(x.float() * (k + 1) + k)
        gi.copy_(gy.float() * (0.5 - k))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(xi, gi)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), k

"""References in 64 bits for the block-scaled fp8 linear and the layer norm in front of it, and how far fp32 arithmetic
may be from them.

Error bounds count roundings: u = 2^-24 is half a step of fp32, and a sum of n terms in any order is off by at most
n u times the sum of the terms' magnitudes (first order; the factor 1.01 below covers the rest)."""
import numpy as np
import torch

from oracle import oracle as O

U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def decode(codes):
    """e4m3fn codes (uint8 or float8 tensor) as fp64, by the oracle's table."""
    table = torch.from_numpy(O.e4m3_decode_table().astype(np.float64)).to(codes.device)
    return table[codes.view(torch.uint8).long()]


def rows(codes, scales):
    """[M, K] codes x [M, G] scales in fp64."""
    g = torch.arange(codes.shape[1], device=codes.device) // 128
    return decode(codes) * scales.double()[:, g]


def matrix(codes, scales):
    """[N, K] codes x [NB, KB] scales in fp64."""
    n = torch.arange(codes.shape[0], device=codes.device) // 128
    k = torch.arange(codes.shape[1], device=codes.device) // 128
    return decode(codes) * scales.double()[n][:, k]


def product_bound(x, w, y, bias, dtype):
    """|error| of y = x w^T + bias, element by element: a block's 128 products are exact and summed with truncation at
    worst (2 u each), its two scales and their use round three times, the blocks and the bias are added in some order.
    A bf16 y's blocks are summed by the fp8 matrix core, which aligns products to the largest of a group and drops what
    lies below its last place: with places down to 2^-18 of the largest (over two million dots of 128 on this GPU the
    error stayed below 2.2e-4 of the sum of magnitudes, 2^-12 = 2.4e-4), 128 products lose at most 128 * 2^-18 = 2^-11
    of the largest, which is at most the sum of the magnitudes."""
    G = -(-x.shape[1] // 128)
    mag = x.abs() @ w.abs().t()
    b = 1.01 * (2 * 128 + 3 + G + 2) * U * mag
    if dtype == torch.bfloat16:
        b = b + 2.0 ** -11 * mag
    if bias is not None:
        b = b + 1.01 * U * (y.abs() + bias.abs())
    return b + HALF_STEP[dtype] * (y.abs() + b) + 2.0 ** -126


def random_rows(gen, M, K, device="cuda"):
    """Codes and scales of M rows: every finite code, scales over several powers of two, some blocks zero."""
    q = torch.randint(0, 256, (M, K), generator=gen, dtype=torch.uint8)
    q[(q & 0x7F) == 0x7F] = 0x38
    s = torch.exp2(torch.empty(M, -(-K // 128)).uniform_(-9, -5, generator=gen))
    if M > 4:
        q[M // 3] = 0
    return q.to(device), s.to(device)


def random_weight(gen, N, K, device="cuda"):
    q = torch.randint(0, 256, (N, K), generator=gen, dtype=torch.uint8)
    q[(q & 0x7F) == 0x7F] = 0xB1
    s = torch.exp2(torch.empty(-(-N // 128), -(-K // 128)).uniform_(-12, -8, generator=gen))
    return q.to(device), s.to(device)


def quantize(x):
    """numpy fp32 [M, K] -> (codes uint8, scales fp32), IEEE divisions and the oracle's encoder."""
    x = np.asarray(x, np.float32)
    M, K = x.shape
    G = -(-K // 128)
    codes, scales = np.empty((M, K), np.uint8), np.empty((M, G), np.float32)
    for g in range(G):
        part = x[:, g * 128:(g + 1) * 128]
        top = np.abs(part).max(axis=1)
        with np.errstate(all="ignore"):
            s = np.maximum((top / np.float32(448)).astype(np.float32), np.float32(2.0 ** -126))
            s = np.where(top == 0, np.float32(1), s)
            q = (part / s[:, None]).astype(np.float32)
            c = O.e4m3_encode(np.clip(np.nan_to_num(q), -448, 448).astype(np.float32)).reshape(part.shape)
        bad = ~np.isfinite(part).all(axis=1)
        c[bad] = 0x7F
        codes[:, g * 128:(g + 1) * 128] = c
        scales[:, g] = np.where(bad, np.float32(np.nan), s)
    return codes, scales


def norm(x, gamma, beta, eps):
    """(y, mean, rstd, bound of |y's error|, bound of |mean's|, relative bound of rstd) in fp64."""
    x = x.double()
    D = x.shape[1]
    mean = x.mean(1, keepdim=True)
    c = x - mean
    var = c.square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    n = D + 4  # terms of a row's sum, the division, and a few roundings around it
    e_mean = 1.01 * n * U * x.abs().mean(1, keepdim=True)
    # (c + d)^2 with |d| <= e_mean + u |c|: mean shift, rounding of c and of the square, the sum
    e_var = 2 * e_mean * c.abs().mean(1, keepdim=True) + e_mean ** 2 + (n + 4) * U * var
    r_rstd = 1.01 * (0.5 * e_var / (var + eps) + 4 * U)
    g, b = gamma.double(), beta.double()
    y = c * rstd * g + b
    e_y = 1.01 * g.abs() * rstd * (e_mean + c.abs() * (r_rstd + 4 * U)) + 2 * U * (y.abs() + b.abs()) + 2.0 ** -126
    return y, mean[:, 0], rstd[:, 0], e_y, e_mean[:, 0] + 2.0 ** -126, r_rstd[:, 0]


def norm_grad(x, mean, rstd, gamma, gy):
    """(gx, dgamma, dbeta) in fp64 for the statistics given, and the bounds of their errors (fp32 results)."""
    x, gy, g = x.double(), gy.double(), gamma.double()
    r = rstd.double()[:, None]
    xh = (x - mean.double()[:, None]) * r
    D, M = x.shape[1], x.shape[0]
    a = gy * g
    c1, c2 = a.mean(1, keepdim=True), (a * xh).mean(1, keepdim=True)
    gx = r * (a - c1 - xh * c2)
    e1 = 1.01 * (D + 3) * U * a.abs().mean(1, keepdim=True)
    e2 = 1.01 * (D + 6) * U * (a * xh).abs().mean(1, keepdim=True)
    e_gx = r * (e1 + xh.abs() * e2 + 8 * U * (a.abs() + c1.abs() + (xh * c2).abs()))
    e_dg = 1.01 * (M + 4) * U * (gy * xh).abs().sum(0)
    e_db = 1.01 * (M + 1) * U * gy.abs().sum(0)
    return gx, (gy * xh).sum(0), gy.sum(0), e_gx + 2.0 ** -126, e_dg + 2.0 ** -126, e_db + 2.0 ** -126


def assert_within(got, want, bound, what):
    got, off = got.double(), (got.double() - want).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all(), what
    assert worst <= 1.0, f"{what}: {worst:.3g} times the bound"

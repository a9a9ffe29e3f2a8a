"""The block-scaled fp8 linear's operators as they are measured: the quantisation of activation rows, the product,
its input gradient, and the layer norm in front of it with its gradient.

Five operators, named in a case's "op":

  quantize   x[M, K] -> e4m3 codes [M, K] and one fp32 scale per row and block of 128 of K
  product    y[M, N] = epi(x W^T + b), x as such codes and scales, W [N, K] e4m3 with a scale per 128 x 128 block
  grad       gx[M, K] = gy W, gy as codes and scales over blocks of 128 of N
  norm       layer norm with its statistics; "codes": the result leaves as quantize's codes and scales
  norm_grad  the gradients of a layer norm's input, gamma and beta

``run`` computes them in their plain form (elementary torch operations in fp32) where ``own`` is false, and with
noeira_amd's kernels where it is true.
"""
import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
EPS = 1e-5
_DT = {"f32": torch.float32, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "bf16": 2}


def listed():
    return [
        # one decoded token's activations ahead of an 11008-wide projection's pair
        {"name": "quantize_step", "op": "quantize", "M": 1, "K": 4096, "x": "bf16"},
        # a training or prefill batch's activations
        {"name": "quantize_batch", "op": "quantize", "M": 8192, "K": 4096, "x": "bf16"},
        # one decoded token through the widest projection: bound by the weight stream
        {"name": "product_row", "op": "product", "M": 1, "K": 4096, "N": 11008, "y": "bf16", "bias": False, "relu": False},
        # a decoder block's MLP at a policy's prompt length: K ends inside a block, N is odd
        {"name": "product_ragged", "op": "product", "M": 135, "K": 960, "N": 2567, "y": "f32", "bias": True, "relu": True},
        # a prompt through a square projection
        {"name": "product_prompt", "op": "product", "M": 1024, "K": 4096, "N": 4096, "y": "bf16", "bias": True, "relu": False},
        # the large-M product: a batch of 8192 rows into 11008 channels
        {"name": "product_batch", "op": "product", "M": 8192, "K": 4096, "N": 11008, "y": "bf16", "bias": False, "relu": False},
        # the gradient that an adapter's training sends back through a frozen 960 -> 2560 projection
        {"name": "grad_adapter", "op": "grad", "M": 256, "K": 960, "N": 2560, "y": "f32"},
        # the same for a batch through 4096 -> 4096
        {"name": "grad_batch", "op": "grad", "M": 8192, "K": 4096, "N": 4096, "y": "bf16"},
        # one token's norm
        {"name": "norm_step", "op": "norm", "M": 1, "K": 960, "x": "f32", "y": "f32"},
        # a batch's norm straight into codes
        {"name": "norm_codes_batch", "op": "norm", "M": 8192, "K": 4096, "x": "bf16", "y": "codes"},
        # a small policy's norm in fp32, rows of odd length
        {"name": "norm_grad_odd", "op": "norm_grad", "M": 333, "K": 1001, "x": "f32"},
        # a batch's norm, backward
        {"name": "norm_grad_batch", "op": "norm_grad", "M": 8192, "K": 4096, "x": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "grad", "grad", "norm", "norm", "norm_grad", "norm_grad"])
    M = _log(rng, 1, 8192)
    if op in ("product", "grad"):
        K = 16 * _log(rng, 4, 688)
        N = _log(rng, 17, 11008) if op == "product" else 16 * _log(rng, 4, 688)
        while M * K * N > 8192 * 4096 * 4096:
            M = max(1, M // 2)
        c = {"op": op, "M": M, "K": K, "N": N, "y": rng.choice(["f32", "bf16"])}
        if op == "product":
            c["bias"] = rng.random() < 0.5
            c["relu"] = rng.random() < 0.3
        return c
    K = _log(rng, 64, 11008)
    while M * K > 8192 * 4096:
        M = max(1, M // 2)
    c = {"op": op, "M": M, "K": K, "x": rng.choice(["f32", "bf16"])}
    if op == "norm":
        c["y"] = rng.choice(["f32", "bf16", "codes"])
    return c


# ---- inputs -------------------------------------------------------------------------------------------------------


def _activations(g, M, K, dtype):
    """Rows as they leave a residual stream: each with a size of its own, a few channels several times the others,
    and now and then a padded row of zeros."""
    x = torch.randn(M, K, generator=g, device="cuda")
    x *= torch.exp(0.5 * torch.randn(M, 1, generator=g, device="cuda"))
    x[:, torch.randperm(K, generator=g, device="cuda")[: max(1, K // 256)]] *= 8.0
    if M >= 64:
        x[torch.randint(0, M, (M // 64,), generator=g, device="cuda")] = 0.0
    return x.to(dtype)


def _weight(g, N, K):
    """e4m3 codes [N, K] and their scales [N / 128, K / 128] of a weight with N(0, 1 / K) values."""
    w = torch.randn(N, K, generator=g, device="cuda") / math.sqrt(K)
    nb, kb = -(-N // BLOCK), -(-K // BLOCK)
    t = torch.nn.functional.pad(w, (0, kb * BLOCK - K, 0, nb * BLOCK - N)).view(nb, BLOCK, kb, BLOCK)
    s = t.abs().amax(dim=(1, 3)) / E4M3_MAX
    q = (t / s[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(nb * BLOCK, kb * BLOCK)[:N, :K]
    return q.to(torch.float8_e4m3fn).contiguous(), s.contiguous()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, M, K = case["op"], case["M"], case["K"]
    st = {"case": case}
    if op in ("product", "grad"):
        N = case["N"]
        st["wq"], st["ws"] = _weight(g, N, K)
        st["xq"], st["xs"] = _quantize(_activations(g, M, K if op == "product" else N, torch.float32))
        st["bias"] = 0.1 * torch.randn(N, generator=g, device="cuda") if case.get("bias") else None
        if own:
            from noeira_amd.qlinear import FP8BlockLinear

            st["layer"] = FP8BlockLinear(K, N, grad=op == "grad")
            st["layer"].set_weight(st["wq"], st["ws"])
        return st
    st["x"] = _activations(g, M, K, _DT[case["x"]])
    if op != "quantize":
        st["x"] += torch.randn(M, 1, generator=g, device="cuda").to(st["x"].dtype)  # a norm's rows have a mean
        st["gamma"] = 1.0 + 0.1 * torch.randn(K, generator=g, device="cuda")
        st["beta"] = 0.1 * torch.randn(K, generator=g, device="cuda")
    if op == "norm_grad":
        st["mean"], st["rstd"] = _statistics(st["x"].float())
        st["gy"] = (torch.randn(M, K, generator=g, device="cuda") * 0.01).to(st["x"].dtype)
    if own and op != "quantize":
        from noeira_amd.norm import LayerNorm

        st["norm"] = LayerNorm(K, eps=EPS)
        st["norm"].set_params(st["gamma"], st["beta"])
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------


def _blocks(x):
    """[M, K] -> [M, G, 128], zeros behind the row's end."""
    G = -(-x.shape[1] // BLOCK)
    return torch.nn.functional.pad(x, (0, G * BLOCK - x.shape[1])).view(x.shape[0], G, BLOCK)


def _quantize(x):
    t = _blocks(x.float())
    amax = t.abs().amax(dim=2)
    # (by a tensor: a division by a number is a product with its rounded reciprocal, which moves codes at the ties)
    s = torch.where(amax > 0, amax / torch.full_like(amax, E4M3_MAX), torch.ones_like(amax))
    q = (t / s[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    return q.view(x.shape[0], -1)[:, : x.shape[1]].to(torch.float8_e4m3fn).contiguous(), s


def _rows(q, s):
    """The values that codes [M, K] and scales [M, G] stand for."""
    return (_blocks(q.float()) * s[:, :, None]).view(q.shape[0], -1)[:, : q.shape[1]]


def _matrix(q, s):
    """The values that a weight's codes [N, K] and scales [N / 128, K / 128] stand for."""
    N, K = q.shape
    return q.float() * s.repeat_interleave(BLOCK, 0)[:N].repeat_interleave(BLOCK, 1)[:, :K]


def _statistics(x):
    mean = x.mean(dim=1, keepdim=True)
    return mean[:, 0], torch.rsqrt((x - mean).square().mean(dim=1) + EPS)


def run(st):
    case = st["case"]
    op = case["op"]
    if op == "quantize":
        if own:
            from noeira_amd.qlinear import quantize_rows_fp8_block

            return quantize_rows_fp8_block(st["x"])
        return _quantize(st["x"])
    if op == "product":
        dt = _DT[case["y"]]
        if own:
            return st["layer"].forward_a8(st["xq"], st["xs"], bias=st["bias"], epilogue="relu" if case["relu"] else "none", out_dtype=dt)
        y = _rows(st["xq"], st["xs"]) @ _matrix(st["wq"], st["ws"]).t()
        if st["bias"] is not None:
            y = y + st["bias"]
        return (torch.where(y > 0, y, torch.zeros_like(y)) if case["relu"] else y).to(dt)
    if op == "grad":
        dt = _DT[case["y"]]
        if own:
            return st["layer"].vjp_a8(st["xq"], st["xs"], out_dtype=dt)
        return (_rows(st["xq"], st["xs"]) @ _matrix(st["wq"], st["ws"])).to(dt)
    if op == "norm":
        if own:
            if case["y"] == "codes":
                return st["norm"].forward_fp8_train(st["x"])
            return st["norm"].forward_train(st["x"], out_dtype=_DT[case["y"]])
        x = st["x"].float()
        mean, rstd = _statistics(x)
        y = (x - mean[:, None]) * rstd[:, None] * st["gamma"] + st["beta"]
        if case["y"] == "codes":
            return (*_quantize(y), mean, rstd)
        return y.to(_DT[case["y"]]), mean, rstd
    if own:
        return st["norm"].vjp(st["x"], st["mean"], st["rstd"], st["gy"])
    x, gy = st["x"].float(), st["gy"].float()
    xhat = (x - st["mean"][:, None]) * st["rstd"][:, None]
    a = gy * st["gamma"]
    gx = st["rstd"][:, None] * (a - a.mean(dim=1, keepdim=True) - xhat * (a * xhat).mean(dim=1, keepdim=True))
    return gx.to(st["x"].dtype), (gy * xhat).sum(dim=0), gy.sum(dim=0)


# ---- in 64 bits, from the definitions -----------------------------------------------------------------------------


def _e4m3(v):
    """The nearest e4m3 value of a float64, ties to the even significand, magnitudes beyond the largest clipped."""
    v = v.clamp(-E4M3_MAX, E4M3_MAX)
    _, e = torch.frexp(v)  # v = m 2^e with 0.5 <= |m| < 1: four significand bits, subnormal steps of 2^-9
    step = torch.ldexp(torch.ones_like(v), (e - 4).clamp(min=-9))
    return torch.round(v / step) * step


def _exact_codes(x):
    """Scales (amax / 448) and code values; the scale and the quotient are each rounded to fp32 by definition."""
    M, K = x.shape
    codes = torch.empty_like(x)
    scales = torch.ones(M, -(-K // BLOCK), dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        part = x[:, b * BLOCK : (b + 1) * BLOCK]
        top = part.abs().max(dim=1).values
        scales[:, b] = torch.where(top == 0, scales[:, b], top / E4M3_MAX)
        s32 = scales[:, b].float().double()
        codes[:, b * BLOCK : (b + 1) * BLOCK] = _e4m3((part / s32[:, None]).float().double())
    return codes, scales


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return _exact_codes(st["x"].double())
    if op in ("product", "grad"):
        K, N = case["K"], case["N"]
        rows, cols = torch.arange(N, device="cuda") // BLOCK, torch.arange(K, device="cuda") // BLOCK
        w = st["wq"].double() * st["ws"].double()[rows][:, cols]
        x = st["xq"].double() * st["xs"].double()[:, rows if op == "grad" else cols]
        if op == "grad":
            return x @ w
        y = x @ w.t()
        if st["bias"] is not None:
            y += st["bias"].double()
        return y.clamp(min=0) if case["relu"] else y
    x = st["x"].double()
    if op == "norm":
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = 1.0 / torch.sqrt(var + EPS)
        y = torch.addcmul(st["beta"].double(), (x - mean[:, None]) * rstd[:, None], st["gamma"].double())
        if case["y"] == "codes":
            return (*_exact_codes(y), mean, rstd)
        return y, mean, rstd
    gy = st["gy"].double()
    K = case["K"]
    r = st["rstd"].double()[:, None]
    z = (x - st["mean"].double()[:, None]) * r
    a = gy * st["gamma"].double()
    gx = r / K * (K * a - a.sum(1, keepdim=True) - z * (a * z).sum(1, keepdim=True))
    return gx, torch.einsum("mk,mk->k", gy, z), gy.sum(0)


def work(case):
    op, M, K = case["op"], case["M"], case["K"]
    G = -(-K // BLOCK)
    if op == "quantize":
        return {"bytes": M * K * (_BYTES[case["x"]] + 1) + 4 * M * G, "flops": 4 * M * K}
    if op in ("product", "grad"):
        N = case["N"]
        B = -(-N // BLOCK)
        a, out, ga = (K, N, G) if op == "product" else (N, K, B)
        n = M * a + 4 * M * ga + N * K + 4 * B * G + M * out * _BYTES[case["y"]]
        return {"bytes": n + (4 * N if case.get("bias") else 0), "flops": 2 * M * N * K}
    if op == "norm":
        es = _BYTES[case["x"]]
        out = M * K + 4 * M * G if case["y"] == "codes" else M * K * _BYTES[case["y"]]
        return {"bytes": M * K * es + out + 8 * K + 8 * M, "flops": 8 * M * K}
    return {"bytes": 3 * M * K * _BYTES[case["x"]] + 12 * K + 8 * M, "flops": 14 * M * K}

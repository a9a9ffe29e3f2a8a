"""Layer norm in front of a quantized linear, over the C ABI.

``LayerNorm`` normalises rows of DIM values and hands them on in the form the next layer takes: fp32 or bf16
(``forward``), or the e4m3 codes and block scales of an ``FP8BlockLinear`` (``forward_fp8``: norm and quantisation in one
launch, the normalised values are never stored).  ``vjp`` is the gradient of its input, gamma and beta.
"""
from __future__ import annotations

from typing import Optional

import numpy as np
import torch

from . import _lib as L
from .qlinear import _FLOATS, _INT32_MAX, _TORCH_DT, _check_dev, _dev_ptr, _need_gpu, _stream_now, _too_many


class LayerNorm:
    """y[M, DIM] = (x - mean) / sqrt(var + eps) * gamma + beta; gamma, beta fp32 [DIM] on the device, ones and zeros
    until ``set_params``."""

    def __init__(self, DIM: int, eps: float = 1e-5):
        if DIM < 1:
            raise L.NQError(L.NQ_ERR_INVALID, "LayerNorm: DIM must be positive")
        if DIM > _INT32_MAX:
            raise _too_many(DIM, "LayerNorm", "values in a row")
        self.DIM, self.eps = int(DIM), float(eps)
        self.gamma = torch.ones((DIM,), dtype=torch.float32, device="cuda")
        self.beta = torch.zeros((DIM,), dtype=torch.float32, device="cuda")

    @classmethod
    def make(cls, DIM: int, eps: float = 1e-5, target: str = "gpu") -> "LayerNorm":
        _need_gpu(target)
        return cls(DIM, eps)

    def set_params(self, gamma, beta):
        """fp32 [DIM] each: arrays or tensors; copied (values only: no part of a graph that a tensor belongs to)."""
        new = []
        for name, v in (("gamma", gamma), ("beta", beta)):
            t = v.detach() if isinstance(v, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(v, dtype=np.float32))
            if tuple(t.shape) != (self.DIM,):
                raise L.NQError(L.NQ_ERR_SIZE, f"LayerNorm.set_params: {name} is {list(t.shape)}, expected [{self.DIM}]")
            new.append(t)
        self.gamma.copy_(new[0])
        self.beta.copy_(new[1])

    def _rows(self, x: torch.Tensor, what: str) -> int:
        _check_dev(x, what, "x", _FLOATS)
        if self.gamma.get_device() != x.get_device():
            raise L.NQError(L.NQ_ERR_INVALID, what + ": x and the norm are on different devices")
        M = x.numel() // self.DIM
        if M * self.DIM != x.numel():
            raise L.NQError(L.NQ_ERR_INVALID, f"{what}: x has {x.numel()} values, not a multiple of DIM = {self.DIM}")
        if M > _INT32_MAX:
            raise _too_many(M, what, "rows")
        return M

    def _like(self, x: torch.Tensor, M: int, dtype: torch.dtype) -> torch.Tensor:
        t = torch.empty_like(x) if dtype is x.dtype else torch.empty_like(x, dtype=dtype)
        return t if x.dim() == 2 and x.shape[1] == self.DIM else t.view(M, self.DIM)

    def _forward(self, x, out, out_dtype, stats, what):
        M = self._rows(x, what)
        if out is not None:
            out_dtype = out.dtype if out_dtype is None else out_dtype
            _check_dev(out, what, "out", out_dtype, M * self.DIM)
        out_dtype = x.dtype if out_dtype is None else out_dtype
        if out_dtype not in _TORCH_DT:
            raise L.NQError(L.NQ_ERR_INVALID, what + ": y must be fp32 or bf16")
        if out is None:
            out = self._like(x, M, out_dtype)
        mean = rstd = None
        if stats:  # (fp32 on x's device, as gamma is; a third of torch.empty's time less)
            mean, rstd = self.gamma.new_empty(M), self.gamma.new_empty(M)
        L.check(L.lib().nq_layer_norm(_dev_ptr(x), _TORCH_DT[x.dtype], _dev_ptr(self.gamma), _dev_ptr(self.beta),
                                      self.eps, _dev_ptr(out), _TORCH_DT[out_dtype], _dev_ptr(mean), _dev_ptr(rstd),
                                      M, self.DIM, _stream_now()))
        return out, mean, rstd

    def forward(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
        """y [M, DIM], of x's type unless `out_dtype` (fp32 or bf16) says otherwise; `out` may be x itself."""
        return self._forward(x, out, out_dtype, False, "LayerNorm.forward")[0]

    def forward_train(self, x: torch.Tensor, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None):
        """(y, mean, rstd): `forward` with the statistics fp32 [M] that ``vjp`` takes."""
        return self._forward(x, out, out_dtype, True, "LayerNorm.forward_train")

    def _forward_fp8(self, x, stats, what):
        M = self._rows(x, what)
        codes = self._like(x, M, torch.float8_e4m3fn)
        scales = self.gamma.new_empty((M, -(-self.DIM // 128)))
        mean = rstd = None
        if stats:  # (fp32 on x's device, as gamma is; a third of torch.empty's time less)
            mean, rstd = self.gamma.new_empty(M), self.gamma.new_empty(M)
        L.check(L.lib().nq_layer_norm_fp8_block(_dev_ptr(x), _TORCH_DT[x.dtype], _dev_ptr(self.gamma), _dev_ptr(self.beta),
                                                self.eps, _dev_ptr(codes), _dev_ptr(scales), _dev_ptr(mean),
                                                _dev_ptr(rstd), M, self.DIM, _stream_now()))
        return codes, scales, mean, rstd

    def forward_fp8(self, x: torch.Tensor):
        """(codes [M, DIM], scales [M, ceil(DIM/128)]): what ``quantize_rows_fp8_block`` makes of the fp32 result."""
        return self._forward_fp8(x, False, "LayerNorm.forward_fp8")[:2]

    def forward_fp8_train(self, x: torch.Tensor):
        """(codes, scales, mean, rstd)."""
        return self._forward_fp8(x, True, "LayerNorm.forward_fp8_train")

    def vjp(self, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, grad_output: torch.Tensor,
            grad_input: Optional[torch.Tensor] = None, params: bool = True):
        """(grad_input [M, DIM] of x's type, dgamma, dbeta fp32 [DIM]) from the forward's input and statistics;
        ``params=False`` (a frozen norm): no sums over the rows, dgamma and dbeta are None."""
        M = self._rows(x, "LayerNorm.vjp")
        _check_dev(grad_output, "LayerNorm.vjp", "grad_output", _FLOATS, M * self.DIM)
        _check_dev(mean, "LayerNorm.vjp", "mean", torch.float32, M)
        _check_dev(rstd, "LayerNorm.vjp", "rstd", torch.float32, M)
        if grad_input is None:
            grad_input = self._like(x, M, x.dtype)
        else:
            _check_dev(grad_input, "LayerNorm.vjp", "grad_input", _FLOATS, M * self.DIM)
        dg = db = ws = None
        n = 0
        if params:
            dg, db = torch.empty_like(self.gamma), torch.empty_like(self.gamma)
            n = L.lib().nq_layer_norm_grad_workspace_bytes(M, self.DIM)
            ws = self.gamma.new_empty(n // 4) if n else None
        L.check(L.lib().nq_layer_norm_grad(_dev_ptr(x), _TORCH_DT[x.dtype], _dev_ptr(mean), _dev_ptr(rstd), _dev_ptr(self.gamma),
                                           _dev_ptr(grad_output), _TORCH_DT[grad_output.dtype], _dev_ptr(grad_input),
                                           _TORCH_DT[grad_input.dtype], _dev_ptr(dg), _dev_ptr(db), M, self.DIM, _dev_ptr(ws),
                                           n, _stream_now()))
        return grad_input, dg, db

"""`rms_norm()`: the residual's addition and the RMS norm in front of a linear layer, with the layer's operand as its output.

No counterpart in the reference.  The quantised outputs are those of `quantize()`: e4m3 with a scale a row, or the NVFP4 operand that
`linear()` takes, without the normalised rows going through memory in bf16.
"""
import torch

from .. import _cuda_ops
from ..native import host_calls
from .utils import align_up, ceil_div

rms_norm_kernel = _cuda_ops.rms_norm


def rms_norm(x, weight=None, eps=1e-6, *, residual=None, precision=None, global_scale=None, keep=False, sf_layout="ac4k"):
    """(x + residual) / sqrt(mean((x + residual)^2) + eps) * weight along the rows of x.

    x: bf16 [M, K] with contiguous rows (any row stride), K at most 32768; weight: [K] bf16 or fp32, None for ones; residual: [M, K] bf16
    or fp32 with contiguous rows.  All arithmetic is fp32 and every output is rounded once.  Returns
      precision None      out bf16 [M, K]
      "fp8e4m3"           out e4m3 [M, align_up(K, 16)], sf fp32 [align_up(M, 16)]: the row's largest value over 448
      "nvfp4"             out u8 [M, align_up(K, 64) // 2], sf e4m3 in `sf_layout`, global_scale (given: a 0-dim fp32 tensor, calibrated, as
                          the largest value is not known before the rows are; sqrt(K) * max|weight| / 2688 holds for any x)
    followed by the result in bf16 as well where `keep` is set (what adapters beside the layer read), and by x + residual in residual's
    type where a residual is given.  A single output comes as a tensor, several as a tuple."""
    if host_calls is not None:
        made = host_calls.rms_norm(x, weight, eps, residual, precision, global_scale, keep, sf_layout)
        if made is not None:
            return made
    if precision not in (None, "fp8e4m3", "nvfp4"):
        raise ValueError(f"unknown precision {precision!r}")
    if sf_layout not in ("ac4k", "128x4"):
        raise ValueError(f"unknown sf_layout {sf_layout!r}")
    if keep and precision is None:
        raise ValueError("keep stands beside a quantised output")
    if (global_scale is not None) != (precision == "nvfp4"):
        raise ValueError("precision \"nvfp4\" takes a global_scale, and no other does")
    if x.ndim != 2:
        raise RuntimeError("x must be a 2d matrix with contiguous rows")
    (m, k), dev = x.shape, x.device
    made, sf = [], None
    if precision is None:
        made.append(torch.empty((m, k), dtype=torch.bfloat16, device=dev))
    elif precision == "fp8e4m3":
        sf = torch.empty((align_up(m, 16),), dtype=torch.float32, device=dev)
        made += [torch.empty((m, align_up(k, 16)), dtype=torch.float8_e4m3fn, device=dev), sf]
    else:
        kt = ceil_div(k, 64)
        sf = torch.empty((kt, align_up(m, 16), 4) if sf_layout == "ac4k" else (ceil_div(m, 128), kt, 32, 4, 4), dtype=torch.float8_e4m3fn, device=dev)
        made += [torch.empty((m, kt * 32), dtype=torch.uint8, device=dev), sf, global_scale]
    normed = torch.empty((m, k), dtype=torch.bfloat16, device=dev) if keep else None
    residual_out = torch.empty((m, k), dtype=residual.dtype, device=dev) if residual is not None else None
    rms_norm_kernel(made[0], sf, normed, residual_out, x, weight, residual, eps, precision, global_scale)
    made += [t for t in (normed, residual_out) if t is not None]
    return made[0] if len(made) == 1 else tuple(made)

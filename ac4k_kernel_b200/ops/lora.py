"""`lora()`: the low-rank adapters of a batch of requests beside a projection that all of them share.

No counterpart in the reference.  The projection is `linear()` on the quantised rows; the adapters read the rows in bf16 (`rms_norm(...,
keep=True)` returns both forms)."""
import torch

from .. import _cuda_ops
from ..native import host_calls

lora_kernel = _cuda_ops.lora


def lora(y, x, a, b, offsets, adapters, scaling=None, *, out=None):
    """y + scaling[j] * (x A_j^T) B_j^T, j the adapter of each row's request.

    y: [T, N] bf16, fp16 or fp32, the projection's output; x: [T, K] bf16, its input; both with contiguous rows.  a: [adapters, R, K] and b:
    [adapters, N, R], bf16, contiguous, R at most 128 (an adapter of a lower rank has zeros behind it).  offsets: int32 [requests + 1],
    ascending: the rows of request i are offsets[i] to offsets[i + 1]; adapters: int32 [requests], the adapter of each, negative for none;
    scaling: fp32 [adapters], None for ones.  Rows without an adapter and rows of no request are those of y.
    out: None, y itself, or a tensor like y that overlaps neither y nor x.  Returns out.

    x A^T is summed in fp32 and its product with B in fp32, with 16 bits of each value of x A^T for a bf16 or fp16 y and all of them for an fp32 y; out
    is rounded once.  A y that `linear()` made in bf16 was rounded there before: where one rounding in all is wanted, give `linear()` an fp32 out."""
    if host_calls is not None:
        made = host_calls.lora(y, x, a, b, offsets, adapters, scaling, out)
        if made is not None:
            return made
    if out is None:
        out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    lora_kernel(out, y, x, a, b, offsets, adapters, scaling)
    return out

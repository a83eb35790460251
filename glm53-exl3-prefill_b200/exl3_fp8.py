"""8-bit layers beside the EXL3 ones: e4m3 weights with one fp32 scale per 128 x 128 block.

Mixed checkpoints keep the shared expert, the dense MLPs, the projections, or a whole expert stack at 8 bits
next to 4-bpw trellis experts (no reference counterpart: the reference runs the trellis ones only).
Activations are quantised on the way in, one scale per row and 128 columns:

    s = max(|x| over the block, 2^-64) / 448        q = e4m3(x / s)         (rounded to nearest, ties to even)

* ``quantize_rows(x)`` — rows to e4m3 and their scales;
* ``quantize_weight(w)`` — a weight matrix (or a stack of them) to e4m3 and its block scales, at load time;
* ``fp8_linear(x, weight, weight_scale)`` — one projection x W^T;
* ``fp8_mlp_prefill(x, mlp, limit)`` — a gated MLP stored as one expert;
* ``fp8_prefill(x, ids, weights, layer, limit)`` — routed experts, the contract of grouped_prefill.

A layer holds ``w13_fp8 [E, 2f, d]`` (gate rows, then up rows), ``w13_scale [E, 2f/128, d/128]``, ``w2_fp8
[E, d, f]``, ``w2_scale [E, d/128, f/128]``.  grouped_prefill, dense_mlp_prefill and moe_block_prefill take such
layers too.  Sums are fp32; a route's sum runs in slot order, so results repeat bit for bit.  Everything runs on
the current stream of the input's device, without a host synchronisation, and can be captured into a CUDA graph.
"""
from __future__ import annotations

import torch

import b200_ext

BLOCK = 128
E4M3_MAX = 448.0


def is_fp8_layer(layer) -> bool:
    return getattr(layer, "w13_fp8", None) is not None


def as_rows(x2d: torch.Tensor) -> torch.Tensor:
    """x2d of any float type and strides as the kernels take it: fp32, fp16 or bf16 in contiguous, separate rows."""
    if x2d.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        x2d = x2d.float()
    if x2d.dim() == 2 and (x2d.shape[1] > 1 and x2d.stride(1) != 1 or x2d.shape[0] > 1 and x2d.stride(0) < x2d.shape[1]):
        x2d = x2d.contiguous()
    return x2d


def quantize_rows(x2d: torch.Tensor, pow2: bool = False):
    """x2d [T, K] (fp32, fp16, bf16; rows may be strided) -> (q e4m3 [T, K], scale fp32 [T, ceil(K / 128)]).
    pow2 takes the least power of two at or above amax / 448 as the scale."""
    return b200_ext.fp8_quantize_rows(x2d, pow2)


def quantize_weight(w: torch.Tensor):
    """w [..., N, K] -> (q e4m3 [..., N, K], scale fp32 [..., ceil(N / 128), ceil(K / 128)]), scale = amax / 448
    over each 128 x 128 block.  Load-time torch code (CPU or GPU); NaN and inf are refused."""
    if not bool(torch.isfinite(w).all()):
        raise RuntimeError("quantize_weight: the weight holds NaN or inf")
    n, k = w.shape[-2:]
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    blocks = torch.nn.functional.pad(w.float(), (0, kb * BLOCK - k, 0, nb * BLOCK - n))
    blocks = blocks.reshape(*w.shape[:-2], nb, BLOCK, kb, BLOCK)
    scale = (blocks.abs().amax(dim=(-3, -1)).double().clamp(min=2.0 ** -64) / E4M3_MAX).float()
    q = (blocks / scale[..., :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    q = q.reshape(*w.shape[:-2], nb * BLOCK, kb * BLOCK)[..., :n, :k].contiguous()
    return q, scale


def fp8_linear(x2d: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               out_dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None) -> torch.Tensor:
    """x2d [T, K], weight e4m3 [N, K], weight_scale fp32 [ceil(N/128), ceil(K/128)] -> x W^T [T, N] as out_dtype
    (float32, float16 or bfloat16), or added into `out` if given.  K must be a multiple of 16; with one token `out`
    may not overlap x (refused)."""
    return b200_ext.fp8_linear(x2d, weight, weight_scale, out, out_dtype)


def fp8_mlp_prefill(x2d: torch.Tensor, mlp, limit: float, out: torch.Tensor | None = None,
                    out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """A gated MLP in the layer layout with one expert -> [T, d] (added into `out` if given)."""
    return b200_ext.fp8_mlp(x2d, mlp.w13_fp8, mlp.w13_scale, mlp.w2_fp8, mlp.w2_scale, float(limit), out, out_dtype)


def fp8_prefill(x2d: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, layer, limit: float,
                out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """x2d [T, d], ids [T, topk] (int64 or int32; ids outside [0, E) add nothing), weights [T, topk]
    -> sum_j weights[t, j] * mlp_{ids[t, j]}(x[t]) as out_dtype [T, d], or added into `out` if given."""
    if ids.dim() == 2 and ids.shape[1] == 0:
        return torch.zeros(x2d.shape, dtype=out_dtype, device=x2d.device) if out is None else out
    return b200_ext.fp8_experts(x2d, ids.contiguous(), weights.contiguous(), layer.w13_fp8, layer.w13_scale, layer.w2_fp8,
                                layer.w2_scale, float(limit), out, out_dtype)

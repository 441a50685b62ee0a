"""The next token from a step's logits on gfx950 (HIP, C ABI): the end of the
serving step whose beginning and middle are ``kernels.rotary`` and ``kernels.paged``.

Random numbers are an input, so a draw can be repeated.  Calls run on the
current stream of the tensors' device, wait for nothing and can be captured.
"""
import functools
import struct

import torch

import spruce_hip

__all__ = ["sample_tokens"]

# struct spruce_sample_tokens_args, field by field.
_SAMPLE_ARGS = struct.Struct("=qqqqqqqqqqqdqddqqqq")


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*shape):
    return spruce_hip.lib().spruce_sample_tokens_workspace_bytes(*shape)


def _setting(x, name, dtype, B, device):
    """(pointer, number) of a setting: one of them stands for it."""
    if not torch.is_tensor(x):
        return 0, x
    if x.dtype != dtype or x.shape != (B,) or not x.is_contiguous():
        raise ValueError(f"{name} must be a number or contiguous {str(dtype)[6:]} [B] = [{B}]")
    if x.device != device:
        raise ValueError(f"{name} must be on the same device as the logits")
    return x.data_ptr(), 0


def sample_tokens(logits, uniform, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, return_logprobs=False):
    """One token of every row of logits x ``[B,V]`` (bf16, f16 or f32; any row stride).

    uniform: a random number u in [0, 1) a row, float32 or float64 ``[B]``.  With the
    weights w_i = exp((x_i - max x) / temperature), a row keeps, in the order of x descending
    (ties by index), the shortest of three prefixes: the first ``top_k`` (0: all);
    of those the fewest whose weights reach ``top_p`` of all of theirs (1: all);
    and those with w_i >= ``min_p``, at least the first each.  Its token is the first i,
    by index, at which the kept weights up to i come to more than u of their sum.

    Each setting is a number, or a tensor ``[B]`` with one of each row (float32,
    top_k int32).  A temperature of 0 takes the largest logit, the first of equal ones.
    NaN logits count as -inf, which is never drawn; beside +inf nothing else is.
    Weights are formed in 64 bits, rounded to a unit (2^-45 of the largest for V up to
    2^18) and added exactly, so no order of additions changes a token.

    Returns tokens int64 ``[B]`` (-1 for a row of nothing but -inf), with
    ``return_logprobs`` also float32 ``[B]``, the log of each token's share of its row's kept
    weights (-inf for token -1).
    """
    device = logits.device
    if logits.dim() != 2:
        raise ValueError("logits must be [B, V]")
    B, V = logits.shape
    code = spruce_hip.dtype_code(logits)
    stride = logits.stride()
    if V < 1:
        raise ValueError("logits must have a column")
    if V > 1 and stride[1] != 1:
        raise ValueError("logits must have a contiguous final dimension")
    if uniform.dtype not in (torch.float32, torch.float64) or uniform.shape != (B,) or not uniform.is_contiguous():
        raise ValueError(f"uniform must be contiguous float32 or float64 [B] = [{B}]")
    if uniform.device != device:
        raise ValueError("uniform must be on the same device as the logits")
    heat, heat1 = _setting(temperature, "temperature", torch.float32, B, device)
    most, most1 = _setting(top_k, "top_k", torch.int32, B, device)
    mass, mass1 = _setting(top_p, "top_p", torch.float32, B, device)
    least, least1 = _setting(min_p, "min_p", torch.float32, B, device)
    if not heat1 >= 0:
        raise ValueError(f"temperature must not be negative, got {heat1}")
    if most1 < 0:
        raise ValueError(f"top_k must not be negative, got {most1}")
    if not 0 <= mass1 <= 1 or not 0 <= least1 <= 1:
        raise ValueError(f"top_p and min_p must be in [0, 1], got {mass1} and {least1}")
    if torch.is_grad_enabled() and logits.requires_grad:
        raise RuntimeError("the draw of a token has no gradient; run it under torch.no_grad()")
    if not logits.is_cuda:
        raise RuntimeError("the sampling HIP backend requires GPU tensors")
    tokens = logits.new_empty_strided((B,), (1,), dtype=torch.int64)
    logprobs = logits.new_empty_strided((B,), (1,), dtype=torch.float32) if return_logprobs else None
    # Rows that nothing bounds, or top_p alone, may be shared by several workgroups.
    alone = most or 0 < most1 < V or least or least1 > 0 or (not heat and heat1 == 0)
    need = 0 if alone else _workspace_bytes(B, V, 1 if mass or mass1 < 1 else 0)
    work = logits.new_empty_strided((need,), (1,), dtype=torch.uint8) if need else None
    with spruce_hip.on_device(device):
        rc = spruce_hip.lib().spruce_sample_tokens(_SAMPLE_ARGS.pack(
            logits.data_ptr(), stride[0] if B > 1 else V, B, V, code, uniform.data_ptr(),
            uniform.dtype == torch.float64, heat, most, mass, least, heat1, min(most1, V), mass1, least1,
            tokens.data_ptr(), logprobs.data_ptr() if return_logprobs else 0, work.data_ptr() if need else 0, need),
            spruce_hip.raw_stream(device.index))
    if rc:
        spruce_hip.check(rc, "spruce_sample_tokens")
    return (tokens, logprobs) if return_logprobs else tokens

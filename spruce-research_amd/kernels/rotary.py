"""Rotary positions and per-head norms of queries and keys on gfx950 (HIP, C ABI).

What stands between a model's projections and the attention calls of this
package, which take normed and rotated queries and keys.  ``rotate_heads`` is
one launch for both; ``rotary_frequencies`` makes the angles per position that
it takes, plain or scaled for long contexts.  Inference only, like the
attention: inputs that need gradients are refused.  (The reference leaves this
step to Transformers' model code.)
"""
import math
import struct

import torch

import spruce_hip

ROTARY_LAYOUTS = ("half", "interleaved")
ROTARY_SCALINGS = (None, "linear", "ntk", "yarn")

__all__ = ["ROTARY_LAYOUTS", "ROTARY_SCALINGS", "rotary_frequencies", "rotate_heads"]


def rotary_frequencies(rotary_dim, base=10000.0, *, scaling=None, factor=1.0, original_length=None,
                       beta_fast=32.0, beta_slow=1.0, device=None):
    """(``inv_freq`` float64 ``[rotary_dim / 2]``, the factor on rotated values).

    Pair i turns by base^(-2i/R) radians per position (R = ``rotary_dim``).
    ``scaling`` stretches a model trained on ``original_length`` positions
    by ``factor``:

    * ``"linear"``: every angle divided by factor;
    * ``"ntk"``: base * factor^(R / (R - 2)), so that the slowest pair turns
      factor times slower and the fastest as before;
    * ``"yarn"`` (Peng et al. 2023): pairs that turn more than ``beta_fast``
      times over ``original_length`` keep their angle, pairs that turn less than
      ``beta_slow`` times are divided by factor, and the share between them is
      linear in the pair's index; rotated values are scaled by
      0.1 ln(factor) + 1.
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be positive and even, got {rotary_dim}")
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"scaling must be one of {ROTARY_SCALINGS}, got {scaling!r}")
    if not base > 1 or not factor >= 1:
        raise ValueError("base must be above 1 and factor at least 1")
    if scaling == "ntk":
        if rotary_dim == 2:
            raise ValueError("ntk scaling needs rotary_dim above 2")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    pair = torch.arange(rotary_dim // 2, dtype=torch.float64)
    inv_freq = base ** (-2.0 * pair / rotary_dim)
    attention = 1.0
    if scaling == "linear":
        inv_freq = inv_freq / factor
    elif scaling == "yarn":
        if not original_length:
            raise ValueError("yarn scaling needs original_length")

        def pair_of(turns):     # the (real) index of the pair that turns so often over original_length
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = max(math.floor(pair_of(beta_fast)), 0)
        high = min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        share = ((pair - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv_freq = inv_freq / factor * share + inv_freq * (1 - share)
        attention = 0.1 * math.log(factor) + 1.0
    return inv_freq.to(device), attention


def _refuse_grad():
    raise RuntimeError("the HIP rotary and paged operators compute no gradients; run them under torch.no_grad()")


_LAYOUT_CODES = {name: code for code, name in enumerate(ROTARY_LAYOUTS)}


def _rotation(inv_freq, layout, head_dim, device):
    """(pointer, rotary_dim, layout code) of checked angles (None: no rotation)."""
    code = _LAYOUT_CODES.get(layout)
    if code is None:
        raise ValueError(f"layout must be one of {ROTARY_LAYOUTS}, got {layout!r}")
    if inv_freq is None:
        return 0, 0, 0
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64 [rotary_dim / 2]")
    if inv_freq.device != device:
        raise ValueError("inv_freq must be on the same device as q and k")
    rotary_dim = 2 * len(inv_freq)
    if rotary_dim > head_dim or rotary_dim % 16:
        raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim {head_dim}, got {rotary_dim}")
    return inv_freq.data_ptr(), rotary_dim, code


def _weights(q_weight, k_weight, head_dim, dtype, device):
    """(pointers of the norm weights, their shared dtype code), after their checks."""
    shared = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w.shape != (head_dim,) or not w.is_contiguous():
            raise ValueError(f"norm weights must be contiguous [{head_dim}]")
        if w.device != device:
            raise ValueError("norm weights must be on the same device as q and k")
        if w.dtype not in (dtype, torch.float32) or shared not in (None, w.dtype):
            raise ValueError("norm weights must share one dtype: float32 or the inputs'")
        shared = w.dtype
    return (0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(),
            2 if shared is None else spruce_hip.DTYPE_CODES[shared])


def _positions(positions, shapes, device):
    """(pointer, row stride, 64 bits or not) of checked positions."""
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if positions.device != device:
        raise ValueError("positions must be on the same device as q and k")
    shape, stride = tuple(positions.shape), positions.stride()
    if shape not in shapes or (shape[-1] > 1 and stride[-1] != 1):
        raise ValueError(f"positions must be {' or '.join(map(str, shapes))} with contiguous tokens, got {shape}")
    return positions.data_ptr(), stride[0] if len(shape) == 2 else 0, positions.dtype == torch.int64


def _needs_grad(q_weight, k_weight, inv_freq):
    return ((q_weight is not None and q_weight.requires_grad) or (k_weight is not None and k_weight.requires_grad)
            or (inv_freq is not None and inv_freq.requires_grad))


# struct spruce_rotate_heads_args, field by field.
_ROTATE_ARGS = struct.Struct("=q4qq4q6qqqqqqqdqqqdq4qq4q")


def rotate_heads(q, k, positions, inv_freq, *, layout="half", factor=1.0, q_weight=None, k_weight=None, eps=1e-6):
    """Norm every head row (where a weight is given), then rotate it by its position.

    q ``[B,Hq,T,D]``, k ``[B,Hkv,T,D]`` (bf16, f16 or f32; any strides with a
    contiguous last dim and 16-byte aligned rows, e.g. the transposed views of
    ``[B,T,H,D]`` projections); positions int32 or int64 ``[B,T]`` or ``[T]``;
    inv_freq float64 ``[R/2]`` from ``rotary_frequencies`` (None: no rotation).

      y = x * (mean(x^2) + eps)^(-1/2) * weight            per head row
      (a, b) <- factor * (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i]

    over the pairs (y_i, y_{i+R/2}) of layout ``"half"`` or (y_2i, y_2i+1) of
    ``"interleaved"``; y_R.. stay as they are.  Angles are formed in 64 bits,
    the rest in 32, rounded once.  Returns (q, k) of the same shapes and dtype,
    laid out as contiguous ``[B,T,H,D]``.
    """
    device, dtype = q.device, q.dtype
    if q.dim() != 4 or k.dim() != 4:
        raise ValueError("q and k must be [B,H,T,D] and match in batch, tokens, and head_dim")
    B, Hq, T, D = q.shape
    Bk, Hkv, Tk, Dk = k.shape
    if Bk != B or Tk != T or Dk != D:
        raise ValueError("q and k must be [B,H,T,D] and match in batch, tokens, and head_dim")
    if k.dtype != dtype:
        raise ValueError("q and k must share one dtype")
    if k.device != device:
        raise ValueError("q and k must be on the same device")
    if D != 128 and D != 64:
        raise ValueError(f"kernel supports head_dim 64 or 128, got {D}")
    qs, ks = q.stride(), k.stride()
    if qs[3] != 1 or ks[3] != 1:
        raise ValueError("q and k must have a contiguous final dimension")
    rotation = _rotation(inv_freq, layout, D, device)
    weights = _weights(q_weight, k_weight, D, dtype, device)
    place = _positions(positions, ((B, T), (T,)), device)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or _needs_grad(q_weight, k_weight, inv_freq)):
        _refuse_grad()
    if not q.is_cuda:
        raise RuntimeError("the rotary HIP backend requires GPU tensors")
    # Laid out [B,T,H,D] from the start: a decoding step's call is host time, and a
    # transposed torch.empty takes 2 us more.
    qos, kos = (T * Hq * D, D, Hq * D, 1), (T * Hkv * D, D, Hkv * D, 1)
    qo, ko = q.new_empty_strided((B, Hq, T, D), qos), q.new_empty_strided((B, Hkv, T, D), kos)
    with spruce_hip.on_device(device):
        rc = spruce_hip.lib().spruce_rotate_heads(_ROTATE_ARGS.pack(
            q.data_ptr(), *qs, k.data_ptr(), *ks, B, Hq, Hkv, T, D, spruce_hip.dtype_code(q), *place, *rotation, factor,
            *weights, eps, qo.data_ptr(), *qos, ko.data_ptr(), *kos),
            spruce_hip.raw_stream(device.index))
    if rc:
        spruce_hip.check(rc, "spruce_rotate_heads")
    return qo, ko

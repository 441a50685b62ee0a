"""Rotary positions and per-head norms of queries and keys on gfx950 (HIP, C ABI).

What stands between a model's projections and the attention calls of this
package, which take normed and rotated queries and keys.  ``rotate_heads`` is
one launch for both; ``rotary_frequencies`` makes the angles per position that
it takes, plain or scaled for long contexts.  Inference only, like the
attention: inputs that need gradients are refused.  (The reference leaves this
step to Transformers' model code.)
"""
import math

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


def _refuse_grad(*tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("the HIP rotary and paged operators compute no gradients; run them under torch.no_grad()")


def _rotation(inv_freq, layout, head_dim, device):
    """(rotary_dim, layout code) of checked angles (None: no rotation)."""
    if layout not in ROTARY_LAYOUTS:
        raise ValueError(f"layout must be one of {ROTARY_LAYOUTS}, got {layout!r}")
    if inv_freq is None:
        return 0, 0
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64 [rotary_dim / 2]")
    if inv_freq.device != device:
        raise ValueError("inv_freq must be on the same device as q and k")
    rotary_dim = 2 * inv_freq.shape[0]
    if rotary_dim > head_dim or rotary_dim % 16:
        raise ValueError(f"rotary_dim must be a multiple of 16 up to head_dim {head_dim}, got {rotary_dim}")
    return rotary_dim, ROTARY_LAYOUTS.index(layout)


def _weights(q_weight, k_weight, head_dim, like):
    """The norm weights' shared dtype code, after their checks."""
    dtype = None
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w.shape != (head_dim,) or not w.is_contiguous():
            raise ValueError(f"norm weights must be contiguous [{head_dim}]")
        if w.device != like.device:
            raise ValueError("norm weights must be on the same device as q and k")
        if w.dtype not in (like.dtype, torch.float32) or dtype not in (None, w.dtype):
            raise ValueError("norm weights must share one dtype: float32 or the inputs'")
        dtype = w.dtype
    return spruce_hip.DTYPE_CODES[dtype or torch.float32]


def _positions(positions, shape, device):
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if positions.device != device:
        raise ValueError("positions must be on the same device as q and k")
    if tuple(positions.shape) not in shape or (positions.shape[-1] > 1 and positions.stride(-1) != 1):
        raise ValueError(f"positions must be {' or '.join(map(str, shape))} with contiguous tokens, "
                         f"got {tuple(positions.shape)}")
    return int(positions.dtype == torch.int64)


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
    as views of contiguous ``[B,T,H,D]`` tensors.
    """
    if q.dim() != 4 or k.dim() != 4 or q.shape[0] != k.shape[0] or q.shape[2:] != k.shape[2:]:
        raise ValueError("q and k must be [B,H,T,D] and match in batch, tokens, and head_dim")
    if q.dtype != k.dtype:
        raise ValueError("q and k must share one dtype")
    if k.device != q.device:
        raise ValueError("q and k must be on the same device")
    B, Hq, T, D = q.shape
    if D not in (64, 128):
        raise ValueError(f"kernel supports head_dim 64 or 128, got {D}")
    if q.stride(-1) != 1 or k.stride(-1) != 1:
        raise ValueError("q and k must have a contiguous final dimension")
    rotary_dim, code = _rotation(inv_freq, layout, D, q.device)
    weight_code = _weights(q_weight, k_weight, D, q)
    pos64 = _positions(positions, ((B, T), (T,)), q.device)
    _refuse_grad(q, k, q_weight, k_weight, inv_freq)
    if not q.is_cuda:
        raise RuntimeError("the rotary HIP backend requires GPU tensors")
    qo = torch.empty((B, T, Hq, D), device=q.device, dtype=q.dtype).transpose(1, 2)
    ko = torch.empty((B, T, k.shape[1], D), device=q.device, dtype=q.dtype).transpose(1, 2)
    with spruce_hip.on_device(q.device):
        rc = spruce_hip.lib().spruce_rotate_heads(
            spruce_hip.ptr(q), spruce_hip.strides(q), spruce_hip.ptr(k), spruce_hip.strides(k),
            B, Hq, k.shape[1], T, D, spruce_hip.dtype_code(q), spruce_hip.ptr(positions),
            positions.stride(0) if positions.dim() == 2 else 0, pos64, spruce_hip.ptr(inv_freq), rotary_dim, code,
            factor, spruce_hip.ptr(q_weight), spruce_hip.ptr(k_weight), weight_code, eps,
            spruce_hip.ptr(qo), spruce_hip.strides(qo), spruce_hip.ptr(ko), spruce_hip.strides(ko),
            spruce_hip.stream_of(q))
    spruce_hip.check(rc, "spruce_rotate_heads")
    return qo, ko

"""Eviction from a paged K/V cache on gfx950 (HIP, C ABI): the attention weight
that each cached key has gathered, and the cache cut down to the keys that
gathered most.

Both calls take the cache and the batch of ``kernels.paged``: pages ``[pages, Hkv,
page_size, D]``, ``page_table`` int32 ``[S, W]``, ``kv_lens`` int32 ``[S]``, read on
the device only.  Masses lie in pages like the keys that they belong to:
``mass_pages`` float32 ``[pages, Hkv, page_size]`` (any strides in which no two
values share memory), so that they go where a sequence's pages go.  A page whose
mass counts belongs to one sequence: of two that share it, either's masses stay.

Keys that were evicted leave no gap: the kept ones stand at positions 0, 1, ..
afterwards, in their old order.  Their rotary positions are those that they were
appended with, so tokens that come later are appended with ``positions`` of their
own (``kernels.paged.append_paged_kv``), which go on from the uncut sequence's.

Calls run on the current stream of the tensors' device, wait for nothing and
can be captured.  Inference only: inputs that need gradients are refused.
"""
import functools
import struct

import torch

import spruce_hip
from kernels.rotary import _refuse_grad

__all__ = ["evict_paged_kv", "paged_key_mass"]

# struct spruce_paged_key_mass_args and spruce_paged_evict_args, field by field.
_MASS_ARGS = struct.Struct("=q3qq4qq3qqqqqqqqqqqqqqdqqq")
_EVICT_ARGS = struct.Struct("=q4qq4qq3qqqqqqqqqqqqqqqqqqqqq")


def _check_pages(k_pages, mass_pages, page_table, kv_lens, device):
    """The shape of checked pages with their masses, and of the table."""
    shape = k_pages.shape
    if len(shape) != 4 or mass_pages.shape != shape[:3]:
        raise ValueError("the pages must be [pages, Hkv, page_size, D] and mass_pages [pages, Hkv, page_size]")
    if mass_pages.dtype != torch.float32:
        raise ValueError("mass_pages must be float32")
    if k_pages.stride()[3] != 1:
        raise ValueError("the pages must have a contiguous final dimension")
    if shape[3] != 128 and shape[3] != 64:
        raise ValueError(f"kernel supports head_dim 64 or 128, got {shape[3]}")
    if page_table.dim() != 2 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be int32 [S, W]")
    S, W = page_table.shape
    if S < 1 or (W > 1 and page_table.stride()[1] != 1):
        raise ValueError("page_table needs a sequence and a contiguous final dimension")
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (S,) or not kv_lens.is_contiguous():
        raise ValueError(f"kv_lens must be contiguous int32 [S] = [{S}]")
    if mass_pages.device != device or page_table.device != device or kv_lens.device != device:
        raise ValueError("the cache and the batch's tensors must be on one device")
    return shape, S, W


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*shape):
    return spruce_hip.lib().spruce_paged_key_mass_workspace_bytes(*shape)


@functools.lru_cache(maxsize=1024)
def _evict_workspace_bytes(*shape):
    return spruce_hip.lib().spruce_paged_evict_workspace_bytes(*shape)


def paged_key_mass(q, k_pages, mass_pages, page_table, q_starts, kv_lens, scale, *, accumulate=True):
    """The attention weight that the new tokens give to their sequences' cached keys.

    q ``[N,Hq,D]`` (bf16 or f16; any strides with a contiguous last dim and 16-byte
    aligned rows), packed by ``q_starts`` int32 ``[S + 1]`` as for
    ``kernels.paged.paged_chunk_attention``, whose weights these are: for key j of KV
    head g the sum, over the new tokens at positions p >= j and the query heads of
    g, of softmax_j(scale q.k_j) over the keys up to p.

    Every sequence with new tokens has the masses of its positions below
    ``kv_lens[s]`` written: those of the new tokens' own are set, of earlier
    positions added to, or set without ``accumulate`` (the weights of a window of last
    tokens, or of the last token alone).  The rest of ``mass_pages`` is left as it was;
    a key without a page gets no weight, what masked keys hold reaches no sum, and a
    token that attends no key gives none.  Weights are formed and added in 32
    bits, in one order whatever the timing.  Returns ``mass_pages``.
    """
    device, dtype = q.device, q.dtype
    if q.dim() != 3:
        raise ValueError("q must be [N, Hq, D] and the pages [pages, Hkv, page_size, D]")
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError(f"the key mass takes bfloat16 or float16, got {dtype}")
    if k_pages.device != device:
        raise ValueError("the cache and the batch's tensors must be on one device")
    shape, S, W = _check_pages(k_pages, mass_pages, page_table, kv_lens, device)
    N, Hq, D = q.shape
    pages, Hkv, page_size = shape[0], shape[1], shape[2]
    if k_pages.dtype != dtype:
        raise ValueError("the pages must have the dtype of q")
    if shape[3] != D:
        raise ValueError("q and the pages must match in head_dim")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("query heads must be divisible by KV heads")
    if q_starts.dtype != torch.int32 or q_starts.shape != (S + 1,) or not q_starts.is_contiguous():
        raise ValueError(f"q_starts must be contiguous int32 [S + 1] = [{S + 1}]")
    if q_starts.device != device:
        raise ValueError("the cache and the batch's tensors must be on one device")
    qs = q.stride()
    if qs[2] != 1:
        raise ValueError("q must have a contiguous final dimension")
    if not 2.0 ** -100 <= scale < float("inf"):
        raise ValueError(f"scale must be at least 2^-100 and finite, got {scale}")
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or mass_pages.requires_grad):
        _refuse_grad()
    if not q.is_cuda:
        raise RuntimeError("the paged HIP backend requires GPU tensors")
    need = _workspace_bytes(N, S, Hq, Hkv, W * page_size)
    work = q.new_empty_strided((need,), (1,), dtype=torch.uint8)
    with spruce_hip.on_device(device):
        rc = spruce_hip.lib().spruce_paged_key_mass(_MASS_ARGS.pack(
            q.data_ptr(), *qs, k_pages.data_ptr(), *k_pages.stride(), mass_pages.data_ptr(), *mass_pages.stride(), pages,
            page_size, page_table.data_ptr(), page_table.stride()[0] if S > 1 else W, W, q_starts.data_ptr(),
            kv_lens.data_ptr(), S, N, Hq, Hkv, D, spruce_hip.DTYPE_CODES[dtype], scale, bool(accumulate),
            work.data_ptr(), need), spruce_hip.raw_stream(device.index))
    if rc:
        spruce_hip.check(rc, "spruce_paged_key_mass")
    return mass_pages


def evict_paged_kv(k_pages, v_pages, mass_pages, page_table, kv_lens, out_table, keep, *, first=0, recent=0):
    """Cut every sequence's cache down to ``keep`` keys a KV head.

    Of the positions below ``kv_lens[s]`` stay the first ``first``, the last
    ``recent``, and of those between the ones with the largest masses, each head its
    own (ties to the lowest position; NaN counts as the lowest); all of them where
    there are no more than ``keep``.  Their keys, values (bf16, f16 or f32, rows
    16-byte aligned) and masses move, in order, into the pages that ``out_table``
    int32 ``[S, W2]`` names: the r-th to slot ``r % page_size`` of page
    ``out_table[s, r // page_size]``.  Those are pages that no sequence reads
    from here, such as free ones (the old pages, shared ones too, keep what they hold),
    or a sequence's own in their old order where it keeps everything.  Positions
    without a page count as the lowest, and where one is kept its new slot keeps what it holds; a
    row whose new page is none does not move.

    Returns (``kept`` int32 ``[S,Hkv,keep]``, the kept positions in ascending order with
    -1 behind them, ``lens`` int32 ``[S]``, the new ``kv_lens``).
    """
    device, dtype = k_pages.device, k_pages.dtype
    shape, S, W = _check_pages(k_pages, mass_pages, page_table, kv_lens, device)
    pages, Hkv, page_size, D = shape
    if v_pages.shape != shape or v_pages.dtype != dtype or v_pages.device != device:
        raise ValueError("k_pages and v_pages must match as [pages, Hkv, page_size, D]")
    if v_pages.stride()[3] != 1:
        raise ValueError("the pages must have a contiguous final dimension")
    code = spruce_hip.dtype_code(k_pages)
    if out_table.dim() != 2 or out_table.dtype != torch.int32 or out_table.shape[0] != S:
        raise ValueError(f"out_table must be int32 [S, W] with S = {S}")
    W2 = out_table.shape[1]
    if W2 > 1 and out_table.stride()[1] != 1:
        raise ValueError("out_table must have a contiguous final dimension")
    if out_table.device != device:
        raise ValueError("the cache and the batch's tensors must be on one device")
    if keep < 1 or first < 0 or recent < 0 or first + recent > keep:
        raise ValueError(f"keep must be positive and first and recent fit into it, got {keep}, {first} and {recent}")
    if torch.is_grad_enabled() and (k_pages.requires_grad or v_pages.requires_grad or mass_pages.requires_grad):
        _refuse_grad()
    if not k_pages.is_cuda:
        raise RuntimeError("the paged HIP backend requires GPU tensors")
    kept = kv_lens.new_empty_strided((S, Hkv, keep), (Hkv * keep, keep, 1))
    lens = kv_lens.new_empty_strided((S,), (1,))
    need = _evict_workspace_bytes(S, Hkv, W * page_size)
    work = kv_lens.new_empty_strided((need,), (1,), dtype=torch.uint8) if need else None
    with spruce_hip.on_device(device):
        rc = spruce_hip.lib().spruce_paged_evict(_EVICT_ARGS.pack(
            k_pages.data_ptr(), *k_pages.stride(), v_pages.data_ptr(), *v_pages.stride(), mass_pages.data_ptr(),
            *mass_pages.stride(), pages, page_size, page_table.data_ptr(), page_table.stride()[0] if S > 1 else W, W,
            kv_lens.data_ptr(), S, Hkv, D, code, out_table.data_ptr(), out_table.stride()[0] if S > 1 else W2, W2,
            keep, first, recent, kept.data_ptr(), lens.data_ptr(), work.data_ptr() if need else 0, need), spruce_hip.raw_stream(device.index))
    if rc:
        spruce_hip.check(rc, "spruce_paged_evict")
    return kept, lens

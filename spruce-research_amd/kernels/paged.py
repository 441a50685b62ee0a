"""Attention over a paged K/V cache on gfx950 (HIP, C ABI): the form of the
sparse-prefill path in which a prompt comes in chunks, or goes on token by
token.

The cache is ``k_pages``, ``v_pages`` ``[pages, Hkv, page_size, D]`` (any
strides with a contiguous last dim, e.g. views of ``[pages, page_size, Hkv, D]``
storage).  A ragged batch of S sequences is described by three device tensors
that every call here takes, and reads on the device only:

* ``page_table`` int32 ``[S, W]``: position p of sequence s lies in slot
  ``p % page_size`` of page ``page_table[s, p // page_size]``; ids outside
  ``[0, pages)`` name no page; one row expanded over sequences that share their
  pages will do;
* ``q_starts`` int32 ``[S + 1]``, ascending: the new tokens of sequence s are rows
  ``q_starts[s] .. q_starts[s + 1]`` of the packed ``[N, H, D]`` tensors; rows behind
  ``q_starts[S]`` belong to no sequence and are left alone;
* ``kv_lens`` int32 ``[S]``: positions in the cache, the new tokens' included, so
  new token i of n stands at position ``kv_lens[s] - n + i``.

Calls run on the current stream of the tensors' device, wait for nothing and
can be captured; a replay goes by what the three tensors then hold.  Inference
only: inputs that need gradients are refused.
"""
import functools
import struct

import torch

import spruce_hip
from kernels.rotary import _needs_grad, _positions, _refuse_grad, _rotation, _weights

__all__ = ["append_paged_kv", "paged_chunk_attention"]

# struct spruce_paged_append_args and spruce_paged_attention_args, field by field.
_APPEND_ARGS = struct.Struct("=q3qq3qq3qq3q5qq4qq4qqqqqqqqqqqqqqdqqqd")
_ATTENTION_ARGS = struct.Struct("=q3qq4qq4qqqqqqqq6qdq4qqqq3qqq")


def _check_cache(k_pages, v_pages, page_table, q_starts, kv_lens, dtype, device):
    """The packed fields of a checked cache and batch (pages to sequences), and its shape."""
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    if len(shape) != 4 or shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must match as [pages, Hkv, page_size, D]")
    if k_pages.dtype != dtype or v_pages.dtype != dtype:
        raise ValueError("the pages must have the dtype of the new tokens")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("k_pages and v_pages must have a contiguous final dimension")
    if page_table.dim() != 2 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be int32 [S, W]")
    S, W = page_table.shape
    ts, step = page_table.stride()
    if S < 1 or (W > 1 and step != 1):
        raise ValueError("page_table needs a sequence and a contiguous final dimension")
    if q_starts.dtype != torch.int32 or q_starts.shape != (S + 1,) or not q_starts.is_contiguous():
        raise ValueError(f"q_starts must be contiguous int32 [S + 1] = [{S + 1}]")
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (S,) or not kv_lens.is_contiguous():
        raise ValueError(f"kv_lens must be contiguous int32 [S] = [{S}]")
    if (k_pages.device != device or v_pages.device != device or page_table.device != device
            or q_starts.device != device or kv_lens.device != device):
        raise ValueError("the cache and the batch's tensors must be on the same device as the new tokens")
    # One sequence's row has no stride that matters.
    fields = (k_pages.data_ptr(), *ks, v_pages.data_ptr(), *vs, shape[0], shape[2], page_table.data_ptr(),
              ts if S > 1 else W, W, q_starts.data_ptr(), kv_lens.data_ptr(), S)
    return fields, shape


def append_paged_kv(k, v, k_pages, v_pages, page_table, q_starts, kv_lens, *, query=None, inv_freq=None,
                    layout="half", factor=1.0, q_weight=None, k_weight=None, eps=1e-6, positions=None):
    """Write the new tokens' keys and values into their pages.

    k, v ``[N,Hkv,D]`` (any strides with a contiguous last dim and 16-byte
    aligned rows, e.g. slices of one fused projection).  The keys are normed
    (``k_weight``) and rotated (``inv_freq``) on the way as
    ``kernels.rotary.rotate_heads`` does it, by their cache positions or by
    ``positions`` (int32 or int64 ``[N]``).  With ``query`` ``[N,Hq,D]`` the queries
    are normed and rotated in the same launch and returned as a new tensor
    (rows of no sequence in it are unspecified); None otherwise.  A token without a
    page is not written.  Two tokens must not share a slot: which of them it then
    holds is unspecified.  bf16, f16 or f32; float32 pages are for a caller's own
    use, ``paged_chunk_attention`` takes the 16-bit types.
    """
    device, dtype = k.device, k.dtype
    if k.dim() != 3 or k.shape != v.shape or v.dtype != dtype or v.device != device:
        raise ValueError("k and v must match as [N, Hkv, D]")
    N, Hkv, D = k.shape
    if D != 128 and D != 64:
        raise ValueError(f"kernel supports head_dim 64 or 128, got {D}")
    cache, pages = _check_cache(k_pages, v_pages, page_table, q_starts, kv_lens, dtype, device)
    if pages[1] != Hkv or pages[3] != D:
        raise ValueError("the pages and the new tokens must match in KV heads and head_dim")
    ks, vs = k.stride(), v.stride()
    if ks[2] != 1 or vs[2] != 1:
        raise ValueError("k and v must have a contiguous final dimension")
    Hq, qs, out = 0, (0, 0, 0), None
    if query is not None:
        if query.dim() != 3 or query.shape[0] != N or query.shape[2] != D or query.dtype != dtype:
            raise ValueError("query must be [N, Hq, D] in the dtype of k")
        if query.device != device:
            raise ValueError("query must be on the same device as k")
        Hq, qs = query.shape[1], query.stride()
        if qs[2] != 1:
            raise ValueError("query must have a contiguous final dimension")
        if Hq < 1:
            raise ValueError("query must have a head")
    rotation = _rotation(inv_freq, layout, D, device)
    weights = _weights(q_weight, k_weight, D, dtype, device)
    place = (0, 0, False) if positions is None else _positions(positions, ((N,),), device)
    if torch.is_grad_enabled() and (
            k.requires_grad or v.requires_grad or k_pages.requires_grad or v_pages.requires_grad
            or (query is not None and query.requires_grad) or _needs_grad(q_weight, k_weight, inv_freq)):
        _refuse_grad()
    if not k.is_cuda:
        raise RuntimeError("the paged HIP backend requires GPU tensors")
    if Hq:
        out = k.new_empty_strided((N, Hq, D), (Hq * D, D, 1))
    with spruce_hip.on_device(device):
        rc = spruce_hip.lib().spruce_paged_append(_APPEND_ARGS.pack(
            query.data_ptr() if Hq else 0, *qs, out.data_ptr() if Hq else 0, Hq * D, D, 1,
            k.data_ptr(), *ks, v.data_ptr(), *vs, N, Hq, Hkv, D, spruce_hip.dtype_code(k), *cache, place[0], place[2],
            *rotation, factor, *weights, eps), spruce_hip.raw_stream(device.index))
    if rc:
        spruce_hip.check(rc, "spruce_paged_append")
    return out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*shape):
    return spruce_hip.lib().spruce_paged_attention_workspace_bytes(*shape)


def paged_chunk_attention(q, k_pages, v_pages, page_table, q_starts, kv_lens, scale, *, indices=None, out=None):
    """Attention of the new tokens over their sequences' cached keys, their own
    (already appended) included: a token at position p attends the positions up to p.

    q ``[N,Hq,D]`` (bf16 or f16; any strides with a contiguous last dim and 16-byte
    aligned rows); Hq a multiple of the pages' Hkv.  indices: optional int32
    ``[S,Hkv,Qc,K]`` block lists; row b of a sequence lists the 64-key blocks
    (of positions ``64 id .. 64 id + 63``) for its new tokens in the b-th
    64-position block that these touch: the slice of a ``selected_blocks``
    layer that belongs to the chunk.  Negative entries are padding, blocks
    behind a token's own are ignored, duplicates attended as often as listed;
    tokens past row Qc attend nothing.

    Returns ``[N,Hq,D]`` (``out`` when given, which must share no memory with the
    inputs; rows of no sequence are left as they were).  A token that attends no key gets zeros, a key without a page no
    weight, and what masked keys and values hold reaches no row.
    """
    device, dtype = q.device, q.dtype
    if q.dim() != 3:
        raise ValueError("q must be [N, Hq, D] and the pages [pages, Hkv, page_size, D]")
    if dtype != torch.bfloat16 and dtype != torch.float16:
        raise ValueError(f"the paged attention takes bfloat16 or float16, got {dtype}")
    N, Hq, D = q.shape
    cache, (_, Hkv, page_size, Dk) = _check_cache(k_pages, v_pages, page_table, q_starts, kv_lens, dtype, device)
    S, W = page_table.shape
    if D != 128 and D != 64:
        raise ValueError(f"kernel supports head_dim 64 or 128, got {D}")
    if Dk != D:
        raise ValueError("q and the pages must match in head_dim")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("query heads must be divisible by KV heads")
    qs = q.stride()
    if qs[2] != 1:
        raise ValueError("q must have a contiguous final dimension")
    if not 0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    lists, K = (0, 0, 0, 0, 1, 0, 0), 0
    if indices is not None:
        if indices.dim() != 4 or tuple(indices.shape[:2]) != (S, Hkv) or indices.dtype != torch.int32:
            raise ValueError("indices must be int32 [S,Hkv,Qc,K]")
        Qc, K = indices.shape[2:]
        if Qc < 1 or K < 1:
            raise ValueError("indices must hold a row and a column")
        strides = indices.stride()
        if strides[3] != 1 and K > 1:
            raise ValueError("indices must have a contiguous final dimension")
        if indices.device != device:
            raise ValueError("indices must be on the same device as q")
        lists = (indices.data_ptr(), *strides[:3], 1, Qc, K)
    if out is not None and (out.shape != q.shape or out.dtype != dtype or out.device != device or out.stride(-1) != 1):
        raise ValueError("out must match q in shape, dtype and device, with a contiguous final dimension")
    if torch.is_grad_enabled() and (q.requires_grad or k_pages.requires_grad or v_pages.requires_grad
                                    or (out is not None and out.requires_grad)):
        _refuse_grad()
    if not q.is_cuda:
        raise RuntimeError("the paged HIP backend requires GPU tensors")
    if out is None:
        out = q.new_empty_strided((N, Hq, D), (Hq * D, D, 1))
    need = _workspace_bytes(N, S, Hq, Hkv, D, W * page_size, K)
    work = q.new_empty_strided((need,), (1,), dtype=torch.uint8)
    with spruce_hip.on_device(device):
        rc = spruce_hip.lib().spruce_paged_attention(_ATTENTION_ARGS.pack(
            q.data_ptr(), *qs, *cache, N, Hq, Hkv, D, spruce_hip.DTYPE_CODES[dtype], scale, *lists,
            out.data_ptr(), *out.stride(), work.data_ptr(), need), spruce_hip.raw_stream(device.index))
    if rc:
        spruce_hip.check(rc, "spruce_paged_attention")
    return out

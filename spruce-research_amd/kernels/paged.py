"""Attention over a paged K/V cache on gfx950 (HIP, C ABI): the form of the
sparse-prefill path in which a prompt comes in chunks, or goes on token by
token.

The cache is ``k_pages``, ``v_pages`` ``[pages, Hkv, page_size, D]`` (any
strides with a contiguous last dim, e.g. views of ``[pages, page_size, Hkv, D]``
storage).  A ragged batch of S sequences is described by three device tensors
that every call here takes, and reads on the device only:

* ``page_table`` int32 ``[S, W]``: position p of sequence s lies in slot
  ``p % page_size`` of page ``page_table[s, p // page_size]``; ids outside
  ``[0, pages)`` name no page;
* ``q_starts`` int32 ``[S + 1]``, ascending: the new tokens of sequence s are rows
  ``q_starts[s] .. q_starts[s + 1]`` of the packed ``[N, H, D]`` tensors; rows behind
  ``q_starts[S]`` belong to no sequence and are left alone;
* ``kv_lens`` int32 ``[S]``: positions in the cache, the new tokens' included, so
  new token i of n stands at position ``kv_lens[s] - n + i``.

Calls run on the current stream of the tensors' device, wait for nothing and
can be captured; a replay goes by what the three tensors then hold.  Inference
only: inputs that need gradients are refused.
"""
import ctypes

import torch

import spruce_hip
from kernels.rotary import _positions, _refuse_grad, _rotation, _weights

__all__ = ["append_paged_kv", "paged_chunk_attention"]

_I64X3 = ctypes.c_int64 * 3


def _check_cache(k_pages, v_pages, page_table, q_starts, kv_lens, like):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
        raise ValueError("k_pages and v_pages must match as [pages, Hkv, page_size, D]")
    if k_pages.dtype != like.dtype or v_pages.dtype != like.dtype:
        raise ValueError("the pages must have the dtype of the new tokens")
    if k_pages.stride(-1) != 1 or v_pages.stride(-1) != 1:
        raise ValueError("k_pages and v_pages must have a contiguous final dimension")
    if page_table.dim() != 2 or page_table.dtype != torch.int32:
        raise ValueError("page_table must be int32 [S, W]")
    S = page_table.shape[0]
    if S < 1 or (page_table.shape[1] > 1 and page_table.stride(1) != 1):
        raise ValueError("page_table needs a sequence and a contiguous final dimension")
    if q_starts.dtype != torch.int32 or q_starts.shape != (S + 1,) or not q_starts.is_contiguous():
        raise ValueError(f"q_starts must be contiguous int32 [S + 1] = [{S + 1}]")
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (S,) or not kv_lens.is_contiguous():
        raise ValueError(f"kv_lens must be contiguous int32 [S] = [{S}]")
    device = like.device
    if (k_pages.device != device or v_pages.device != device or page_table.device != device
            or q_starts.device != device or kv_lens.device != device):
        raise ValueError("the cache and the batch's tensors must be on the same device as the new tokens")
    return S


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
    holds is unspecified.
    """
    if k.dim() != 3 or k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
        raise ValueError("k and v must match as [N, Hkv, D]")
    N, Hkv, D = k.shape
    if D not in (64, 128):
        raise ValueError(f"kernel supports head_dim 64 or 128, got {D}")
    S = _check_cache(k_pages, v_pages, page_table, q_starts, kv_lens, k)
    if k_pages.shape[1] != Hkv or k_pages.shape[3] != D:
        raise ValueError("the pages and the new tokens must match in KV heads and head_dim")
    if k.stride(-1) != 1 or v.stride(-1) != 1:
        raise ValueError("k and v must have a contiguous final dimension")
    Hq, out = 0, None
    if query is not None:
        if query.dim() != 3 or query.shape[0] != N or query.shape[2] != D or query.dtype != k.dtype:
            raise ValueError("query must be [N, Hq, D] in the dtype of k")
        if query.device != k.device:
            raise ValueError("query must be on the same device as k")
        if query.stride(-1) != 1:
            raise ValueError("query must have a contiguous final dimension")
        Hq = query.shape[1]
        if Hq < 1:
            raise ValueError("query must have a head")
    rotary_dim, code = _rotation(inv_freq, layout, D, k.device)
    weight_code = _weights(q_weight, k_weight, D, k)
    pos64 = 0 if positions is None else _positions(positions, ((N,),), k.device)
    _refuse_grad(k, v, query, k_pages, v_pages, q_weight, k_weight, inv_freq)
    if not k.is_cuda:
        raise RuntimeError("the paged HIP backend requires GPU tensors")
    if query is not None:
        out = torch.empty((N, Hq, D), device=k.device, dtype=k.dtype)
    with spruce_hip.on_device(k.device):
        rc = spruce_hip.lib().spruce_paged_append(
            spruce_hip.ptr(query), _I64X3(*query.stride()) if Hq else None, spruce_hip.ptr(out),
            _I64X3(*out.stride()) if Hq else None,
            spruce_hip.ptr(k), _I64X3(*k.stride()), spruce_hip.ptr(v), _I64X3(*v.stride()),
            N, Hq, Hkv, D, spruce_hip.dtype_code(k),
            spruce_hip.ptr(k_pages), spruce_hip.strides(k_pages), spruce_hip.ptr(v_pages), spruce_hip.strides(v_pages),
            k_pages.shape[0], k_pages.shape[2], spruce_hip.ptr(page_table), page_table.stride(0), page_table.shape[1],
            spruce_hip.ptr(q_starts), spruce_hip.ptr(kv_lens), S, spruce_hip.ptr(positions), pos64,
            spruce_hip.ptr(inv_freq), rotary_dim, code, factor, spruce_hip.ptr(q_weight), spruce_hip.ptr(k_weight),
            weight_code, eps, spruce_hip.stream_of(k))
    spruce_hip.check(rc, "spruce_paged_append")
    return out


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

    Returns ``[N,Hq,D]`` (``out`` when given; rows of no sequence are left as they
    were).  A token that attends no key gets zeros, a key without a page no
    weight, and what masked keys and values hold reaches no row.
    """
    if q.dim() != 3 or k_pages.dim() != 4:
        raise ValueError("q must be [N, Hq, D] and the pages [pages, Hkv, page_size, D]")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"the paged attention takes bfloat16 or float16, got {q.dtype}")
    N, Hq, D = q.shape
    S = _check_cache(k_pages, v_pages, page_table, q_starts, kv_lens, q)
    pages, Hkv, page_size, _ = k_pages.shape
    if D not in (64, 128):
        raise ValueError(f"kernel supports head_dim 64 or 128, got {D}")
    if k_pages.shape[3] != D:
        raise ValueError("q and the pages must match in head_dim")
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise ValueError("query heads must be divisible by KV heads")
    if q.stride(-1) != 1:
        raise ValueError("q must have a contiguous final dimension")
    if not 0 < scale < float("inf"):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    Qc = K = 0
    if indices is not None:
        if indices.dim() != 4 or tuple(indices.shape[:2]) != (S, Hkv) or indices.dtype != torch.int32:
            raise ValueError("indices must be int32 [S,Hkv,Qc,K]")
        Qc, K = indices.shape[2:]
        if Qc < 1 or K < 1:
            raise ValueError("indices must hold a row and a column")
        if indices.stride(-1) != 1 and K > 1:
            raise ValueError("indices must have a contiguous final dimension")
        if indices.device != q.device:
            raise ValueError("indices must be on the same device as q")
    if out is not None:
        if out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.stride(-1) != 1:
            raise ValueError("out must match q in shape, dtype and device, with a contiguous final dimension")
    _refuse_grad(q, k_pages, v_pages, out)
    if not q.is_cuda:
        raise RuntimeError("the paged HIP backend requires GPU tensors")
    if out is None:
        out = torch.empty((N, Hq, D), device=q.device, dtype=q.dtype)
    lib = spruce_hip.lib()
    need = lib.spruce_paged_attention_workspace_bytes(N, S, Hq, Hkv, D, page_table.shape[1] * page_size, K)
    work = torch.empty(need, device=q.device, dtype=torch.uint8)
    with spruce_hip.on_device(q.device):
        rc = lib.spruce_paged_attention(
            spruce_hip.ptr(q), _I64X3(*q.stride()), spruce_hip.ptr(k_pages), spruce_hip.strides(k_pages),
            spruce_hip.ptr(v_pages), spruce_hip.strides(v_pages), pages, page_size,
            spruce_hip.ptr(page_table), page_table.stride(0), page_table.shape[1], spruce_hip.ptr(q_starts),
            spruce_hip.ptr(kv_lens), S, N, Hq, Hkv, D, scale, spruce_hip.DTYPE_CODES[q.dtype],
            spruce_hip.ptr(indices), None if indices is None else spruce_hip.strides(indices), Qc, K,
            spruce_hip.ptr(out), _I64X3(*out.stride()), spruce_hip.ptr(work), need, spruce_hip.stream_of(q))
    spruce_hip.check(rc, "spruce_paged_attention")
    return out

"""Rotary frequencies and the refusals of the rotary and append calls: the
checks come before the GPU is touched, so these run without one."""
import math
import os
import re

import pytest
import torch

import spruce_hip
from kernels import paged, rotary
from kernels.paged import append_paged_kv, paged_chunk_attention
from kernels.rotary import rotary_frequencies, rotate_heads


def test_plain_linear_and_ntk_frequencies():
    R, base = 64, 1e6
    plain, factor = rotary_frequencies(R, base)
    assert plain.dtype == torch.float64 and factor == 1.0
    for i in (0, 1, 17, 31):
        assert plain[i].item() == pytest.approx(base ** (-2 * i / R), rel=1e-14)
    linear, factor = rotary_frequencies(R, base, scaling="linear", factor=4.0)
    assert factor == 1.0 and torch.equal(linear, plain / 4.0)
    ntk, factor = rotary_frequencies(R, base, scaling="ntk", factor=4.0)
    # The fastest pair turns as before, the slowest four times slower.
    assert factor == 1.0 and ntk[0].item() == 1.0
    assert ntk[-1].item() == pytest.approx(plain[-1].item() / 4.0, rel=1e-12)


@pytest.mark.parametrize("dim,base,factor,length", [(128, 1e6, 4.0, 32768), (64, 1e4, 16.0, 2048)])
def test_yarn_frequencies(dim, base, factor, length):
    plain, _ = rotary_frequencies(dim, base)
    yarn, attention = rotary_frequencies(dim, base, scaling="yarn", factor=factor, original_length=length)
    assert attention == pytest.approx(0.1 * math.log(factor) + 1.0)
    turns = plain * length / (2 * math.pi)
    ratio = plain / yarn
    # Away from the two borders (an index either way, for the rounding of their places).
    fast, slow = (turns > 32 * base ** (2 / dim)), (turns < base ** (-4 / dim))
    assert fast.any() and slow.any()
    assert torch.allclose(ratio[fast], torch.ones_like(ratio[fast]), rtol=1e-12)
    assert torch.allclose(ratio[slow], torch.full_like(ratio[slow], factor), rtol=1e-12)
    assert (ratio[1:] >= ratio[:-1] - 1e-12).all()


def test_yarn_agrees_with_transformers():
    rope = pytest.importorskip("transformers.modeling_rope_utils")
    from transformers import Qwen2Config
    config = Qwen2Config(hidden_size=512, num_attention_heads=4, max_position_embeddings=131072, rope_theta=1e6,
                         rope_scaling={"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768})
    want, attention = rope.ROPE_INIT_FUNCTIONS["yarn"](config, torch.device("cpu"))
    got, factor = rotary_frequencies(128, 1e6, scaling="yarn", factor=4.0, original_length=32768)
    assert factor == pytest.approx(attention, rel=1e-6)
    assert torch.allclose(got.float(), want, rtol=1e-5, atol=0)


def test_frequency_refusals():
    for kwargs, message in ((dict(rotary_dim=0), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"),
                            (dict(rotary_dim=64, scaling="other"), "scaling must be"),
                            (dict(rotary_dim=64, factor=0.5), "factor"), (dict(rotary_dim=64, base=1.0), "base"),
                            (dict(rotary_dim=64, scaling="yarn", factor=2.0), "original_length"),
                            (dict(rotary_dim=2, scaling="ntk", factor=2.0), "rotary_dim above 2")):
        with pytest.raises(ValueError, match=message):
            rotary_frequencies(**kwargs)


def _rotate(B=1, T=3, Hq=4, Hkv=2, D=64, dtype=torch.bfloat16, k=None, q=None, positions=None, R=64, **kwargs):
    q = torch.zeros(B, Hq, T, D, dtype=dtype) if q is None else q
    k = torch.zeros(B, Hkv, T, D, dtype=dtype) if k is None else k
    positions = torch.arange(T) if positions is None else positions
    return rotate_heads(q, k, positions, rotary_frequencies(R)[0] if R else None, **kwargs)


def test_rotate_refusals():
    bf = torch.bfloat16
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(R=72), "rotary_dim"), (dict(R=128), "rotary_dim"),
                            (dict(layout="other"), "layout must be"),
                            (dict(k=torch.zeros(1, 2, 4, 64, dtype=bf)), "match in batch"),
                            (dict(k=torch.zeros(1, 2, 3, 64)), "share one dtype"),
                            (dict(q=torch.zeros(1, 4, 64, 3, dtype=bf).transpose(2, 3)), "contiguous final"),
                            (dict(positions=torch.zeros(3)), "int32 or int64"),
                            (dict(positions=torch.zeros(4, dtype=torch.int32)), "positions must be"),
                            (dict(positions=torch.zeros(6, dtype=torch.int32)[::2]), "contiguous tokens"),
                            (dict(q_weight=torch.ones(63)), "norm weights"),
                            (dict(q_weight=torch.ones(64, dtype=torch.float16)), "share one dtype"),
                            (dict(q_weight=torch.ones(64), k_weight=torch.ones(64, dtype=bf)), "share one dtype")):
        with pytest.raises(ValueError, match=message):
            _rotate(**kwargs)
    with pytest.raises(ValueError, match="float64"):
        rotate_heads(torch.zeros(1, 4, 3, 64), torch.zeros(1, 2, 3, 64), torch.arange(3), torch.ones(32))
    with pytest.raises(RuntimeError, match="requires GPU tensors"):
        _rotate()
    grad = torch.zeros(1, 4, 3, 64, dtype=bf, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        _rotate(q=grad)
    with torch.no_grad(), pytest.raises(RuntimeError, match="requires GPU tensors"):
        _rotate(q=grad)


def _append(N=3, Hkv=2, D=64, dtype=torch.bfloat16, S=2, W=4, page=16, **change):
    args = dict(k=torch.zeros(N, Hkv, D, dtype=dtype), v=torch.zeros(N, Hkv, D, dtype=dtype),
                k_pages=torch.zeros(5, Hkv, page, D, dtype=dtype), v_pages=torch.zeros(5, Hkv, page, D, dtype=dtype),
                page_table=torch.zeros(S, W, dtype=torch.int32), q_starts=torch.zeros(S + 1, dtype=torch.int32),
                kv_lens=torch.zeros(S, dtype=torch.int32))
    args.update(change)
    return append_paged_kv(**args)


def test_append_refusals():
    bf, i32 = torch.bfloat16, torch.int32
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"),
                            (dict(v=torch.zeros(4, 2, 64, dtype=bf)), "k and v must match"),
                            (dict(v_pages=torch.zeros(5, 2, 8, 64, dtype=bf)), "k_pages and v_pages must match"),
                            (dict(k_pages=torch.zeros(5, 2, 16, 64), v_pages=torch.zeros(5, 2, 16, 64)), "dtype"),
                            (dict(k_pages=torch.zeros(5, 3, 16, 64, dtype=bf),
                                  v_pages=torch.zeros(5, 3, 16, 64, dtype=bf)), "match in KV heads"),
                            (dict(page_table=torch.zeros(2, 4)), "page_table must be int32"),
                            (dict(page_table=torch.zeros(4, 2, dtype=i32).T), "contiguous final"),
                            (dict(q_starts=torch.zeros(2, dtype=i32)), "q_starts"),
                            (dict(kv_lens=torch.zeros(2)), "kv_lens"),
                            (dict(query=torch.zeros(2, 4, 64, dtype=bf)), "query must be"),
                            (dict(query=torch.zeros(3, 0, 64, dtype=bf)), "must have a head"),
                            (dict(positions=torch.zeros(1, 3, dtype=i32)), "positions must be")):
        with pytest.raises(ValueError, match=message):
            _append(**kwargs)
    with pytest.raises(RuntimeError, match="requires GPU tensors"):
        _append()
    with pytest.raises(RuntimeError, match="no gradients"):
        _append(k=torch.zeros(3, 2, 64, dtype=bf, requires_grad=True))


FAKE = 1 << 20  # never dereferenced: validation fails first


def _call(entry, layout, fields):
    return getattr(spruce_hip.lib(), entry)(layout.pack(*fields), None)


def test_entry_points_refuse_before_the_launch():
    def rotate(D=128, dtype=0, R=128, layout=0, wd=2, qs=(0, 128, 512, 1), B=1, q=FAKE, freq=FAKE, w=0):
        return _call("spruce_rotate_heads", rotary._ROTATE_ARGS, (
            q, *qs, FAKE, 0, 128, 256, 1, B, 4, 2, 8, D, dtype, FAKE, 0, 0, freq, R, layout, 1.0, w, 0, wd, 1e-6,
            FAKE, 0, 128, 512, 1, FAKE, 0, 128, 256, 1))
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(dtype=3), "dtype"), (dict(R=24), "rotary_dim"),
                            (dict(R=144), "rotary_dim"), (dict(layout=2), "layout"), (dict(wd=1), "norm weights"),
                            (dict(w=FAKE + 4), "norm weights must be 16-byte"),
                            (dict(qs=(0, 128, 512, 2)), "contiguous final"), (dict(qs=(0, 100, 512, 1)), "16-byte"),
                            (dict(q=FAKE + 2), "16-byte"), (dict(q=0), "non-null"),
                            (dict(freq=0), "inv_freq"), (dict(B=-1), "invalid shape")):
        assert rotate(**kwargs) == -1, kwargs
        assert message in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())
    assert rotate(B=0) == 0
    assert spruce_hip.lib().spruce_rotate_heads(None, None) == -1

    def append(N=8, Hq=4, page=16, pages=9, width=4, stride=4, S=2, table=FAKE, q=FAKE, kps=(4096, 2048, 128, 1)):
        return _call("spruce_paged_append", paged._APPEND_ARGS, (
            q, 512, 128, 1, FAKE, 512, 128, 1, FAKE, 256, 128, 1, FAKE, 256, 128, 1, N, Hq, 2, 128, 0, FAKE, *kps,
            FAKE, 4096, 2048, 128, 1, pages, page, table, stride, width, FAKE, FAKE, S, 0, 0, 0, 0, 0, 1.0, 0, 0, 2,
            1e-6))
    for kwargs, message in ((dict(page=0), "page size"), (dict(S=0), "sequences"), (dict(stride=3), "overlap"),
                            (dict(width=1 << 28, stride=1 << 28), "2^31"), (dict(pages=-1), "page count"),
                            (dict(N=-1), "token count"), (dict(table=0), "non-null"), (dict(q=0), "non-null"),
                            (dict(kps=(4096, 2048, 100, 1)), "16-byte")):
        assert append(**kwargs) == -1, kwargs
        assert message in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())
    assert append(N=0) == 0
    assert spruce_hip.lib().spruce_paged_append(None, None) == -1


def test_argument_blocks_match_the_header():
    # The packed fields, in order: pointers, integers and arrays are 8 bytes each, doubles "d".
    text = open(os.path.join(os.path.dirname(spruce_hip.LIB_PATH), "..", "..", "include", "spruce_hip.h")).read()
    for name, layout in (("rotate_heads", rotary._ROTATE_ARGS), ("paged_append", paged._APPEND_ARGS),
                         ("paged_attention", paged._ATTENTION_ARGS)):
        body = re.search(r"typedef struct spruce_%s_args \{(.*?)\} spruce" % name, text, re.S).group(1)
        kinds = ""
        for line in body.strip().split(";"):
            for field in filter(None, (f.strip() for f in line.split(","))):
                size = re.search(r"\[(\d)\]", field)
                kinds += ("d" if line.strip().startswith("double") else "q") * (int(size.group(1)) if size else 1)
        code = re.sub(r"(\d)q", lambda m: "q" * int(m.group(1)), layout.format.lstrip("="))
        assert code == kinds, name


def test_page_division_by_multiplication():
    # prepare_batch's constants: l = ceil(log2(page)), magic = floor(2^(31 + l) / page) + 1.
    top = (1 << 31) - 1
    for page in [1, 2, 3, 5, 7, 16, 48, 100, 641, 4095, 4096, 4097, (1 << 29) + 1, (1 << 30) - 1]:
        shift = (page - 1).bit_length()
        magic = (1 << (31 + shift)) // page + 1
        assert magic < 1 << 32
        for k in [0, 1, 2, 3, 1000, top // page - 1, top // page]:
            for p in (k * page - 1, k * page, k * page + 1, k * page + page - 1, top):
                if 0 <= p <= top:
                    assert (p * magic) >> (31 + shift) == p // page, (page, p)


def _attend(N=3, Hq=4, Hkv=2, D=64, dtype=torch.bfloat16, S=2, W=4, page=16, scale=0.1, indices=None, out=None,
            **change):
    args = dict(q=torch.zeros(N, Hq, D, dtype=dtype), k_pages=torch.zeros(5, Hkv, page, D, dtype=dtype),
                v_pages=torch.zeros(5, Hkv, page, D, dtype=dtype), page_table=torch.zeros(S, W, dtype=torch.int32),
                q_starts=torch.zeros(S + 1, dtype=torch.int32), kv_lens=torch.zeros(S, dtype=torch.int32))
    args.update(change)
    return paged_chunk_attention(scale=scale, indices=indices, out=out, **args)


def test_attention_refusals():
    bf, i32 = torch.bfloat16, torch.int32
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(dtype=torch.float32), "bfloat16 or float16"),
                            (dict(Hq=3), "divisible"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                            (dict(scale=float("nan")), "scale"),
                            (dict(q=torch.zeros(3, 64, dtype=bf)), "q must be"),
                            (dict(q=torch.zeros(3, 64, 4, dtype=bf).transpose(1, 2)), "contiguous final"),
                            (dict(k_pages=torch.zeros(5, 2, 16, 128, dtype=bf),
                                  v_pages=torch.zeros(5, 2, 16, 128, dtype=bf)), "match in head_dim"),
                            (dict(kv_lens=torch.zeros(3, dtype=i32)), "kv_lens"),
                            (dict(indices=torch.zeros(2, 2, 1, 3)), "indices must be int32"),
                            (dict(indices=torch.zeros(2, 1, 1, 3, dtype=i32)), "indices must be int32"),
                            (dict(indices=torch.zeros(2, 2, 1, 0, dtype=i32)), "a row and a column"),
                            (dict(indices=torch.zeros(2, 2, 3, 4, dtype=i32).transpose(2, 3)), "contiguous final"),
                            (dict(out=torch.zeros(3, 4, 64)), "out must match")):
        with pytest.raises(ValueError, match=message):
            _attend(**kwargs)
    with pytest.raises(RuntimeError, match="requires GPU tensors"):
        _attend()
    with pytest.raises(RuntimeError, match="no gradients"):
        _attend(q=torch.zeros(3, 4, 64, dtype=bf, requires_grad=True))


def test_attention_entry_point_refuses_before_the_launch():
    need = spruce_hip.lib().spruce_paged_attention_workspace_bytes(8, 2, 4, 2, 128, 64, 0)
    assert need > 0 and need % 16 == 0

    def call(D=128, dtype=0, Hq=4, scale=0.1, qs=(512, 128, 1), K=0, idx=0, is_=(1, 1, 1, 1), Qc=1, ws=FAKE,
             ws_bytes=need, width=4, N=8, q=FAKE):
        return _call("spruce_paged_attention", paged._ATTENTION_ARGS, (
            q, *qs, FAKE, 4096, 2048, 128, 1, FAKE, 4096, 2048, 128, 1, 9, 16, FAKE, 4, width, FAKE, FAKE, 2, N, Hq, 2, D,
            dtype, scale, idx, *is_, Qc, K, FAKE, 512, 128, 1, ws, ws_bytes))
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(dtype=2), "bf16 or f16"),
                            (dict(Hq=5), "divisible"), (dict(Hq=130), "at most 64"), (dict(scale=0.0), "scale"),
                            (dict(scale=float("inf")), "scale"), (dict(qs=(512, 128, 2)), "contiguous final"),
                            (dict(qs=(500, 128, 1)), "16-byte"), (dict(K=4), "indices"),
                            (dict(K=4, idx=FAKE, is_=(1, 1, 1, 2)), "contiguous final"), (dict(K=-1), "list width"),
                            (dict(ws=0), "workspace"), (dict(ws_bytes=need - 4), "workspace too small"),
                            (dict(ws=FAKE + 4), "workspace must be 16-byte"),
                            (dict(width=5), "overlap"), (dict(N=-1), "token count"), (dict(q=0), "non-null")):
        assert call(**kwargs) == -1, kwargs
        assert message in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())
    assert call(N=0) == 0
    assert spruce_hip.lib().spruce_paged_attention(None, None) == -1


def test_outputs_that_overlap_themselves_are_refused():
    def append(kps=(4096, 2048, 128, 1), vps=(4096, 2048, 128, 1), pages=9, page=16):
        return _call("spruce_paged_append", paged._APPEND_ARGS, (
            0, 0, 0, 1, 0, 0, 0, 1, FAKE, 256, 128, 1, FAKE, 256, 128, 1, 8, 0, 2, 128, 0, FAKE, *kps, FAKE, *vps, pages,
            page, FAKE, 4, 4, FAKE, FAKE, 2, 0, 0, 0, 0, 0, 1.0, 0, 0, 2, 1e-6))

    need = spruce_hip.lib().spruce_paged_attention_workspace_bytes(8, 2, 4, 2, 128, 64, 0)

    def attend(os=(512, 128, 1)):
        return _call("spruce_paged_attention", paged._ATTENTION_ARGS, (
            FAKE, 512, 128, 1, FAKE, 4096, 2048, 128, 1, FAKE, 4096, 2048, 128, 1, 9, 16, FAKE, 4, 4, FAKE, FAKE, 2, 8, 4,
            2, 128, 0, 0.1, 0, 1, 1, 1, 1, 1, 0, FAKE, *os, FAKE, need))
    for call, kwargs in ((append, dict(kps=(0, 2048, 128, 1))), (append, dict(kps=(4096, 0, 128, 1))),
                         (append, dict(vps=(4096, 2048, 64, 1))), (attend, dict(os=(0, 128, 1))),
                         (attend, dict(os=(512, 64, 1)))):
        assert call(**kwargs) == -1, kwargs
        assert "overlap" in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())


def test_outputs_whose_dims_step_over_one_another_are_refused():
    # Each stride holds a row, yet rows of two dims meet.
    def rotate(qos=(0, 128, 512, 1), kos=(0, 128, 256, 1), B=1):
        return _call("spruce_rotate_heads", rotary._ROTATE_ARGS, (
            FAKE, 0, 128, 512, 1, FAKE, 0, 128, 256, 1, B, 4, 2, 8, 128, 0, FAKE, 0, 0, FAKE, 128, 0, 1.0, 0, 0, 2, 1e-6,
            FAKE, *qos, FAKE, *kos))

    def append(kps=(4096, 2048, 128, 1), vps=(4096, 2048, 128, 1), qos=(512, 128, 1), pages=9, page=16):
        return _call("spruce_paged_append", paged._APPEND_ARGS, (
            FAKE, 512, 128, 1, FAKE, *qos, FAKE, 256, 128, 1, FAKE, 256, 128, 1, 8, 4, 2, 128, 0, FAKE, *kps, FAKE, *vps,
            pages, page, FAKE, 4, 4, FAKE, FAKE, 2, 0, 0, 0, 0, 0, 1.0, 0, 0, 2, 1e-6))

    need = spruce_hip.lib().spruce_paged_attention_workspace_bytes(8, 2, 4, 2, 128, 64, 0)

    def attend(os):
        return _call("spruce_paged_attention", paged._ATTENTION_ARGS, (
            FAKE, 512, 128, 1, FAKE, 4096, 2048, 128, 1, FAKE, 4096, 2048, 128, 1, 9, 16, FAKE, 4, 4, FAKE, FAKE, 2, 8, 4,
            2, 128, 0, 0.1, 0, 1, 1, 1, 1, 1, 0, FAKE, *os, FAKE, need))
    for call, kwargs in ((append, dict(kps=(128, 128, 128, 1))), (append, dict(kps=(4096, 128, 128, 1))),
                         (append, dict(vps=(2048, 2048, 128, 1))), (append, dict(vps=(4096, 1920, 128, 1))),
                         (append, dict(kps=(2048, 128, 2048, 1))), (append, dict(qos=(128, 128, 1))),
                         (append, dict(qos=(384, 128, 1))), (append, dict(kps=(1 << 62, 128, 256, 1))),
                         (attend, dict(os=(128, 128, 1))), (attend, dict(os=(128, 512, 1))),
                         (attend, dict(os=(504, 128, 1))), (rotate, dict(qos=(0, 128, 128, 1))),
                         (rotate, dict(qos=(0, 128, 384, 1))), (rotate, dict(kos=(0, 512, 128, 1))),
                         (rotate, dict(B=2)), (rotate, dict(B=2, qos=(3968, 128, 512, 1), kos=(2048, 128, 256, 1)))):
        assert call(**kwargs) == -1, kwargs
        assert "overlap" in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())


def test_one_table_row_for_all_sequences_is_taken():
    need = spruce_hip.lib().spruce_paged_attention_workspace_bytes(8, 2, 4, 2, 128, 64, 0)
    for stride, want in ((0, 0), (4, 0), (3, -1), (-4, -1)):       # no new token: the checks alone
        assert _call("spruce_paged_append", paged._APPEND_ARGS, (
            0, 0, 0, 1, 0, 0, 0, 1, FAKE, 256, 128, 1, FAKE, 256, 128, 1, 0, 0, 2, 128, 0, FAKE, 4096, 2048, 128, 1, FAKE,
            4096, 2048, 128, 1, 9, 16, FAKE, stride, 4, FAKE, FAKE, 2, 0, 0, 0, 0, 0, 1.0, 0, 0, 2, 1e-6)) == want
        assert _call("spruce_paged_attention", paged._ATTENTION_ARGS, (
            FAKE, 512, 128, 1, FAKE, 4096, 2048, 128, 1, FAKE, 4096, 2048, 128, 1, 9, 16, FAKE, stride, 4, FAKE, FAKE, 2, 0,
            4, 2, 128, 0, 0.1, 0, 1, 1, 1, 1, 1, 0, FAKE, 512, 128, 1, FAKE, need)) == want


@pytest.mark.parametrize("N,S,lists", [(40000, 2, 0), (40000, 9, 0), (60000, 3, 64)])
def test_single_tokens_beside_a_large_chunk_are_shared_out(N, S, lists):
    # The chunk's tiles go whole; those of the other sequences are few, of a token each, and their keys are
    # shared out, for which the workspace holds two slots of 32 rows a workgroup.
    Hq, Hkv, D = 32, 8, 128
    got = spruce_hip.lib().spruce_paged_attention_workspace_bytes(N, S, Hq, Hkv, D, 131072, lists)
    assert got >= 2 * 256 * 32 * (D + 2) * 4


def test_scales_whose_product_leaves_32_bits_are_refused():
    # exp(scale x) is formed as exp2(scale log2(e) x): an infinite factor would make NaN of a score of zero.
    need = spruce_hip.lib().spruce_paged_attention_workspace_bytes(8, 2, 4, 2, 128, 64, 0)
    for scale, N, want in ((2.5e38, 8, -1), (3.4e38, 8, -1), (1e39, 8, -1), (1e-50, 8, -1), (2.3e38, 0, 0), (1e-30, 0, 0)):
        assert _call("spruce_paged_attention", paged._ATTENTION_ARGS, (
            FAKE, 512, 128, 1, FAKE, 4096, 2048, 128, 1, FAKE, 4096, 2048, 128, 1, 9, 16, FAKE, 4, 4, FAKE, FAKE, 2, N,
            4, 2, 128, 0, scale, 0, 1, 1, 1, 1, 1, 0, FAKE, 512, 128, 1, FAKE, need)) == want, scale
        assert want == 0 or "scale must be positive" in spruce_hip.last_error()

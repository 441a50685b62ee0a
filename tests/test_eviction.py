"""Refusals of the key mass, the eviction and the sampling, on the CPU."""
import os
import re

import pytest
import torch

import spruce_hip
from kernels import eviction, sampling
from kernels.eviction import evict_paged_kv, paged_key_mass
from kernels.sampling import sample_tokens

BF, I32 = torch.bfloat16, torch.int32
FAKE = 1 << 20  # never dereferenced: validation fails first


def _mass(N=3, Hq=4, Hkv=2, D=64, dtype=BF, S=2, W=4, page=16, scale=0.1, **change):
    args = dict(q=torch.zeros(N, Hq, D, dtype=dtype), k_pages=torch.zeros(5, Hkv, page, D, dtype=dtype),
                mass_pages=torch.zeros(5, Hkv, page), page_table=torch.zeros(S, W, dtype=I32),
                q_starts=torch.zeros(S + 1, dtype=I32), kv_lens=torch.zeros(S, dtype=I32))
    args.update(change)
    return paged_key_mass(scale=scale, **args)


def test_mass_refusals():
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(dtype=torch.float32), "bfloat16 or float16"),
                            (dict(Hq=3), "divisible"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"),
                            (dict(scale=1e-31), "scale"), (dict(q=torch.zeros(3, 64, dtype=BF)), "q must be"),
                            (dict(q=torch.zeros(3, 64, 4, dtype=BF).transpose(1, 2)), "contiguous final"),
                            (dict(k_pages=torch.zeros(5, 2, 16, 128, dtype=BF)), "match in head_dim"),
                            (dict(k_pages=torch.zeros(5, 2, 16, 64, dtype=torch.float16)), "dtype of q"),
                            (dict(k_pages=torch.zeros(5, 2, 64, 16, dtype=BF).transpose(2, 3)), "contiguous final"),
                            (dict(mass_pages=torch.zeros(5, 2, 8)), "mass_pages"),
                            (dict(mass_pages=torch.zeros(5, 2, 16, dtype=BF)), "mass_pages must be float32"),
                            (dict(page_table=torch.zeros(2, 4)), "page_table must be int32"),
                            (dict(page_table=torch.zeros(4, 2, dtype=I32).T), "contiguous final"),
                            (dict(q_starts=torch.zeros(2, dtype=I32)), "q_starts"),
                            (dict(kv_lens=torch.zeros(3, dtype=I32)), "kv_lens")):
        with pytest.raises(ValueError, match=message):
            _mass(**kwargs)
    with pytest.raises(RuntimeError, match="requires GPU tensors"):
        _mass()
    grad = torch.zeros(3, 4, 64, dtype=BF, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        _mass(q=grad)
    with torch.no_grad(), pytest.raises(RuntimeError, match="requires GPU tensors"):
        _mass(q=grad)


def _evict(Hkv=2, D=64, dtype=BF, S=2, W=4, W2=2, page=16, keep=20, **change):
    args = dict(k_pages=torch.zeros(5, Hkv, page, D, dtype=dtype), v_pages=torch.zeros(5, Hkv, page, D, dtype=dtype),
                mass_pages=torch.zeros(5, Hkv, page), page_table=torch.zeros(S, W, dtype=I32),
                kv_lens=torch.zeros(S, dtype=I32), out_table=torch.zeros(S, W2, dtype=I32))
    args.update(change)
    return evict_paged_kv(keep=keep, **args)


def test_evict_refusals():
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(dtype=torch.float64), "unsupported dtype"),
                            (dict(v_pages=torch.zeros(5, 2, 16, 64)), "must match"),
                            (dict(v_pages=torch.zeros(5, 2, 64, 16, dtype=BF).transpose(2, 3)), "contiguous final"),
                            (dict(mass_pages=torch.zeros(4, 2, 16)), "mass_pages"),
                            (dict(page_table=torch.zeros(2, 4)), "page_table must be int32"),
                            (dict(kv_lens=torch.zeros(2)), "kv_lens"),
                            (dict(out_table=torch.zeros(3, 2, dtype=I32)), "out_table must be int32"),
                            (dict(out_table=torch.zeros(2, 2)), "out_table must be int32"),
                            (dict(out_table=torch.zeros(2, 2, dtype=I32).T), "contiguous final"),
                            (dict(keep=0), "keep must be"), (dict(first=-1), "keep must be"),
                            (dict(first=11, recent=10), "keep must be")):
        with pytest.raises(ValueError, match=message):
            _evict(**kwargs)
    with pytest.raises(RuntimeError, match="requires GPU tensors"):
        _evict(first=10, recent=10)
    with pytest.raises(RuntimeError, match="no gradients"):
        _evict(k_pages=torch.zeros(5, 2, 16, 64, dtype=BF, requires_grad=True))


def _sample(B=3, V=7, dtype=torch.float32, **change):
    args = dict(logits=torch.zeros(B, V, dtype=dtype), uniform=torch.zeros(B))
    args.update(change)
    return sample_tokens(**args)


def test_sample_refusals():
    for kwargs, message in ((dict(dtype=torch.float64), "unsupported dtype"), (dict(V=0), "a column"),
                            (dict(logits=torch.zeros(3)), r"logits must be \[B, V\]"),
                            (dict(logits=torch.zeros(7, 3).T), "contiguous final"),
                            (dict(uniform=torch.zeros(2)), "uniform"), (dict(uniform=torch.zeros(3, dtype=BF)), "uniform"),
                            (dict(uniform=torch.zeros(6)[::2]), "uniform"),
                            (dict(temperature=-0.5), "temperature"), (dict(temperature=float("nan")), "temperature"),
                            (dict(temperature=torch.ones(2)), "temperature must be"),
                            (dict(top_k=-1), "top_k"), (dict(top_k=torch.ones(3)), "top_k must be"),
                            (dict(top_p=1.5), "top_p"), (dict(top_p=float("nan")), "top_p"),
                            (dict(min_p=-0.1), "min_p"), (dict(min_p=torch.ones(3, dtype=BF)), "min_p must be")):
        with pytest.raises(ValueError, match=message):
            _sample(**kwargs)
    with pytest.raises(RuntimeError, match="requires GPU tensors"):
        _sample()
    with pytest.raises(RuntimeError, match="no gradient"):
        _sample(logits=torch.zeros(3, 7, requires_grad=True))


def _call(entry, layout, fields):
    return getattr(spruce_hip.lib(), entry)(layout.pack(*fields), None)


def test_entry_points_refuse_before_the_launch():
    need = spruce_hip.lib().spruce_paged_key_mass_workspace_bytes(8, 2, 4, 2, 64)
    assert need > 0

    def mass(D=128, dtype=0, Hq=4, scale=0.1, qs=(512, 128, 1), mps=(32, 16, 1), ws=FAKE, ws_bytes=need, width=4, N=8,
             q=FAKE, at=FAKE, S=2, page=16):
        return _call("spruce_paged_key_mass", eviction._MASS_ARGS, (
            q, *qs, FAKE, 4096, 2048, 128, 1, at, *mps, 9, page, FAKE, 4, width, FAKE, FAKE, S, N, Hq, 2, D, dtype, scale,
            1, ws, ws_bytes))
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(dtype=2), "bf16 or f16"),
                            (dict(Hq=5), "divisible"), (dict(Hq=130), "at most 64"), (dict(scale=0.0), "scale"),
                            (dict(scale=3e38), "scale"), (dict(scale=2.0 ** -101), "scale"),
                            (dict(qs=(512, 128, 2)), "contiguous final"), (dict(qs=(500, 128, 1)), "16-byte"),
                            (dict(mps=(16, 16, 1)), "overlap"), (dict(mps=(32, 16, 0)), "overlap"),
                            (dict(at=FAKE + 2), "4-byte"), (dict(at=0), "non-null"), (dict(q=0), "non-null"),
                            (dict(ws=0), "workspace"), (dict(ws_bytes=need - 4), "workspace too small"),
                            (dict(ws=FAKE + 4), "workspace must be 16-byte"), (dict(width=5), "overlap"),
                            (dict(N=-1), "token count"), (dict(S=0), "sequences"), (dict(page=0), "page size")):
        assert mass(**kwargs) == -1, kwargs
        assert message in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())
    assert mass(N=0) == 0
    assert spruce_hip.lib().spruce_paged_key_mass(None, None) == -1

    def evict(D=128, dtype=0, Hkv=2, keep=20, first=2, recent=3, kps=(4096, 2048, 128, 1), mps=(32, 16, 1), stride=2,
              width=2, out=FAKE, at=FAKE, k=FAKE, kept=FAKE, S=2, page=16):
        return _call("spruce_paged_evict", eviction._EVICT_ARGS, (
            k, *kps, FAKE, 4096, 2048, 128, 1, at, *mps, 9, page, FAKE, 4, 4, FAKE, S, Hkv, D, dtype, out, stride, width,
            keep, first, recent, kept, FAKE, 0, 0))
    for kwargs, message in ((dict(D=96), "head_dim 64 or 128"), (dict(dtype=3), "dtype"), (dict(Hkv=0), "KV head"),
                            (dict(keep=0), "keep"), (dict(keep=1 << 30), "keep"), (dict(first=-1), "first"),
                            (dict(first=18), "first"), (dict(kps=(4096, 2048, 128, 2)), "contiguous final"),
                            (dict(kps=(4096, 2048, 100, 1)), "16-byte"), (dict(kps=(2048, 2048, 128, 1)), "overlap"),
                            (dict(mps=(32, 8, 1)), "overlap"), (dict(k=FAKE + 2), "16-byte"), (dict(k=0), "non-null"),
                            (dict(at=FAKE + 1), "4-byte"), (dict(out=0), "non-null"), (dict(kept=0), "non-null"),
                            (dict(width=1, stride=1), "out_table must hold"), (dict(stride=1), "overlap"),
                            (dict(S=0), "sequences"), (dict(page=0), "page size")):
        assert evict(**kwargs) == -1, kwargs
        assert message in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())
    assert spruce_hip.lib().spruce_paged_evict(None, None) == -1

    def sample(B=2, V=9, dtype=2, logits=FAKE, u=FAKE, out=FAKE, heat=1.0, k=0, p=1.0, m=0.0):
        return _call("spruce_sample_tokens", sampling._SAMPLE_ARGS, (
            logits, V, B, V, dtype, u, 0, 0, 0, 0, 0, heat, k, p, m, out, 0, 0, 0))
    for kwargs, message in ((dict(dtype=3), "dtype"), (dict(V=0), "vocabulary"), (dict(V=2088961), "vocabulary"),
                            (dict(B=-1), "row count"), (dict(logits=0), "non-null"), (dict(u=0), "non-null"),
                            (dict(out=0), "non-null"), (dict(logits=FAKE + 2), "aligned"), (dict(heat=-1.0), "temperature"),
                            (dict(heat=float("nan")), "temperature"), (dict(k=-1), "top_k"), (dict(p=1.1), "top_p"),
                            (dict(m=-0.5), "min_p")):
        assert sample(**kwargs) == -1, kwargs
        assert message in spruce_hip.last_error(), (kwargs, spruce_hip.last_error())
    assert sample(B=0) == 0
    assert spruce_hip.lib().spruce_sample_tokens(None, None) == -1


def test_workspaces_are_checked_before_the_launch():
    lib = spruce_hip.lib()
    # A few long rows are shared, many, short or bounded ones are not.
    assert lib.spruce_sample_tokens_workspace_bytes(2, 70000, 1) > lib.spruce_sample_tokens_workspace_bytes(1, 70000, 1) > 0
    assert lib.spruce_sample_tokens_workspace_bytes(2, 40000, 0) > 0 == lib.spruce_sample_tokens_workspace_bytes(2, 40000, 1)
    for B, V in ((129, 70000), (2, 1000), (0, 70000), (-1, 70000), (2, 0), (1 << 40, 70000), (2, 1 << 40)):
        assert lib.spruce_sample_tokens_workspace_bytes(B, V, 0) == 0

    def sample(work, size, V=70000, p=0.9):
        return _call("spruce_sample_tokens", sampling._SAMPLE_ARGS, (
            FAKE, V, 2, V, 0, FAKE, 0, 0, 0, 0, 0, 1.0, 0, p, 0.0, FAKE, 0, work, size))
    need = lib.spruce_sample_tokens_workspace_bytes(2, 70000, 1)
    for args, message in (((0, need), "too small"), ((FAKE, need - 1), "too small"), ((FAKE, 0), "too small"),
                          ((FAKE + 8, need), "16-byte"), ((FAKE, 64, 40000, 1.0), "too small")):
        assert sample(*args) == -1, args
        assert message in spruce_hip.last_error(), (args, spruce_hip.last_error())
    assert lib.spruce_paged_evict_workspace_bytes(2, 2, 32768) == 0
    need = lib.spruce_paged_evict_workspace_bytes(2, 2, 32784)

    def evict(work, size):
        return _call("spruce_paged_evict", eviction._EVICT_ARGS, (
            FAKE, 4096, 2048, 128, 1, FAKE, 4096, 2048, 128, 1, FAKE, 32, 16, 1, 9, 16, FAKE, 2049, 2049, FAKE, 2, 2, 128, 0,
            FAKE, 2, 2, 20, 2, 3, FAKE, FAKE, work, size))
    for args, message in (((0, need), "too small"), ((FAKE, need - 1), "too small"), ((FAKE + 8, need), "16-byte")):
        assert evict(*args) == -1, args
        assert message in spruce_hip.last_error(), (args, spruce_hip.last_error())


def test_argument_blocks_match_the_header():
    # The packed fields, in order: pointers, integers and arrays are 8 bytes each, doubles "d".
    text = open(os.path.join(os.path.dirname(spruce_hip.LIB_PATH), "..", "..", "include", "spruce_hip.h")).read()
    for name, layout in (("paged_key_mass", eviction._MASS_ARGS), ("paged_evict", eviction._EVICT_ARGS),
                         ("sample_tokens", sampling._SAMPLE_ARGS)):
        body = re.search(r"typedef struct spruce_%s_args \{(.*?)\} spruce" % name, text, re.S).group(1)
        kinds = ""
        for line in body.strip().split(";"):
            for field in filter(None, (f.strip() for f in line.split(","))):
                size = re.search(r"\[(\d)\]", field)
                kinds += ("d" if line.strip().startswith("double") else "q") * (int(size.group(1)) if size else 1)
        code = re.sub(r"(\d)q", lambda m: "q" * int(m.group(1)), layout.format.lstrip("="))
        assert code == kinds, name


def test_mass_workspaces_of_the_largest_calls():
    # More scores than 63 bits count (queries of one row for all tokens take no memory): the sums of the two passes.
    size = spruce_hip.lib().spruce_paged_key_mass_workspace_bytes
    for N, Hq in ((1 << 24, 512), (1 << 25, 256), ((1 << 25) + 77, 511)):
        assert size(N, 16, Hq, Hq, (1 << 31) - 1024) >= 8 * N * Hq
    for keys in (-1, 1 << 31, 1 << 40):
        assert size(8, 2, 4, 2, keys) == 0


def test_mass_workspaces_have_room_for_what_few_rows_need():
    # Scores are kept of sequences of up to 32 packed rows: beside longer ones 8 tokens each of four heads a KV head.
    size = spruce_hip.lib().spruce_paged_key_mass_workspace_bytes
    scores = 16 * 8 * 32 * 12000 * 4
    assert scores <= size(640, 16, 32, 8, 12000) <= 1.2 * scores
    assert size(640, 16, 32, 8, 12000) < size(640, 80, 32, 8, 12000)     # 640 tokens of which each may count

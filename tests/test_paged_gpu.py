"""Attention of new tokens over a paged cache on the GPU against a plain form in
64 bits, and the serving step (append, then attention) against the dense one.

The bar of an output o = sum_j p_j v_j / sum_j p_j, with A = sum_j p_j |v_j| / sum_j p_j:
  eps(type) / 2 * |o|      the output's rounding;
  eps(type) / 2 * A        each weight's rounding to the matrix cores' type;
  4 e A                    the 32-bit scores: e = 2^-24 (D + 4) max_j scale sum_d |q_d k_jd| (D products and
                           sums, the scaling and the exponent's argument) + 2^-21 (the exponential and the sums
                           of 32-bit weights), in numerator and denominator;
and for float16 2^-25 (|o|'s smallest step) and 2^-25 sum_j |v_j| / sum_j p_j (weights below its
smallest normal number, relative to the row's largest one).
"""
import pytest
import torch

from kernels.direct_index import direct_index_sparse_prefill
from kernels.paged import append_paged_kv, paged_chunk_attention
from kernels.rotary import rotary_frequencies, rotate_heads
from test_rotary_gpu import make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make_cache(gen, total, Hkv, page, D, dtype, slot_major=True):
    shape = (total, page, Hkv, D) if slot_major else (total, Hkv, page, D)
    k, v = (torch.randn(shape, generator=gen, device=DEV).to(dtype) for _ in range(2))
    return (k.transpose(1, 2), v.transpose(1, 2)) if slot_major else (k, v)


def attend64(q, kp, vp, table, new, kv, scale, lists=None, starts=None):
    """(o, bar) of every row of the sequences' tokens, in 64 bits; lists [S, Hkv, Qc, K] or None."""
    page, Hkv, D = kp.shape[2], kp.shape[1], kp.shape[3]
    Hq = q.shape[1]
    G = Hq // Hkv
    half = torch.finfo(q.dtype).eps / 2
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bar = torch.zeros_like(out)
    row = 0 if starts is None else None
    for s, (n, m) in enumerate(zip(new, kv)):
        at = row if starts is None else starts[s]
        if starts is None:
            row += n
        if n == 0:
            continue
        keys = torch.arange(min(max(m, 0), table.shape[1] * page), device=q.device)
        ids = table[s].long()[keys // page]
        have = (ids >= 0) & (ids < kp.shape[0])
        ids = torch.where(have, ids, 0)
        pos = torch.arange(m - n, m, device=q.device)
        for g in range(Hkv):
            k = kp[ids, g, keys % page].double()
            v = vp[ids, g, keys % page].double()
            seen = have & (keys <= pos[:, None])
            weight = seen.double()
            if lists is not None:
                base = (m - n) // 64
                for i, p in enumerate(pos.tolist()):
                    b = p // 64 - base
                    listed = lists[s, g, b].tolist() if b < lists.shape[2] else []
                    count = torch.zeros(len(keys) // 64 + 2, dtype=torch.float64)
                    for j in listed:
                        if 0 <= j <= p // 64:
                            count[j] += 1
                    weight[i] *= count.to(q.device)[keys // 64]
            for h in range(g * G, (g + 1) * G):
                x = q[at:at + n, h].double()
                score = scale * x @ k.T
                score = score.masked_fill(weight == 0, -torch.inf)
                top = score.amax(-1, keepdim=True) if len(keys) else torch.zeros(n, 1, device=q.device).double()
                top = torch.where(torch.isinf(top), 0.0, top)
                p = (score - top).exp() * weight
                total = p.sum(-1, keepdim=True)
                safe = torch.where(weight[..., None] == 0, 0.0, v) if not bool(torch.isfinite(v).all()) else v
                num = (p[..., None] * safe).sum(1) if safe.dim() == 3 else p @ safe
                away = (p[..., None] * safe.abs()).sum(1) if safe.dim() == 3 else p @ safe.abs()
                size = total.clamp(min=1e-300)
                o = torch.where(total == 0, 0.0, num / size)
                A = torch.where(total == 0, 0.0, away / size)
                worst = scale * (x.abs() @ k.abs().T).masked_fill(weight == 0, 0.0)
                worst = worst.amax(-1, keepdim=True) if len(keys) else torch.zeros_like(total)
                e = 2.0 ** -24 * (D + 4) * worst + 2.0 ** -21
                b = half * o.abs() * (1 + half) + A * (half + 4 * e)
                if q.dtype == torch.float16:
                    all_v = (weight[..., None] * safe.abs()).sum(1) if safe.dim() == 3 else weight @ safe.abs()
                    b = b + 2.0 ** -25 * (1 + torch.where(total == 0, 0.0, all_v / size))
                out[at:at + n, h], bar[at:at + n, h] = o, b
    return out, bar


def check(got, want, bar, what=""):
    off = (got.double() - want).abs()
    fine = (off <= bar) | (torch.isnan(got) & torch.isnan(want)) | (got.double() == want)
    assert bool(fine.all()), (what, float((off - bar).nan_to_num(nan=9e9).max()), (~fine).nonzero()[:4].tolist())


CASES = [
    # new, kv, page, Hq, Hkv, D, slot_major
    ([1], [1], 16, 8, 2, 128, True),
    ([1], [517], 16, 8, 2, 128, True),
    ([1, 1, 1, 1], [64, 65, 1, 2000], 32, 28, 4, 128, False),
    ([1] * 70, [3 + 37 * s for s in range(70)], 16, 12, 2, 64, True),
    ([4, 4, 1, 0, 3], [900, 4, 77, 50, 1500], 32, 16, 8, 64, True),
    ([9, 2], [300, 4096], 48, 28, 4, 128, True),
    ([5], [200], 1, 4, 4, 128, False),
    ([3], [130], 7, 64, 1, 64, True),
    ([64], [64], 64, 8, 2, 128, True),
    ([97, 130], [97, 1000], 64, 28, 4, 128, True),
    ([333], [5000], 128, 12, 2, 128, False),
    ([65, 1, 700], [1000, 33, 700], 16, 16, 8, 64, True),
    ([200], [64 * 20 + 13], 256, 5, 1, 128, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,kv,page,Hq,Hkv,D,slot_major", CASES)
def test_attention(new, kv, page, Hq, Hkv, D, slot_major, dtype):
    print(f"case new={new[:6]} kv={kv[:6]} page={page} {Hq}/{Hkv} D={D} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(sum(new) + page)
    table, starts, lens, total = make_batch(page, new, kv, page)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype, slot_major)
    N = sum(new) + 2
    q = torch.randn(N, Hq + 1, D, generator=gen, device=DEV).to(dtype)[:, 1:]
    out = torch.full((N, Hq, D), 5.0, device=DEV, dtype=dtype)
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5, out=out)
    assert got is out and bool((out[-2:] == 5.0).all())
    want, bar = attend64(q, kp, vp, table, new, kv, D ** -0.5)
    check(out[:-2], want[:-2], bar[:-2])
    again = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5)
    assert torch.equal(again[:-2], out[:-2])


def _lists(seed, new, kv, Hkv, K, empty=True):
    """Random rows over all blocks: duplicates, padding anywhere, blocks behind the token's, empty rows."""
    gen = torch.Generator().manual_seed(seed)
    Qc = max((m - 1) // 64 - (m - n) // 64 + 1 for n, m in zip(new, kv) if n)
    nb = max((m + 63) // 64 for m in kv)
    idx = torch.randint(-2, nb + 2, (len(new), Hkv, Qc, K), generator=gen, dtype=torch.int32)
    if empty:
        idx[0, 0, 0] = -1
    return idx


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,kv,page,Hq,Hkv,D,K", [
    ([1], [700], 16, 8, 2, 128, 4),
    ([1, 1, 5], [64, 2000, 66], 32, 28, 4, 128, 9),
    ([64], [640], 64, 8, 2, 64, 3),
    ([130], [1000], 64, 28, 4, 128, 6),
    ([300, 77], [900, 77], 48, 12, 2, 128, 40),
    ([200], [3000], 128, 16, 8, 64, 1),
])
def test_listed_blocks(new, kv, page, Hq, Hkv, D, K, dtype):
    print(f"case new={new} kv={kv} page={page} {Hq}/{Hkv} D={D} K={K} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(sum(new) + page)
    table, starts, lens, total = make_batch(page, new, kv, page)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(dtype)
    idx = _lists(K, new, kv, Hkv, K)
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5, indices=idx.to(DEV))
    want, bar = attend64(q, kp, vp, table, new, kv, D ** -0.5, idx)
    check(got, want, bar)
    # Rows that the lists do not reach attend nothing.
    short = idx[:, :, :1].to(DEV)
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5, indices=short)
    want, bar = attend64(q, kp, vp, table, new, kv, D ** -0.5, short.cpu())
    check(got, want, bar)


@pytest.mark.parametrize("new", [1, 5, 70])
def test_nothing_of_masked_keys_gets_through(new):
    # Stale slots behind a sequence's end, other pages and later tokens of the chunk hold NaN and infinities.
    page, Hkv, D = 16, 2, 128
    for dtype in (torch.bfloat16, torch.float16):
        for kv in (new, 200, 1000 + new):
            if kv < new:
                continue
            gen = torch.Generator(device=DEV).manual_seed(kv)
            table, starts, lens, total = make_batch(kv, [new], [kv], page)
            kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
            q = torch.randn(new, 8, D, generator=gen, device=DEV).to(dtype)
            pos = torch.arange(total * page, device=DEV).view(total, page)
            own = torch.full((total, page), -1, device=DEV)
            for i, t in enumerate(table[0].tolist()):
                own[t] = i * page + pos[0]
            stale = (own < 0) | (own >= kv)
            kp.transpose(1, 2)[stale] = float("nan")
            vp.transpose(1, 2)[stale] = float("inf")
            last = own == kv - 1           # the last token sees itself alone
            if new > 1:
                kp.transpose(1, 2)[last] = float("nan")
                vp.transpose(1, 2)[last] = float("-inf")
            got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5)
            assert bool(torch.isfinite(got[:-1] if new > 1 else got).all()), (new, kv, dtype)
            if new > 1:
                assert bool(torch.isnan(got[-1]).all())
            clean_k, clean_v = kp.nan_to_num(0.0), vp.nan_to_num(0.0, 0.0, 0.0)
            want, bar = attend64(q, clean_k, clean_v, table, [new], [kv], D ** -0.5)
            keep = slice(0, new - 1) if new > 1 else slice(0, 1)
            check(got[keep], want[keep], bar[keep], (new, kv, dtype))


def test_lengths_that_do_not_fit_and_missing_pages():
    page, Hkv, D, dtype = 16, 2, 64, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(4)
    table, _, _, total = make_batch(9, [1, 1, 1, 1], [96, 96, 96, 96], page)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    table[1, 2] = -1
    table[1, 5] = total
    table[2] = -5                       # no page at all: zeros
    # Rows 0-2 and 63.. belong to no sequence; sequence 0 has 20 new tokens and 5 positions, sequence 3 more
    # positions than its table row.
    new, kv, starts = [20, 20, 10, 10], [5, 90, 50, 120], [3, 23, 43, 53]
    q = torch.randn(66, 4, D, generator=gen, device=DEV).to(dtype)
    out = torch.full_like(q, 5.0)
    paged_chunk_attention(q, kp, vp, table, torch.tensor([*starts, 63], dtype=torch.int32, device=DEV),
                          torch.tensor(kv, dtype=torch.int32, device=DEV), 0.125, out=out)
    want, bar = attend64(q, kp, vp, table, new, kv, 0.125, starts=starts)
    check(out[3:63], want[3:63], bar[3:63])
    assert bool((out[:3] == 5.0).all()) and bool((out[63:] == 5.0).all())
    assert bool((out[3:18] == 0).all()) and bool((out[43:53] == 0).all())
    # No position, no page and no column at all.
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    two = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    for t in (table[:1], table[:1, :0]):
        assert bool((paged_chunk_attention(q[:2], kp, vp, t, two, none, 0.125) == 0).all())
    empty = torch.empty(0, Hkv, page, D, device=DEV, dtype=dtype)
    assert bool((paged_chunk_attention(q[:2], empty, empty, table[:1], two, none + 9, 0.125) == 0).all())
    assert paged_chunk_attention(q[:0], kp, vp, table[:1], none.repeat(2), none, 0.125).shape == (0, 4, D)


def test_hostile_starts_stay_in_bounds():
    # Starts that overlap, go backwards or leave the packed rows: rows are unspecified, memory behind them is not.
    page, dtype = 16, torch.bfloat16
    table, _, _, total = make_batch(1, [1] * 4, [80] * 4, page)
    kp, vp = make_cache(torch.Generator(device=DEV).manual_seed(0), total, 2, page, 64, dtype)
    q = torch.randn(40, 4, 64, device=DEV, dtype=dtype)
    lens = torch.tensor([80, 80, -3, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    for starts in ([0, 40, 0, 40, 0], [-7, 100, 3, 2 ** 31 - 1, 5], [40, 30, 20, 10, 0], [-(2 ** 31), 0, 10, 20, 900]):
        big = torch.full((60, 4, 64), 5.0, device=DEV, dtype=dtype)
        at = torch.tensor(starts, dtype=torch.int32, device=DEV)
        paged_chunk_attention(q, kp, vp, table, at, lens, 0.125, out=big[10:50])
        assert bool((big[:10] == 5.0).all()) and bool((big[50:] == 5.0).all())
        kq, vq = (torch.full((total + 2, 2, page, 64), 5.0, device=DEV, dtype=dtype) for _ in range(2))
        append_paged_kv(q[:, :2], q[:, 2:], kq[1:-1], vq[1:-1], table, at, lens)
        for x in (kq, vq):
            assert bool((x[0] == 5.0).all()) and bool((x[-1] == 5.0).all())


def test_extreme_scores():
    # Scores far apart (one key takes all), all equal, and all far below zero.
    page, D = 32, 64
    table, starts, lens, total = make_batch(3, [2, 1], [400, 300], page)
    gen = torch.Generator(device=DEV).manual_seed(8)
    kp, vp = make_cache(gen, total, 1, page, D, torch.bfloat16)
    q = torch.randn(3, 4, D, generator=gen, device=DEV).to(torch.bfloat16)
    for f in (200.0, 0.0, -200.0):
        got = paged_chunk_attention((q.abs() * f).to(torch.bfloat16), kp.abs(), vp, table, starts, lens, 1.0)
        want, bar = attend64((q.abs() * f).to(torch.bfloat16), kp.abs(), vp, table, [2, 1], [400, 300], 1.0)
        check(got, want, bar, f)


def test_streams_graphs_and_two_calls_at_once():
    page, Hkv, D, dtype = 16, 4, 128, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(2)
    new, kv = [1] * 6, [33, 1200, 77, 5000, 16, 2048]
    table, starts, lens, total = make_batch(6, new, [5000] * 6, page)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    q = [torch.randn(6, 28, D, generator=gen, device=DEV).to(dtype) for _ in range(2)]
    want = [paged_chunk_attention(x, kp, vp, table, starts, lens, 0.08) for x in q]
    streams = [torch.cuda.Stream() for _ in q]
    got = []
    for stream, x in zip(streams, q):
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            got.append(paged_chunk_attention(x, kp, vp, table, starts, lens, 0.08))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Two graphs over the same tensors; replays follow the lengths that the tensors then hold.
    k, v = (torch.randn(6, Hkv, D, generator=gen, device=DEV).to(dtype) for _ in range(2))
    inv_freq = rotary_frequencies(D, device=DEV)[0]
    graphs, outs = [], []
    for x in q:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            turned = append_paged_kv(k, v, kp, vp, table, starts, lens, query=x, inv_freq=inv_freq)
            outs.append(paged_chunk_attention(turned, kp, vp, table, starts, lens, 0.08))
        graphs.append(graph)
    for step in range(3):
        lens.copy_(torch.tensor([m + 700 * step for m in kv[:1]] + [m + step for m in kv[1:3]] + [5000 - step] + kv[4:],
                                dtype=torch.int32))
        for i in (0, 1):
            graphs[i].replay()
            torch.cuda.synchronize()
            turned = append_paged_kv(k, v, kp, vp, table, starts, lens, query=q[i], inv_freq=inv_freq)
            eager = paged_chunk_attention(turned, kp, vp, table, starts, lens, 0.08)
            assert torch.equal(outs[i], eager), (step, i)
            k.mul_(1.01)


def test_chunks_and_tokens_agree_with_the_whole_prompt():
    # A prompt taken in ragged chunks and then token by token, appended and attended, against the dense
    # operators over the whole of it: norms, rotation and block lists included.
    T, Hq, Hkv, D, page, dtype = 333, 8, 2, 128, 16, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(0)
    q, k, v = (torch.randn(T, H, D, generator=gen, device=DEV).to(dtype) for H in (Hq, Hkv, Hkv))
    qw, kw = (1 + 0.1 * torch.randn(D, generator=gen, device=DEV) for _ in range(2))
    inv_freq, factor = rotary_frequencies(D, 1e6, scaling="yarn", factor=4.0, original_length=128, device=DEV)
    turn = dict(inv_freq=inv_freq, factor=factor, q_weight=qw, k_weight=kw)
    nb = (T + 63) // 64
    idx = torch.full((1, Hkv, nb, 3), -1, dtype=torch.int32)
    for b in range(nb):
        idx[0, :, b, :2] = torch.tensor([0, b]) if b else torch.tensor([0, -1])
        idx[0, 1, b, 2] = b // 2 if b > 3 else -1
    idx = idx.to(DEV)
    qr, kr = rotate_heads(q[None].transpose(1, 2), k[None].transpose(1, 2), torch.arange(T, device=DEV), **turn)
    whole = direct_index_sparse_prefill(qr, kr, v[None].transpose(1, 2), idx, D ** -0.5)[0]
    table, _, _, total = make_batch(1, [T], [T], page)
    kp, vp = (torch.zeros(total, page, Hkv, D, device=DEV, dtype=dtype).transpose(1, 2) for _ in range(2))
    parts, at = [], 0
    for n in (130, 100, 60, 40, 1, 1, 1):
        starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        lens = torch.tensor([at + n], dtype=torch.int32, device=DEV)
        turned = append_paged_kv(k[at:at + n], v[at:at + n], kp, vp, table, starts, lens, query=q[at:at + n], **turn)
        assert torch.equal(turned, qr[0].transpose(0, 1)[at:at + n])
        rows = idx[:, :, at // 64:(at + n - 1) // 64 + 1]
        parts.append(paged_chunk_attention(turned, kp, vp, table, starts, lens, D ** -0.5, indices=rows))
        at += n
    assert at == T
    want, bar = attend64(qr[0].transpose(0, 1), kp, vp, table, [T], [T], D ** -0.5, idx.cpu())
    check(torch.cat(parts), want, bar)
    check(whole, want, bar)       # the dense operator's own sums obey the same bar


@pytest.mark.parametrize("new,kv,page,Hq,Hkv,D", [
    ([1] * 70, [1 + 13 * s for s in range(70)], 16, 8, 2, 128),                  # few keys: a tile a workgroup
    ([33] * 66, [33 + 7 * s for s in range(66)], 32, 14, 2, 64),
    ([33] * 66, [1500 - 20 * s for s in range(66)], 32, 14, 2, 64),              # many keys: shared out
    ([33, 1] * 33, [1500 - 20 * s for s in range(66)], 48, 14, 2, 128),          # both kinds, page ends within tiles
    ([1, 2, 5], [1500, 1100, 1300], 16, 40, 40, 64),                             # heads that do not divide the CUs
    ([70], [1200], 64, 40, 40, 64),
    ([1100], [1100], 64, 128, 2, 64),                                            # many tiles: each whole
    ([9], [300], 16, 8, 2, 128),                                                 # two tiles of few rows
    ([9], [3001], 16, 8, 2, 64),
    ([9, 6, 1, 8] * 4, [1100 + 61 * s for s in range(16)], 48, 28, 4, 128),      # a second tile would read the keys again
    ([2, 4, 3] * 30, [1030 + 11 * s for s in range(90)], 16, 14, 2, 64),         # a whole tile for each of many sequences
])
def test_ways_to_share_the_work(new, kv, page, Hq, Hkv, D):
    print(f"case new={new[:4]} kv={kv[:4]} page={page} {Hq}/{Hkv} D={D}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(sum(kv))
    table, starts, lens, total = make_batch(7, new, kv, page)
    kp, vp = make_cache(gen, total, Hkv, page, D, torch.bfloat16)
    q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(torch.bfloat16)
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5)
    want, bar = attend64(q, kp, vp, table, new, kv, D ** -0.5)
    check(got, want, bar)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_many_sequences_of_many_heads(dtype):
    # Enough row tiles that no sequence is split, of sequences that could be.
    S, H, D, page = 130, 128, 64, 32
    gen = torch.Generator(device=DEV).manual_seed(1)
    kv = [1100 - s for s in range(S)]
    table, starts, lens, total = make_batch(5, [1] * S, kv, page)
    kp, vp = make_cache(gen, total, H, page, D, dtype, False)
    q = torch.randn(S, H, D, generator=gen, device=DEV).to(dtype)
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, 0.125).double()
    half = torch.finfo(dtype).eps / 2
    for s in range(S):
        at = torch.arange(kv[s], device=DEV)
        ids = table[s].long()[at // page]
        k, v = (x[ids, :, at % page].double() for x in (kp, vp))       # [kv, H, D]
        x = q[s].double()
        score = 0.125 * (x * k).sum(-1)
        p = torch.softmax(score, 0)[..., None]
        want, away = (p * v).sum(0), (p * v.abs()).sum(0)
        e = 2.0 ** -24 * (D + 4) * 0.125 * (x.abs() * k.abs()).sum(-1).amax(0)[:, None] + 2.0 ** -21
        bar = half * want.abs() * (1 + half) + away * (half + 4 * e)
        if dtype == torch.float16:
            top = torch.exp(score - score.amax(0)).sum(0)[:, None]
            bar = bar + 2.0 ** -25 * (1 + v.abs().sum(0) / top)
        assert bool(((got[s] - want).abs() <= bar).all()), s


@pytest.mark.parametrize("new", [3, 200])
def test_pages_whose_rows_overlap(new):
    # Slots 72 values apart with rows of 128: read as they lie.
    page, Hkv, D, kv = 64, 2, 128, 1300
    gen = torch.Generator(device=DEV).manual_seed(3)
    table, starts, lens, total = make_batch(2, [new], [kv], page)
    span = page * 72 + D
    kp, vp = (torch.randn(total * Hkv * span, generator=gen, device=DEV).to(torch.bfloat16)
              .as_strided((total, Hkv, page, D), (Hkv * span, span, 72, 1)) for _ in range(2))
    q = torch.randn(new, 8, D, generator=gen, device=DEV).to(torch.bfloat16)
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5)
    want, bar = attend64(q, kp.contiguous(), vp.contiguous(), table, [new], [kv], D ** -0.5)
    check(got, want, bar)


@pytest.mark.parametrize("page", [64, 48])
def test_offsets_past_32_bits(page):
    # The sequences' pages are the last of a cache of more than 2^31 elements.
    Hkv, D, dtype = 2, 128, torch.bfloat16
    total = (1 << 31) // (page * Hkv * D) + 200
    gen = torch.Generator(device=DEV).manual_seed(page)
    new, kv = [2, 170], [90, 1100]
    table, starts, lens, used = make_batch(1, new, kv, page)
    kp, vp = (torch.empty(total, page, Hkv, D, device=DEV, dtype=dtype).transpose(1, 2) for _ in range(2))
    for x in (kp, vp):
        x[-used:] = torch.randn(used, Hkv, page, D, generator=gen, device=DEV).to(dtype)
    far = torch.where((table >= 0) & (table < used), table + (total - used), table)
    N = sum(new)
    q, k, v = (torch.randn(N, H, D, generator=gen, device=DEV).to(dtype) for H in (8, Hkv, Hkv))
    near = [x[-used:].clone() for x in (kp, vp)]
    append_paged_kv(k, v, *near, table, starts, lens)
    append_paged_kv(k, v, kp, vp, far, starts, lens)
    assert torch.equal(kp[-used:], near[0]) and torch.equal(vp[-used:], near[1])
    got = paged_chunk_attention(q, kp, vp, far, starts, lens, D ** -0.5)
    assert torch.equal(got, paged_chunk_attention(q, *near, table, starts, lens, D ** -0.5))
    want, bar = attend64(q, *near, table, new, kv, D ** -0.5)
    check(got, want, bar)


def check_exact(got, want, bar, what=""):
    """As check, with rows that are finite, infinite or NaN wherever the 64-bit form's are."""
    want_t = want.to(got.dtype).double()
    finite = torch.isfinite(want)
    off = (got.double() - want).abs()
    fine = torch.where(finite, torch.isfinite(got) & (off <= bar),
                       (torch.isnan(got) & torch.isnan(want)) | (got.double() == want_t))
    assert bool(fine.all()), (what, int((~fine).sum()), (~fine).nonzero()[:4].tolist())


def attend_with_bad_slots(new, kv, page, Hq, Hkv, D, dtype, bad, lists=None, width=None, nan_keys=()):
    """Positions `bad` of every sequence hold infinite values, `nan_keys` NaN keys; slots of no token hold NaN."""
    gen = torch.Generator(device=DEV).manual_seed(sum(new) + sum(kv) + page)
    table, starts, lens, total = make_batch(page, new, kv, page, width=width)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(dtype)
    used = torch.zeros(total, page, dtype=torch.bool, device=DEV)
    for s, m in enumerate(kv):
        at = torch.arange(m, device=DEV)
        used[table[s].long()[at // page], at % page] = True
        for j in bad:
            if j < m:
                vp[int(table[s, j // page]), :, j % page] = float("inf") if j % 2 else float("-inf")
        for j in nan_keys:
            if j < m:
                kp[int(table[s, j // page]), :, j % page] = float("nan")
    kp.transpose(1, 2)[~used] = float("nan")
    vp.transpose(1, 2)[~used] = float("nan")
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5,
                                indices=None if lists is None else lists.to(DEV))
    want, bar = attend64(q, kp, vp, table, new, kv, D ** -0.5, lists)
    check_exact(got, want, bar, (new, kv, page, D, dtype, bad))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,kv,bad", [
    (64, 66, [65]),         # a wave's rows stand on both sides of the block border at 64
    (64, 66, [64, 65]),
    (70, 66, [2]),          # the first rows have no position at all
    (70, 66, [1, 65]),
    (130, 1155, [1088, 1090, 1154]),
])
def test_values_of_the_next_block_reach_no_earlier_row(new, kv, bad, page, dtype):
    print(f"case new={new} kv={kv} page={page} bad={bad} {dtype}", flush=True)
    attend_with_bad_slots([new], [kv], page, 8, 2, 128, dtype, bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("new,kv,bad,nan_keys,width", [
    ([1, 3, 5], [700, 66, 1010], [63, 64, 65, 1008], [1009], 64),          # few rows, whole tiles
    ([1, 3, 5], [700, 66, 1010], [0, 64, 1007], [], 130),                  # the same, shared out
    ([5, 4, 1], [2000, 3, 1301], [1, 1995, 1997, 1300], [1999], 130),
    ([70, 130], [200, 1000], [129, 192, 870, 960, 961], [999], 64),        # many rows, whole tiles
    ([70, 130], [200, 1000], [130, 191, 193, 869, 999], [], 130),          # the same, shared out
    ([131, 66], [1279, 64], [1149, 1151, 1152, 1216, 1217, 3], [1278], 130),
])
def test_bad_values_at_any_place(new, kv, bad, nan_keys, width, page, D, dtype):
    # Seen, they show; unseen, they do not.  `width` pages of 16: up to 1024 positions tiles go whole.
    print(f"case new={new} kv={kv} page={page} D={D} width={width} {dtype}", flush=True)
    # (1008 positions are 21 pages of 48, and 1010 a page more: shared out there.)
    pages = max(width * 16 // page, (max(kv) + page - 1) // page)
    attend_with_bad_slots(new, kv, page, 8, 2, D, dtype, bad, width=pages, nan_keys=nan_keys)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,kv,bad,K", [
    ([1, 3], [700, 66], [63, 64, 699], 6),
    ([1, 3], [700, 1366], [1, 640, 1363, 1364], 20),
    ([70, 40], [200, 1000], [131, 191, 192, 961, 999], 6),
    ([70, 40], [200, 1000], [129, 960, 961], 20),
])
def test_bad_values_in_listed_blocks(new, kv, bad, K, page, D, dtype):
    print(f"case new={new} kv={kv} page={page} D={D} K={K} {dtype}", flush=True)
    attend_with_bad_slots(new, kv, page, 8, 2, D, dtype, bad, lists=_lists(K + D, new, kv, 2, K))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,kv,page,Hq,Hkv,D,K", [
    ([1, 2, 5], [700, 2000, 1300], 16, 8, 2, 128, 40),     # few rows, the lists shared out
    ([1, 4], [1300, 3000], 32, 16, 8, 64, 300),            # more than 64 items a wave
    ([3], [1000], 64, 14, 2, 64, 521),
    ([70, 33], [1500, 3000], 64, 8, 2, 128, 90),           # many rows, more than 64 items
    ([70, 33], [1500, 3000], 48, 28, 4, 64, 131),
])
def test_long_lists(new, kv, page, Hq, Hkv, D, K, dtype):
    print(f"case new={new} kv={kv} page={page} {Hq}/{Hkv} D={D} K={K} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(sum(new) + page)
    table, starts, lens, total = make_batch(page, new, kv, page)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(dtype)
    idx = _lists(K, new, kv, Hkv, K)
    idx[:, :, :, K // 4:K // 2] = -1        # whole rounds of padding in the middle
    idx[-1, -1, 0, :-1] = -1                # one entry, the last
    idx[-1, -1, 0, -1] = 0
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5, indices=idx.to(DEV))
    want, bar = attend64(q, kp, vp, table, new, kv, D ** -0.5, idx)
    check(got, want, bar)


@pytest.mark.parametrize("page", [16, 64])
def test_one_table_row_for_all_sequences(page):
    # Sequences that share their pages: an expanded row, against a table that repeats it.
    Hkv, D, dtype = 2, 128, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(page)
    new, kv = [1, 70, 3], [1300, 900, 1303]
    row, _, _, total = make_batch(3, [1], [1400], page)
    starts = torch.tensor([0, 1, 71, 74], dtype=torch.int32, device=DEV)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    q, k, v = (torch.randn(sum(new), H, D, generator=gen, device=DEV).to(dtype) for H in (8, Hkv, Hkv))
    shared, whole = row.expand(3, -1), row.repeat(3, 1)
    assert shared.stride(0) == 0
    caches = [(kp, vp), (kp.clone(), vp.clone())]
    starts_own = torch.tensor([0, 0, 70, 70], dtype=torch.int32, device=DEV)    # one sequence writes
    for table, (a, b) in zip((shared, whole), caches):
        append_paged_kv(k, v, a, b, table, starts_own, lens)
    assert torch.equal(caches[0][0], caches[1][0]) and torch.equal(caches[0][1], caches[1][1])
    got = paged_chunk_attention(q, kp, vp, shared, starts, lens, D ** -0.5)
    assert torch.equal(got, paged_chunk_attention(q, kp, vp, whole, starts, lens, D ** -0.5))
    want, bar = attend64(q, kp, vp, whole, new, kv, D ** -0.5)
    check(got, want, bar)


@pytest.mark.parametrize("lists", [False, True])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new,kv,Hq,Hkv,D", [
    ([150, 64, 64, 1], [900, 95, 640, 300], 2, 2, 64),      # two tiles of few rows, across a block border
    ([150, 16, 17, 1, 0], [900, 71, 640, 300, 9], 8, 2, 128),
    ([150, 21, 22, 2], [150, 700, 80, 900], 6, 2, 64),
    ([90] + [8] * 20, [700] + [67 + 40 * s for s in range(20)], 8, 2, 64),       # one tile each
    ([1, 2, 1, 3], [700, 66, 900, 64], 40, 1, 64),          # a token of 40 rows
    ([9, 1], [500, 900], 64, 1, 128),
    ([2, 1] * 20, [64 + 20 * s for s in range(40)], 33, 1, 64),                  # none has few rows
])
def test_mixed_batches_at_the_kinds_border(new, kv, Hq, Hkv, D, page, lists):
    # Both with whole tiles (up to 1024 positions, 16 blocks) and shared out.
    gen = torch.Generator(device=DEV).manual_seed(sum(kv))
    for width, K in ((1024 // page, 5), (2048 // page, 33)):
        print(f"case new={new[:5]} kv={kv[:5]} {Hq}/{Hkv} D={D} page={page} lists={lists} width={width}", flush=True)
        table, starts, lens, total = make_batch(7, new, kv, page, width=width)
        kp, vp = make_cache(gen, total, Hkv, page, D, torch.bfloat16)
        q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(torch.bfloat16)
        idx = _lists(K, new, kv, Hkv, K) if lists else None
        out = torch.full((sum(new), Hq, D), 5.0, device=DEV, dtype=torch.bfloat16)
        paged_chunk_attention(q, kp, vp, table, starts, lens, D ** -0.5, out=out,
                              indices=None if idx is None else idx.to(DEV))
        want, bar = attend64(q, kp, vp, table, new, kv, D ** -0.5, idx)
        check(out, want, bar)


@pytest.mark.parametrize("page,new,kv", [(16, 1, 1000), (16, 3, 20000), (64, 70, 1000), (16, 70, 1000), (64, 70, 20000)])
@pytest.mark.parametrize("gap", [12.0, 16.0, 18.0])
def test_float16_weights_far_below_the_largest(gap, page, new, kv):
    # One key, with a value of zero, takes nearly all of the weight; the output is what the many others, `gap`
    # below it, add up to.  Each of their weights w = exp(-gap) times the largest is rounded to 16 bits after a
    # factor of 2^7: by 2^-11 of it where it stays normal (2^-14 and above), by 2^-25 / 2^7 below.
    Hkv, D = 2, 64
    gen = torch.Generator(device=DEV).manual_seed(new)
    table, starts, lens, total = make_batch(2, [new], [kv], page)
    kp, vp = make_cache(gen, total, Hkv, page, D, torch.float16)
    kp.zero_()
    vp.copy_((1 + 0.25 * torch.rand(vp.shape, generator=gen, device=DEV)).half())
    at = 3
    kp[int(table[0, at // page]), :, at % page, 0] = gap
    vp[int(table[0, at // page]), :, at % page] = 0
    q = torch.zeros(new, 8, D, device=DEV, dtype=torch.float16)
    q[..., 0] = 1.0
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, 1.0).double()
    keys = torch.arange(kv, device=DEV)
    v = vp[table[0].long()[keys // page], :, keys % page].double()                  # [kv, Hkv, D]
    w = torch.exp(torch.tensor(-gap, dtype=torch.float64)).item()
    each = max(2.0 ** -11, 2.0 ** -32 / w) if w * 2 ** 7 < 2.0 ** -14 else 2.0 ** -11
    sums = v.cumsum(0)
    for i in range(new):
        n = kv - new + i + 1
        want = (w * sums[n - 1] / (1 + w * (n - 1))).repeat_interleave(4, 0)
        # the weights; the output's rounding; 32-bit sums of positive terms (as in the file's bar, 4 e)
        bar = want * (each + 2.0 ** -11 + 4 * (2.0 ** -24 * (D + 4) * gap + 2.0 ** -21)) + 2.0 ** -25
        assert bool(((got[i] - want).abs() <= bar).all()), (i, float(((got[i] - want).abs() / bar).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,new,kv", [(16, 3, 300), (16, 3, 3000), (64, 70, 900), (16, 70, 900), (64, 70, 3000)])
@pytest.mark.parametrize("size", [2.0 ** 8, 2.0 ** 9, 2.0 ** 10, 2.0 ** 14])
def test_scores_whose_own_rounding_is_large(size, page, new, kv, dtype):
    # Scores of some size^2 D, whose steps in 32 bits are up to 4096: a row is the value of its largest score where
    # that stands alone by more than the products' own error, 2^-24 (D + 4) of it, and some mean of values in any case.
    Hkv, D = 2, 128
    gen = torch.Generator(device=DEV).manual_seed(kv)
    table, starts, lens, total = make_batch(2, [new], [kv], page)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    near = torch.rand(kp.shape, generator=gen, device=DEV) * 2.0 ** -9
    kp.copy_((size * (1 + near)).to(dtype))
    q = (size * (1 + torch.rand(new, 8, D, generator=gen, device=DEV))).to(dtype)
    got = paged_chunk_attention(q, kp, vp, table, starts, lens, 1.0).double()
    keys = torch.arange(kv, device=DEV)
    ids, at = table[0].long()[keys // page], keys % page
    k, v = (x[ids, :, at].double().repeat_interleave(4, 1) for x in (kp, vp))          # [kv, 8, D]
    alone = 0
    for i in range(new):
        n = kv - new + i + 1
        score = (q[i].double() * k[:n]).sum(-1)                                           # [n, 8]
        top, where = score.max(0)
        gap = top - score.scatter(0, where[None], -torch.inf).max(0).values
        low, high = v[:n].amin(0), v[:n].amax(0)
        half = torch.finfo(dtype).eps / 2
        slack = 3 * half * v[:n].abs().amax(0) + 2.0 ** -25
        assert bool(((got[i] >= low - slack) & (got[i] <= high + slack)).all()), i
        one = gap > 4 * 2.0 ** -24 * (D + 4) * top + 40
        alone += int(one.sum())
        want = v[where, torch.arange(8, device=DEV)]
        assert bool(((got[i] - want).abs() <= 3 * half * want.abs() + 2.0 ** -25)[one].all()), i
    print(f"{alone} of {8 * new} rows of one key", flush=True)

"""Key masses of a paged cache and the eviction by them on the GPU, against plain forms in 64 bits.

The bar of a mass m_j = sum_r p_rj over rows r, p_rj = exp(s_rj) / sum_j exp(s_rj):
  p_rj (exp(2 e_r) - 1), e_r = 2^-24 (D + 4) (2 max_j scale sum_d |q_d k_jd| + ln(keys)): the 32-bit scores, D
      products and sums beside a reference of the scores' size, which the row's sum has too (its logarithm
      among it), and the exponents' arguments;
  m_j (2^-21 + 2^-24 (keys / 32 + 32) + 2^-24 (rows / 2 + 32)): the two exponentials, the
      additions of a row's sum (16 at a time, then once per 32 keys) and of a key's (at most rows / 2 in a lane);
  2^-24 of the sum of old and new where it is added to an old value, and 2^-126 a row for
      what is too small for 32 bits.
"""
import math

import pytest
import torch

from kernels.eviction import evict_paged_kv, paged_key_mass
from kernels.paged import append_paged_kv, paged_chunk_attention
from kernels.rotary import rotary_frequencies
from kernels.sampling import sample_tokens
from test_paged_gpu import make_cache
from test_rotary_gpu import make_batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def mass64(q, kp, table, new, kv, scale, starts=None):
    """(mass, bar) [S, Hkv, positions] of this call's weights, in 64 bits."""
    page, Hkv, D = kp.shape[2], kp.shape[1], kp.shape[3]
    G = q.shape[1] // Hkv
    L = table.shape[1] * page
    out = torch.zeros(len(new), Hkv, L, dtype=torch.float64, device=q.device)
    bar = torch.zeros_like(out)
    row = 0
    for s, (n, m) in enumerate(zip(new, kv)):
        at = row if starts is None else starts[s]
        row += n
        keys = torch.arange(min(max(m, 0), L), device=q.device)
        if n == 0 or len(keys) == 0:
            continue
        ids = table[s].long()[keys // page]
        have = (ids >= 0) & (ids < kp.shape[0])
        ids = torch.where(have, ids, 0)
        pos = torch.arange(m - n, m, device=q.device)
        seen = have & (keys <= pos[:, None])
        for g in range(Hkv):
            k = kp[ids, g, keys % page].double()
            for h in range(g * G, (g + 1) * G):
                x = q[at:at + n, h].double()
                score = (scale * x @ k.T).masked_fill(~seen, -torch.inf)
                top = score.amax(-1, keepdim=True)
                p = (score - torch.where(torch.isinf(top), 0.0, top)).exp().masked_fill(~seen, 0.0)
                p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
                worst = (scale * x.abs() @ k.abs().T).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
                e = 2.0 ** -24 * (D + 4) * (2 * worst + math.log(len(keys)))
                out[s, g, :len(keys)] += p.sum(0)
                bar[s, g, :len(keys)] += (p * torch.expm1(2 * e)).sum(0)
        rows = n * G
        bar[s, :, :len(keys)] += out[s, :, :len(keys)] * (2.0 ** -21 + 2.0 ** -24 * (len(keys) / 32 + rows / 2 + 64))
        bar[s, :, :len(keys)] += rows * 2.0 ** -126
    return out, bar


def places(table, kv, page, pages):
    """(sequence, position, page, slot) of the positions below kv that have a page."""
    rows = []
    for s, m in enumerate(kv):
        for j, t in enumerate(table[s].tolist()):
            if 0 <= t < pages:
                rows += [(s, p, t, p - j * page) for p in range(j * page, min((j + 1) * page, m))]
    return [torch.tensor(c, device=DEV) for c in zip(*rows)] if rows else [torch.zeros(0, dtype=torch.long, device=DEV)] * 4


def check_mass(mp, before, q, kp, table, new, kv, scale, accumulate, starts=None):
    want, bar = mass64(q, kp, table, new, kv, scale, starts)
    s, p, t, slot = places(table, [m if n else 0 for n, m in zip(new, kv)], kp.shape[2], kp.shape[0])
    full = before.clone()
    got, exact, off = mp[t, :, slot].double(), want[s, :, p], bar[s, :, p]
    if accumulate:
        first_new = torch.tensor([m - n for n, m in zip(new, kv)], device=DEV)
        old = torch.where((p < first_new[s])[:, None], before[t, :, slot].double(), 0.0)
        exact = exact + old
        off = off + exact.abs() * 2.0 ** -24
    assert bool(((got - exact).abs() <= off).all()), float(((got - exact).abs() / off.clamp(min=1e-300)).max())
    full[t, :, slot] = mp[t, :, slot]
    assert torch.equal(full, mp)        # nothing else was written


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
    ([1, 1], [9000, 20011], 16, 28, 4, 128, True),
    ([40, 33], [9000, 5003], 32, 16, 8, 64, True),
    ([600], [600], 16, 64, 1, 64, False),
    ([1500, 2], [1500, 40], 48, 14, 2, 128, True),
    # Sequences without new tokens beside long ones.
    ([9, 0, 0, 0, 0, 0, 0, 0, 0, 0], [700] * 10, 32, 8, 2, 128, True),
    ([0] * 30 + [60] + [0] * 40, [33] * 30 + [1500] + [7] * 40, 16, 16, 4, 64, False),
    ([0, 1, 33, 0, 1, 0, 40, 0, 0, 1], [500] * 10, 16, 4, 4, 64, True),
    # Few rows as 32 columns.
    ([4, 3], [900, 2000], 32, 28, 4, 128, False),
    ([1, 1, 1], [333, 64, 3000], 16, 32, 1, 64, True),
    # Both ways in one call, past the sequences that a wave looks at together.
    ([1] * 41 + [50] + [2] * 40, [300 + s for s in range(41)] + [1200] + [90] * 40, 16, 8, 2, 64, True),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new,kv,page,Hq,Hkv,D,slot_major", CASES)
def test_mass(new, kv, page, Hq, Hkv, D, slot_major, dtype):
    print(f"case new={new[:6]} kv={kv[:6]} page={page} {Hq}/{Hkv} D={D} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(sum(new) + page)
    table, starts, lens, total = make_batch(page, new, kv, page)
    kp = make_cache(gen, total, Hkv, page, D, dtype, slot_major)[0]
    q = (2 * torch.randn(sum(new) + 2, Hq + 1, D, generator=gen, device=DEV)).to(dtype)[:, 1:]
    before = torch.rand(total, Hkv, page, generator=gen, device=DEV)
    for accumulate in (False, True):
        mp = before.clone()
        assert paged_key_mass(q, kp, mp, table, starts, lens, D ** -0.5, accumulate=accumulate) is mp
        check_mass(mp, before, q, kp, table, new, kv, D ** -0.5, accumulate)
        again = before.clone()
        paged_key_mass(q, kp, again, table, starts, lens, D ** -0.5, accumulate=accumulate)
        assert torch.equal(mp, again)


@pytest.mark.parametrize("new", [1, 5, 70, 300])
def test_nothing_of_masked_keys_gets_through(new):
    page, Hkv, D = 16, 2, 128
    for dtype in (torch.bfloat16, torch.float16):
        for kv in (new, 200, 1000 + new):
            if kv < new:
                continue
            gen = torch.Generator(device=DEV).manual_seed(kv)
            table, starts, lens, total = make_batch(kv, [new], [kv], page)
            kp = make_cache(gen, total, Hkv, page, D, dtype)[0]
            q = torch.randn(new, 8, D, generator=gen, device=DEV).to(dtype)
            own = torch.full((total, page), -1, device=DEV)
            for i, t in enumerate(table[0].tolist()):
                own[t] = i * page + torch.arange(page, device=DEV)
            kp.transpose(1, 2)[(own < 0) | (own >= kv)] = float("nan")
            mp = torch.full((total, Hkv, page), float("nan"), device=DEV)
            paged_key_mass(q, kp, mp, table, starts, lens, D ** -0.5, accumulate=False)
            check_mass(mp.nan_to_num(7.0), torch.full_like(mp, 7.0), q, kp.nan_to_num(0.0), table, [new], [kv], D ** -0.5,
                       False)
            if new == 1:
                continue
            # The last token sees the last key, whose weights are NaN; all rows before it stay as they are.
            kp.transpose(1, 2)[own == kv - 1] = float("nan")
            paged_key_mass(q[:-1], kp, mp, table, starts.clamp(max=new - 1), lens - 1, D ** -0.5, accumulate=False)
            t, slot = int(table[0, (kv - 1) // page]), (kv - 1) % page
            first = mp.clone()
            paged_key_mass(q[:-1], kp.nan_to_num(0.0), mp, table, starts.clamp(max=new - 1), lens - 1, D ** -0.5,
                           accumulate=False)
            first[t, :, slot] = mp[t, :, slot] = 0.0
            assert torch.equal(first.nan_to_num(7.0), mp.nan_to_num(7.0))
            # A NaN key reaches every key that its row sees.
            paged_key_mass(q, kp, mp, table, starts, lens, D ** -0.5, accumulate=False)
            s, p, t, slot = places(table, [kv], page, total)
            assert bool(torch.isnan(mp[t, :, slot]).all())


def test_lengths_that_do_not_fit_and_missing_pages():
    page, Hkv, D, dtype = 16, 2, 64, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(4)
    table, _, _, total = make_batch(9, [1, 1, 1, 1], [96, 96, 96, 96], page)
    kp = make_cache(gen, total, Hkv, page, D, dtype)[0]
    table[1, 2] = -1
    table[1, 5] = total
    table[2] = -5
    # Rows 0-2 and 63.. belong to no sequence; sequence 0 has 20 new tokens and 5 positions, sequence 3 more
    # positions than its table row.
    new, kv, starts = [20, 20, 10, 10], [5, 90, 50, 120], [3, 23, 43, 53]
    q = torch.randn(66, 4, D, generator=gen, device=DEV).to(dtype)
    at = torch.tensor([*starts, 63], dtype=torch.int32, device=DEV)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    before = torch.rand(total, Hkv, page, generator=gen, device=DEV)
    for accumulate in (False, True):
        mp = before.clone()
        paged_key_mass(q, kp, mp, table, at, lens, 0.125, accumulate=accumulate)
        check_mass(mp, before, q, kp, table, new, kv, 0.125, accumulate, starts)
    # No new token, no position, no page and no column at all: nothing is written.
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    two = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
    mp = before.clone()
    for t, length in ((table[:1], none), (table[:1, :0], none + 9), (table[2:3], none + 9)):
        paged_key_mass(q[:2], kp, mp, t, two, length, 0.125)
    paged_key_mass(q[:0], kp, mp, table[:1], none.repeat(2), none + 9, 0.125)
    empty = torch.empty(0, Hkv, page, D, device=DEV, dtype=dtype)
    paged_key_mass(q[:2], empty, torch.empty(0, Hkv, page, device=DEV), table[:1], two, none + 9, 0.125)
    assert torch.equal(mp, before)


def test_single_tokens_of_wide_tables():
    # As many scores as the tables have room for would not fit into a workspace: two passes over the keys.
    new, kv, page, dtype = [1] * 64, [1 + 5 * s for s in range(64)], 64, torch.bfloat16
    table, starts, lens, total = make_batch(1, new, kv, page, width=2500)
    gen = torch.Generator(device=DEV).manual_seed(6)
    kp = make_cache(gen, total, 4, page, 64, dtype)[0]
    q = torch.randn(64, 28, 64, generator=gen, device=DEV).to(dtype)
    before = torch.rand(total, 4, page, generator=gen, device=DEV)
    for accumulate in (False, True):
        mp = before.clone()
        paged_key_mass(q, kp, mp, table, starts, lens, 0.125, accumulate=accumulate)
        check_mass(mp, before, q, kp, table, new, kv, 0.125, accumulate)


def test_hostile_starts_stay_in_bounds():
    page, dtype = 16, torch.bfloat16
    table, _, _, total = make_batch(1, [1] * 4, [80] * 4, page)
    kp = make_cache(torch.Generator(device=DEV).manual_seed(0), total, 2, page, 64, dtype)[0]
    q = torch.randn(40, 4, 64, device=DEV, dtype=dtype)
    lens = torch.tensor([80, 80, -3, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    for starts in ([0, 40, 0, 40, 0], [-7, 100, 3, 2 ** 31 - 1, 5], [40, 30, 20, 10, 0], [-(2 ** 31), 0, 10, 20, 900]):
        mp = torch.full((total + 2, 2, page), 5.0, device=DEV)
        at = torch.tensor(starts, dtype=torch.int32, device=DEV)
        paged_key_mass(q, kp, mp[1:-1], table, at, lens, 0.125)
        assert bool((mp[0] == 5.0).all()) and bool((mp[-1] == 5.0).all())


@pytest.mark.parametrize("new,kv", [([2, 1], [400, 300]), ([150], [400])])
def test_extreme_scores(new, kv):
    page, D, Hq = 32, 64, 4
    table, starts, lens, total = make_batch(3, new, kv, page)
    gen = torch.Generator(device=DEV).manual_seed(8)
    kp = make_cache(gen, total, 1, page, D, torch.bfloat16)[0].abs()
    q = torch.randn(sum(new), Hq, D, generator=gen, device=DEV).to(torch.bfloat16).abs()
    zero = torch.zeros(total, 1, page, device=DEV)
    for f in (0.0, 1.0, -1.0, 20.0, -20.0):
        x = (q * f).to(torch.bfloat16)
        mp = zero.clone()
        paged_key_mass(x, kp, mp, table, starts, lens, 1.0, accumulate=False)
        check_mass(mp, zero, x, kp, table, new, kv, 1.0, False)
    # One key far above all others, by more than 32 bits err: it has each row's weight, whole.
    for at, size in ((0, 1e3), (77, 1e10), (kv[0] - new[0], 1e16)):
        spiked = kp.clone() * 0.01
        spiked[int(table[0, at // page]), 0, at % page] = size
        x = (q + 0.5).to(torch.bfloat16)
        mp = zero.clone()
        paged_key_mass(x, spiked, mp, table, starts, lens, 1.0, accumulate=False)
        rows = new[0] * Hq
        got = mp[int(table[0, at // page]), 0, at % page].double()
        assert abs(float(got) - rows) <= rows * 2.0 ** -20, (at, size, float(got))
        s, p, t, slot = places(table[:1], [kv[0]], page, total)
        assert float(mp[t, 0, slot].sum() - got) <= 2.0 ** -20


def test_mass_of_other_layouts_and_far_pages():
    # Masses in [pages, page, Hkv] storage with a gap; a page 2^31 elements away.
    page, Hkv, D, dtype, new, kv = 64, 2, 64, torch.float16, [3, 70], [130, 200]
    gen = torch.Generator(device=DEV).manual_seed(1)
    table, starts, lens, total = make_batch(2, new, kv, page, spare=0)
    step = (2 ** 31 + 4096) // (total - 1)
    step -= step % 64
    storage = torch.empty(step * (total - 1) + page * Hkv * D + 4096, dtype=dtype, device=DEV)
    kp = storage.as_strided((total, Hkv, page, D), (step, D, Hkv * D, 1))
    kp.copy_(torch.randn(total, Hkv, page, D, generator=gen, device=DEV))
    q = torch.randn(sum(new), 6, D, generator=gen, device=DEV).to(dtype)
    wide = torch.rand(total, page, Hkv + 3, generator=gen, device=DEV)
    mp = wide[:, :, 1:1 + Hkv].transpose(1, 2)
    before = mp.clone()
    kept = wide.clone()
    paged_key_mass(q, kp, mp, table, starts, lens, 0.125)
    check_mass(mp.contiguous(), before.contiguous(), q, kp, table, new, kv, 0.125, True)
    assert torch.equal(wide[:, :, 0], kept[:, :, 0]) and torch.equal(wide[:, :, 1 + Hkv:], kept[:, :, 1 + Hkv:])


# ------------------------------------------------------------------ eviction


def evict_plain(kp, vp, mp, table, kv, out_table, keep, first, recent):
    """The eviction as one reads it, a row at a time."""
    S, Hkv, page = table.shape[0], kp.shape[1], kp.shape[2]
    kept = torch.full((S, Hkv, keep), -1, dtype=torch.int32)
    lens, pages, cap = [], kp.shape[0], table.shape[1] * page
    kq, vq, mq = kp.clone(), vp.clone(), mp.clone()
    tab, out, mass = table.tolist(), out_table.tolist(), mp.cpu()
    for s in range(S):
        m = min(max(kv[s], 0), cap)
        lens.append(min(m, keep))
        for g in range(Hkv):
            def weight(p):
                t = tab[s][p // page]
                x = float(mass[t, g, p % page]) if 0 <= t < pages else float("nan")
                return -math.inf if x != x else x
            if m <= keep:
                chosen = list(range(m))
            else:
                free = list(range(first, m - recent))
                free.sort(key=lambda p: (-weight(p), p))
                chosen = sorted(list(range(first)) + free[:keep - first - recent] + list(range(m - recent, m)))
            kept[s, g, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
            r = [(tab[s][p // page], p % page, out[s][i // page], i % page) for i, p in enumerate(chosen)]
            r = [x for x in r if 0 <= x[0] < pages and 0 <= x[2] < pages]
            if r:
                a, b, c, d = (torch.tensor(x, device=kp.device) for x in zip(*r))
                kq[c, g, d], vq[c, g, d], mq[c, g, d] = kp[a, g, b], vp[a, g, b], mp[a, g, b]
    return kept, lens, kq, vq, mq


def bits(x):
    return x.contiguous().view(torch.int16 if x.element_size() == 2 else torch.int32)


@pytest.mark.parametrize("kv,keep,first,recent,page,Hkv,D,dtype,ties", [
    ([1], 1, 0, 0, 16, 1, 64, torch.bfloat16, False),
    ([2], 1, 0, 0, 1, 2, 128, torch.float16, False),
    ([2], 1, 0, 1, 16, 2, 128, torch.float16, False),
    ([700], 256, 4, 32, 16, 2, 128, torch.bfloat16, False),
    ([700, 3, 0, 256, 257], 256, 4, 32, 16, 3, 64, torch.float32, True),
    ([1000], 36, 4, 32, 48, 2, 128, torch.float32, False),
    ([5000, 900], 777, 0, 0, 7, 2, 64, torch.float16, True),
    ([9001], 9000, 1, 1, 64, 1, 128, torch.bfloat16, False),
    ([9001], 9000, 0, 0, 256, 2, 64, torch.bfloat16, True),
    ([2500] * 3, 100, 0, 99, 16, 2, 64, torch.float16, False),
    ([40011], 2, 0, 0, 64, 2, 64, torch.float16, True),
])
def test_evict(kv, keep, first, recent, page, Hkv, D, dtype, ties):
    gen = torch.Generator(device=DEV).manual_seed(keep)
    spans = kv + [min(m, keep) for m in kv]
    both, _, _, total = make_batch(keep, [1] * len(spans), spans, page)
    S = len(kv)
    table, out = both[:S], both[S:, :max(1, (keep + page - 1) // page)]
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype, keep % 2 == 0)
    mp = torch.randn(total, Hkv, page, generator=gen, device=DEV).exp()
    if ties:
        mp = (mp * 2).round() / 2 - 0.5
        mp[mp == 0.5] = -0.0
        mp[torch.rand(mp.shape, generator=gen, device=DEV) < 0.02] = float("nan")
        mp[torch.rand(mp.shape, generator=gen, device=DEV) < 0.02] = float("-inf")
        mp[torch.rand(mp.shape, generator=gen, device=DEV) < 0.001] = float("inf")
    want = evict_plain(kp, vp, mp, table, kv, out, keep, first, recent)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    kept, new_lens = evict_paged_kv(kp, vp, mp, table, lens, out, keep, first=first, recent=recent)
    assert torch.equal(kept.cpu(), want[0]) and new_lens.tolist() == want[1]
    for got, exact in zip((kp, vp, mp), want[2:]):
        assert torch.equal(bits(got), bits(exact))


def test_evict_without_pages_and_in_place():
    page, Hkv, D = 16, 2, 64
    gen = torch.Generator(device=DEV).manual_seed(0)
    both, _, _, total = make_batch(1, [1] * 6, [200, 200, 90, 64, 64, 90], page)
    kp, vp = make_cache(gen, total, Hkv, page, D, torch.bfloat16)
    mp = torch.rand(total, Hkv, page, generator=gen, device=DEV)
    table, out = both[:3].clone(), both[3:, :6].clone()
    table[0, 3] = -1            # 16 positions without a page, all below the rest
    table[1, 0] = total         # `first` lies in no page: those rows do not move
    out[1, 1] = -7              # nowhere to move to
    out[2] = table[2, :6]       # kept whole: in place
    kv, keep = [200, 900, 60], 64
    want = evict_plain(kp, vp, mp, table, kv, out, keep, 2, 20)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    kept, new_lens = evict_paged_kv(kp, vp, mp, table, lens, out, keep, first=2, recent=20)
    assert torch.equal(kept.cpu(), want[0]) and new_lens.tolist() == want[1] == [64, 64, 60]
    for got, exact in zip((kp, vp, mp), want[2:]):
        assert torch.equal(bits(got), bits(exact))
    # Lengths below zero and tables of no column: nothing is kept.
    kept, new_lens = evict_paged_kv(kp, vp, mp, table, lens * 0 - 5, out, keep)
    assert bool((kept == -1).all()) and new_lens.tolist() == [0, 0, 0]
    kept, new_lens = evict_paged_kv(kp, vp, mp, table[:, :0], lens, out[:, :0], keep)
    assert bool((kept == -1).all()) and new_lens.tolist() == [0, 0, 0]


@pytest.mark.parametrize("cols", [6, 1200, 2100])
def test_evict_where_no_pages_are(cols):
    # A cache of no page, tables on either side of what one workgroup holds: the lowest positions stay.
    page, Hkv, D = 16, 2, 64
    none = torch.empty(0, Hkv, page, D, dtype=torch.bfloat16, device=DEV)
    mass = torch.empty(0, Hkv, page, device=DEV)
    table = torch.zeros(2, cols, dtype=torch.int32, device=DEV)
    lens = torch.tensor([cols * page, 20], dtype=torch.int32, device=DEV)
    kept, new_lens = evict_paged_kv(none, none.clone(), mass, table, lens, table, 40, first=1, recent=9)
    want = list(range(31)) + list(range(cols * page - 9, cols * page))
    assert kept[0].tolist() == [want] * Hkv and new_lens.tolist() == [40, 20]
    assert kept[1].tolist() == [list(range(20)) + [-1] * 20] * Hkv


@pytest.mark.parametrize("kv", [[4096, 4095, 4097], [16384, 9000, 301], [16385, 16384, 8193], [32768, 301],
                                [32769, 32768, 8192, 300], [40960, 40961, 24577]])
def test_evict_at_the_borders_of_its_parts(kv):
    # Positions that one workgroup holds, and that a part of a longer table has.
    page, Hkv, D, keep = 1, 2, 64, 300
    gen = torch.Generator(device=DEV).manual_seed(kv[0])
    both, _, _, total = make_batch(4, [1] * (2 * len(kv)), kv + [keep] * len(kv), page)
    table, out = both[:len(kv)], both[len(kv):, :keep]
    kp, vp = make_cache(gen, total, Hkv, page, D, torch.bfloat16)
    mp = (torch.rand(total, Hkv, page, generator=gen, device=DEV) * 100).round()
    want = evict_plain(kp, vp, mp, table, kv, out, keep, 3, 5)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    kept, new_lens = evict_paged_kv(kp, vp, mp, table, lens, out, keep, first=3, recent=5)
    assert torch.equal(kept.cpu(), want[0]) and new_lens.tolist() == want[1]
    for got, exact in zip((kp, vp, mp), want[2:]):
        assert torch.equal(bits(got), bits(exact))


def test_evict_long_and_far():
    # A long sequence against the sort of torch, and pages past 2^31 elements.
    page, Hkv, D, kv, keep, dtype = 64, 2, 64, 131072 + 77, 30001, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(5)
    both, _, _, total = make_batch(2, [1, 1], [kv, keep], page, spare=0)
    wide = page * Hkv * D + 2 ** 31 // total
    wide -= wide % 64
    storage = torch.empty(wide * total, dtype=dtype, device=DEV)
    kp = storage.as_strided((total, Hkv, page, D), (wide, page * D, D, 1))
    kp.copy_(torch.randn(total, Hkv, page, D, generator=gen, device=DEV))
    vp = torch.randn(total, Hkv, page, D, generator=gen, device=DEV).to(dtype)
    mp = torch.rand(total, Hkv, page, generator=gen, device=DEV).mul_(5000).round_()
    table, out = both[:1], both[1:, :(keep + page - 1) // page]
    p = torch.arange(kv, device=DEV)
    at, slot = table[0].long()[p // page], p % page
    weight = mp[at, :, slot].T.clone()
    weight[:, :10] = weight[:, kv - 333:] = float("inf")
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices[:, :keep].sort(dim=-1).values
    want = [[x[at[o], g, slot[o]].clone() for g, o in enumerate(order)] for x in (kp, vp, mp)]
    lens = torch.tensor([kv], dtype=torch.int32, device=DEV)
    kept, new_lens = evict_paged_kv(kp, vp, mp, table, lens, out, keep, first=10, recent=333)
    assert torch.equal(kept[0].long(), order) and new_lens.tolist() == [keep]
    r = torch.arange(keep, device=DEV)
    to, slot = out[0].long()[r // page], r % page
    for x, rows in zip((kp, vp, mp), want):
        for g in range(Hkv):
            assert torch.equal(x[to, g, slot], rows[g])


# ------------------------------------------------------------------ together


def test_streams_graphs_and_two_calls_at_once():
    page, Hkv, D, dtype, keep = 16, 4, 128, torch.bfloat16, 300
    gen = torch.Generator(device=DEV).manual_seed(2)
    new, kv = [1] * 6, [33, 1200, 77, 5000, 16, 2048]
    both, _, _, total = make_batch(6, [1] * 12, [5000] * 6 + [keep] * 6, page)
    table, out = both[:6], both[6:, :(keep + page - 1) // page]
    starts = torch.arange(7, dtype=torch.int32, device=DEV)
    lens = torch.tensor(kv, dtype=torch.int32, device=DEV)
    kp, vp = make_cache(gen, total, Hkv, page, D, dtype)
    q = [torch.randn(6, 28, D, generator=gen, device=DEV).to(dtype) for _ in range(2)]
    x = torch.randn(6, 5003, generator=gen, device=DEV)
    u = torch.rand(6, generator=gen, device=DEV)

    def step(i, mp):
        paged_key_mass(q[i], kp, mp, table, starts, lens, 0.08)
        token = sample_tokens(x, u, temperature=0.9, top_p=0.9, return_logprobs=True)
        return (*evict_paged_kv(kp, vp, mp, table, lens, out, keep, first=3, recent=9), *token)
    zero = [torch.rand(total, Hkv, page, generator=gen, device=DEV) for _ in q]
    mps = [z.clone() for z in zero]
    want = []
    for i in (0, 1):
        want.append([*(t.clone() for t in step(i, mps[i])), mps[i].clone()])
    streams, got = [torch.cuda.Stream() for _ in q], []
    for i, stream in enumerate(streams):
        mps[i].copy_(zero[i])
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            paged_key_mass(q[i], kp, mps[i], table, starts, lens, 0.08)
            got.append(sample_tokens(x, u, temperature=0.9, top_p=0.9))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert torch.equal(got[i], want[i][2])
    # Two graphs over the same tensors; replays follow what the tensors then hold.
    graphs, outs = [], []
    for i in (0, 1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(i, mps[i]))
        graphs.append(graph)
    for turn in range(3):
        lens.copy_(torch.tensor([m + 400 * turn if m < 4000 else 5000 - turn for m in kv], dtype=torch.int32))
        u.add_(0.31).frac_()
        for i in (0, 1):
            mps[i].copy_(zero[i])
            graphs[i].replay()
            torch.cuda.synchronize()
            mine = zero[i].clone()
            eager = step(i, mine)
            assert torch.equal(mine, mps[i])
            for a, b in zip(outs[i], eager):
                assert torch.equal(a, b), (turn, i)


def test_one_row_of_tables_for_all_and_empty_batches():
    # A table's row expanded over sequences of different lengths (a shared prompt), whose masses are set by one
    # of them at a time; sequences of which none has a token.
    page, Hq, Hkv, D, dtype = 16, 8, 2, 64, torch.float16
    gen = torch.Generator(device=DEV).manual_seed(7)
    table, _, _, total = make_batch(9, [1], [600], page)
    kp = make_cache(gen, total, Hkv, page, D, dtype)[0]
    q = torch.randn(7, Hq, D, generator=gen, device=DEV).to(dtype)
    before = torch.rand(total, Hkv, page, generator=gen, device=DEV)
    lens = torch.tensor([600, 433, 20], dtype=torch.int32, device=DEV)
    for who in range(3):
        new = [7 if s == who else 0 for s in range(3)]
        starts = torch.tensor([0, *new]).cumsum(0).to(torch.int32).to(DEV)
        mp = before.clone()
        paged_key_mass(q, kp, mp, table.expand(3, -1), starts, lens, 0.125)
        check_mass(mp, before, q, kp, table.expand(3, -1), new, [600, 433, 20], 0.125, True)
    mp = before.clone()
    paged_key_mass(q, kp, mp, table.expand(3, -1), starts * 0, lens, 0.125)
    paged_key_mass(q[:0], kp, mp, table.expand(3, -1), starts * 0, lens, 0.125)
    assert torch.equal(mp, before)


def test_a_cut_cache_serves_on():
    # A prompt's masses, its cache cut down, then tokens decoded over what is left: against attention over the kept
    # keys alone.  What is asked for is the run; its parts' values are tested above.
    Hq, Hkv, D, page, T, keep, dtype = 8, 2, 128, 16, 500, 120, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(3)
    both, _, _, total = make_batch(1, [1, 1], [T, keep + 16], page)
    table, out = both[:1], both[1:, :(keep + 16 + page - 1) // page]
    kp, vp = (torch.zeros(total, page, Hkv, D, device=DEV, dtype=dtype).transpose(1, 2) for _ in range(2))
    mp = torch.zeros(total, Hkv, page, device=DEV)
    inv_freq = rotary_frequencies(D, device=DEV)[0]
    qkv = torch.randn(T + 4, Hq + 2 * Hkv, D, generator=gen, device=DEV).to(dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    at = 0
    for n in (300, 199, 1):
        starts = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        lens = torch.tensor([at + n], dtype=torch.int32, device=DEV)
        turned = append_paged_kv(k[at:at + n], v[at:at + n], kp, vp, table, starts, lens, query=q[at:at + n],
                                 inv_freq=inv_freq)
        paged_chunk_attention(turned, kp, vp, table, starts, lens, D ** -0.5)
        paged_key_mass(turned, kp, mp, table, starts, lens, D ** -0.5)
        at += n
    s, p, t, slot = places(table, [T], page, total)
    gathered = mp[t, :, slot].sum(dtype=torch.float64)
    assert abs(float(gathered) - T * Hq) <= T * Hq * 2.0 ** -12        # every row gave a weight of one
    kept, lens = evict_paged_kv(kp, vp, mp, table, lens, out, keep, first=4, recent=16)
    assert lens.tolist() == [keep]
    full_k, full_v = (torch.stack([x[table[0].long()[kept[0, g].long() // page], g, kept[0, g].long() % page]
                                   for g in range(Hkv)]) for x in (kp, vp))
    starts = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    W = torch.randn(Hq * D, 999, generator=gen, device=DEV) * 0.02
    for i in range(T, T + 4):
        lens = lens + 1
        position = torch.tensor([i], device=DEV)
        turned = append_paged_kv(k[i:i + 1], v[i:i + 1], kp, vp, out, starts, lens, query=q[i:i + 1], inv_freq=inv_freq,
                                 positions=position)
        r = int(lens) - 1
        page_at = int(out[0, r // page])
        full_k = torch.cat((full_k, kp[page_at, :, r % page][:, None]), dim=1)
        full_v = torch.cat((full_v, vp[page_at, :, r % page][:, None]), dim=1)
        o = paged_chunk_attention(turned, kp, vp, out, starts, lens, D ** -0.5)
        a = torch.softmax((turned.view(Hkv, Hq // Hkv, D).double() @ full_k.double().transpose(1, 2)) * D ** -0.5, dim=-1)
        want = (a @ full_v.double()).view(1, Hq, D)
        assert float((o.double() - want).abs().max()) <= 2.0 ** -7 * float(full_v.abs().max())
        mp_before = mp.clone()
        paged_key_mass(turned, kp, mp, out, starts, lens, D ** -0.5)
        s, p, t, slot = places(out, [int(lens)], page, total)
        added = mp[t, :, slot].double() - torch.where((p < r)[:, None], mp_before[t, :, slot], 0.0).double()
        want = a.sum(1)[:, p].T
        assert float((added - want).abs().max()) <= 2.0 ** -14 * Hq * 4 + 2.0 ** -23 * float(mp[t, :, slot].max())
        token = sample_tokens(o.view(1, -1).float() @ W, torch.rand(1, generator=gen, device=DEV), top_k=50, top_p=0.9)
        assert 0 <= int(token) < 999


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,new,kv,at", [(8, 2, 3, 40, 1), (8, 2, 5, 700, 0), (28, 4, 4, 1500, 2), (8, 2, 70, 300, 30),
                                              (16, 8, 300, 1000, 100), (4, 4, 600, 600, 599), (8, 2, 64, 64, 0)])
def test_a_token_of_nan_reaches_only_keys_it_sees(Hq, Hkv, new, kv, at, dtype):
    # Its weights are NaN: those of the keys up to its position, and of no later token's.
    page, D = 16, 64
    gen = torch.Generator(device=DEV).manual_seed(new)
    table, starts, lens, total = make_batch(kv, [new], [kv], page)
    kp = make_cache(gen, total, Hkv, page, D, dtype)[0]
    q = (2 * torch.randn(new, Hq, D, generator=gen, device=DEV)).to(dtype)
    G = Hq // Hkv
    for bad in (float("nan"), float("inf")):
        q[at, G - 1] = bad          # (an infinite query's products are of both signs, their sum NaN)
        mp = torch.zeros(total, Hkv, page, device=DEV)
        paged_key_mass(q, kp, mp, table, starts, lens, D ** -0.5)
        plain = q.clone()
        plain[at, G - 1] = 0.0
        want, bar = mass64(plain, kp, table, [new], [kv], D ** -0.5)
        _, p, t, slot = places(table, [kv], page, total)
        later, got = p > kv - new + at, mp[t, :, slot].double()
        assert bool(torch.isnan(got[~later, 0]).all())
        off = (got - want[0, :, p].T).abs() <= bar[0, :, p].T
        assert bool(off[later].all()) and bool(off[:, 1:].all())


def test_masses_of_many_equal_weights():
    # 57344 rows that attend the same 1999 keys alike, at weights of 1 / 1999: summed up in one line they are off by
    # up to half a step each, all the same way (3e-4 of the mass here).  Counted in 2^-24 of a mass: the
    # logarithm of the row's sum, 11 bits, times ln 2 at four roundings (31), the two exponentials (4), sums of 32
    # at a time (32), these added up with what is rounded off carried on, and the halves (4).
    page, Hq, Hkv, D, new, dtype = 1999, 56, 8, 64, 8192, torch.bfloat16
    gen = torch.Generator(device=DEV).manual_seed(0)
    table = torch.full((1, 66), -1, dtype=torch.int32, device=DEV)     # one page, room for many
    table[0, 0] = 0
    kp = torch.randn(1, Hkv, page, D, generator=gen, device=DEV).to(dtype)
    q = torch.zeros(new, Hq, D, device=DEV, dtype=dtype)
    starts = torch.tensor([0, new], dtype=torch.int32, device=DEV)
    lens = torch.tensor([2000 + new], dtype=torch.int32, device=DEV)
    mp = torch.zeros(1, Hkv, page, device=DEV)
    paged_key_mass(q, kp, mp, table, starts, lens, 0.125)
    want = new * (Hq // Hkv) / page
    assert float((mp.double() / want - 1).abs().max()) <= 71 * 2.0 ** -24


def test_the_masses_of_a_chunk_come_to_its_rows():
    # Every row gives a weight of one.  What its roundings make of that goes either way and averages out over the rows:
    # six of scores and references of up to 128, half a step each, at scale 0.0884, come to a deviation of under 2^-19
    # a row, six of which are allowed.  What all rows have alike, the exponential's and the logarithm's own errors,
    # is in their sums as in their weights: 2^-23 is left for it.
    new, kv, page, Hq, Hkv, D = 512, 4000, 64, 32, 4, 128
    for dtype in (torch.bfloat16, torch.float16):
        gen = torch.Generator(device=DEV).manual_seed(1)
        table, starts, lens, total = make_batch(8, [new], [kv], page)
        kp = make_cache(gen, total, Hkv, page, D, dtype)[0]
        q = (0.5 * torch.randn(new, Hq, D, generator=gen, device=DEV)).to(dtype)
        mp = torch.zeros(total, Hkv, page, device=DEV)
        paged_key_mass(q, kp, mp, table, starts, lens, D ** -0.5)
        rows = new * Hq
        assert abs(float(mp.double().sum()) / rows - 1) <= 2.0 ** -23 + 6 * 2.0 ** -19 / math.sqrt(rows)


@pytest.mark.parametrize("new,kv,page,Hq,Hkv,D", [
    ([1, 60, 3, 0, 200, 4, 2, 5, 1, 1], [900, 60, 3, 50, 1000, 700, 333, 90, 1, 2000], 32, 16, 2, 64),
    ([0] * 9 + [500] + [2] * 3, [40] * 9 + [500] + [77, 2, 1500], 16, 28, 4, 128),
    ([(7 * s) % 4 for s in range(66)] + [300, 0, 1, 3, 130, 2], [200 + 5 * s for s in range(72)], 16, 32, 4, 64),
    ([300] + [1] * 130, [777] + [90 + s for s in range(130)], 48, 32, 1, 64),
])
def test_few_rows_beside_more_tokens_than_they_have_room_for(new, kv, page, Hq, Hkv, D):
    assert sum(new) > len(new) * (32 // (Hq // Hkv)) and len(new) > 8
    gen = torch.Generator(device=DEV).manual_seed(sum(new))
    for dtype in (torch.bfloat16, torch.float16):
        table, starts, lens, total = make_batch(page, new, kv, page)
        kp = make_cache(gen, total, Hkv, page, D, dtype)[0]
        q = (2 * torch.randn(sum(new), Hq, D, generator=gen, device=DEV)).to(dtype)
        before = torch.rand(total, Hkv, page, generator=gen, device=DEV)
        for accumulate in (False, True):
            mp = before.clone()
            paged_key_mass(q, kp, mp, table, starts, lens, D ** -0.5, accumulate=accumulate)
            check_mass(mp, before, q, kp, table, new, kv, D ** -0.5, accumulate)


def test_hostile_starts_of_many_sequences_stay_in_bounds():
    # As above, with places of their own for the few rows: sequences that overlap, go back and leave the batch.
    page, dtype, S = 16, torch.bfloat16, 12
    table, _, _, total = make_batch(1, [1] * S, [80] * S, page)
    kp = make_cache(torch.Generator(device=DEV).manual_seed(0), total, 2, page, 64, dtype)[0]
    q = torch.randn(400, 4, 64, device=DEV, dtype=dtype)
    lens = torch.tensor([80, 80, -3, 2 ** 31 - 1] * 3, dtype=torch.int32, device=DEV)
    for starts in ([0, 16, 0, 16] * 3 + [0], [0, 1, 17, 33] * 3 + [400], [396, 400, 2 ** 31 - 1, -7] * 3 + [16],
                   [400 - 33 * s for s in range(13)]):
        mp = torch.full((total + 2, 2, page), 5.0, device=DEV)
        at = torch.tensor(starts, dtype=torch.int32, device=DEV)
        paged_key_mass(q, kp, mp[1:-1], table, at, lens, 0.125)
        assert bool((mp[0] == 5.0).all()) and bool((mp[-1] == 5.0).all())

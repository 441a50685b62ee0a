"""Head norms with rotary positions, and the append to a paged cache, on the
GPU against a plain form in 64 bits.

The bar, per value: half a step of the output type, eps(type) / 2 of the value
(for float16 at least half of its smallest step, 2^-25), and the 32-bit
arithmetic before it.  That is bounded by 28 units of 2^-24 of
factor * (|a| + |b|), a and b the normed pair: 10 for the mean of squares
(16 sequential and up to 3 pairwise additions, halved by the square root), 5 for
root, reciprocal and the two products with it and the weight (an input's widening
is exact), 4 for the sine or cosine (the angle's fraction of a turn rounded to 32
bits is off by up to 2^-26 turns = 1.6 units, the function by up to 2), 1 for the factor, 3 for two products
and a sum; 5 in reserve for the functions' last bits.  Values that are not rotated stand
for a = x, b = 0; without a norm and a rotation they are the input's bits.
"""
import pytest
import torch

from kernels.paged import append_paged_kv
from kernels.rotary import rotary_frequencies, rotate_heads

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6


def turn64(x, weight, positions, inv_freq, layout, factor=1.0, eps=EPS):
    """(values, |a| + |b|) of [..., H, D] rows at positions [...], in 64 bits."""
    y = x.double()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    size = y.abs()
    if inv_freq is None:
        return y, size
    R = 2 * inv_freq.numel()
    angle = (positions.double()[..., None] * inv_freq)[..., None, :]
    c, s = angle.cos() * factor, angle.sin() * factor
    out, size = y.clone(), size.clone()
    one, two = (slice(0, R // 2), slice(R // 2, R)) if layout == "half" else (slice(0, R, 2), slice(1, R, 2))
    a, b = y[..., one], y[..., two]
    out[..., one], out[..., two] = a * c - b * s, b * c + a * s
    size[..., one] = size[..., two] = (a.abs() + b.abs()) * max(factor, 1.0)
    return out, size


def check(got, want, size, what=""):
    half = torch.finfo(got.dtype).eps / 2
    bar = want.abs() * half * (1 + half) + size * 28 * 2.0 ** -24 + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((off <= bar).all()), (what, float((off / bar.clamp(min=1e-300)).max()))


def _heads(gen, B, T, H, D, dtype, form):
    """[B, H, T, D] in one of the storages that callers have."""
    if form == "bthd":
        return torch.randn(B, T, H, D, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    if form == "bhtd":
        return torch.randn(B, H, T, D, generator=gen, device=DEV).to(dtype)
    return torch.randn(B, T, H + 3, D + 16, generator=gen, device=DEV).to(dtype)[:, :, 1:H + 1, 16:].transpose(1, 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,Hq,Hkv,D,R,layout,norm,form,first", [
    (1, 1, 28, 4, 128, 128, "half", "both", "bthd", 100003),
    (1, 1, 1, 1, 64, 16, "interleaved", "none", "bhtd", 0),
    (2, 77, 12, 2, 128, 128, "interleaved", "both", "bthd", 5),
    (3, 65, 5, 5, 64, 32, "half", "q", "slice", 1000003),
    (1, 333, 9, 3, 128, 48, "half", "k", "slice", 0),
    (2, 130, 16, 8, 64, 64, "half", "none", "bhtd", 77),
    (1, 1029, 28, 4, 128, 64, "interleaved", "f32", "bthd", 4000000),
    (1, 50, 17, 1, 64, 64, "interleaved", "both", "slice", 0),
    (2, 9, 8, 2, 128, 0, "half", "both", "bthd", 0),
])
def test_rotate_heads(B, T, Hq, Hkv, D, R, layout, norm, form, first, dtype):
    print(f"case {B} {T} {Hq}/{Hkv} D={D} R={R} {layout} {norm} {form} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(B * 1000 + T)
    q, k = (_heads(gen, B, T, H, D, dtype, form) for H in (Hq, Hkv))
    weight = (1 + 0.2 * torch.randn(2, D, generator=gen, device=DEV)).to(torch.float32 if norm == "f32" else dtype)
    qw = weight[0].contiguous() if norm in ("both", "q", "f32") else None
    kw = weight[1].contiguous() if norm in ("both", "k", "f32") else None
    pos = first + torch.arange(T, device=DEV)
    if B > 1:
        pos = pos + 31 * torch.arange(B, device=DEV)[:, None]
    if layout == "half":
        pos = pos.to(torch.int32)
    inv_freq = rotary_frequencies(R, 1e6, device=DEV)[0] if R else None
    qo, ko = rotate_heads(q, k, pos, inv_freq, layout=layout, factor=1.25, q_weight=qw, k_weight=kw, eps=EPS)
    assert qo.transpose(1, 2).is_contiguous() and ko.transpose(1, 2).is_contiguous()
    rows = pos.expand(B, T)
    for got, x, w in ((qo, q, qw), (ko, k, kw)):
        want, size = turn64(x.transpose(1, 2), w, rows, inv_freq, layout, 1.25)
        check(got.transpose(1, 2), want, size)
        if w is None:     # what is neither normed nor turned keeps its bits
            assert torch.equal(got[..., R:], x[..., R:])


def test_rotate_far_and_negative_positions():
    # int64 positions past 2^31 and below zero: the angle keeps its place on the circle.
    pos = torch.tensor([0, -1, -100000, (1 << 31) + 7, (1 << 33) + 12345], device=DEV)
    gen = torch.Generator(device=DEV).manual_seed(3)
    q, k = (torch.randn(1, H, 5, 64, generator=gen, device=DEV) for H in (2, 1))
    inv_freq = rotary_frequencies(64, 1e4, device=DEV)[0]
    qo, _ = rotate_heads(q, k, pos, inv_freq)
    # In turns the product p * inv_freq / (2 pi) has up to 31 bits before the point and 2^-22 after it here:
    # 2^33 * 2^-53 * 2 * 2 pi = 1.2e-5 radians at the farthest position, on both sides.
    want, size = turn64(q.transpose(1, 2), None, pos[None], inv_freq, "half")
    off = (qo.transpose(1, 2).double() - want).abs()
    assert bool((off <= size * (3e-5 + 28 * 2.0 ** -24)).all())
    near = off[:, :3] <= size[:, :3] * 28 * 2.0 ** -24 + want[:, :3].abs() * 2.0 ** -24
    assert bool(near.all())


def test_rotate_special_values():
    # A NaN or infinity stays in its own head row; a zero row normed is zero.
    q = torch.ones(1, 4, 3, 64, device=DEV, dtype=torch.bfloat16)
    q[0, 1, 1, 5] = float("nan")
    q[0, 2, 0, 7] = float("inf")
    q[0, 3] = 0
    inv_freq = rotary_frequencies(64, 1e4, device=DEV)[0]
    qo, ko = rotate_heads(q, q, torch.arange(3, device=DEV), inv_freq, q_weight=torch.ones(64, device=DEV))
    bad = ~torch.isfinite(qo).all(-1)[0]
    assert bad.nonzero().tolist() == [[1, 1], [2, 0]]
    assert bool((qo[0, 3] == 0).all())
    hurt = ~torch.isfinite(ko)[0]
    assert sorted(set(map(tuple, hurt.nonzero()[:, :2].tolist()))) == [(1, 1), (2, 0)]


def test_rotate_empty_and_on_another_stream():
    inv_freq = rotary_frequencies(64, 1e4, device=DEV)[0]
    qo, ko = rotate_heads(torch.empty(2, 4, 0, 64, device=DEV), torch.empty(2, 2, 0, 64, device=DEV),
                          torch.empty(2, 0, device=DEV, dtype=torch.int32), inv_freq)
    assert qo.shape == (2, 4, 0, 64) and ko.shape == (2, 2, 0, 64)
    q = torch.randn(1, 4, 500, 64, device=DEV)
    pos = torch.arange(500, device=DEV)
    want = rotate_heads(q, q, pos, inv_freq)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = rotate_heads(q, q, pos, inv_freq)[0]
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


# ------------------------------------------------------------------ append


def make_batch(seed, new, kv, page, spare=3, width=None):
    """(page_table, q_starts, kv_lens, pages): random page ids, -1 behind a sequence's own."""
    counts = [(n + page - 1) // page for n in kv]
    total = sum(counts) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    W = max([1, *counts]) if width is None else width
    table = torch.full((len(new), W), -1, dtype=torch.int32)
    for s, c in enumerate(counts):
        for i in range(c):
            table[s, i] = order.pop()
    starts = torch.tensor([0, *new]).cumsum(0).to(torch.int32)
    return table.to(DEV), starts.to(DEV), torch.tensor(kv, dtype=torch.int32, device=DEV), total


def _pages(total, Hkv, page, D, dtype, slot_major, fill=7.0):
    if slot_major:
        return torch.full((total, page, Hkv, D), fill, device=DEV, dtype=dtype).transpose(1, 2)
    return torch.full((total, Hkv, page, D), fill, device=DEV, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("new,kv,page,Hq,Hkv,D,R,layout,norm,slot_major", [
    ([1], [1], 16, 28, 4, 128, 128, "half", True, True),
    ([1, 1, 1, 1, 1], [1, 17, 16, 300, 15], 16, 12, 2, 128, 128, "interleaved", False, False),
    ([5, 0, 64, 1, 77], [5, 9, 64, 33, 200], 32, 16, 8, 64, 32, "half", True, True),
    ([130, 3], [130, 2000], 48, 6, 3, 128, 64, "half", True, False),
    ([333], [1000], 1, 4, 4, 64, 64, "interleaved", True, True),
    ([40, 50], [40, 50], 64, 0, 2, 128, 0, "half", False, True),
    ([2] * 150, list(range(2, 152)), 8, 8, 1, 64, 16, "half", False, True),
])
def test_append(new, kv, page, Hq, Hkv, D, R, layout, norm, slot_major, dtype):
    print(f"case new={new[:6]} kv={kv[:6]} page={page} {Hq}/{Hkv} D={D} R={R} {layout} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(len(new) + page)
    table, starts, lens, total = make_batch(page, new, kv, page)
    tail = 3     # rows behind the last sequence
    N = sum(new) + tail
    qkv = torch.randn(N, Hq + 2 * Hkv, D, generator=gen, device=DEV).to(dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    weight = (1 + 0.2 * torch.randn(2, D, generator=gen, device=DEV)).to(dtype)
    qw, kw = (weight[0].contiguous(), weight[1].contiguous()) if norm else (None, None)
    inv_freq = rotary_frequencies(R, 1e6, device=DEV)[0] if R else None
    kp, vp = (_pages(total, Hkv, page, D, dtype, slot_major) for _ in range(2))
    out = append_paged_kv(k, v, kp, vp, table, starts, lens, query=q if Hq else None, inv_freq=inv_freq,
                          layout=layout, q_weight=qw, k_weight=kw, eps=EPS)
    pos = torch.cat([torch.arange(m - n, m) for n, m in zip(new, kv)]).to(DEV)
    seq = torch.cat([torch.full((n,), s) for s, n in enumerate(new)]).to(DEV)
    at, slot = table.long()[seq, pos // page], pos % page
    want, size = turn64(k[:-tail], kw, pos, inv_freq, layout)
    check(kp[at, :, slot], want, size, "keys")
    assert torch.equal(vp[at, :, slot], v[:-tail])
    if Hq:
        check(out[:-tail], *turn64(q[:-tail], qw, pos, inv_freq, layout), "queries")
    else:
        assert out is None
    # Every other slot is as it was.
    for pages in (kp, vp):
        rest = torch.ones(total, page, dtype=torch.bool, device=DEV)
        rest[at, slot] = False
        assert bool((pages.transpose(1, 2)[rest] == 7.0).all())


def test_append_own_positions_and_missing_pages():
    gen = torch.Generator(device=DEV).manual_seed(1)
    table, starts, lens, total = make_batch(2, [40, 30], [40, 100], 16)
    table[0, 1] = -1               # no page for positions 16..31 of sequence 0
    table[1, 5] = total            # nor for 80..95 of sequence 1
    k, v = (torch.randn(70, 2, 64, generator=gen, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    q = torch.randn(70, 4, 64, generator=gen, device=DEV, dtype=torch.bfloat16)
    kp, vp = (_pages(total, 2, 16, 64, torch.bfloat16, True) for _ in range(2))
    inv_freq = rotary_frequencies(64, 1e4, device=DEV)[0]
    own = torch.randint(0, 1 << 20, (70,), generator=gen, device=DEV)
    out = append_paged_kv(k, v, kp, vp, table, starts, lens, query=q, inv_freq=inv_freq, positions=own)
    check(out, *turn64(q, None, own, inv_freq, "half"))
    pos = torch.cat([torch.arange(40), torch.arange(70, 100)]).to(DEV)
    seq = torch.tensor([0] * 40 + [1] * 30, device=DEV)
    have = ~(((seq == 0) & (pos // 16 == 1)) | ((seq == 1) & (pos // 16 == 5)))
    at, slot = table.long()[seq, pos // 16][have], pos[have] % 16
    check(kp[at, :, slot], *turn64(k[have], None, own[have], inv_freq, "half"))
    written = torch.zeros(total, 16, dtype=torch.bool, device=DEV)
    written[at, slot] = True
    for pages in (kp, vp):
        assert bool((pages.transpose(1, 2)[~written] == 7.0).all())


def test_append_lengths_that_do_not_fit():
    # More new tokens than the cache has, a cache longer than the table, starts that leave rows in front:
    # only the tokens with a slot are written, and rows of no sequence are left alone.
    table, _, _, total = make_batch(5, [1, 1, 1], [32, 32, 32], 16)
    starts = torch.tensor([2, 10, 20, 30], dtype=torch.int32, device=DEV)
    lens = torch.tensor([5, 35, 8], dtype=torch.int32, device=DEV)     # 8, 10 and 10 new tokens
    k = torch.randn(33, 1, 64, device=DEV, dtype=torch.float16)
    v = torch.randn(33, 1, 64, device=DEV, dtype=torch.float16)
    kp, vp = (_pages(total, 1, 16, 64, torch.float16, False) for _ in range(2))
    append_paged_kv(k, v, kp, vp, table, starts, lens)
    want_k, want_v = (_pages(total, 1, 16, 64, torch.float16, False) for _ in range(2))
    for s, (a, b, n) in enumerate(((2, 10, 5), (10, 20, 35), (20, 30, 8))):
        for t in range(a, b):
            p = n - b + t
            if 0 <= p < 32:
                want_k[table[s, p // 16], :, p % 16] = k[t]
                want_v[table[s, p // 16], :, p % 16] = v[t]
    assert torch.equal(kp, want_k) and torch.equal(vp, want_v)


def test_rotate_offsets_past_32_bits():
    # The last tokens of more than 2^31 elements, as those tokens alone.
    T, H, D, last = (1 << 31) // (28 * 128) + 33, 28, 128, 40
    q = torch.empty(1, T, H, D, device=DEV, dtype=torch.bfloat16).transpose(1, 2)
    q[:, :, -last:] = torch.randn(1, H, last, D, device=DEV).to(torch.bfloat16)
    k = torch.randn(1, 2, T, D, device=DEV).to(torch.bfloat16)
    pos = torch.arange(T, device=DEV)
    inv_freq = rotary_frequencies(D, device=DEV)[0]
    qo, ko = rotate_heads(q, k, pos, inv_freq)
    qs, ks = rotate_heads(q[:, :, -last:], k[:, :, -last:], pos[-last:], inv_freq)
    assert torch.equal(qo[:, :, -last:], qs) and torch.equal(ko[:, :, -last:], ks)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_calls_equal_their_parts(dtype):
    # Rows that go past the caches hold the bits of those that do not.
    T, Hq, Hkv, D, page = 20011, 28, 4, 128, 64
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = (torch.randn(1, T, H, D, generator=gen, device=DEV).to(dtype).transpose(1, 2) for H in (Hq, Hkv, Hkv))
    w = (1 + 0.1 * torch.randn(D, generator=gen, device=DEV)).to(dtype)
    inv_freq = rotary_frequencies(D, device=DEV)[0]
    pos = torch.arange(T, device=DEV)
    qo, ko = rotate_heads(q, k, pos, inv_freq, q_weight=w, k_weight=w)
    parts = [rotate_heads(q[:, :, a:a + 5000], k[:, :, a:a + 5000], pos[a:a + 5000], inv_freq, q_weight=w, k_weight=w)
             for a in range(0, T, 5000)]
    assert torch.equal(qo, torch.cat([x for x, _ in parts], 2)) and torch.equal(ko, torch.cat([x for _, x in parts], 2))
    pages = -(-T // page)
    table = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)[None]
    kp, vp = (torch.zeros(pages, Hkv, page, D, device=DEV, dtype=dtype) for _ in range(2))
    turned = append_paged_kv(k[0].transpose(0, 1), v[0].transpose(0, 1), kp, vp, table,
                             torch.tensor([0, T], dtype=torch.int32, device=DEV),
                             torch.tensor([T], dtype=torch.int32, device=DEV), query=q[0].transpose(0, 1),
                             inv_freq=inv_freq, q_weight=w, k_weight=w)
    assert torch.equal(turned, qo[0].transpose(0, 1))
    back = [x[table[0].long()].transpose(1, 2).reshape(-1, Hkv, D)[:T] for x in (kp, vp)]
    assert torch.equal(back[0], ko[0].transpose(0, 1)) and torch.equal(back[1], v[0].transpose(0, 1))

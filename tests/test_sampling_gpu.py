"""The draw of tokens on the GPU against the definition in 64 bits.

A token is right if its interval of the running sums of kept weights, in the oracle's 64 bits, holds u times their
total to within off(V) of that total, and the same for the ends of the prefixes: a row in which an end lies within that
is not judged.  Weights are rounded to units of 2^-(63 - ceil(log2 V)) of the largest, which is one: V of them are off by
V / 2 units where they all round one way, as equal ones do (70000 weights of e^-29 beside one: 1.9e-9 at units of
2^-42), and 2^-30 covers the exponentials, whose polynomial is off by 2^-44, and the oracle's own sums.  Log-
probabilities are off by a rounding of float32 and the same.
"""
import math

import pytest
import torch

from kernels.sampling import sample_tokens

pytestmark = pytest.mark.gpu
DEV = "cuda"


def off(V):
    return 2.0 ** -30 + V / 2 * 2.0 ** -min(52, 63 - (V - 1).bit_length())


def kept64(x, T, k, p, floor):
    """(weights of the kept, zeros elsewhere, whether a border is too near) of one row, in 64 bits on the CPU."""
    x = torch.where(torch.isnan(x), -torch.inf, x.double())
    V, top = x.numel(), x.max()
    EPS = off(V)
    if top == -torch.inf:
        return torch.zeros_like(x), False
    order = torch.sort(x, descending=True, stable=True).indices
    w = torch.zeros_like(x)
    if not T > 0:
        w[order[0]] = 1.0
        return w, False
    xs = x[order]
    ws = (xs == top).double() if top == torch.inf else torch.exp((xs - top) / T if math.isfinite(T) else (xs - top) * 0.0)
    ws = torch.where(xs == -torch.inf, 0.0, ws)
    keep = torch.ones(V, dtype=torch.bool)
    close = False
    if 0 < k < V:
        keep[k:] = False
    if p < 1:
        ws = ws * keep
        before, mass = ws.cumsum(0) - ws, p * ws.sum()
        # (Weights of one each, as at an infinite temperature: their sums are whole numbers on either side, and
        # half of an even number of them is met exactly, which leaves no doubt.)
        whole = bool(((ws == 0) | (ws == 1)).all()) and p == 0.5
        close |= not whole and bool((((before - mass).abs() < EPS * ws.sum()) & (ws > 0))[1:].any()) and p > 0
        out = before >= mass
        out[0] = False
        keep &= ~out
    close |= bool(((ws - floor).abs() < 1e-12)[1:].any()) and floor > 0 and floor < 1
    low = ws < min(floor, 1.0)
    low[0] = False
    keep &= ~low
    w[order] = ws * keep
    return w, close


def check(x, u, tokens, logprobs, T=1.0, k=0, p=1.0, floor=0.0):
    x, u, tokens, logprobs = x.float().cpu(), u.double().cpu(), tokens.cpu(), logprobs.double().cpu()
    assert tokens.dtype == torch.int64
    unsure, EPS = 0, off(x.shape[1])
    for b in range(len(tokens)):
        row = [float(v[b]) if torch.is_tensor(v) else v for v in (T, k, p, floor)]
        w, close = kept64(x[b], row[0], int(row[1]), row[2], row[3])
        t, total = int(tokens[b]), w.sum()
        if total == 0:
            assert t == -1 and logprobs[b] == -math.inf
            continue
        unsure += close
        if close:
            continue
        at = w.cumsum(0)
        assert 0 <= t < x.shape[1] and w[t] > 0, (b, t, row)
        target = min(max(float(u[b]), 0.0), 1.0) * total
        assert at[t] - w[t] <= target + EPS * total and target - EPS * total <= at[t], (b, t, row)
        want = math.log(w[t] / total)
        assert abs(float(logprobs[b]) - want) <= abs(want) * 2.0 ** -23 + EPS, (b, float(logprobs[b]), want)
    return unsure


def logits(gen, B, V, dtype, spread=3.0):
    x = torch.randn(B, V, generator=gen, device=DEV) * spread
    at = torch.rand(B, V, generator=gen, device=DEV).topk(min(V, 20), dim=-1).indices
    x.scatter_add_(1, at, 8 * torch.rand(B, at.shape[1], generator=gen, device=DEV))
    return x.to(dtype)


SETTINGS = [
    dict(), dict(temperature=0.0), dict(temperature=0.3), dict(temperature=2.5), dict(top_k=1), dict(top_k=7),
    dict(top_k=2000), dict(top_p=0.0), dict(top_p=0.3), dict(top_p=0.95), dict(top_p=0.999, temperature=2.0),
    dict(min_p=0.05), dict(min_p=1.0), dict(top_k=50, top_p=0.9, min_p=0.01, temperature=0.8),
    dict(top_k=3000, top_p=0.99, temperature=3.0), dict(top_k=10 ** 12, top_p=0.5),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (2, 63), (5, 1000), (4, 8191), (2, 32003), (3, 150001), (1, 262144)])
def test_sample(B, V, dtype):
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = logits(gen, B, V, dtype)
    unsure = 0
    for setting in SETTINGS:
        print(f"case {B}x{V} {dtype} {setting}", flush=True)
        u = torch.rand(B, generator=gen, device=DEV)
        tokens, logprobs = sample_tokens(x, u, return_logprobs=True, **setting)
        assert torch.equal(sample_tokens(x, u, **setting), tokens)
        names = dict(temperature="T", top_k="k", top_p="p", min_p="floor")
        unsure += check(x, u, tokens, logprobs, **{names[n]: v for n, v in setting.items()})
    assert unsure <= 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_of_their_own(dtype):
    B, V = 40, 4099
    gen = torch.Generator(device=DEV).manual_seed(0)
    wide = logits(gen, B, V + 9, dtype)
    x = wide[:, 3:3 + V]               # rows that begin anywhere
    r = torch.rand(4, B, generator=gen, device=DEV)
    heat = torch.where(torch.arange(B, device=DEV) % 5 == 4, 0.0, 0.2 + 2 * r[0])
    heat[7] = -1.0                      # not above zero: the largest
    k = (r[1] * 60).to(torch.int32)
    k[3], k[5] = -4, 2 ** 31 - 1        # all
    p = (r[2] * 1.2).clamp(max=1.0)
    floor = (r[3] - 0.5).clamp(min=0.0) * 0.1
    for u in (torch.rand(B, generator=gen, device=DEV), torch.rand(B, generator=gen, device=DEV, dtype=torch.float64)):
        tokens, logprobs = sample_tokens(x, u, temperature=heat, top_k=k, top_p=p, min_p=floor, return_logprobs=True)
        assert check(x, u, tokens, logprobs, T=heat, k=k, p=p, floor=floor) == 0


def test_every_share_is_drawn():
    # Evenly spaced random numbers draw every token as often as its share says, to within one, in index order.
    V, n = 500, 4096
    gen = torch.Generator(device=DEV).manual_seed(9)
    x = logits(gen, 1, V, torch.float32, 1.0)
    u = (torch.arange(n, device=DEV, dtype=torch.float64) + 0.5) / n
    for k, p in ((0, 1.0), (40, 0.9)):
        tokens = sample_tokens(x.expand(n, V), u, top_k=k, top_p=p).cpu()
        assert bool((tokens[1:] >= tokens[:-1]).all())
        w, _ = kept64(x[0].cpu(), 1.0, k, p, 0.0)
        count = torch.bincount(tokens, minlength=V).double()
        assert float((count - n * w / w.sum()).abs().max()) <= 1.0 + 1e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_masked_rows_and_numbers_that_are_none(dtype):
    V, inf, lowest = 5000, float("inf"), torch.finfo(dtype).min
    gen = torch.Generator(device=DEV).manual_seed(2)
    x = logits(gen, 10, V, dtype)
    x[0] = -inf                                # nothing
    x[1] = float("nan")
    x[2, 1:] = -inf                            # one
    x[3, :-1] = lowest                         # masked by the type's lowest value
    x[4, ::2] = float("nan")
    x[5, 77], x[5, 4000] = inf, inf            # two that outweigh everything
    x[6] = lowest                              # all alike
    x[7, 100:] = lowest
    x[8, 100:] = -inf
    x[9, 50] = torch.finfo(dtype).max
    names = dict(temperature="T", top_k="k", top_p="p", min_p="floor")
    for setting in (dict(), dict(top_p=0.7), dict(top_k=200), dict(top_k=300, top_p=0.9, temperature=1.5),
                    dict(min_p=0.1), dict(temperature=0.0), dict(temperature=inf), dict(temperature=inf, top_p=0.5),
                    dict(temperature=1e-30, top_p=0.5), dict(temperature=1e30, top_k=1000)):
        for v in (0.0, 0.5, 0.999, 1.0 - 2.0 ** -24):
            u = torch.full((10,), v, device=DEV)
            tokens, logprobs = sample_tokens(x, u, return_logprobs=True, **setting)
            unsure = check(x, u, tokens, logprobs, **{names[n]: s for n, s in setting.items()})
            assert unsure <= 4, setting
    # Random numbers out of range take the first and the last of the kept.
    for v, near in ((-3.0, 0.0), (1.0, 1 - 2.0 ** -53), (7.0, 1 - 2.0 ** -53), (float("nan"), 0.0)):
        a = sample_tokens(x, torch.full((10,), v, device=DEV, dtype=torch.float64), top_k=30)
        b = sample_tokens(x, torch.full((10,), near, device=DEV, dtype=torch.float64), top_k=30)
        assert torch.equal(a, b)


@pytest.mark.parametrize("V", [9000, 70001])
def test_crowds_and_ties(V):
    # More of one value, or close together, than are sorted at once; far from an outlier, which sets the bins.
    gen = torch.Generator(device=DEV).manual_seed(V)
    base = torch.rand(V, generator=gen, device=DEV)
    rows = [torch.zeros(V, device=DEV), (base * 3).floor(), base * 1e-3, base * 1e-3, base * 1e-6 + 1.0,
            torch.where(base < 0.6, 1.0, base)]
    x = torch.stack(rows)
    x[3, 17], x[4, 5], x[5, 9] = 8.0, 30.0, 12.0
    x[3, 40] = -20.0
    names = dict(temperature="T", top_k="k", top_p="p", min_p="floor")
    for setting in (dict(top_k=1), dict(top_k=4097), dict(top_k=V - 1), dict(top_p=0.5), dict(top_p=0.25, top_k=6000),
                    dict(top_p=0.999, temperature=5.0), dict(top_p=0.75, min_p=0.5)):
        for v in (0.0, 0.37, 0.99999):
            u = torch.full((len(rows),), v, device=DEV)
            tokens, logprobs = sample_tokens(x, u, return_logprobs=True, **setting)
            # (Shares of equal weights may end a prefix exactly: those rows go by the count below.)
            check(x, u, tokens, logprobs, **{names[n]: s for n, s in setting.items()})
    # Ties go to the lowest index: of equal weights the first k, and as many as reach the share.
    last = torch.full((1,), 1 - 2.0 ** -24, device=DEV)
    for k in (1, 5, 4096, 5000, V - 1):
        assert int(sample_tokens(x[:1], last, top_k=k)) == k - 1
    even = torch.zeros(1, 8192, device=DEV)
    for p, n in ((0.5, 4096), (0.25, 2048), (0.125 + 2.0 ** -13, 1025), (1 - 2.0 ** -13, 8191), (2.0 ** -14, 1)):
        assert int(sample_tokens(even, last, top_p=p)) == n - 1
    assert int(sample_tokens(even, last, top_p=0.5, top_k=1000)) == 499


def test_the_largest_vocabulary_and_many_rows():
    V = 2088960
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = logits(gen, 2, V, torch.bfloat16)
    for setting in (dict(), dict(top_p=0.9), dict(top_k=100)):
        u = torch.rand(2, generator=gen, device=DEV)
        tokens, logprobs = sample_tokens(x, u, return_logprobs=True, **setting)
        check(x, u, tokens, logprobs, k=setting.get("top_k", 0), p=setting.get("top_p", 1.0))
    with pytest.raises(ValueError, match="vocabulary"):
        sample_tokens(torch.zeros(1, V + 1, device=DEV), torch.zeros(1, device=DEV))
    # Rows past 2^31 elements, and one row for all.
    B, V = 70000, 40000
    x = torch.zeros(1, V, device=DEV, dtype=torch.float16)
    u = torch.rand(B, generator=gen, device=DEV)
    tokens = sample_tokens(x.expand(B, V), u)
    assert torch.equal(tokens, (u.double() * V).floor().long())
    x = torch.zeros(B, V, device=DEV, dtype=torch.float16)
    x[-1, 123] = 60.0
    tokens = sample_tokens(x, u, temperature=0.5)
    assert int(tokens[-1]) == 123 and torch.equal(tokens[:-1], (u[:-1].double() * V).floor().long())
    assert sample_tokens(x[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [65536, 70001, 131071])
def test_shared_rows_draw_as_lone_ones(V, dtype):
    # A few long rows are shared by workgroups, many are not.  Weights are whole units, so tokens and sums are
    # the same to the last bit.
    inf, lowest = float("inf"), torch.finfo(dtype).min
    gen = torch.Generator(device=DEV).manual_seed(V)
    wide = logits(gen, 16, V + 5, dtype)
    x = wide[:, 3:3 + V]                        # rows that begin anywhere
    x[0] = -inf
    x[1], x[1, V - 1] = float("nan"), 0.5       # one, in the last part
    x[2, 100], x[2, V - 2] = inf, inf
    x[3] = 1.0                                  # all alike: the bin of an end holds more than a list
    x[4] = lowest
    x[5, :-1] = lowest
    x[6] = (torch.rand(V, generator=gen, device=DEV) * 3).floor().to(dtype)
    x[7, 5] = 60.0                              # peaked: a short list
    x[8, 1000:] = -inf                          # parts with nothing
    x[9] = (x[9].float() * 0.01).to(dtype)      # flat
    B = x.shape[0]
    heat = torch.full((B,), 0.8, device=DEV)
    heat[10], heat[11], heat[12], heat[13] = 0.0, 3.0, inf, 1e-30
    mass = torch.rand(B, generator=gen, device=DEV)
    mass[14], mass[15], mass[11] = 1.0, 0.0, 0.999
    many = x.repeat(9, 1)
    for v in (0.0, 0.4, 1.0 - 2.0 ** -24):
        u = torch.full((9 * B,), v, device=DEV)
        for setting in (dict(), dict(top_p=0.9), dict(top_p=0.3, temperature=2.0), dict(temperature=heat),
                        dict(temperature=heat, top_p=mass)):
            long = {n: s.repeat(9) if torch.is_tensor(s) else s for n, s in setting.items()}
            tokens, logprobs = sample_tokens(x, u[:B], return_logprobs=True, **setting)
            lone, alone = sample_tokens(many, u, return_logprobs=True, **long)
            for i in range(9):
                assert torch.equal(lone[i * B:i * B + B], tokens), setting
                assert torch.equal(alone[i * B:i * B + B], logprobs), setting


def test_shared_rows_in_a_graph():
    B, V = 3, 100003
    gen = torch.Generator(device=DEV).manual_seed(4)
    x, u = logits(gen, B, V, torch.bfloat16), torch.rand(B, generator=gen, device=DEV)
    sample_tokens(x, u, top_p=0.9)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        free = sample_tokens(x, u)
        some = sample_tokens(x, u, top_p=0.9)
    for i in range(5):
        x.copy_(logits(gen, B, V, torch.bfloat16, spread=0.1 + i))
        u.copy_(torch.rand(B, generator=gen, device=DEV))
        graph.replay()
        got = free.clone(), some.clone()
        torch.cuda.synchronize()
        assert torch.equal(got[0], sample_tokens(x, u)) and torch.equal(got[1], sample_tokens(x, u, top_p=0.9))


@pytest.mark.parametrize("B,V", [(3, 150001), (40, 70000)])
def test_shared_rows_time_after_time(B, V):
    # Calls that follow one another in one workspace, each with other settings: nothing of the last one's is left.
    gen = torch.Generator(device=DEV).manual_seed(B)
    x, u = logits(gen, B, V, torch.float16), torch.rand(B, generator=gen, device=DEV)
    many, all_u = x.repeat(129 // B + 1, 1), u.repeat(129 // B + 1)
    settings = [dict(top_p=p, temperature=t) for t in (0.7, 1.0, 2.0) for p in (0.5, 0.95, 0.999, 1.0)]
    want = [[y[:B] for y in sample_tokens(many, all_u, return_logprobs=True, **s)] for s in settings]
    got = []
    for _ in range(20):
        for s in settings:
            got.append(sample_tokens(x, u, return_logprobs=True, **s))
    for i, (tokens, logprobs) in enumerate(got):
        exact = want[i % len(settings)]
        assert torch.equal(tokens, exact[0]) and torch.equal(logprobs, exact[1]), (i, settings[i % len(settings)])


def test_other_layouts():
    # Rows one by one, one row for all, a batch of another batch's rows, a vocabulary of one.
    gen = torch.Generator(device=DEV).manual_seed(12)
    x, u = logits(gen, 6, 70007, torch.bfloat16), torch.rand(6, generator=gen, device=DEV)
    for setting in (dict(), dict(top_p=0.8), dict(top_k=40, top_p=0.8)):
        tokens = sample_tokens(x, u, **setting)
        for b in range(6):
            assert int(sample_tokens(x[b:b + 1], u[b:b + 1], **setting)) == int(tokens[b])
        assert torch.equal(sample_tokens(x[::2], u[::2].contiguous(), **setting), tokens[::2])
        assert torch.equal(sample_tokens(x[2:3].expand(6, -1), u, **setting),
                           sample_tokens(x[2:3].repeat(6, 1), u, **setting))
    assert sample_tokens(x[:, 5:6], u, top_p=0.5).tolist() == [0] * 6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", ["ends", "behind", "between", "least"])
def test_top_k_past_the_logits_that_are_there(rows, dtype):
    # More of the lowest logit than a list holds, the rest of the row masked: top_k from below their number to the
    # whole row.
    V, inf = 20000, float("inf")
    gen = torch.Generator(device=DEV).manual_seed(6)
    x = torch.full((3, V), -inf, device=DEV)
    if rows == "ends":
        x[0, :10000], x[1, :5000], x[2, :17000] = 0.0, -2.0, 1.0
    elif rows == "behind":
        x[0, 10000:], x[1, 15000:], x[2, 3001:] = 0.0, -2.0, 1.0
    elif rows == "between":
        x[0, ::2], x[1, 1::3], x[2, 5::2] = 0.0, -2.0, 1.0
    else:       # 2000 different logits above the many of the lowest
        for r, n in enumerate((4500, 9000, 16000)):
            at = torch.randperm(V, generator=gen, device=DEV)[:2000 + n]
            x[r, at] = -1.0
            x[r, at[:2000]] = 4 * torch.rand(2000, generator=gen, device=DEV)
    x = x.to(dtype)
    there = (x > -inf).sum(dim=1).tolist()
    last = [int((x[r] > -inf).nonzero()[-1]) for r in range(3)]
    counts = sorted({k for n in there for k in (n - 1, n, n + 1)} | {4000, 18500, V - 1})
    names = dict(top_p="p", min_p="floor")
    for k in counts:
        each = torch.tensor([k, there[1] + 100, V - 1], dtype=torch.int32, device=DEV)
        for setting in (dict(), dict(top_p=0.5), dict(top_p=0.83127), dict(min_p=0.02)):
            print(f"case {rows} {dtype} top_k={k} {setting}", flush=True)
            for v in (0.0, 0.37, 1.0 - 2.0 ** -24):
                u = torch.full((3,), v, device=DEV)
                for top_k in (k, each):
                    tokens, logprobs = sample_tokens(x, u, top_k=top_k, return_logprobs=True, **setting)
                    check(x, u, tokens, logprobs, k=top_k, **{names[n]: s for n, s in setting.items()})
                    if not setting and v > 0.9 and rows != "least":
                        want = [last[r] for r in range(3) if (k if top_k is k else int(each[r])) >= there[r]]
                        assert [t for r, t in enumerate(tokens.tolist())
                                if (k if top_k is k else int(each[r])) >= there[r]] == want


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [50, 700, 9001])
def test_min_p_where_the_temperature_leaves_all_alike(V, dtype):
    # The logarithm of min_p times a temperature says nothing of weights that are one, or one to the last bits.
    inf = float("inf")
    gen = torch.Generator(device=DEV).manual_seed(V)
    x = logits(gen, 4, V, dtype)
    x[1, ::3] = -inf
    x[2] = x[2] * 0.0 + 5.0
    x[3, 7] = torch.finfo(dtype).max
    heats = [inf, 1e30, 2.0 ** 70]
    for heat in heats + [torch.tensor([inf, 1e25, 1e35, inf], device=DEV)]:
        for floor in (1.0, 1.0 - 2.0 ** -24, 0.5, torch.tensor([1.0, 1.0, 0.75, 1.0], device=DEV)):
            for v in (0.0, 0.6, 1.0 - 2.0 ** -24):
                u = torch.full((4,), v, device=DEV)
                tokens, logprobs = sample_tokens(x, u, temperature=heat, min_p=floor, return_logprobs=True)
                check(x, u, tokens, logprobs, T=heat, floor=floor)
    # All but the masked have the same share.
    tokens = sample_tokens(x, torch.full((4,), 1.0 - 2.0 ** -24, device=DEV), temperature=inf, min_p=1.0)
    assert tokens.tolist() == [V - 1, V - 1 if (V - 1) % 3 else V - 2, V - 1, V - 1]

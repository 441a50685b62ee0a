"""Performance cases of what a decoding loop over a paged K/V cache needs beside
its attention: the attention weight that each cached key has gathered, the
eviction of the keys that gathered least, and the draw of the next token.

A case is a dict of plain values; ``op`` names the operator:

* ``mass``    the softmax weights of each sequence's new tokens on its cached
  keys, summed over the tokens and over the query heads of each KV head
  (``add``: onto what earlier chunks gave);
* ``evict``   of each sequence and KV head the ``first`` and the ``recent`` positions
  and the heaviest others are kept, ``keep`` in all, and move in order into
  other pages (sequences of no more move whole);
* ``sample``  one token a row from logits with temperature, top-k, top-p and
  min-p, given a random number a row; ``mixed``: other values in every row,
  as a server's batch has them.

Sequences of a ragged batch have lengths spread between a fifth and the whole
of ``kv`` (and of ``new``), the same for every seed; pages are handed out in
random order.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
_DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_EB = {"bf16": 2, "f16": 2, "f32": 4}
_HEADS = ((28, 4), (12, 2), (8, 2), (16, 8), (32, 8))


def listed():
    return [
        # The next token of one short conversation: launch and latency.
        {"name": "mass_short", "op": "mass", "S": 1, "new": 1, "kv": 517, "Hq": 8, "Hkv": 2, "D": 128, "page": 16,
         "add": False, "dtype": "f16"},
        # The next token of 64 conversations of ragged lengths.
        {"name": "mass_64", "op": "mass", "S": 64, "new": 1, "kv": 32768, "Hq": 28, "Hkv": 4, "D": 128, "page": 16,
         "add": False, "dtype": "bf16"},
        # The last tokens of four long prompts, as the window that decides what to keep of them.
        {"name": "mass_window", "op": "mass", "S": 4, "new": 40, "kv": 33000, "Hq": 16, "Hkv": 8, "D": 64, "page": 32,
         "add": False, "dtype": "f16"},
        # A chunk of a long prompt, added to what the earlier chunks gave.
        {"name": "mass_chunk", "op": "mass", "S": 1, "new": 4096, "kv": 32768, "Hq": 28, "Hkv": 4, "D": 128,
         "page": 64, "add": True, "dtype": "bf16"},
        # One short conversation past a small budget: launch and latency.
        {"name": "evict_short", "op": "evict", "S": 1, "kv": 700, "keep": 256, "first": 4, "recent": 32, "Hkv": 2,
         "D": 128, "page": 16, "dtype": "f16"},
        # Odd sizes, float32 pages, narrow heads.
        {"name": "evict_odd", "op": "evict", "S": 5, "kv": 20011, "keep": 1531, "first": 1, "recent": 0, "Hkv": 8,
         "D": 64, "page": 48, "dtype": "f32"},
        # 64 conversations of ragged lengths, the shorter ones moved whole.
        {"name": "evict_64", "op": "evict", "S": 64, "kv": 16384, "keep": 4096, "first": 16, "recent": 512, "Hkv": 4,
         "D": 128, "page": 16, "dtype": "bf16"},
        # One very long prompt cut to a quarter.
        {"name": "evict_128k", "op": "evict", "S": 1, "kv": 131072, "keep": 32768, "first": 64, "recent": 2048,
         "Hkv": 4, "D": 128, "page": 64, "dtype": "bf16"},
        # One conversation's next token.
        {"name": "sample_one", "op": "sample", "B": 1, "V": 32003, "temperature": 0.7, "top_k": 50, "top_p": 0.95,
         "min_p": 0.0, "mixed": False, "dtype": "f16"},
        # A batch whose rows all ask for something else, an odd vocabulary.
        {"name": "sample_mixed", "op": "sample", "B": 24, "V": 50021, "temperature": 0.9, "top_k": 1000, "top_p": 0.9,
         "min_p": 0.02, "mixed": True, "dtype": "bf16"},
        # A batch drawn from its nuclei.
        {"name": "sample_nucleus", "op": "sample", "B": 64, "V": 150016, "temperature": 0.8, "top_k": 0,
         "top_p": 0.95, "min_p": 0.0, "mixed": False, "dtype": "bf16"},
        # A large batch of rollouts at temperature 1, with nothing but a floor.
        {"name": "sample_plain", "op": "sample", "B": 256, "V": 131072, "temperature": 1.0, "top_k": 0, "top_p": 1.0,
         "min_p": 0.001, "mixed": False, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("mass", "mass", "evict", "evict", "sample", "sample"))
    if op == "sample":
        case = {"op": op, "B": _log(rng, 1, 128), "V": _log(rng, 500, 200000), "mixed": rng.random() < 0.4,
                "temperature": rng.choice((0.5, 0.8, 1.0, 1.3)), "top_k": rng.choice((0, 0, 20, _log(rng, 1, 3000))),
                "top_p": rng.choice((1.0, 0.9, 0.95, rng.uniform(0.05, 0.99))),
                "min_p": rng.choice((0.0, 0.0, 0.05, 0.002)), "dtype": rng.choice(("bf16", "f16", "f32"))}
        return case
    Hq, Hkv = rng.choice(_HEADS)
    D, page = rng.choice((128, 128, 64)), rng.choice((16, 32, 48, 64, 128, 256))
    case = {"op": op, "Hkv": Hkv, "D": D, "page": page, "dtype": rng.choice(("bf16", "bf16", "f16"))}
    if op == "evict":
        S = rng.choice((1, 1, 3, 8, 64))
        kv = _log(rng, 100, 131072 if S == 1 else 131072 // S)
        keep = max(8, int(kv * rng.uniform(0.05, 0.7)))
        case.update(S=S, kv=kv, keep=keep, first=rng.choice((0, 4, min(64, keep // 4))),
                    recent=rng.randint(0, keep // 2))
        return case
    S = rng.choice((1, 2, 4, 16, 64))
    new = {"one": 1, "few": rng.randint(2, 40)}.get(rng.choice(("one", "few", "chunk"))) or _log(rng, 41, 2048 // min(S, 8))
    S = S if new < 10 else min(S, 4)
    case.update(S=S, new=new, kv=max(new, _log(rng, 200, 16384 if S > 16 else 30000)), Hq=Hq, add=rng.random() < 0.3)
    return case


# ------------------------------------------------------------------ shapes


def _lengths(case):
    """(new, kv) of every sequence: ragged, the longest as long as the case says."""
    out = []
    for s in range(case["S"]):
        f = 1.0 - 0.8 * ((s * 0.6180339887498949) % 1.0)
        g = 1.0 - 0.8 * ((s * 0.7548776662466927) % 1.0)
        n = max(1, round(case.get("new", 1) * g))
        out.append((n, max(n, round(case["kv"] * f))))
    return out


def work(case):
    eb = _EB[case["dtype"]]
    if case["op"] == "sample":
        # An exponential and a sum a logit.
        return {"bytes": case["B"] * (case["V"] * eb + 16), "flops": 2 * case["B"] * case["V"]}
    lens, Hkv, D = _lengths(case), case["Hkv"], case["D"]
    keys = sum(kv for _, kv in lens)
    pages = sum((kv + case["page"] - 1) // case["page"] for _, kv in lens)
    if case["op"] == "evict":
        kept = sum(min(kv, case["keep"]) for _, kv in lens)
        # Every mass read; a kept key: its row and its value's read and written, its mass and position written.
        return {"bytes": 4 * Hkv * keys + Hkv * kept * (4 * D * eb + 8) + 4 * pages, "flops": Hkv * keys}
    n = sum(a for a, _ in lens)
    pairs = sum(a * (kv - a) + a * (a + 1) / 2 for a, kv in lens)
    return {"bytes": n * case["Hq"] * D * eb + keys * Hkv * (D * eb + (8 if case["add"] else 4)) + 4 * pages,
            "flops": 2 * D * case["Hq"] * pairs}


# ------------------------------------------------------------------ inputs


def _tables(gen, counts, spare):
    """A row of random page ids for each count of ``counts`` (lists of equal length), -1 behind it; pages in all."""
    total = sum(sum(c) for c in counts) + spare
    order = torch.randperm(total, generator=gen, device=DEV)
    tables, at = [], 0
    for c in counts:
        c = torch.tensor(c, device=DEV)
        col = torch.arange(int(c.max()), device=DEV)
        first = at + torch.cumsum(c, 0) - c
        slot = (first[:, None] + col).clamp(max=total - 1)
        tables.append(torch.where(col < c[:, None], order[slot], -1).to(torch.int32).contiguous())
        at += int(c.sum())
    return tables, total


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = _DT[case["dtype"]]
    st = {"case": case}
    if case["op"] == "sample":
        B, V = case["B"], case["V"]
        # A language model's row: many small logits, a few tens that stand out, more or less so.
        x = torch.randn(B, V, generator=gen, device=DEV) * 2.0
        likely = torch.rand(B, V, generator=gen, device=DEV).topk(min(V, 40), dim=-1).indices
        sharp = 6.0 + 10.0 * torch.rand(B, 1, generator=gen, device=DEV)
        x.scatter_add_(1, likely, sharp * torch.rand(B, likely.shape[1], generator=gen, device=DEV))
        st["logits"] = x.to(dt)
        st["uniform"] = torch.rand(B, generator=gen, device=DEV)
        if case["mixed"]:
            r = torch.rand(4, B, generator=gen, device=DEV)
            greedy = torch.arange(B, device=DEV) % 8 == 7
            st["temperature"] = torch.where(greedy, 0.0, case["temperature"] * (0.5 + r[0]))
            st["top_k"] = torch.where(r[1] < 0.3, 0.0, case["top_k"] * r[1]).round().to(torch.int32)
            st["top_p"] = torch.where(r[2] < 0.3, 1.0, case["top_p"] * (0.5 + 0.5 * r[2]))
            st["min_p"] = torch.where(r[3] < 0.5, 0.0, case["min_p"] * r[3])
        else:
            for name in ("temperature", "top_k", "top_p", "min_p"):
                st[name] = case[name]
        return st
    lens, page, Hkv, D = _lengths(case), case["page"], case["Hkv"], case["D"]
    S = len(lens)
    counts = [[(kv + page - 1) // page for _, kv in lens]]
    if case["op"] == "evict":
        counts.append([(min(kv, case["keep"]) + page - 1) // page for _, kv in lens])
    tables, total = _tables(gen, counts, 8)
    st["page_table"] = tables[0]
    st["kv_lens"] = torch.tensor([kv for _, kv in lens], dtype=torch.int32, device=DEV)
    # [pages, Hkv, page, D] views of [pages, page, Hkv, D] storage.
    st["k_pages"] = torch.randn(total, page, Hkv, D, generator=gen, device=DEV, dtype=dt).transpose(1, 2)
    if case["op"] == "evict":
        st["out_table"] = tables[1]
        st["v_pages"] = torch.randn(total, page, Hkv, D, generator=gen, device=DEV, dtype=dt).transpose(1, 2)
        # Weights spread over many sizes; some keys that nothing attended.
        mass = torch.exp(2.0 * torch.randn(total, Hkv, page, generator=gen, device=DEV))
        idle = torch.rand(total, Hkv, page, generator=gen, device=DEV) < 0.05
        st["mass_pages"] = mass.masked_fill_(idle, 0.0)
        return st
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    st["q_starts"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
    st["q"] = (2.0 * torch.randn(starts[-1], case["Hq"], D, generator=gen, device=DEV)).to(dt)
    st["mass_pages"] = torch.zeros(total, Hkv, page, device=DEV)
    if case["add"]:
        st["before"] = torch.rand(total, Hkv, page, generator=gen, device=DEV)
    st["new"] = max(n for n, _ in lens)
    return st


# ------------------------------------------------------------------ the framework's operators


def _run_own(st):
    case = st["case"]
    if "kernels.eviction" not in sys.modules:
        pkg = os.path.join(os.getcwd(), "spruce-research_amd")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
    if case["op"] == "sample":
        from kernels.sampling import sample_tokens
        return sample_tokens(st["logits"], st["uniform"], temperature=st["temperature"], top_k=st["top_k"],
                             top_p=st["top_p"], min_p=st["min_p"], return_logprobs=True)
    if case["op"] == "evict":
        from kernels.eviction import evict_paged_kv
        kept, lens = evict_paged_kv(st["k_pages"], st["v_pages"], st["mass_pages"], st["page_table"], st["kv_lens"],
                                    st["out_table"], case["keep"], first=case["first"], recent=case["recent"])
        return kept, lens, st["k_pages"], st["v_pages"], st["mass_pages"]
    from kernels.eviction import paged_key_mass
    if case["add"]:     # what the earlier chunks gave: a pass adds to it, and may run again
        st["mass_pages"].copy_(st["before"])
    return paged_key_mass(st["q"], st["k_pages"], st["mass_pages"], st["page_table"], st["q_starts"], st["kv_lens"],
                          case["D"] ** -0.5, accumulate=case["add"])


# ------------------------------------------------------------------ plain forms


def _plain_mass(st):
    case = st["case"]
    q, table, lens = st["q"], st["page_table"].long(), st["kv_lens"].long()
    N, Hq, D = q.shape
    S, Hkv, page, T = table.shape[0], case["Hkv"], case["page"], st["new"]
    G, L = Hq // Hkv, table.shape[1] * page
    if case["add"]:
        st["mass_pages"].copy_(st["before"])
    # Sequences padded to the longest: queries [S, Hkv, T*G, D], keys [S, Hkv, D, L].
    starts = st["q_starts"].long()
    new = starts[1:] - starts[:-1]
    n = torch.arange(N, device=DEV)
    seq = torch.searchsorted(starts[1:].contiguous(), n, right=True)
    qp = torch.zeros(S, T, Hq, D, device=DEV)
    qp[seq, n - starts[seq]] = q.float()
    qp = qp.view(S, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hkv, T * G, D)
    keys = st["k_pages"][table.clamp(min=0)].float().permute(0, 2, 4, 1, 3).reshape(S, Hkv, D, L)
    row = torch.arange(T, device=DEV)
    key_pos = torch.arange(L, device=DEV)
    first_new = (lens - new)[:, None]
    seen = (key_pos <= (first_new + row)[..., None]) & (row < new[:, None])[..., None]      # [S, T, L]
    scores = torch.matmul(qp, keys).mul_(D ** -0.5).view(S, Hkv, T, G, L)
    scores.masked_fill_(~seen[:, None, :, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    scores.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
    scores.div_(scores.sum(dim=-1, keepdim=True).clamp(min=1e-30))
    now = scores.sum(dim=(2, 3))                                                            # [S, Hkv, L]
    # Into the sequences' pages: new positions hold this pass's weight alone.
    s, pos = torch.nonzero(key_pos < lens[:, None], as_tuple=True)
    at, slot = table[s, pos // page], pos % page
    value = now[s, :, pos]
    if case["add"]:
        value = value + torch.where((pos < first_new[s, 0])[:, None], st["mass_pages"][at, :, slot], 0.0)
    st["mass_pages"][at, :, slot] = value
    return st["mass_pages"]


def _plain_evict(st):
    case = st["case"]
    table, out_table, lens = st["page_table"].long(), st["out_table"].long(), st["kv_lens"].long()
    page, keep = case["page"], case["keep"]
    S, L = table.shape[0], table.shape[1] * page
    mass = st["mass_pages"][table.clamp(min=0)].permute(0, 2, 1, 3).reshape(S, case["Hkv"], L)
    pos = torch.arange(L, device=DEV)
    held = (pos < case["first"]) | (pos >= lens[:, None] - case["recent"])                  # [S, L]
    weight = mass.masked_fill(held[:, None], float("inf")).masked_fill((pos >= lens[:, None])[:, None], float("-inf"))
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices[..., :keep]
    K = order.shape[-1]
    new_lens = lens.clamp(max=keep)
    order = torch.where(torch.arange(K, device=DEV) < new_lens[:, None, None], order, L).sort(dim=-1).values
    kept = torch.where(order < L, order, -1)
    if K < keep:
        kept = torch.cat((kept, kept.new_full((S, kept.shape[1], keep - K), -1)), dim=-1)
    s, g, r = torch.nonzero(kept >= 0, as_tuple=True)
    p = kept[s, g, r]
    src, slot, dst, to = table[s, p // page], p % page, out_table[s, r // page], r % page
    for pages in (st["k_pages"], st["v_pages"], st["mass_pages"]):
        pages[dst, g, to] = pages[src, g, slot]
    return kept.to(torch.int32), new_lens.to(torch.int32), st["k_pages"], st["v_pages"], st["mass_pages"]


def _column(x, B, dtype=torch.float64):
    return (x if torch.is_tensor(x) else torch.full((B,), x, dtype=torch.float64, device=DEV)).to(dtype)[:, None]


def _plain_sample(st):
    x = st["logits"].double()
    B, V = x.shape
    temperature, top_p, min_p = (_column(st[n], B) for n in ("temperature", "top_p", "min_p"))
    top_k = _column(st["top_k"], B, torch.int64)
    xs, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((xs - xs[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    rank = torch.arange(V, device=DEV)
    keep = rank < torch.where((top_k <= 0) | (top_k > V), V, top_k)
    w = w * keep
    before = torch.cumsum(w, dim=-1) - w
    keep = keep & ((top_p >= 1) | (before < top_p * w.sum(dim=-1, keepdim=True)) | (rank == 0))
    keep = keep & ((w >= min_p) | (rank == 0))
    keep = keep & ((temperature > 0) | (rank == 0))
    w = torch.zeros_like(x).scatter_(1, order, w * keep)
    total = w.sum(dim=-1, keepdim=True)
    found = (torch.cumsum(w, dim=-1) <= st["uniform"].double()[:, None] * total).sum(dim=-1, keepdim=True)
    last = torch.where(w > 0, rank, -1).amax(dim=-1, keepdim=True)
    token = torch.minimum(found, last)
    return token[:, 0], torch.log(w.gather(1, token) / total)[:, 0].float()


def run(st):
    if own:
        return _run_own(st)
    return {"mass": _plain_mass, "evict": _plain_evict, "sample": _plain_sample}[st["case"]["op"]](st)


# ------------------------------------------------------------------ 64 bits


def _exact_mass(case, st):
    lens, page, starts = _lengths(case), case["page"], st["q_starts"].tolist()
    G = case["Hq"] // case["Hkv"]
    out = st["before"].double() if case["add"] else st["mass_pages"].double()
    for s, (n, kv) in enumerate(lens):
        p = torch.arange(kv, device=DEV)
        at = st["page_table"][s].long()[p // page]
        for g in range(case["Hkv"]):
            k = st["k_pages"][at, g, p % page].double()
            total = torch.zeros(kv, dtype=torch.float64, device=DEV)
            for r in range(0, n, 256):
                t = torch.arange(r, min(n, r + 256), device=DEV)
                hide = p > (kv - n + t)[:, None]
                for h in range(g * G, (g + 1) * G):
                    a = st["q"][starts[s] + t, h].double() @ k.T / math.sqrt(case["D"])
                    total += torch.softmax(a.masked_fill(hide, -math.inf), dim=-1).sum(dim=0)
            if case["add"]:
                total[:kv - n] += out[at, g, p % page][:kv - n]
            out[at, g, p % page] = total
    return out


def _exact_evict(case, st):
    page, keep = case["page"], case["keep"]
    kp, vp, mp = st["k_pages"].double(), st["v_pages"].double(), st["mass_pages"].double()
    kept = torch.full((case["S"], case["Hkv"], keep), -1, dtype=torch.int32, device=DEV)
    for s, (_, kv) in enumerate(_lengths(case)):
        k = min(kv, keep)
        everything = torch.arange(kv, device=DEV)
        free = everything[case["first"]:max(case["first"], kv - case["recent"])] if kv > keep else everything[:0]
        at = st["page_table"][s].long()
        for g in range(case["Hkv"]):
            if kv > keep:
                m = mp[at[free // page], g, free % page]
                # Twice stably sorted: by position as it lies, then by weight.
                best = free[torch.argsort(-m, stable=True)[:k - (kv - len(free))]]
                picked = torch.ones(kv, dtype=torch.bool, device=DEV)
                picked[free] = False
                picked[best] = True
                p = everything[picked]
            else:
                p = everything
            r = torch.arange(k, device=DEV)
            to = st["out_table"][s].long()[r // page]
            kept[s, g, :k] = p.to(torch.int32)
            kp[to, g, r % page] = kp[at[p // page], g, p % page]
            vp[to, g, r % page] = vp[at[p // page], g, p % page]
            mp[to, g, r % page] = mp[at[p // page], g, p % page]
    return kept, st["kv_lens"].clamp(max=keep), kp, vp, mp


def _exact_sample(case, st):
    tokens, logprobs = [], []
    for b in range(case["B"]):
        T, k, p, floor = (float(v[b] if torch.is_tensor(v) else v)
                          for v in (st[n] for n in ("temperature", "top_k", "top_p", "min_p")))
        x = st["logits"][b].double()
        if T == 0:
            tokens.append(int((x == x.max()).nonzero()[0]))
            logprobs.append(0.0)
            continue
        logp = torch.log_softmax(x / T, dim=-1)
        ids = torch.argsort(x, descending=True, stable=True)
        if 0 < k < len(ids):
            ids = ids[:int(k)]
        if p < 1:
            share = torch.softmax(x[ids] / T, dim=-1)
            reached = torch.cumsum(share, dim=0) >= p
            ids = ids[:int(reached.nonzero()[0]) + 1] if bool(reached.any()) else ids
        ids = ids[torch.exp(logp[ids] - logp[ids[0]]) >= floor].sort().values
        prob = torch.softmax(x[ids] / T, dim=-1)
        past = (torch.cumsum(prob, dim=0) > float(st["uniform"][b])).nonzero()
        at = int(past[0]) if len(past) else len(ids) - 1
        tokens.append(int(ids[at]))
        logprobs.append(float(torch.log(prob[at])))
    return torch.tensor(tokens, device=DEV), torch.tensor(logprobs, dtype=torch.float64, device=DEV)


def exact(case, seed):
    st = prepare(case, seed)
    return {"mass": _exact_mass, "evict": _exact_evict, "sample": _exact_sample}[case["op"]](case, st)

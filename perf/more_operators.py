"""Many answers to one prompt, drafted and verified: the operators that batched serving over a 4-bit paged KV cache needs for them, as cases
that can be timed.

rope      query and key rows of a ragged batch turned by their positions, either layout, a part of the head, scaled frequencies
fork      sequences continued from others: full pages shared, a partly filled one copied, in all layers
compact   the pages in use to the front of the pool, tables and free stack after them
shared    attention of a batch whose sequences share their first pages, those computed once for all
verify    drafted tokens against the target's probabilities, from given random numbers

`own` false: elementary torch operations; true: the framework's entry points.  `listed()` holds the cases that are looked at by
name, `draw()` further ones of the same ranges, `prepare()` makes what a program has in hand before the call, `run()` is one pass,
`work()` what it cannot do without, `exact()` the result in 64 bits.

The cache: pages of 64 rows, (n_pages, kv_heads, page bytes of a head) bytes for the keys and the same for the values.  A block of 32
channels of a row is one fp16 scale d and 32 numbers -8 .. 7 in two's complement nibbles.  A head's part of a page is its quants,
then its scales, [row / 4][block][row % 4].  Keys: [row][8-channel group of a block][block][4 bytes], the low nibbles channels 0 .. 3
of the group, the high ones 4 .. 7.  Values: [block][channel % 16][row, reordered], the low nibbles channels 0 .. 15 of the block, the
high ones 16 .. 31; row 16 s + 4 g + i lies at 16 g + 4 s + i.  Shapes are those of caten_amd.synth and of the repository's size benchmark.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

PAGE = 64  # rows of a page
GPT2, LLAMA_1B, LLAMA_7B, LLAMA_70B = (12, 12, 64), (32, 4, 64), (32, 32, 128), (64, 8, 128)  # query heads, key / value heads, head size


def listed():
    return [
        # a small server's decode step: one row each of 48 sequences, slices of a fused q/k/v product; bound by latency
        dict(name="rope 1.1b 48 rows", family="rope", rows=48, h=32, kv=4, dh=64, rotary=64, halves=0, factor=1.0, longest=2048),
        # prompts of a server with long contexts (70B shape), frequencies scaled by parts
        dict(name="rope 70b 6001 rows", family="rope", rows=6001, h=64, kv=8, dh=128, rotary=128, halves=1, factor=8.0, longest=120000),
        # eight answers to one prompt with GPT-2: one parent, 12 layers
        dict(name="fork gpt2 1 into 8", family="fork", parents=1, forks=8, layers=12, kv=12, dh=64, longest=900, table=16),
        # 24 prompts with four answers each, 22 layers (1.1B shape)
        dict(name="fork 1.1b 24 into 96", family="fork", parents=24, forks=96, layers=22, kv=4, dh=64, longest=2000, table=32),
        # a small server's pool after a night's requests, 12 layers of GPT-2
        dict(name="compact gpt2 200 pages", family="compact", pages=200, used=0.6, n=12, layers=12, kv=12, dh=64, table=16),
        # a larger pool, before a part of it is given back
        dict(name="compact 70b 500 pages", family="compact", pages=500, used=0.5, n=30, layers=16, kv=8, dh=128, table=32),
        # eight answers to one prompt with GPT-2: latency counts
        dict(name="shared gpt2 8 answers", family="shared", h=12, kv=12, dh=64, groups=1, members=8, prefix=900, tail=200, rows=1, shape=1),
        # 64 samples of one long prompt, keys and values for every head (7B shape)
        dict(name="shared 7b 64 samples", family="shared", h=32, kv=32, dh=128, groups=1, members=64, prefix=4100, tail=400, rows=1, shape=2),
        # three system prompts with some dozen conversations each, five rows a sequence: a token and four drafted ones (70B shape)
        dict(name="shared 70b drafts", family="shared", h=64, kv=8, dh=128, groups=3, members=14, prefix=9000, tail=1500, rows=5, shape=3),
        # one conversation with GPT-2's vocabulary, four drafted tokens
        dict(name="verify gpt2 1x4", family="verify", n=1, drafts=4, vocab=50257),
        # sequences with and without drafts, up to seven
        dict(name="verify llama 48x7", family="verify", n=48, drafts=7, vocab=32000),
        # a vocabulary of 128256
        dict(name="verify 128k 64x4", family="verify", n=64, drafts=4, vocab=128256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["rope", "fork", "compact", "shared", "shared", "shared", "verify"])
    if family == "rope":
        h, kv, dh = rng.choice([GPT2, LLAMA_1B, LLAMA_7B, LLAMA_70B, (6, 2, 32), (10, 5, 80), (21, 3, 96)])
        rotary = rng.choice([dh, dh, dh // 2, dh // 4])
        return dict(family=family, rows=_log(rng, 1, min(6000, 6000 * 9216 // ((h + kv) * dh))), h=h, kv=kv, dh=dh, rotary=rotary, halves=rng.choice([0, 1]),
                    factor=rng.choice([1.0, 2.0, 8.0]), longest=_log(rng, 500, 500000))
    if family in ("fork", "compact"):
        h, kv, dh = rng.choice([GPT2, LLAMA_1B, (32, 8, 128), (6, 2, 32)])
        table, layers = rng.choice([16, 32]), rng.randint(2, 16)
        if family == "fork":
            parents = _log(rng, 1, 20)
            return dict(family=family, parents=parents, forks=_log(rng, 1, 80), layers=layers, kv=kv, dh=dh, longest=_log(rng, 65, table * PAGE), table=table)
        n = _log(rng, 1, 30)
        return dict(family=family, pages=_log(rng, 40, 450), used=round(rng.uniform(0.1, 0.9), 2), n=n, layers=layers, kv=kv, dh=dh, table=table)
    if family == "shared":
        h, kv, dh = rng.choice([GPT2, LLAMA_1B, LLAMA_7B, LLAMA_70B, (6, 2, 32), (10, 5, 64), (21, 3, 128)])
        rows = rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 9, 60)])
        groups = rng.choice([1, 1, 2, 3, _log(rng, 4, 12)])
        members = _log(rng, 1, max(2, min(64, 250 // (groups * rows))))
        prefix = _log(rng, 50, max(100, min(20000, 30_000_000 // (groups * members * rows * h * dh // 64), 20_000_000 // (groups * kv * dh))))
        tail = _log(rng, 10, max(20, min(1500, 20_000_000 // (groups * members * kv * dh))))
        return dict(family=family, h=h, kv=kv, dh=dh, groups=groups, members=members, prefix=prefix, tail=max(tail, rows), rows=rows, shape=rng.randint(10, 1 << 20))
    vocab, drafts = rng.choice([50257, 32000, _log(rng, 1000, 130000)]), rng.choice([0, 1, 2, 4, 5, 7, 12])
    return dict(family=family, n=_log(rng, 1, max(1, min(64, 40_000_000 // (vocab * (drafts + 1))))), drafts=drafts, vocab=vocab)


# ---------------------------------------------------------------------------------------------------------------------
# the format of the cache, with torch


def _head_bytes(dh):
    return PAGE * dh // 2 + PAGE * (dh // 32) * 2


def _shared_workspace_bytes(rows, h, dh):  # what cthip_sdpa_shared_paged_q4_workspace says
    return 4 * (4096 + 131072 * (dh + 2) + 2 * rows * h)


def _compact_workspace_bytes(n_pages):  # what cthip_kv_compact_paged_q4_workspace says
    return 64 + 8 * n_pages


def _verify_workspace_bytes(n):  # what cthip_draft_verify_workspace says
    return 2048 * n


def _quantise(x):
    """Rows (..., dh) -> (numbers -8 .. 7 (..., dh) as int8, scales (..., dh / 32) as fp16)."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    hi, lo = b.amax(-1), b.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) / -8.0).half()
    q = torch.floor(b / d.float().unsqueeze(-1) + 8.5).clamp(0, 15) - 8
    return q.to(torch.int8).reshape(x.shape), d


def _bytes_of(lo, hi):
    return (lo.to(torch.uint8) & 15) | ((hi.to(torch.uint8) & 15) << 4)


def _page_bytes(q, d, keys):
    """(..., 64, dh) numbers and (..., 64, dh / 32) scales of whole pages -> (..., bytes of a head's part of a page)."""
    lead, dh = q.shape[:-2], q.shape[-1]
    nb = dh // 32
    if keys:  # row, block, group, half, 4
        t = q.reshape(*lead, 64, nb, 4, 2, 4)
        quants = _bytes_of(t[..., 0, :], t[..., 1, :]).transpose(-3, -2)
    else:  # s, g, i, block, half, 16 -> block, channel, g, s, i
        t = q.reshape(*lead, 4, 4, 4, nb, 2, 16)
        k = len(lead)
        quants = _bytes_of(t[..., 0, :], t[..., 1, :]).permute(*range(k), k + 3, k + 4, k + 1, k, k + 2)
    scales = d.reshape(*lead, 16, 4, nb).transpose(-1, -2).contiguous().view(torch.uint8)
    return torch.cat([quants.reshape(*lead, -1), scales.reshape(*lead, -1)], -1)


def _page_values(pages, dh, keys):
    """(..., bytes of a head's part of a page) -> (..., 64, dh) in fp32."""
    lead, nb = pages.shape[:-1], dh // 32
    quants, scales = pages[..., : 32 * dh], pages[..., 32 * dh:]
    both = torch.stack([((quants & 15) ^ 8).to(torch.int8) - 8, ((quants >> 4) ^ 8).to(torch.int8) - 8], -1).float()
    k = len(lead)
    if keys:  # row, group, block, 4, half -> row, block, group, half, 4
        t = both.reshape(*lead, 64, 4, nb, 4, 2).permute(*range(k), k, k + 2, k + 1, k + 4, k + 3)
    else:  # block, channel, g, s, i, half -> s, g, i, block, half, channel
        t = both.reshape(*lead, nb, 16, 4, 4, 4, 2).permute(*range(k), k + 3, k + 2, k + 4, k, k + 5, k + 1)
    d = scales.contiguous().view(torch.float16).reshape(*lead, 16, nb, 4).transpose(-1, -2).reshape(*lead, 64, nb, 1).float()
    return (t.reshape(*lead, 64, nb, 32) * d).reshape(*lead, 64, dh)


def _random_pool(g, n_pages, kv, dh, keys):
    """Pages of rows as a model's projections give them: channels of different sizes, keys with some that stand out."""
    out = torch.empty(n_pages, kv, _head_bytes(dh), dtype=torch.uint8, device="cuda")
    spread = torch.exp(0.5 * torch.randn(kv, 1, dh, generator=g, device="cuda"))
    offset = 0.5 * torch.randn(kv, 1, dh, generator=g, device="cuda") * (1.0 if keys else 0.0)
    step = max(1, (1 << 25) // (kv * 64 * dh))
    for first in range(0, n_pages, step):
        count = min(step, n_pages - first)
        rows = torch.randn(count, kv, 64, dh, generator=g, device="cuda").mul_(spread * 0.7).add_(offset)
        out[first:first + count] = _page_bytes(*_quantise(rows), keys)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# inputs


def _groups(case):
    """Of a case of shared prefixes, by the case alone: (the group's prefix, [(rows of the cache, query rows) of each sequence])."""
    r, out = random.Random(case["shape"]), []
    for i in range(case["groups"]):
        prefix = case["prefix"] if i == 0 else _log(r, max(1, case["prefix"] // 3), case["prefix"])
        members = case["members"] if i == 0 else _log(r, 1, case["members"])
        seqs = []
        for j in range(members):
            rows = case["rows"] if r.random() < 0.7 or j == 0 else r.randint(1, case["rows"])
            seqs.append((prefix + max(rows, case["tail"] if j == 0 else _log(r, 1, case["tail"])), 0 if j % 9 == 8 else rows))  # (every ninth sits this step out)
        out.append((prefix, seqs))
    return out


def _drafts(case):
    """Drafted tokens of each sequence, by the case alone."""
    r, most = random.Random(case["vocab"] + case["n"]), case["drafts"]
    return [most if i == 0 else r.choice([most, most, r.randint(0, most)]) for i in range(case["n"])]


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _empty(*shape, dtype=torch.int32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def _frequencies(case):
    """Angles a position of each pair of channels; scaled by parts: pairs that turn less than once over a trained length of 8192 by the factor,
    those that turn more than four times not at all."""
    f = 10000.0 ** (-np.arange(case["rotary"] // 2, dtype=np.float64) * 2 / case["rotary"])
    turns = 8192 * f / (2 * math.pi)
    keep = np.clip((turns - 1.0) / 3.0, 0.0, 1.0)
    return f * (keep + (1 - keep) / case["factor"])


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    r = random.Random(seed)
    s = dict(case)
    family = case["family"]
    if family == "rope":
        rows, h, kv, dh = (case[x] for x in ("rows", "h", "kv", "dh"))
        width = (h + 2 * kv) * dh  # a row of the fused product: q, then k, then v
        fused = torch.randn(rows, width, generator=g, device="cuda").mul_(torch.exp(0.5 * torch.randn(width, generator=g, device="cuda")))
        position = [] if rows > 64 else [r.randrange(case["longest"]) for _ in range(rows)]  # a decode step, or pieces of prompts
        while len(position) < rows:
            first, n = r.randrange(case["longest"]), r.randint(1, 1500)
            position += list(range(first, first + n))
        return dict(s, fused=fused, width=width, q=fused[:, : h * dh], k=fused[:, h * dh:][:, : kv * dh], positions=_i32(position[:rows]),
                    frequencies=torch.from_numpy(_frequencies(case)).cuda(), magnitude=1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0,
                    q_out=_empty(rows, h * dh, dtype=torch.float32), k_out=_empty(rows, kv * dh, dtype=torch.float32))
    if family == "fork":
        p, f, layers, kv, dh, table = (case[x] for x in ("parents", "forks", "layers", "kv", "dh", "table"))
        n = p + f  # the parents, then what they are forked into
        lens = [_log(r, 1, case["longest"]) for _ in range(p)]
        have = [-(-v // PAGE) for v in lens]
        n_pages = p * -(-case["longest"] // PAGE) + f + 5
        pages = list(range(n_pages))
        r.shuffle(pages)
        tables = np.full((n, table), -1, np.int32)
        for i, c in enumerate(have):
            tables[i, :c] = [pages.pop() for _ in range(c)]
        parents = [j * p // f for j in range(f)]
        at = [r.choice([lens[i], lens[i], lens[i], r.randint(0, lens[i])]) for i in parents]  # most from where the parent ends
        pool = [torch.randint(0, 256, (layers, n_pages, kv, _head_bytes(dh)), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
        return dict(s, n=n, n_pages=n_pages, tables=torch.from_numpy(tables).cuda(), lens=_i32(lens + [0] * f), parents=_i32(parents), children=_i32(r.sample(range(p, n), f)),
                    at=_i32(at), free=_i32(pages), n_free=_i32([len(pages)]), k_pages=pool[0], v_pages=pool[1], n_free_out=_empty(1), refused=_empty(f))
    if family == "compact":
        n_pages, n, layers, kv, dh, table = (case[x] for x in ("pages", "n", "layers", "kv", "dh", "table"))
        ids = r.sample(range(n_pages), max(1, int(n_pages * case["used"])))
        shared = [ids.pop() for _ in range(min(3, len(ids) - 1))]  # the pages of a prompt that all begin with
        lens, tables = [], np.full((n, table), -1, np.int32)
        for i in range(n):
            c = min(table - len(shared), len(ids), -(-len(ids) // (n - i)))
            tables[i, :len(shared) + c] = shared + [ids.pop() for _ in range(c)]
            lens.append((len(shared) + c) * PAGE - r.randrange(PAGE))
        pool = [torch.randint(0, 256, (layers, n_pages, kv, _head_bytes(dh)), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
        return dict(s, lens=_i32([max(v, 0) for v in lens]), tables=torch.from_numpy(tables).cuda(), k_pages=pool[0], v_pages=pool[1], tables_out=_empty(n, table), free=_empty(n_pages),
                    n_free=_empty(1), workspace=torch.zeros(_compact_workspace_bytes(n_pages) // 4, dtype=torch.int32, device="cuda"))
    if family == "shared":
        h, kv, dh = case["h"], case["kv"], case["dh"]
        groups = _groups(case)
        seqs = [t for _, m in groups for t in m]
        lens, rows = [t for t, _ in seqs], [q for _, q in seqs]
        stride = -(-max(lens) // PAGE)
        pages = list(range(sum(p // PAGE + sum(-(-t // PAGE) - p // PAGE for t, _ in m) for p, m in groups) + 3))
        n_pages = len(pages)
        r.shuffle(pages)
        tables, i = np.full((len(seqs), stride), -1, np.int32), 0
        for p, m in groups:
            first = [pages.pop() for _ in range(p // PAGE)]  # a page that the prompt does not fill is each sequence's own
            for t, _ in m:
                tables[i, : -(-t // PAGE)] = first + [pages.pop() for _ in range(-(-t // PAGE) - p // PAGE)]
                i += 1
        total = sum(rows)
        q = torch.randn(total, (h + 2 * kv) * dh, generator=g, device="cuda")[:, : h * dh]  # the first part of the fused rows
        cuts = np.concatenate([[0], np.cumsum([len(m) for _, m in groups])]).tolist()
        return dict(s, q=q, q_stride=(h + 2 * kv) * dh, tables=torch.from_numpy(tables).cuda(), stride=stride, n_pages=n_pages, total=total, n=len(seqs), lens=_i32(lens),
                    starts=_i32(np.concatenate([[0], np.cumsum(rows)]).tolist()), most=max(rows), cuts=_i32(cuts), prefixes=_i32([p for p, _ in groups]),
                    most_pages=max(p for p, _ in groups) // PAGE, most_tail=max(-(-t // PAGE) - p // PAGE for p, m in groups for t, _ in m),
                    most_group=max(sum(q for _, q in m) for _, m in groups),
                    k_pages=_random_pool(g, n_pages, kv, dh, True), v_pages=_random_pool(g, n_pages, kv, dh, False), out=_empty(total, h * dh, dtype=torch.float32),
                    workspace=torch.zeros(_shared_workspace_bytes(total, h, dh) // 4, dtype=torch.int32, device="cuda"))
    n, vocab = case["n"], case["vocab"]
    drafts = _drafts(case)
    starts = np.concatenate([[0], np.cumsum([d + 1 for d in drafts])])
    rows = int(starts[-1])
    # a draft model that is near the target, each token drawn from the draft's probabilities
    logits = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.5)
    draft = torch.softmax(logits, -1)
    target = torch.softmax(logits.add_(torch.randn(rows, vocab, generator=g, device="cuda").mul_(0.7)), -1)
    tokens = torch.cat([torch.zeros(1, 1, dtype=torch.int64, device="cuda"), torch.multinomial(draft, 1, generator=g)])[:rows].view(-1).int()  # row j + 1's was drawn from row j
    lens = [d + 1 + r.randint(0, 2000) for d in drafts]
    return dict(s, rows=rows, target=target, draft=draft, tokens=tokens, uniforms=torch.rand(rows, generator=g, device="cuda"), starts=_i32(starts.tolist()), lens=_i32(lens),
                positions=_i32([t - d - 1 + j for t, d in zip(lens, drafts) for j in range(d + 1)]), most=max(drafts), tokens_out=_empty(rows), accepted=_empty(n), lens_out=_empty(n),
                workspace=torch.zeros(_verify_workspace_bytes(n) // 4, dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------------------------------------------------------------
# the operators with elementary torch operations


def _rope(s):
    angle = s["positions"].double().unsqueeze(1) * s["frequencies"]
    cos, sin = (torch.cos(angle) * s["magnitude"]).float().unsqueeze(1), (torch.sin(angle) * s["magnitude"]).float().unsqueeze(1)

    def turned(x, heads):
        x = x.reshape(s["rows"], heads, s["dh"])
        part, rest = x[..., : s["rotary"]], x[..., s["rotary"]:]
        if s["halves"]:
            a, b = part.chunk(2, -1)
            return torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1).view(s["rows"], -1)
        a, b = part[..., 0::2], part[..., 1::2]
        return torch.cat([torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2), rest], -1).view(s["rows"], -1)

    return [turned(s["q"], s["h"]), turned(s["k"], s["kv"])]


def _fork(s):
    n, table = s["n"], s["table"]
    parent, child, at, n_free = s["parents"].long(), s["children"].long(), s["at"].long(), s["n_free"].long()
    f = torch.arange(parent.numel(), device="cuda")
    ok = (parent >= 0) & (parent < n) & (child >= 0) & (child < n)
    p, c = parent.clamp(0, n - 1), child.clamp(0, n - 1)
    again = ((child.unsqueeze(1) == child) & (f.unsqueeze(0) < f.unsqueeze(1))).any(1)
    ok = ok & (at >= 0) & (at <= s["lens"][p]) & ~(child.unsqueeze(1) == parent).any(1) & ~again
    need = ok & (at % PAGE > 0)
    taken = need.long().cumsum(0)
    ok = ok & (~need | (taken <= n_free))
    page = s["free"][(n_free - taken).clamp(0, s["free"].numel() - 1)]
    full = (at // PAGE).unsqueeze(1)
    column = torch.arange(table, device="cuda")
    rows = torch.where(column < full, s["tables"][p], torch.where((column == full) & need.unsqueeze(1), page.unsqueeze(1), s["tables"][c]))
    do = torch.nonzero(ok).view(-1)
    tables, lens = s["tables"].clone(), s["lens"].clone()
    tables[c[do]] = rows[do]
    lens[c[do]] = at[do].int()
    do = torch.nonzero(ok & need).view(-1)
    src, dst = s["tables"][p[do], full[do, 0]].long(), page[do].long()
    for name in ("k_pages", "v_pages"):
        s[name][:, dst] = s[name][:, src]
    return dict(tables=tables, lens=lens, n_free=(n_free - (ok & need).sum()).int(), refused=(~ok).int(), k_pages=s["k_pages"], v_pages=s["v_pages"])


def _compact(s):
    n_pages, lens = s["pages"], s["lens"].long()
    there = torch.arange(s["table"], device="cuda") < ((lens + PAGE - 1) // PAGE).unsqueeze(1)
    there = there & (s["tables"] >= 0) & (s["tables"] < n_pages)
    used = torch.zeros(n_pages, dtype=torch.bool, device="cuda")
    used[s["tables"][there].long()] = True
    count = used.sum()
    page = torch.arange(n_pages, device="cuda")
    src, dst = torch.nonzero(used & (page >= count)).view(-1), torch.nonzero(~used & (page < count)).view(-1)
    to = page.clone()
    to[src] = dst
    tables = torch.where(there, to[s["tables"].long().clamp(0, n_pages - 1)].int(), s["tables"])
    for name in ("k_pages", "v_pages"):
        s[name][:, dst] = s[name][:, src]
    free = torch.where(page < n_pages - count, n_pages - 1 - page, torch.full_like(page, -1)).int()
    return dict(tables=tables, free=free, n_free=(n_pages - count).int().view(1), k_pages=s["k_pages"], v_pages=s["v_pages"])


def _shared(s):
    h, kv, dh, n, most, stride = s["h"], s["kv"], s["dh"], s["n"], s["most"], s["stride"]
    lens, starts, cuts = s["lens"].long(), s["starts"].long(), s["cuts"].long()
    rows, groups = starts[1:] - starts[:-1], cuts.numel() - 1
    group = torch.searchsorted(cuts, torch.arange(n, device="cuda"), right=True) - 1
    pages = (s["prefixes"].long() // PAGE)
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1

    def weighed(slots, first, q_at, seen):
        """Query rows q_at (b, m) against the rows of the pages (b, p); seen(key) -> whether: maxima, sums, sums of values."""
        k, v = (_page_values(s[name][slots.clamp(min=0)], dh, keys).transpose(1, 2).reshape(slots.shape[0], kv, -1, dh) for name, keys in (("k_pages", True), ("v_pages", False)))
        b, m = q_at.shape
        q = s["q"][q_at.clamp(0, s["total"] - 1)].reshape(b, m, kv, h // kv, dh).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, dh)
        score = (q @ k.transpose(-1, -2) / math.sqrt(dh)).view(b, kv, h // kv, m, -1)
        key = first.view(-1, 1, 1) + torch.arange(k.shape[2], device="cuda")
        score = score.masked_fill(~seen(key).view(b, 1, 1, m, -1), -math.inf)
        top = score.amax(-1, keepdim=True)
        p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
        o = (p.reshape(b, kv, -1, p.shape[-1]) @ v).view(b, kv, h // kv, m, dh)
        return [x.permute(0, 3, 1, 2, 4).reshape(b * m, h, -1) for x in (top, p.sum(-1, keepdim=True), o)]

    # the shared pages, a group's rows together
    page = torch.arange(max(s["most_pages"], 1), device="cuda")
    g_rows = starts[cuts[1:]] - starts[cuts[:-1]]
    slot = torch.arange(s["most_group"], device="cuda")
    a = weighed(s["tables"].long()[cuts[:-1]][:, : page.numel()], torch.zeros_like(pages), starts[cuts[:-1]].unsqueeze(1) + slot,
                lambda key: (key < (pages * PAGE).view(-1, 1, 1)) & (slot < g_rows.unsqueeze(1)).unsqueeze(-1))
    # what each sequence has behind them
    skip = pages[group]
    page = skip.unsqueeze(1) + torch.arange(s["most_tail"], device="cuda")
    slot_own = torch.arange(most, device="cuda")
    position = (lens - rows).unsqueeze(1) + slot_own
    b = weighed(s["tables"].long().gather(1, page.clamp(max=stride - 1)), skip * PAGE, starts[:-1].unsqueeze(1) + slot_own,
                lambda key: (key <= position.unsqueeze(-1)) & (slot_own < rows.unsqueeze(1)).unsqueeze(-1))
    at_a, at_b = group[seq] * s["most_group"] + row - starts[cuts[group[seq]]], seq * most + row - starts[seq]
    (m1, l1, o1), (m2, l2, o2) = [x[at_a] for x in a], [x[at_b] for x in b]
    top = torch.maximum(m1, m2)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    w1, w2 = torch.exp(m1 - top), torch.exp(m2 - top)
    total = w1 * l1 + w2 * l2
    return torch.where(total > 0, (w1 * o1 + w2 * o2) / total, torch.zeros_like(o1)).view(s["total"], h * dh)


def _verify(s):
    n, most, rows, vocab = s["n"], s["most"], s["rows"], s["vocab"]
    starts, lens = s["starts"].long(), s["lens"].long()
    drafts = starts[1:] - starts[:-1] - 1
    slot = torch.arange(most + 1, device="cuda")
    at = (starts[:-1].unsqueeze(1) + slot).clamp(max=rows - 1)  # row of target and draft that slot's draft is held against
    token = s["tokens"].long()[(at + 1).clamp(max=rows - 1)]
    p, q = s["target"][at, token].double(), s["draft"][at, token].double()
    good = (s["uniforms"][at].double() * q < p) & (slot < drafts.unsqueeze(1))
    accepted = good.long().cumprod(1).sum(1)
    last = starts[:-1] + accepted
    p, q = s["target"][last].double(), s["draft"][last].double()
    w = torch.where((accepted < drafts).unsqueeze(1), (p - q).clamp(min=0), p)
    w = torch.where((w.sum(1, keepdim=True) > 0), w, p)
    total = w.cumsum(1)
    drawn = (total <= s["uniforms"][starts[1:] - 1].double().unsqueeze(1) * total[:, -1:]).sum(1)
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    j = row - starts[seq]
    kept = s["tokens"].long()[(row + 1).clamp(max=rows - 1)]
    out = torch.where(j < accepted[seq], kept, torch.where(j == accepted[seq], drawn[seq], torch.full_like(row, -1)))
    return dict(tokens=out.int(), accepted=accepted.int(), lens=(lens - (drafts - accepted)).int())


# ---------------------------------------------------------------------------------------------------------------------
# one pass


def _own(s):
    from caten_amd import _lib

    lib, check, p = _lib.init(), _lib.check, {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if s["family"] == "rope":
        check(lib.cthip_rope_rows(p["q_out"], s["h"] * s["dh"], p["k_out"], s["kv"] * s["dh"], p["q"], s["width"], p["k"], s["width"], p["positions"], s["rows"], s["h"], s["kv"], s["dh"],
                                  s["rotary"], s["halves"], p["frequencies"], s["magnitude"]))
        return [s["q_out"], s["k_out"]]
    if s["family"] == "fork":
        check(lib.cthip_kv_fork_paged_q4(p["tables"], s["table"], p["lens"], s["n"], p["n_free_out"], p["refused"], p["k_pages"], p["v_pages"], s["layers"], s["n_pages"], p["parents"],
                                         p["children"], p["at"], s["forks"], p["free"], p["n_free"], s["kv"], s["dh"]))
        return dict(tables=s["tables"], lens=s["lens"], n_free=s["n_free_out"], refused=s["refused"], k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["family"] == "compact":
        check(lib.cthip_kv_compact_paged_q4(p["tables_out"], p["free"], p["n_free"], p["k_pages"], p["v_pages"], s["layers"], s["pages"], p["tables"], s["table"], p["lens"], s["n"],
                                            s["kv"], s["dh"], p["workspace"]))
        return dict(tables=s["tables_out"], free=s["free"], n_free=s["n_free"], k_pages=s["k_pages"], v_pages=s["v_pages"])
    if s["family"] == "shared":
        check(lib.cthip_sdpa_shared_paged_q4(p["out"], p["q"], s["q_stride"], p["k_pages"], p["v_pages"], s["n_pages"], p["tables"], s["stride"], p["lens"], p["starts"], s["n"], s["total"],
                                             p["cuts"], p["prefixes"], s["groups"], s["h"], s["kv"], s["dh"], p["workspace"]))
        return s["out"]
    check(lib.cthip_draft_verify(p["tokens_out"], p["accepted"], p["lens_out"], p["target"], s["vocab"], p["draft"], s["vocab"], p["tokens"], p["uniforms"], p["starts"], p["positions"],
                                 p["lens"], s["n"], s["rows"], s["vocab"], p["workspace"]))
    return dict(tokens=s["tokens_out"], accepted=s["accepted"], lens=s["lens_out"])


def run(state):
    if own:
        return _own(state)
    return {"rope": _rope, "fork": _fork, "compact": _compact, "shared": _shared, "verify": _verify}[state["family"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    if case["family"] == "rope":
        size = float(case["rows"] * (case["h"] + case["kv"]) * case["dh"])
        return {"bytes": 8.0 * size + 4.0 * case["rows"] + 4.0 * case["rotary"], "flops": 3.0 * size * case["rotary"] / case["dh"]}
    if case["family"] == "fork":  # nearly every child copies a page of keys and one of values a layer
        page = case["kv"] * _head_bytes(case["dh"])
        return {"bytes": case["forks"] * (4.0 * case["layers"] * page + 4.0 * case["longest"] / PAGE), "flops": 0.0}
    if case["family"] == "compact":  # of the pages in use, those that lie behind their number
        page = case["kv"] * _head_bytes(case["dh"])
        return {"bytes": 4.0 * case["layers"] * page * case["pages"] * case["used"] * (1 - case["used"]) + 8.0 * case["n"] * case["table"] + 4.0 * case["pages"], "flops": 0.0}
    if case["family"] == "shared":
        keys, pairs, rows = 0, 0.0, 0
        for p, m in _groups(case):
            keys += p // PAGE * PAGE + sum(t - p // PAGE * PAGE for t, _ in m)
            pairs += sum(q * (t - q) + q * (q + 1) / 2 for t, q in m)
            rows += sum(q for _, q in m)
        return {"bytes": 2 * 9 / 16 * case["kv"] * case["dh"] * keys + 8.0 * rows * case["h"] * case["dh"], "flops": 4.0 * case["h"] * case["dh"] * pairs}
    # the row that a token is drawn from, of target and, behind a rejection, of draft
    return {"bytes": case["n"] * (8.0 if case["drafts"] else 4.0) * case["vocab"] + 40.0 * (sum(_drafts(case)) + case["n"]), "flops": 3.0 * case["n"] * case["vocab"]}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits


def _exact_pages(pages, dh, keys):
    """(m, kv, bytes) -> (m * 64, kv, dh): every value from its own byte and its own scale."""
    row, ch = torch.arange(64, device="cuda").view(-1, 1), torch.arange(dh, device="cuda").view(1, -1)
    block, inner = ch // 32, ch % 32
    if keys:
        byte, high = row * (dh // 2) + (inner // 8) * (dh // 8) + block * 4 + inner % 4, (inner % 8) >= 4
    else:
        byte, high = (block * 16 + inner % 16) * 64 + (row % 16) // 4 * 16 + row // 16 * 4 + row % 4, inner >= 16
    number = pages[:, :, byte.reshape(-1)].to(torch.int16)
    number = torch.where((high | (byte < 0)).reshape(-1), number >> 4, number & 15)
    number = torch.where(number >= 8, number - 16, number).double()
    at = 32 * dh + 2 * ((row // 4 * (dh // 32) + block) * 4 + row % 4).reshape(-1)
    bits = pages[:, :, at].to(torch.int32) | (pages[:, :, at + 1].to(torch.int32) << 8)
    return (number * bits.to(torch.int16).view(torch.float16).double()).view(-1, pages.shape[1], 64, dh).transpose(1, 2).reshape(-1, pages.shape[1], dh)


def exact(case, seed):
    if case["family"] not in ("rope", "shared"):
        return None  # whole numbers and bytes are held to the plain form's
    s = prepare(case, seed)
    if case["family"] == "rope":
        half, out = case["rotary"] // 2, []
        at = torch.arange(half, device="cuda")
        first, second = (at, at + half) if case["halves"] else (2 * at, 2 * at + 1)
        turn = torch.polar(torch.full((), s["magnitude"], dtype=torch.float64, device="cuda"), s["positions"].double().view(-1, 1, 1) * s["frequencies"].view(1, 1, -1))
        for x, heads in ((s["q"], case["h"]), (s["k"], case["kv"])):
            y = x.double().reshape(case["rows"], heads, case["dh"]).clone()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y[..., first], y[..., second] = z.real, z.imag
            out.append(y.view(case["rows"], -1))
        return out
    h, kv, dh = case["h"], case["kv"], case["dh"]
    lens, starts = s["lens"].tolist(), s["starts"].tolist()
    out = torch.zeros(s["total"], kv, h // kv, dh, dtype=torch.float64, device="cuda")
    for i, t in enumerate(lens):  # each sequence by its own table alone
        r0, r1 = starts[i], starts[i + 1]
        if r1 == r0:
            continue
        pages = s["tables"][i, : -(-t // PAGE)].long()
        k, v = _exact_pages(s["k_pages"][pages], dh, True)[:t], _exact_pages(s["v_pages"][pages], dh, False)[:t]
        hidden = torch.arange(t, device="cuda") > torch.arange(t - (r1 - r0), t, device="cuda").view(-1, 1)
        q = s["q"][r0:r1].double().view(-1, kv, h // kv, dh)
        for j in range(kv):
            w = torch.softmax((q[:, j].transpose(0, 1) @ k[:, j].T.contiguous() * dh ** -0.5).masked_fill(hidden, -math.inf), -1)
            out[r0:r1, j] = (w @ v[:, j].contiguous()).transpose(0, 1)
    return out.view(s["total"], -1)

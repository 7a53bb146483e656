"""Batched serving and beam search over a paged KV cache held in 4 bits: the operators of one step, as cases that can be timed.

plan      block tables and slot maps from the requests' lengths
append    key and value rows into the cache by their slots, and what the cache then holds of them
attention a ragged batch of query rows over the cache
select    the next beams out of beams x vocabulary
reorder   block tables, partly filled pages and token histories follow the beams

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
        # a small server's decode step: 64 sequences, each with one new token; bound by latency
        dict(name="plan decode 64", family="plan", n=64, new=1, longest=2048, table=32),
        # a full server taking up prompts: ragged pieces, some sequences with nothing new
        dict(name="plan prompts 500", family="plan", n=500, new=300, longest=7000, table=128),
        # the rows of a decode step, slices of a fused q/k/v product: GPT-2 heads, 48 sequences
        dict(name="append gpt2 48 rows", family="append", rows=48, kv=12, dh=64, q_heads=12, n=48),
        # the rows of prompts, eight heads of 128 (a 70B shape)
        dict(name="append 70b 6001 rows", family="append", rows=6001, kv=8, dh=128, q_heads=64, n=7),
        # one conversation with GPT-2 small: the smallest attention there is
        dict(name="attention gpt2 one 701", family="attention", h=12, kv=12, dh=64, n=1, lo=701, hi=701, rows=1, shape=1),
        # a server's decode step over conversations of very different lengths, some slots idle (70B shape)
        dict(name="attention 70b ragged 32", family="attention", h=64, kv=8, dh=128, n=32, lo=150, hi=20000, rows=1, shape=2),
        # keys and values for every head (7B shape), eight conversations
        dict(name="attention 7b batch 8", family="attention", h=32, kv=32, dh=128, n=8, lo=1500, hi=5000, rows=1, shape=3),
        # pieces of prompts behind what is cached, next to sequences that decode (1.1B shape)
        dict(name="attention 1.1b prompts", family="attention", h=32, kv=4, dh=64, n=5, lo=900, hi=3500, rows=700, shape=4),
        # beam search with GPT-2: four beams of one request
        dict(name="select gpt2 1x4", family="select", n=1, beams=4, vocab=50257, done=0),
        # beam search as a service: 48 requests with eight beams, some of them finished
        dict(name="select llama 48x8", family="select", n=48, beams=8, vocab=32000, done=1),
        # the four beams of one request, 12 layers of GPT-2
        dict(name="reorder gpt2 1x4", family="reorder", n=1, beams=4, layers=12, kv=12, dh=64, longest=900, table=16),
        # 24 requests with six beams, 22 layers (1.1B shape)
        dict(name="reorder 1.1b 24x6", family="reorder", n=24, beams=6, layers=22, kv=4, dh=64, longest=2000, table=32),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["plan", "append", "attention", "attention", "attention", "select", "reorder"])
    if family == "plan":
        n, table = _log(rng, 1, 600), rng.choice([16, 32, 128, 160])
        return dict(family=family, n=n, new=rng.choice([1, 1, _log(rng, 2, 300)]), longest=_log(rng, 200, table * PAGE - 1000), table=table)
    if family == "append":
        h, kv, dh = rng.choice([GPT2, LLAMA_1B, LLAMA_7B, LLAMA_70B, (5, 5, 32)])
        n = _log(rng, 1, 64)
        return dict(family=family, rows=_log(rng, n, min(6000, 6000 * 1024 // (kv * dh))) if n < 64 else n, kv=kv, dh=dh, q_heads=h, n=n)
    if family == "attention":
        h, kv, dh = rng.choice([GPT2, LLAMA_1B, LLAMA_7B, LLAMA_70B, (6, 2, 32), (10, 5, 64), (21, 3, 128)])
        rows = rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 500)])
        most = 60_000_000 // (kv * dh) if rows == 1 else 8000 if rows < 10 else 2500  # rows of the cache, all sequences
        n = _log(rng, 1, min(64, most // 200))
        hi = _log(rng, 100, most // n)
        return dict(family=family, h=h, kv=kv, dh=dh, n=n, lo=max(1, int(hi * rng.uniform(0.05, 1.0))), hi=hi, rows=rows, shape=rng.randint(10, 1 << 20))
    if family == "select":
        beams, vocab = rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), rng.choice([50257, 32000, _log(rng, 1000, 130000)])
        return dict(family=family, n=_log(rng, 1, max(1, min(64, 12_000_000 // (beams * vocab)))), beams=beams, vocab=vocab, done=rng.choice([0, 1]))
    h, kv, dh = rng.choice([GPT2, LLAMA_1B, (32, 8, 128)])
    table = rng.choice([16, 32])
    return dict(family=family, n=_log(rng, 1, 12), beams=rng.choice([2, 3, 4, 5, 8]), layers=rng.randint(2, 12), kv=kv, dh=dh, longest=_log(rng, 65, table * PAGE), table=table)


# ---------------------------------------------------------------------------------------------------------------------
# the format of the cache, with torch


def _head_bytes(dh):
    return PAGE * dh // 2 + PAGE * (dh // 32) * 2


def _workspace_bytes(dh):  # what cthip_sdpa_paged_q4_workspace says
    return 4 * (2048 + 2048 * 16 * (dh + 2))


def _select_workspace_bytes(n, beams):  # what cthip_beam_select_workspace says
    return 256 + 4 * n + n * beams * 32 * (24 + 8 * beams)


def _quantise(x):
    """Rows (..., dh) -> (numbers -8 .. 7 (..., dh) as int8, scales (..., dh / 32) as fp16)."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    hi, lo = b.amax(-1), b.amin(-1)
    d = (torch.where(hi >= -lo, hi, lo) / -8.0).clamp(-65504.0, 65504.0).half()
    d = torch.where(torch.isfinite(b).all(-1), d, torch.full_like(d, math.nan))
    # in 64 bits: whether a value lies below a border between two levels is decided on the value itself
    q = torch.floor(b.double() / d.double().unsqueeze(-1) + 8.5).clamp(0, 15)
    q = torch.where((d != 0).unsqueeze(-1) & torch.isfinite(q), q, torch.full_like(q, 8.0)) - 8
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


def _lens(case):
    """Rows of the cache and query rows of each sequence of an attention case, by the case alone."""
    r, n = random.Random(case["shape"]), case["n"]
    lens = [case["hi"] if i == 0 else _log(r, case["lo"], case["hi"]) for i in range(n)]
    rows = [min(lens[i], case["rows"] if i == 0 or case["rows"] == 1 else r.choice([1, r.randint(1, case["rows"])])) for i in range(n)]
    for i in range(7, n, 8):  # idle slots
        lens[i], rows[i] = 0, 0
    return lens, rows


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _empty(*shape, dtype=torch.int32):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    r = random.Random(seed)
    s = dict(case)
    if case["family"] == "plan":
        n, table = case["n"], case["table"]
        cap = table * PAGE
        lens = [min(cap, _log(r, 1, case["longest"])) for _ in range(n)]
        new = [1 if case["new"] == 1 else r.choice([0, 1, r.randint(1, case["new"])]) for _ in range(n)]
        have = [-(-v // PAGE) for v in lens]
        want = sum(max(0, -(-(a + b) // PAGE) - h) for a, b, h in zip(lens, new, have))
        pages = list(range(sum(have) + want + 100))
        r.shuffle(pages)
        tables = np.full((n, table), -1, np.int32)
        for i, h in enumerate(have):
            tables[i, :h] = [pages.pop() for _ in range(h)]
        max_rows = n * case["new"]
        return dict(s, lens=_i32(lens), new_lens=_i32(new), free=_i32(pages), n_free=_i32([len(pages)]), tables=torch.from_numpy(tables).cuda(), max_rows=max_rows,
                    slots=_empty(max_rows), positions=_empty(max_rows), starts=_empty(n + 1), lens_out=_empty(n), n_free_out=_empty(1), refused=_empty(1))
    if case["family"] == "append":
        kv, dh, rows, n = case["kv"], case["dh"], case["rows"], case["n"]
        width = case["q_heads"] * dh + 2 * kv * dh  # a row of the fused product: q, then k, then v
        fused = torch.randn(rows, width, generator=g, device="cuda").mul_(torch.exp(0.5 * torch.randn(width, generator=g, device="cuda")))
        # the sequences' new rows, each behind what its sequence holds, in pages in any order
        cuts = sorted(r.sample(range(1, rows), n - 1)) if n > 1 else []
        counts = [b - a for a, b in zip([0] + cuts, cuts + [rows])]
        pages = list(range(sum(-(-c // PAGE) + 1 for c in counts) + 20))
        n_pages = len(pages)
        r.shuffle(pages)
        slots = []
        for c in counts:
            at = r.randrange(PAGE)
            mine = [pages.pop() for _ in range(-(-(at + c) // PAGE))]
            slots += [mine[(at + j) // PAGE] * PAGE + (at + j) % PAGE for j in range(c)]
        pool = [torch.zeros(n_pages, kv, _head_bytes(dh), dtype=torch.uint8, device="cuda") for _ in range(2)]
        return dict(s, fused=fused, width=width, k=fused[:, case["q_heads"] * dh:][:, : kv * dh], v=fused[:, (case["q_heads"] + kv) * dh:], slots=_i32(slots), n_pages=n_pages,
                    k_pages=pool[0], v_pages=pool[1], k_back=_empty(rows, kv * dh, dtype=torch.float32), v_back=_empty(rows, kv * dh, dtype=torch.float32))
    if case["family"] == "attention":
        lens, rows = _lens(case)
        h, kv, dh, n = case["h"], case["kv"], case["dh"], case["n"]
        stride = max(1, -(-max(lens) // PAGE))
        pages = list(range(sum(-(-v // PAGE) for v in lens) + 3))
        n_pages = len(pages)
        r.shuffle(pages)
        tables = np.full((n, stride), -1, np.int32)
        for i, v in enumerate(lens):
            c = -(-v // PAGE)
            tables[i, :c] = [pages.pop() for _ in range(c)]
        total = sum(rows)
        q = torch.randn(total, (h + 2 * kv) * dh, generator=g, device="cuda")[:, : h * dh]  # the first part of the fused rows
        return dict(s, q=q, q_stride=(h + 2 * kv) * dh, tables=torch.from_numpy(tables).cuda(), stride=stride, n_pages=n_pages, total=total,
                    lens=_i32(lens), starts=_i32(np.concatenate([[0], np.cumsum(rows)]).tolist()), most=max(rows),
                    k_pages=_random_pool(g, n_pages, kv, dh, True), v_pages=_random_pool(g, n_pages, kv, dh, False),
                    out=_empty(total, h * dh, dtype=torch.float32), workspace=torch.zeros(_workspace_bytes(dh) // 4, dtype=torch.int32, device="cuda"))
    if case["family"] == "select":
        n, k, v = case["n"], case["beams"], case["vocab"]
        logits = torch.randn(n * k, v, generator=g, device="cuda").mul_(2.5)
        logits[:, ::97] = -math.inf  # tokens that a program forbids
        scores = torch.rand(n, k, generator=g, device="cuda").mul_(-15.0).sort(1, descending=True).values.contiguous()
        done = (torch.rand(n, k, generator=g, device="cuda") < 0.15).int() if case["done"] else torch.zeros(n, k, dtype=torch.int32, device="cuda")
        return dict(s, logits=logits, scores=scores, finished=done, eos=v - 1, tokens=_empty(n, k), parents=_empty(n, k), scores_out=_empty(n, k, dtype=torch.float32),
                    finished_out=_empty(n, k), workspace=torch.zeros(_select_workspace_bytes(n, k) // 4, dtype=torch.int32, device="cuda"))
    n, k, layers, kv, dh, table = (case[x] for x in ("n", "beams", "layers", "kv", "dh", "table"))
    lens = [_log(r, 1, case["longest"]) for _ in range(n)]
    n_pages = n * (case["longest"] // PAGE + k)
    pages = list(range(n_pages))
    r.shuffle(pages)
    tables = np.full((n * k, table), -1, np.int32)
    for i, v in enumerate(lens):  # full pages belong to all beams, the last one to each
        tables[i * k:(i + 1) * k, : v // PAGE] = [pages.pop() for _ in range(v // PAGE)]
        if v % PAGE:
            tables[i * k:(i + 1) * k, v // PAGE] = [pages.pop() for _ in range(k)]
    parents = [[r.choice([j, r.randrange(k)]) for j in range(k)] for _ in range(n)]
    pool = [torch.randint(0, 256, (layers, n_pages, kv, _head_bytes(dh)), generator=g, device="cuda", dtype=torch.uint8) for _ in range(2)]
    cols = 200
    return dict(s, tables=torch.from_numpy(tables).cuda(), lens=_i32(lens), parents=_i32(parents), k_pages=pool[0], v_pages=pool[1], n_pages=n_pages, tables_out=_empty(n * k, table),
                cols=cols, step=_i32([r.randrange(cols)]), tokens=_i32([[r.randrange(32000) for _ in range(k)] for _ in range(n)]),
                history=torch.randint(0, 32000, (n * k, cols), generator=g, device="cuda", dtype=torch.int32), history_out=_empty(n * k, cols))


# ---------------------------------------------------------------------------------------------------------------------
# the operators with elementary torch operations


def _plan(s):
    cap, lens, new = s["table"] * PAGE, s["lens"].long(), s["new_lens"].long()
    starts = torch.cat([new.new_zeros(1), new.clamp(min=0).cumsum(0)])
    ok = (lens >= 0) & (new >= 0) & (lens + new <= cap) & (starts[1:] <= s["max_rows"])
    have = (lens + PAGE - 1) // PAGE
    need = torch.where(ok, (lens + new + PAGE - 1) // PAGE - have, torch.zeros_like(lens))
    total, n_free = need.cumsum(0), s["n_free"].long()
    ok = ok & ((need == 0) | (total <= n_free))
    column = torch.arange(s["table"], device="cuda").unsqueeze(0) - have.unsqueeze(1)
    at = (n_free - 1 - ((total - need).unsqueeze(1) + column)).clamp(0, s["free"].numel() - 1)
    tables = torch.where(ok.unsqueeze(1) & (column >= 0) & (column < need.unsqueeze(1)), s["free"][at], s["tables"])
    row = torch.arange(s["max_rows"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True).clamp(max=s["n"]) - 1
    pos = lens[seq] + row - starts[seq]
    there = ok[seq] & (row < starts[-1])
    page = tables[seq, (pos // PAGE).clamp(0, s["table"] - 1)]
    minus = torch.full_like(pos, -1)
    used = torch.where(ok, need, torch.zeros_like(need)).sum()
    return dict(slots=torch.where(there & (page >= 0), page * PAGE + pos % PAGE, minus).int(), positions=torch.where(there, pos, minus).int(), starts=starts.int(),
                tables=tables, lens=torch.where(ok, lens + new, lens).int(), n_free=(n_free - used).int(), refused=(~ok).sum().reshape(1).int())


def _append(s):
    kv, dh = s["kv"], s["dh"]
    slot = s["slots"].long()
    page, row = slot // PAGE, slot % PAGE
    # the places of a row's bytes in its page: those that a page numbered by row holds at this row
    place = torch.arange(64, device="cuda").view(64, 1)
    nb = dh // 32
    k_at = place * (dh // 2) + torch.arange(dh // 2, device="cuda")
    v_at = torch.arange(dh // 2, device="cuda") * 64 + (place // 4 % 4) * 16 + place // 16 * 4 + place % 4
    d_at = 32 * dh + ((place // 4 * nb + torch.arange(nb, device="cuda")).unsqueeze(-1) * 4 + (place % 4).unsqueeze(-1)) * 2 + torch.arange(2, device="cuda")
    back = []
    for name, at, keys in (("k", k_at, True), ("v", v_at, False)):
        q, d = _quantise(s[name].reshape(-1, kv, dh))
        t = q.reshape(-1, kv, nb, 4, 2, 4) if keys else q.reshape(-1, kv, nb, 2, 16)
        b = _bytes_of(t[..., 0, :], t[..., 1, :])
        b = (b.transpose(-3, -2) if keys else b).reshape(-1, kv, dh // 2)
        b = torch.cat([b, d.contiguous().view(torch.uint8).reshape(-1, kv, nb * 2)], -1)
        where = torch.cat([at[row], d_at[row].reshape(-1, nb * 2)], -1)
        s[name + "_pages"][page.view(-1, 1, 1), torch.arange(kv, device="cuda").view(1, -1, 1), where.unsqueeze(1)] = b
        back.append((q.float().reshape(-1, kv, nb, 32) * d.float().unsqueeze(-1)).reshape(-1, kv * dh))
    return back


def _attention(s):
    h, kv, dh, n, most = s["h"], s["kv"], s["dh"], s["n"], s["most"]
    lens, starts = s["lens"].long(), s["starts"].long()
    page = s["tables"].long().clamp(min=0)
    k, v = (_page_values(s[name][page], dh, keys).transpose(1, 2).reshape(n, kv, -1, dh) for name, keys in (("k_pages", True), ("v_pages", False)))
    rows = starts[1:] - starts[:-1]
    slot = torch.arange(most, device="cuda")
    at = (starts[:-1].unsqueeze(1) + slot).clamp(max=s["total"] - 1)
    q = s["q"][at].reshape(n, most, kv, h // kv, dh).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, dh)
    score = (q @ k.transpose(-1, -2) / math.sqrt(dh)).view(n, kv, h // kv, most, -1)
    pos = (lens - rows).unsqueeze(1) + slot  # of each query row
    seen = (torch.arange(k.shape[2], device="cuda") <= pos.unsqueeze(-1)) & (slot < rows.unsqueeze(1)).unsqueeze(-1)
    score = score.masked_fill(~seen.view(n, 1, 1, most, -1), -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    o = (p.reshape(n, kv, -1, p.shape[-1]) @ v).view(n, kv, h // kv, most, dh).permute(0, 3, 1, 2, 4).reshape(n * most, h * dh)
    row = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(starts, row, right=True) - 1
    return o[seq * most + row - starts[seq]]


def _select(s):
    n, k, v = s["n"], s["beams"], s["vocab"]
    x = s["logits"].double().view(n, k, v)
    top = x.amax(-1, keepdim=True)
    x = x - top
    score = s["scores"].double().unsqueeze(-1) + (x - torch.log(torch.exp(x).sum(-1, keepdim=True)))
    done = s["finished"].bool().unsqueeze(-1)
    ends = torch.arange(v, device="cuda") == s["eos"]
    score = torch.where(done, torch.where(ends, s["scores"].double().unsqueeze(-1), torch.full_like(score, -math.inf)), score).view(n, k * v)
    least = score.topk(k, dim=1).values[:, -1:]
    over, level = score > least, score == least
    kept = over | (level & (level.cumsum(1) <= k - over.sum(1, keepdim=True)))  # of equal ones the first
    first = torch.where(kept, k * v - torch.arange(k * v, device="cuda"), torch.zeros((), dtype=torch.int64, device="cuda")).topk(k, dim=1).values
    at = k * v - first  # rising
    best, order = score.gather(1, at).sort(dim=1, descending=True, stable=True)
    at = at.gather(1, order)
    parents, tokens = at // v, at % v
    return dict(tokens=tokens.int(), parents=parents.int(), scores=best.float(), finished=(s["finished"].gather(1, parents).bool() | (tokens == s["eos"])).int())


def _reorder(s):
    n, k = s["n"], s["beams"]
    child = torch.arange(k, device="cuda")
    base = torch.arange(n, device="cuda").unsqueeze(1) * k
    parent = s["parents"].long()
    lens = s["lens"].long()
    same = parent.unsqueeze(2) == parent.unsqueeze(1)  # [i, j]: children of one parent
    further = (same & (child.unsqueeze(0) < child.unsqueeze(1))).any(2)  # not the first of its parent
    dead = ~(parent.unsqueeze(1) == child.view(1, -1, 1)).any(2)
    rank = further.cumsum(1) - 1
    free = torch.where(dead, child, child + k).sort(1).values  # the dead beams, rising
    source = torch.where(further, free.gather(1, rank.clamp(min=0)).clamp(max=k - 1), parent)  # whose last page the child gets
    last = (lens // PAGE).unsqueeze(1).expand(n, k)
    column = torch.arange(s["table"], device="cuda").view(1, 1, -1)
    take = torch.where(column < last.unsqueeze(2), parent.unsqueeze(2), torch.where((column == last.unsqueeze(2)) & (lens % PAGE > 0).view(n, 1, 1), source.unsqueeze(2), child.view(1, k, 1)))
    tables = s["tables"].gather(0, (base.unsqueeze(2) + take).view(n * k, -1))
    at = last.clamp(max=s["table"] - 1).reshape(-1)
    from_page = s["tables"].long()[(base + parent).view(-1), at]
    to_page = tables.long()[torch.arange(n * k, device="cuda"), at]
    copies = torch.nonzero((further & (lens % PAGE > 0).unsqueeze(1)).view(-1)).view(-1)
    for name in ("k_pages", "v_pages"):
        s[name][:, to_page[copies]] = s[name][:, from_page[copies]]
    history = s["history"][(base + parent).view(-1)]
    history = torch.where(torch.arange(s["cols"], device="cuda") == s["step"], s["tokens"].view(-1, 1), history)
    return dict(tables=tables, history=history, k_pages=s["k_pages"], v_pages=s["v_pages"])


# ---------------------------------------------------------------------------------------------------------------------
# one pass


def _own(s):
    from caten_amd import _lib

    lib, check, p = _lib.init(), _lib.check, {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if s["family"] == "plan":
        check(lib.cthip_kv_plan_paged(p["slots"], p["positions"], p["starts"], p["tables"], s["table"], p["lens_out"], p["n_free_out"], p["refused"], p["lens"], p["new_lens"], s["n"],
                                      p["free"], p["n_free"], s["max_rows"]))
        return dict(slots=s["slots"], positions=s["positions"], starts=s["starts"], tables=s["tables"], lens=s["lens_out"], n_free=s["n_free_out"], refused=s["refused"])
    if s["family"] == "append":
        check(lib.cthip_kv_append_paged_q4(p["k_pages"], p["v_pages"], p["k"], p["v"], s["width"], s["width"], p["slots"], s["rows"], s["n_pages"], s["kv"], s["dh"]))
        check(lib.cthip_kv_rows_paged_q4(p["k_back"], p["v_back"], p["k_pages"], p["v_pages"], p["slots"], s["rows"], s["n_pages"], s["kv"], s["dh"]))
        return [s["k_back"], s["v_back"]]
    if s["family"] == "attention":
        check(lib.cthip_sdpa_paged_q4(p["out"], p["q"], s["q_stride"], p["k_pages"], p["v_pages"], s["n_pages"], p["tables"], s["stride"], p["lens"], p["starts"], s["n"], s["total"],
                                      s["h"], s["kv"], s["dh"], p["workspace"]))
        return s["out"]
    if s["family"] == "select":
        check(lib.cthip_beam_select(p["tokens"], p["parents"], p["scores_out"], p["finished_out"], p["logits"], s["vocab"], p["scores"], p["finished"], s["n"], s["beams"], s["vocab"], s["eos"],
                                    p["workspace"]))
        return dict(tokens=s["tokens"], parents=s["parents"], scores=s["scores_out"], finished=s["finished_out"])
    check(lib.cthip_beam_reorder_paged_q4(p["tables_out"], p["history_out"], p["k_pages"], p["v_pages"], s["layers"], s["n_pages"], p["tables"], s["table"], p["lens"], p["parents"],
                                          s["n"], s["beams"], s["kv"], s["dh"], p["history"], s["cols"], p["tokens"], p["step"]))
    return dict(tables=s["tables_out"], history=s["history_out"], k_pages=s["k_pages"], v_pages=s["v_pages"])


def run(state):
    if own:
        return _own(state)
    return {"plan": _plan, "append": _append, "attention": _attention, "select": _select, "reorder": _reorder}[state["family"]](state)


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    if case["family"] == "plan":
        rows = case["n"] * (1 if case["new"] == 1 else (1 + case["new"] / 2) / 3)
        return {"bytes": 8.0 * case["n"] * case["new"] + rows / 8 + 16.0 * case["n"], "flops": 0.0}
    if case["family"] == "append":  # rows in, packed rows out; packed rows in, values out
        size = 2.0 * case["rows"] * case["kv"] * case["dh"]
        return {"bytes": size * (8 + 2 * 9 / 16) + 8.0 * case["rows"], "flops": 4.0 * size}
    if case["family"] == "attention":
        lens, rows = _lens(case)
        pairs = sum(r * (t - r) + r * (r + 1) / 2 for t, r in zip(lens, rows))
        return {"bytes": 2 * 9 / 16 * case["kv"] * case["dh"] * sum(lens) + 8.0 * sum(rows) * case["h"] * case["dh"], "flops": 4.0 * case["h"] * case["dh"] * pairs}
    if case["family"] == "select":
        size = case["n"] * case["beams"]
        return {"bytes": 4.0 * size * case["vocab"] + 28.0 * size, "flops": 4.0 * size * case["vocab"]}
    size = case["n"] * case["beams"]
    # about two children in seven are copies, of two pages a layer
    return {"bytes": 8.0 * size * (case["table"] + 200) + size * 2 / 7 * 4 * case["layers"] * case["kv"] * _head_bytes(case["dh"]), "flops": 0.0}


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
    s = prepare(case, seed)
    if case["family"] == "append":
        out = []
        for name in "kv":
            x = s[name].double().reshape(-1, 32)
            m = x.gather(1, x.abs().argmax(1, keepdim=True))
            d = (m / -8).half().double()
            out.append((d * (torch.floor(x / torch.where(d == 0, torch.ones_like(d), d) + 8.5).clamp(0, 15) - 8)).view(case["rows"], -1))
        return out
    if case["family"] == "attention":
        h, kv, dh, scale = case["h"], case["kv"], case["dh"], case["dh"] ** -0.5
        lens, starts, out = s["lens"].tolist(), s["starts"].tolist(), torch.zeros(s["total"], h, dh, dtype=torch.float64, device="cuda")
        for i, t in enumerate(lens):
            r0, r1 = starts[i], starts[i + 1]
            if r1 == r0:
                continue
            pages = s["tables"][i, : -(-t // PAGE)].long()
            k, v = _exact_pages(s["k_pages"][pages], dh, True)[:t], _exact_pages(s["v_pages"][pages], dh, False)[:t]
            hidden = torch.arange(t, device="cuda") > torch.arange(t - (r1 - r0), t, device="cuda").view(-1, 1)
            q = s["q"][r0:r1].double().view(-1, h, dh)
            for j in range(h):
                w = torch.softmax((q[:, j] @ k[:, j // (h // kv)].T * scale).masked_fill(hidden, -math.inf), -1)
                out[r0:r1, j] = w @ v[:, j // (h // kv)]
        return out.view(s["total"], -1)
    if case["family"] == "select":
        n, k, v = case["n"], case["beams"], case["vocab"]
        lp = torch.log_softmax(s["logits"].double(), -1).view(n, k, v) + s["scores"].double().unsqueeze(-1)
        done = s["finished"].bool()
        lp[done] = -math.inf
        lp[..., s["eos"]] = torch.where(done, s["scores"].double(), lp[..., s["eos"]])
        # whole numbers are held to the plain form's
        return dict(tokens=None, parents=None, scores=lp.view(n, -1).topk(k, 1).values, finished=None)
    return None

"""Operators of a serving step over the paged K/V cache, as they are measured: their cases, plain forms and sizes.

What stands between a fused projection and the next token, for many sequences out of one pool of pages (include/gpu.h):

  gpu_paged_rotate_append     norms the queries and keys of each head, rotates them to their rows' places and writes the keys and values
                              to the pool, in one pass
  gpu_paged_bounds            keeps, for each page and KV head, the least and the largest value of every key element
  gpu_paged_sparse_attention  scores the pages of a sequence for each query by those bounds, takes the best `blocks` of them (a few
                              first and recent ones always) and attends to their rows alone
  gpu_sample                  draws each row's token from its logits with temperature, top-k, top-p and min-p, by a given random number

With `own` false, run() computes them by elementary torch operations, else by the library's kernels.
"""
import math
import random

import numpy as np
import torch

own = False

BF16, BYTES = 2, 3  # TcmPagedCache.kind
EPS = 1e-6


def _paged(name, op, kind, heads, page, seqs, new, length, norm=True, rotary=128, theta=1e6, blocks=0, first=0, recent=0, layout=1):
    """heads: (query heads, KV heads, head size); new, length: the smallest and largest of a sequence."""
    return {"name": name, "op": op, "kind": kind, "qheads": heads[0], "kvheads": heads[1], "dim": heads[2], "page": page,
            "seqs": seqs, "new_min": new[0], "new_max": new[1], "len_min": length[0], "len_max": length[1], "norm": norm,
            "rotary": rotary, "theta": theta, "blocks": blocks, "first": first, "recent": recent, "layout": layout}


def _sample(name, rows, vocab, mode, pad=0, coarse=False, layout=1):
    """pad: floats between rows; coarse: logits as a 16-bit readout leaves them, with many equal ones."""
    return {"name": name, "op": "sample", "rows": rows, "vocab": vocab, "mode": mode, "pad": pad, "coarse": coarse, "layout": layout}


def listed():
    qwen, vocab = (12, 2, 128), 151936  # this repository's decoder
    return [
        # One chat session decoding: the smallest call, one token normed, rotated, written and read back.
        _paged("rotate 1x300 bytes", "rotate", BYTES, qwen, 16, 1, (1, 1), (300, 300)),
        # Prompts of many lengths, small heads of their own K and V, no norm, a quarter of each head rotated.
        _paged("rotate 24 ragged bf16", "rotate", BF16, (8, 8, 64), 48, 24, (1, 1500), (40, 6000), norm=False, rotary=16, theta=1e4, layout=6),
        # Prompt chunks.
        _paged("rotate 16x2048 bytes", "rotate", BYTES, qwen, 64, 16, (1000, 2048), (1000, 8192), layout=7),
        # Sessions moved into the pool: the bounds of all their pages.
        _paged("bounds 8x16384 bf16", "bounds", BF16, qwen, 128, 8, (9000, 16384), (1, 1), layout=8),
        # One long session decoding over 32 of its 512 pages: from the projection to the attention's output.
        _paged("step 1x32749 bytes", "step", BYTES, qwen, 64, 1, (1, 1), (32749, 32749), blocks=32, first=1, recent=2),
        # The batched decoder's workload, 64 sessions of 128 to 8192 rows; the short ones are attended to whole.
        _paged("step 64x8192 bytes", "step", BYTES, qwen, 64, 64, (1, 1), (128, 8192), blocks=32, first=1, recent=2, layout=2),
        # Long documents in BF16 and small pages: 64 of 1024.
        _paged("sparse 16x32768 bf16", "attend", BF16, qwen, 32, 16, (1, 1), (20000, 32768), blocks=64, first=1, recent=4, layout=3),
        # A drafted continuation being verified: five tokens a sequence, each with pages of its own.
        _paged("sparse 32x5 bf16", "attend", BF16, (32, 8, 128), 32, 32, (5, 5), (900, 4100), blocks=40, first=2, recent=2, layout=5),
        # A prompt's next chunk over a long cache, every query over 64 of 512 pages.
        _paged("sparse 512 on 32768 bytes", "attend", BYTES, qwen, 64, 1, (512, 512), (32768, 32768), blocks=64, first=1, recent=2),
        # One session's next token, as a chat samples it.
        _sample("sample 1x151936", 1, vocab, "chat"),
        # A batch of requests that each bring settings of their own, over a 16-bit readout; some rows have masked tokens.
        _sample("sample 64x151936 mixed", 64, vocab, "mixed", coarse=True, layout=2),
        # The largest: top-p alone, where no small k bounds what is kept.
        _sample("sample 256x151936 nucleus", 256, vocab, "nucleus"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    while True:
        op = rng.choice(["rotate", "rotate", "bounds", "step", "step", "attend", "attend", "sample", "sample", "sample"])
        layout = rng.randrange(1 << 20)
        if op == "sample":
            c = _sample("", _spread(rng, 1, 256), _spread(rng, 2, 151936), rng.choice(["chat", "mixed", "nucleus", "plain"]),
                        rng.choice([0, 0, 1, 64]), rng.random() < 0.5, layout)
            del c["name"]
            return c
        heads = rng.choice([(12, 2, 128), (12, 2, 128), (32, 8, 128), (8, 1, 128), (4, 4, 128), (8, 8, 64), (10, 2, 64), (14, 2, 64)])
        seqs, dim = _spread(rng, 1, 64), heads[2]
        if op == "step":
            new = (1, 1)
        elif op == "attend":
            top = rng.choice([1, _spread(rng, 2, 8), _spread(rng, 9, 512)])
            new = (rng.choice([1, top]), top)
        else:
            new = (1, _spread(rng, 1, 16384 if op == "bounds" else 4096))
        top = _spread(rng, max(new[1], 600 if op in ("step", "attend") else 2), 32768)
        c = _paged("", op, rng.choice([BF16, BYTES]), heads, rng.choice([16, 24, 32, 48, 64, 100, 128]), seqs, new, (_spread(rng, 1, top), top),
                   norm=rng.random() < 0.6, rotary=rng.choice([dim, dim, dim // 2, dim // 4, 20, 0]), theta=rng.choice([1e4, 5e5, 1e6]), layout=layout)
        del c["name"]
        if op in ("step", "attend"):
            c["first"], c["recent"] = rng.choice([0, 1, 2]), rng.choice([1, 2, 5])
            c["blocks"] = c["first"] + c["recent"] + _spread(rng, 1, 64)
        news, lengths = _extents(c)
        rows, kv = int(lengths.sum()), heads[1]
        gathered = seqs * int(news.max()) * kv * c["blocks"] * c["page"] * dim
        scores = seqs * heads[0] * int(news.max()) * -(-int(lengths.max()) // c["page"])
        # No dearer than the largest listed case, and within what the plain forms' padding can hold.
        if rows * kv * dim < 2e8 and int(news.sum()) * (heads[0] + 2 * kv) * dim < 4.3e7 and gathered < 5.4e8 and scores < 5e7 \
                and seqs * int(lengths.max()) * kv * dim < 4e8:
            return c


def _extents(c):
    """Each sequence's new rows and its length, from the case alone."""
    rng = random.Random(c["layout"])
    news = [_spread(rng, c["new_min"], c["new_max"]) for _ in range(c["seqs"])]
    news[rng.randrange(c["seqs"])] = c["new_max"]
    lengths = [max(n, _spread(rng, c["len_min"], c["len_max"])) for n in news]
    return np.array(news), np.array(lengths)


def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 32), "flops": 0}
    news, lengths = _extents(case)
    kv, d, qh, page = case["kvheads"], case["dim"], case["qheads"], case["page"]
    row = kv * (2 * d * 2 if case["kind"] == BF16 else 2 * (d + 4))  # a cached row's bytes, K and V
    rows, values, bound = int(news.sum()), kv * d * 2 * 4, kv * 2 * d * 2
    total = flops = 0
    if case["op"] in ("rotate", "step"):
        total += rows * (values + 2 * qh * d * 4 + row)
    if case["op"] == "rotate" and case["kind"] == BYTES:
        total += rows * (values + row)
    if case["op"] in ("bounds", "step"):
        for n, length in zip(news.tolist(), lengths.tolist()):
            a = (length - n) // page
            total += (length - a * page) * row // 2 + (-(-length // page) - a) * bound
    if case["op"] in ("attend", "step"):
        for n, length in zip(news.tolist(), lengths.tolist()):
            at = np.arange(length - n, length)
            pages = at // page + 1
            seen = (np.minimum(pages, case["blocks"]) - 1) * page + at % page + 1
            scored = np.where(pages > case["blocks"], pages - case["first"] - case["recent"], 0)
            # One query's pages at least are read, whatever the others share with it.
            total += int(seen.max()) * row + int(scored.max()) * bound + n * qh * d * 4 * (2 if case["op"] == "attend" else 1)
            flops += int(4 * d * qh * seen.sum() + 2 * d * qh * scored.sum())
    return {"bytes": total, "flops": flops}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return _prepare_sample(dict(case), g) if case["op"] == "sample" else _prepare_paged(dict(case), g)


def _prepare_sample(c, g):
    rows, vocab, rng = c["rows"], c["vocab"], random.Random(c["layout"])
    full = torch.empty(rows, vocab + c["pad"], device="cuda")
    full.normal_(generator=g)
    # A readout's logits: a broad body, some rows peaked and some flat, a few tokens far ahead.
    full *= torch.tensor([math.exp(rng.uniform(math.log(0.7), math.log(3.5))) for _ in range(rows)], device="cuda").view(-1, 1)
    at = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    full.scatter_add_(1, at, 6 * torch.rand(rows, 24, generator=g, device="cuda"))
    if c["coarse"]:
        full = full.to(torch.bfloat16).float()
    p = np.zeros(rows, dtype=[("temperature", "f4"), ("top_k", "i4"), ("top_p", "f4"), ("min_p", "f4")])
    for r in range(rows):
        kind = c["mode"] if c["mode"] != "mixed" else rng.choice(["chat", "nucleus", "plain", "top-k", "min-p", "greedy", "masked"])
        p[r] = {"chat": (0.7, 40, 0.95, 0.0), "nucleus": (1.0, 0, 0.9, 0.0), "plain": (1.0, 0, 1.0, 0.0), "top-k": (1.3, 1000, 1.0, 0.0),
                "min-p": (1.5, 0, 1.0, 0.05), "greedy": (0.0, 0, 1.0, 0.0), "masked": (0.9, 0, 0.98, 0.01)}[kind]
        if kind == "masked" and vocab > 40:  # a grammar allows few tokens here
            full[r].masked_fill_(torch.rand(vocab + c["pad"], generator=g, device="cuda") > 20.0 / vocab, -math.inf)
            full[r, at[r, 0]] = 1.5
    host = torch.from_numpy(np.ascontiguousarray(p).view(np.int32).reshape(rows, 4).copy())
    return {"case": c, "logits": full[:, :vocab], "params": host.cuda(), "temperature": torch.from_numpy(p["temperature"].copy()).cuda(),
            "top_k": torch.from_numpy(p["top_k"].copy()).cuda(), "top_p": torch.from_numpy(p["top_p"].copy()).cuda(),
            "min_p": torch.from_numpy(p["min_p"].copy()).cuda(), "uniforms": torch.rand(rows, generator=g, device="cuda"),
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_paged(c, g):
    news, lengths = _extents(c)
    seqs, page, kv, d, qh = c["seqs"], c["page"], c["kvheads"], c["dim"], c["qheads"]
    need = -(-lengths // page)
    pages = int(need.sum()) + max(2, int(need.sum()) // 16)
    stride = int(need.max()) + 1
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((seqs, stride), -1, dtype=torch.int32)
    held = torch.zeros(seqs, stride, dtype=torch.bool)
    for s in range(seqs):
        held[s, :int(need[s])] = True
    table, held = table.cuda(), held.cuda()
    table[held] = order[:int(need.sum())]
    starts = np.concatenate([[0], np.cumsum(news)])
    st = {
        "case": c, "pages": pages, "rows": int(starts[-1]), "max_new": int(news.max()), "max_length": int(lengths.max()),
        "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"),
        "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"),
        "table": table, "stride": stride, "status": torch.zeros(1, dtype=torch.int32, device="cuda"),
        "bounds": torch.zeros(pages, kv, 2, d, dtype=torch.bfloat16, device="cuda"),
    }
    shape = (pages, kv, page, d)
    rand = lambda *size: torch.randn(*size, generator=g, device="cuda")  # noqa: E731
    dtype = torch.int8 if c["kind"] == BYTES else torch.bfloat16
    if c["op"] == "rotate":  # the pool starts empty
        pool = [torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2)]
        scales = torch.zeros(2, pages, kv, page, device="cuda")
    else:  # rows of a page are alike, as neighbouring keys are, and of unlike size
        pool = [torch.empty(shape, dtype=dtype, device="cuda") for _ in range(2)]
        scales = torch.exp(rand(2, pages, kv, page) * 0.3) * 0.025
        for t in pool:
            for a in range(0, pages, 4096):
                n = min(4096, pages - a)
                x = rand(n, kv, 1, d) * 0.8 + rand(n, *shape[1:]) * 0.6
                t[a:a + n] = (x * 40).round_().clamp_(-127, 127).to(torch.int8) if c["kind"] == BYTES else x * torch.exp(rand(n, kv, page, 1) * 0.3)
        # What no sequence holds (free pages, the rows behind a sequence's last) is never visible, whatever it contains.
        free = torch.ones(pages, page, dtype=torch.bool, device="cuda")
        at = torch.arange(stride * page, device="cuda").view(1, stride, page) < st["lengths"].view(-1, 1, 1)
        free[table[held].long()] = ~at.expand(seqs, stride, page)[held]
        if c["kind"] == BYTES:
            scales.masked_fill_(free.view(1, pages, 1, page), math.nan)
        else:
            for t in pool:
                t.masked_fill_(free.view(pages, 1, page, 1), math.nan)
    st["keys"], st["values"], st["scales"] = pool[0], pool[1], scales
    if c["op"] in ("attend", "step"):
        _plain_bounds(st, torch.zeros_like(st["lengths"], dtype=torch.int64))
    if c["op"] != "bounds":  # rows of a fused projection: queries, keys, values
        st["qkv"] = rand(st["rows"], (qh + 2 * kv) * d) * torch.exp(rand(st["rows"], 1) * 0.2)
        st["qnorm"], st["knorm"] = 1 + 0.1 * rand(d), 1 + 0.1 * rand(d)
    return st


# ---------------------------------------------------------------- the plain forms
def _new_rows(st):
    """Of each new row: its sequence, and its place there."""
    r = torch.arange(st["rows"], device="cuda")
    s = (torch.searchsorted(st["starts"], r, right=True, out_int32=True) - 1).long()
    return s, st["lengths"].long()[s] - st["starts"].long()[s + 1] + r


def _slots(st, s, j):
    """Page and row in it of row j of sequence s; the page is -1 where there is none."""
    page = st["case"]["page"]
    return st["table"].long()[s, (j // page).clamp(0, st["stride"] - 1)], j % page


def _plain_turn(st, x, weight, at):
    """x [rows, heads, dim], each head normed and its first elements rotated to the row's place. Angles reach tens of thousands, and the
    keys are rounded to few bits behind this, so it is done in 64 bits and rounded once to 32."""
    c = st["case"]
    x = x.double()
    if c["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + float(np.float32(EPS))) * weight.double()
    if c["rotary"]:
        half = c["rotary"] // 2
        rate = float(np.float32(c["theta"])) ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        angle = at.double().view(-1, 1, 1) * rate
        cos, sin = torch.cos(angle), torch.sin(angle)
        a, b = x[..., :half], x[..., half:2 * half]
        x = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1)
    return x.float()


def _plain_rotate(st):
    c = st["case"]
    kv, d, qh = c["kvheads"], c["dim"], c["qheads"]
    s, at = _new_rows(st)
    p, o = _slots(st, s, at)
    x = st["qkv"].view(-1, qh + 2 * kv, d)
    for kind, (pool, y) in enumerate(((st["keys"], _plain_turn(st, x[:, qh:qh + kv], st["knorm"], at)), (st["values"], x[:, qh + kv:]))):
        if c["kind"] == BYTES:
            m = y.abs().amax(-1)
            scale = torch.where(m > 0, m / torch.full_like(m, 127), torch.ones_like(m))
            y = y / scale.unsqueeze(-1)
            pool[p, :, o] = (torch.sign(y) * torch.floor(y.abs() + 0.5)).clamp(-127, 127).to(torch.int8)
            st["scales"][kind][p, :, o] = scale
        else:
            pool[p, :, o] = y.to(torch.bfloat16)
    return _plain_turn(st, x[:, :qh], st["qnorm"], at)


def _plain_rows(st, kind, p, o):
    """FP32 values of the pool's rows (p, o): [..., kvheads, dim]."""
    x = (st["keys"], st["values"])[kind][p, :, o].float()
    return x * st["scales"][kind][p, :, o].unsqueeze(-1) if st["case"]["kind"] == BYTES else x


def _outward(x, up):
    """64-bit values as BF16, rounded up or down, by way of FP32 rounded the same way."""
    near = x.float()
    wrong = near.double() < x if up else near.double() > x
    i = torch.where(wrong, torch.nextafter(near, torch.full_like(near, math.inf if up else -math.inf)), near).contiguous().view(torch.int32)
    away = ((i & 65535) != 0) & ((i >= 0) == up)
    return (((i & -65536) + away.int() * 65536) >> 16).to(torch.int16).view(torch.bfloat16)


def _plain_bounds(st, first=None):
    """The bounds of all pages that hold a row from place `first` on; where it is None, a new row."""
    page, length = st["case"]["page"], st["lengths"].long()
    if first is None:
        first, most = length - (st["starts"][1:] - st["starts"][:-1]).long(), st["max_new"] // page + 2
    else:
        most = st["max_length"] // page + 1
    last = (length - 1) // page
    j = torch.minimum((first // page).view(-1, 1) + torch.arange(most, device="cuda"), last.view(-1, 1))  # the last one again where there are fewer
    rows = j.unsqueeze(-1) * page + torch.arange(page, device="cuda")  # [seqs, most, page]
    p, o = _slots(st, torch.arange(len(length), device="cuda").view(-1, 1, 1), rows)
    there = (rows < length.view(-1, 1, 1))[..., None, None]
    x = st["keys"][p, :, o].double()
    if st["case"]["kind"] == BYTES:
        x *= st["scales"][0][p, :, o].unsqueeze(-1)
    st["bounds"][p[..., 0], :, 0] = _outward(torch.where(there, x, math.inf).amin(2), False)
    st["bounds"][p[..., 0], :, 1] = _outward(torch.where(there, x, -math.inf).amax(2), True)


def _plain_select(st, q, at, last):
    """The pages of each query and KV head, ascending, -1 behind the last: [seqs, new rows, kvheads, blocks]. q [seqs, n, kvheads, group, dim],
    at [seqs, n] the queries' places, last [seqs] the last page. In 64 bits: two pages' scores may lie next to one another."""
    c = st["case"]
    page, blocks = c["page"], c["blocks"]
    pages = st["max_length"] // page + 1
    j = torch.arange(pages, device="cuda")
    ids = st["table"].long()[:, :pages].clamp(min=0)
    bounds = torch.where((j <= last.view(-1, 1))[..., None, None, None], st["bounds"][ids].double(), 0.0)  # [seqs, pages, kvheads, 2, dim]
    q = q.permute(0, 2, 1, 3, 4).double()
    low, high = bounds[:, :, :, 0].permute(0, 2, 3, 1).unsqueeze(2), bounds[:, :, :, 1].permute(0, 2, 3, 1).unsqueeze(2)
    score = (torch.matmul(q.clamp(max=0), low) + torch.matmul(q.clamp(min=0), high)).amax(3).permute(0, 2, 1, 3)  # [seqs, n, kvheads, pages]
    own_page = (at // page)[:, :, None, None]
    score = torch.where((j < c["first"]) | (j > own_page - c["recent"]), math.inf, score)
    score = torch.where(j > own_page, -math.inf, score)
    best = torch.sort(score, dim=-1, descending=True, stable=True)[1][..., :blocks]
    rank = torch.arange(best.shape[-1], device="cuda")
    best = torch.sort(torch.where(rank <= own_page, best, 1 << 30), -1)[0]
    best = torch.where(best == 1 << 30, -1, best)
    return torch.nn.functional.pad(best, (0, blocks - best.shape[-1]), value=-1)


def _plain_attend(st, q):
    c = st["case"]
    kv, d, qh, page = c["kvheads"], c["dim"], c["qheads"], c["page"]
    n, seqs, group = st["max_new"], c["seqs"], qh // kv
    s, place = _new_rows(st)
    i = torch.arange(st["rows"], device="cuda") - st["starts"].long()[s]
    x = torch.zeros(seqs, n, kv, group, d, device="cuda")
    x[s, i] = q.reshape(-1, kv, group, d)
    at = torch.zeros(seqs, n, dtype=torch.int64, device="cuda")
    at[s, i] = place
    chosen = _plain_select(st, x, at, (st["lengths"].long() - 1) // page)  # [seqs, n, kvheads, blocks]
    rows = chosen.unsqueeze(-1) * page + torch.arange(page, device="cuda")
    there = (chosen.unsqueeze(-1) >= 0) & (rows <= at[:, :, None, None, None])
    ids = st["table"].long()[torch.arange(seqs, device="cuda").view(-1, 1, 1, 1), chosen.clamp(min=0)]
    head = torch.arange(kv, device="cuda").view(1, 1, -1, 1)
    k, v = st["keys"][ids, head].float(), st["values"][ids, head].float()  # [seqs, n, kvheads, blocks, page, dim]
    if c["kind"] == BYTES:
        k, v = k * st["scales"][0][ids, head].unsqueeze(-1), v * st["scales"][1][ids, head].unsqueeze(-1)
    k, v = (torch.where(there.unsqueeze(-1), y, 0.0).view(seqs, n, kv, -1, d) for y in (k, v))
    w = torch.matmul(x, k.transpose(-1, -2)) / math.sqrt(d)
    w = w.masked_fill_(~there.view(seqs, n, kv, 1, -1), -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    out = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    return {"out": out.view(seqs, n, qh, d)[s, i], "selected": chosen[s, i].int()}


def _plain_sample(st):
    logits, p = st["logits"], st["temperature"].double().view(-1, 1)
    greedy = p == 0
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    x = (x - top) / torch.where(greedy, 1.0, p)
    live = logits > -math.inf
    order = torch.sort(logits, dim=-1, descending=True, stable=True)[1]
    w = torch.exp(x)
    ranked = torch.gather(w, 1, order)
    count = live.sum(-1, keepdim=True)
    k = st["top_k"].long().view(-1, 1)
    n = torch.where(k > 0, torch.minimum(k, count), count)
    rank = torch.arange(x.shape[1], device="cuda")
    mass = torch.cumsum(torch.where(rank < n, ranked, 0.0), -1)
    share = st["top_p"].double().view(-1, 1)
    n = torch.where(share < 1, torch.minimum(n, (mass < share * mass[:, -1:]).sum(-1, keepdim=True) + 1), n)
    least = st["min_p"].double().view(-1, 1)
    n = torch.where(least > 0, torch.minimum(n, (ranked >= least).sum(-1, keepdim=True)), n)
    n = torch.where(greedy, 1, n)
    kept = torch.zeros_like(live).scatter_(1, order, rank < n)
    w = torch.where(kept, w, 0.0)
    total = torch.cumsum(w, -1)
    target = st["uniforms"].double().view(-1, 1) * total[:, -1:]
    ids = (total <= target).sum(-1, keepdim=True)
    logprob = torch.gather(x, 1, ids) - torch.log(total[:, -1:])
    return {"ids": ids.int().view(-1), "kept": n.int().view(-1), "logprobs": torch.where(greedy, 0.0, logprob).float().view(-1)}


# ---------------------------------------------------------------- the library's kernels
_gpu = []  # the program's one handle: it owns the workspaces


def _handles(st):
    """The descriptors that a program keeps beside its pool and batch."""
    if "lib" not in st:
        import cmachine_b200 as cm
        c = st["case"]
        st["lib"] = cm.lib()
        if not _gpu:
            _gpu.append(st["lib"].gpu_open())
        st["gpu"] = _gpu[0]
        if c["op"] != "sample":
            st["cache"] = cm.PagedCache(c["kind"], st["pages"], c["page"], c["kvheads"], c["dim"], st["keys"].data_ptr(),
                                        st["values"].data_ptr(), st["scales"].data_ptr())
            st["batch"] = cm.PagedBatch(c["seqs"], st["rows"], st["max_new"], st["max_length"], st["starts"].data_ptr(),
                                        st["lengths"].data_ptr(), st["table"].data_ptr(), st["stride"])
            if "qkv" in st:
                st["turn"] = cm.HeadRotation(st["qnorm"].data_ptr() if c["norm"] else None, st["knorm"].data_ptr() if c["norm"] else None,
                                             EPS, c["theta"], c["rotary"])
    return st["lib"]


def _own_rotate(st):
    L, c = _handles(st), st["case"]
    q = torch.empty(st["rows"], c["qheads"], c["dim"], device="cuda")
    at = st["qkv"].data_ptr()
    k = at + c["qheads"] * c["dim"] * 4
    if L.gpu_paged_rotate_append(st["cache"], st["batch"], st["turn"], q.data_ptr(), q.stride(0), at, k, k + c["kvheads"] * c["dim"] * 4,
                                 st["qkv"].stride(0), c["qheads"], st["status"].data_ptr()):
        raise RuntimeError("gpu_paged_rotate_append refused")
    return q


def _own_read(st):
    L, c = _handles(st), st["case"]
    k, v = (torch.empty(st["rows"], c["kvheads"], c["dim"], device="cuda") for _ in range(2))
    if L.gpu_paged_read(st["cache"], st["batch"], k.data_ptr(), v.data_ptr(), k.stride(0), st["status"].data_ptr()):
        raise RuntimeError("gpu_paged_read refused")
    return {"k": k, "v": v}


def _own_bounds(st):
    L = _handles(st)
    if L.gpu_paged_bounds(st["cache"], st["batch"], st["bounds"].data_ptr(), st["status"].data_ptr()):
        raise RuntimeError("gpu_paged_bounds refused")


def _own_attend(st, q, stride):
    L, c = _handles(st), st["case"]
    out = torch.empty(st["rows"], c["qheads"], c["dim"], device="cuda")
    chosen = torch.empty(st["rows"], c["kvheads"], c["blocks"], dtype=torch.int32, device="cuda")
    if L.gpu_paged_sparse_attention(st["gpu"], out.data_ptr(), out.stride(0), q.data_ptr(), stride, st["cache"], st["batch"],
                                    st["bounds"].data_ptr(), c["qheads"], c["blocks"], c["first"], c["recent"], chosen.data_ptr(),
                                    st["status"].data_ptr()):
        raise RuntimeError("gpu_paged_sparse_attention refused")
    return {"out": out, "selected": chosen}


def _own_sample(st):
    L, c = _handles(st), st["case"]
    ids, kept = (torch.empty(c["rows"], dtype=torch.int32, device="cuda") for _ in range(2))
    logprobs = torch.empty(c["rows"], device="cuda")
    if L.gpu_sample(st["gpu"], ids.data_ptr(), logprobs.data_ptr(), kept.data_ptr(), st["logits"].data_ptr(), c["vocab"] + c["pad"],
                    c["rows"], c["vocab"], st["params"].data_ptr(), st["uniforms"].data_ptr(), st["status"].data_ptr()):
        raise RuntimeError("gpu_sample refused")
    return {"ids": ids, "kept": kept, "logprobs": logprobs}


def _stored(st):
    """What a rotate case gives back of the pool: its own buffers, or the new rows as the values that their bytes stand for."""
    if st["case"]["kind"] == BF16:
        return {"keys": st["keys"], "values": st["values"]}
    if own:
        return _own_read(st)
    p, o = _slots(st, *_new_rows(st))
    return {"k": _plain_rows(st, 0, p, o), "v": _plain_rows(st, 1, p, o)}


def run(state):
    c = state["case"]
    if c["op"] == "sample":
        return _own_sample(state) if own else _plain_sample(state)
    q = None
    if c["op"] in ("rotate", "step"):
        q = _own_rotate(state) if own else _plain_rotate(state)
        if c["op"] == "rotate":
            return {"q": q, **_stored(state)}
    if c["op"] in ("bounds", "step"):
        if own:
            _own_bounds(state)
        else:
            _plain_bounds(state)
        if c["op"] == "bounds":
            return {"bounds": state["bounds"]}
    width = c["qheads"] * c["dim"]
    if own:
        got = _own_attend(state, state["qkv"] if q is None else q, state["qkv"].stride(0) if q is None else width)
    else:
        got = _plain_attend(state, state["qkv"][:, :width] if q is None else q)
    return got if q is None else {"q": q, **got}


# ---------------------------------------------------------------- the definitions in 64 bits
def _codec64(x, kind):
    """What rows of single-precision values stand for once stored. The codec is defined by single-precision divisions; a 64-bit
    quotient of single-precision numbers rounds to the same single-precision number."""
    if kind == BF16:
        return x.to(torch.bfloat16).double()
    m = x.abs().amax(-1, keepdim=True)
    scale = torch.where(m > 0, m / 127.0, torch.ones_like(m)).float().double()
    y = (x / scale).float().double()
    return torch.trunc(y + torch.where(y < 0, -0.5, 0.5)).clamp(-127, 127) * scale


def _turn64(st, a, b, lo, hi, weight, first):
    """Heads lo..hi of rows a..b of the fused projection, normed and turned as complex numbers; the first row stands at place `first`."""
    c = st["case"]
    d, half = c["dim"], c["rotary"] // 2
    x = st["qkv"][a:b, lo * d:hi * d].reshape(b - a, hi - lo, d).double()
    if c["norm"]:
        size = torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / d
        x = x * weight.double() * (size + float(np.float32(EPS))) ** -0.5
    if half:
        rate = torch.exp(torch.arange(half, dtype=torch.float64, device="cuda") * (-math.log(float(np.float32(c["theta"]))) / half))
        angle = torch.outer(torch.arange(first, first + b - a, dtype=torch.float64, device="cuda"), rate)
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * torch.polar(torch.ones_like(angle), angle).unsqueeze(1)
        x = torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)
    return x


def _held(st, s, kind, lo, hi):
    """Rows [lo, hi) of sequence s in 64 bits: [kvheads, hi - lo, dim]."""
    page = st["case"]["page"]
    a, b = lo // page, -(-hi // page)
    ids = st["table"][s, a:b].long()
    x = (st["keys"], st["values"])[kind][ids].double()  # [pages, kvheads, page, dim]
    if st["case"]["kind"] == BYTES:
        x = x * st["scales"][kind][ids].double().unsqueeze(-1)
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[3])[:, lo - a * page:hi - a * page]


def _bf16_towards(x, up):
    """The BF16 number next to each 64-bit value on the side asked for: the nearest, or its neighbour."""
    near = x.float().to(torch.bfloat16)
    wrong = near.double() < x if up else near.double() > x
    return torch.where(wrong, torch.nextafter(near, torch.full_like(near, math.inf if up else -math.inf)), near)


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["op"] == "sample":
        return _exact_sample(st)
    kv, d, qh, page = c["kvheads"], c["dim"], c["qheads"], c["page"]
    starts, lengths = st["starts"].tolist(), st["lengths"].tolist()
    spans = [(s, starts[s], starts[s + 1], lengths[s] - (starts[s + 1] - starts[s]), lengths[s]) for s in range(c["seqs"])]
    if c["op"] == "rotate":
        q = torch.cat([_turn64(st, a, b, 0, qh, st["qnorm"], first) for _, a, b, first, _ in spans])
        k = torch.cat([_turn64(st, a, b, qh, qh + kv, st["knorm"], first) for _, a, b, first, _ in spans])
        v = st["qkv"][:, (qh + kv) * d:].reshape(-1, kv, d)
        k, v = _codec64(k.float().double(), c["kind"]), _codec64(v.double(), c["kind"])
        if c["kind"] == BYTES:
            return {"q": q, "k": k, "v": v}
        pools = [torch.zeros(st["keys"].shape, dtype=torch.float64, device="cuda") for _ in range(2)]
        for s, a, b, first, length in spans:
            j = torch.arange(first, length, device="cuda")
            ids = st["table"][s].long()[j // page]
            pools[0][ids, :, j % page], pools[1][ids, :, j % page] = k[a:b], v[a:b]
        return {"q": q, "keys": pools[0], "values": pools[1]}
    if c["op"] == "bounds":
        out = st["bounds"].double()
        for s, _, _, first, length in spans:
            a = first // page
            x = _held(st, s, 0, a * page, length)  # [kvheads, rows, dim]
            pad = -x.shape[1] % page
            for side, fill in enumerate((math.inf, -math.inf)):
                y = torch.nn.functional.pad(x, (0, 0, 0, pad), value=fill).view(kv, -1, page, d)
                y = y.amax(2) if side else y.amin(2)
                out[st["table"][s, a:a + y.shape[1]].long(), :, side] = _bf16_towards(y, bool(side)).double().transpose(0, 1)
        return {"bounds": out}
    out = torch.zeros(st["rows"], qh, d, dtype=torch.float64, device="cuda")
    chosen = torch.full((st["rows"], kv, c["blocks"]), -1, dtype=torch.int64, device="cuda")
    turned = []
    for s, a, b, first, length in spans:
        k, v = _held(st, s, 0, 0, length), _held(st, s, 1, 0, length)
        if c["op"] == "step":
            turned.append(_turn64(st, a, b, 0, qh, st["qnorm"], first))
            q = turned[-1].float().double()
            k[:, first:] = _codec64(_turn64(st, a, b, qh, qh + kv, st["knorm"], first).float().double(), c["kind"]).transpose(0, 1)
            v[:, first:] = _codec64(st["qkv"][a:b, (qh + kv) * d:].double().view(-1, kv, d), c["kind"]).transpose(0, 1)
        else:
            q = st["qkv"][a:b, :qh * d].double().view(-1, qh, d)
        whole = length // page  # pages that bounds are asked of
        y = k[:, :whole * page].view(kv, whole, page, d)
        low, high = _bf16_towards(y.amin(2), False).double(), _bf16_towards(y.amax(2), True).double()
        mid, reach = (low + high) / 2, (high - low) / 2  # the most of q . x in a box: at its middle, and |q| from there
        for h in range(kv):
            x = q[:, h * (qh // kv):(h + 1) * (qh // kv)]
            score = (x @ mid[h].T + x.abs() @ reach[h].T).amax(1)  # [new rows, pages]
            for r in range(b - a):
                at = first + r
                mine = at // page
                pages = list(range(mine + 1))
                if mine + 1 > c["blocks"]:
                    lo, hi = c["first"], mine - c["recent"] + 1
                    want = c["blocks"] - c["first"] - c["recent"]
                    rank = torch.argsort(score[r, lo:hi], descending=True, stable=True)[:want] + lo
                    pages = sorted(list(range(lo)) + rank.tolist() + list(range(hi, mine + 1)))
                ids = torch.tensor(pages, device="cuda")
                chosen[a + r, h, :len(pages)] = ids
                rows = (ids.view(-1, 1) * page + torch.arange(page, device="cuda")).view(-1)
                rows = rows[:(len(pages) - 1) * page + at % page + 1]
                w = torch.softmax(x[r] @ k[h, rows].T / math.sqrt(d), -1)
                out[a + r, h * (qh // kv):(h + 1) * (qh // kv)] = w @ v[h, rows]
    got = {"out": out, "selected": chosen}
    return {"q": torch.cat(turned), **got} if c["op"] == "step" else got


def _exact_sample(st):
    ids, kept, logprobs = [], [], []
    for r in range(st["case"]["rows"]):
        t, k, share, least = (float(st[name][r]) for name in ("temperature", "top_k", "top_p", "min_p"))
        x = st["logits"][r].double()
        if t == 0:
            ids.append(int((x == x.max()).nonzero()[0]))
            kept.append(1)
            logprobs.append(0.0)
            continue
        x = (x - x.max()) / t
        order = torch.argsort(-x, stable=True)[:int((x > -math.inf).sum())]
        if k > 0:
            order = order[:int(k)]
        w = torch.exp(x[order])
        n = len(order)
        if share < 1:
            n = min(n, int(torch.searchsorted(torch.cumsum(w, 0), share * w.sum())) + 1)
        if least > 0:
            n = min(n, int((w >= least).sum()))
        order = torch.sort(order[:n])[0]
        total = torch.cumsum(torch.exp(x[order]), 0)
        at = min(n - 1, int(torch.searchsorted(total, float(st["uniforms"][r]) * total[-1], right=True)))
        ids.append(int(order[at]))
        kept.append(n)
        logprobs.append(float(x[order[at]] - torch.log(total[-1])))
    return {"ids": torch.tensor(ids), "kept": torch.tensor(kept), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}

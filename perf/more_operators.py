"""Cases of the operators on a paged key/value cache in 16 bits: storing rows,
attention of new tokens over the cached sequences (one token a sequence, a few,
or a chunk of a prompt), the weight that each cached token gets from them, and
eviction of the tokens with the least of it.

K and V are [pages, kv_heads, page_size, head_dim]; block_table [batch,
max_pages] names the pages of each sequence, token j of sequence b lies in page
block_table[b, j / page_size].  The new tokens are the last q_len[b] of the
kv_len[b] ones.  With e[r, j] the softmax weight of query row r (of any query
head that reads kv head h) on token j,

    key_weights[b, h, j] = decay * (what was there) + sum over r of e[r, j]

in pages as well, [pages, kv_heads, page_size] in 32 bits; decay is 0 here, so
that a pass can be repeated.  Eviction keeps min(kv_len, budget) tokens of each
(sequence, kv head): the first `sinks`, the last `recent`, and of the others
those of the largest weight (of equal ones the earliest), in their order, and
moves their rows of K, V and weights to tokens 0, 1, .. of the pages of
`out_table` (the sequence's own pages without one; here others, so that a pass
can be repeated).
"""
import math
import random

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _attend(name, dtype, batch, heads, kv_heads, head_dim, kv_min, kv_max, page, q_len=1, ragged_q=False, alibi=False, window=-1,
            cap=0.0, weights=False):
    return {"name": name, "kind": "attend", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "kv_min": kv_min, "kv_max": kv_max, "page": page, "q_len": q_len, "ragged_q": ragged_q,
            "alibi": alibi, "window": window, "cap": cap, "weights": weights}


def _evict(name, dtype, batch, kv_heads, head_dim, kv_min, kv_max, page, budget, recent, sinks):
    return {"name": name, "kind": "evict", "dtype": dtype, "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim,
            "kv_min": kv_min, "kv_max": kv_max, "page": page, "budget": budget, "recent": recent, "sinks": sinks}


def _store(name, dtype, batch, rows, kv_heads, head_dim, page, start_min=0, start_max=0, ragged=False):
    return {"name": name, "kind": "store", "dtype": dtype, "batch": batch, "rows": rows, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "start_min": start_min, "start_max": start_max, "ragged": ragged}


def listed():
    return [
        # one short sequence, the first tokens of an answer: latency
        _attend("step_one_short", "fp16", 1, 8, 2, 64, 77, 77, 16),
        # a decode step of a serving batch, grouped-query heads, mixed lengths
        _attend("step_batch_gqa", "bf16", 32, 32, 8, 128, 1001, 8191, 64),
        # one long document, a single sequence
        _attend("step_one_long", "fp16", 1, 32, 8, 128, 131071, 131071, 128),
        # several proposed tokens a sequence checked at once, ragged, some sequences new, ALiBi as in the benchmark's decode
        _attend("verify_alibi", "bf16", 16, 32, 8, 128, 0, 4096, 64, q_len=5, ragged_q=True, alibi=True),
        # the next chunk of a long prompt over what is cached of it
        _attend("chunk_long", "bf16", 1, 32, 8, 128, 34816, 34816, 64, q_len=2048),
        # chunks of two prompts, wide heads, a sliding window and soft-capped scores
        _attend("chunk_window_cap", "bf16", 2, 16, 8, 256, 2500, 4097, 32, q_len=512, window=1023, cap=50.0),
        # a decode step that also notes what each cached token weighs
        _attend("step_weights", "bf16", 16, 32, 8, 128, 2000, 8191, 64, weights=True),
        # ragged chunks of prompts that note it, a kv head for each query head, the smallest pages
        _attend("chunk_weights", "fp16", 3, 16, 16, 64, 700, 6000, 16, q_len=700, ragged_q=True, weights=True),
        # a serving batch cut back to a quarter of its tokens
        _evict("evict_batch", "bf16", 32, 8, 128, 2500, 4096, 64, 1024, 128, 4),
        # one long document cut back to an eighth
        _evict("evict_long", "fp16", 1, 8, 128, 131071, 131071, 128, 16384, 1024, 4),
        # the new token's keys and values of a decode step
        _store("store_token", "bf16", 64, 1, 8, 128, 64, 255, 4095),
        # the prompts of a prefill (the benchmark's causal prefill shape)
        _store("store_prompt", "bf16", 8, 2048, 32, 128, 64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["step", "step", "chunk", "chunk", "evict", "store"])
    dtype = rng.choice(["fp16", "bf16"])
    d = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
    if kind in ("step", "chunk"):
        group = rng.choice([1, 2, 3, 4, 7, 8]) if kv_heads <= 8 else 1
        batch = _log(rng, 1, 64 if kind == "step" else 8)
        q_len = rng.choice([1, 1, rng.randint(2, 8)]) if kind == "step" else _log(rng, 9, 2048)
        most = min(131072, int(3e8) // (batch * kv_heads * d), int(1.5e11) // (batch * kv_heads * group * d * q_len))
        kv_max = _log(rng, min(16, most), max(17, most))
        kv_min = rng.choice([0, kv_max // 2, kv_max])
        window = rng.choice([-1, -1, rng.randint(1, kv_max)])
        c = _attend("", dtype, batch, kv_heads * group, kv_heads, d, kv_min, kv_max, page, q_len, q_len > 1 and rng.random() < 0.5,
                    rng.random() < 0.25, window, rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.3)
    elif kind == "evict":
        batch = _log(rng, 1, 32)
        kv_max = _log(rng, 16, max(17, min(131072, int(1.5e8) // (batch * kv_heads * d))))
        budget = rng.randint(1, max(1, kv_max // rng.choice([1, 2, 8])))
        recent = rng.randint(0, budget // 2)
        c = _evict("", dtype, batch, kv_heads, d, rng.choice([0, kv_max // 2, kv_max]), kv_max, page, budget, recent,
                   rng.randint(0, min(4, budget - recent)))
    else:
        batch = _log(rng, 1, 64)
        rows = _log(rng, 1, max(2, min(8192, int(6e7) // (batch * kv_heads * d))))
        start = rng.choice([0, rng.randint(0, 2000)])
        c = _store("", dtype, batch, rows, kv_heads, d, page, start // 2, start, rng.random() < 0.5)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers evenly from lo to hi, in an order that only n gives."""
    v = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(v)
    return v


def _kv_lens(case):
    return _spread(case["kv_min"], case["kv_max"], case["batch"])


def _q_lens(case):
    b, n = case["batch"], case["q_len"]
    return _spread(max(1, n // 4), n, b)[::-1] if case["ragged_q"] else [n] * b


def _rows(case):
    b, n = case["batch"], case["rows"]
    return _spread(case["start_min"], case["start_max"], b), _spread(n // 2, n, b)[::-1] if case["ragged"] else [n] * b


def _table(need, order, dev):
    """A table whose sequence i owns the next need[i] pages of `order`."""
    table = torch.zeros(len(need), max(max(need), 1), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table


def prepare(case, seed):
    dev, t = "cuda", DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    b, page, hk, d = case["batch"], case["page"], case["kv_heads"], case["head_dim"]

    def normal(*shape, spread=1.0):  # normal values, as in the repository's workloads
        return torch.randn(*shape, generator=gen, device=dev, dtype=t).mul_(spread)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=dev)

    s = {"case": case}
    if case["kind"] == "store":
        # the pages before the first row are one shared page (a common prompt): nothing is written there
        first, count = _rows(case)
        lo = [f // page for f in first]
        need = [-(-(f + n) // page) - p if n else 0 for f, n, p in zip(first, count, lo)]
        order = torch.randperm(sum(need), generator=gen, device=dev).int() + 1
        own_pages = _table(need, order, dev)
        s["table"] = torch.zeros(b, max(max(p + n for p, n in zip(lo, need)), 1), dtype=torch.int32, device=dev)
        for i in range(b):
            s["table"][i, lo[i]:lo[i] + need[i]] = own_pages[i, :need[i]]
        s["k_cache"], s["v_cache"] = (torch.zeros(sum(need) + 1, hk, page, d, dtype=t, device=dev) for _ in range(2))
        s["k"], s["v"] = normal(b, case["rows"], hk, d), normal(b, case["rows"], hk, d, spread=0.7)
        s["start"], s["lens"] = ints(first), ints(count)
        return s
    lens = _kv_lens(case)
    need = [-(-n // page) for n in lens]
    extra = b * -(-case["budget"] // page) if case["kind"] == "evict" else 3
    pages = sum(need) + extra
    s["table"] = _table(need, torch.randperm(sum(need), generator=gen, device=dev).int(), dev)
    s["lens"] = ints(lens)
    s["k_cache"], s["v_cache"] = normal(pages, hk, page, d), normal(pages, hk, page, d, spread=0.7)
    if case["kind"] == "evict":
        # weights as they add up: over several powers of ten, a tenth of them 0
        w = torch.exp(2.0 * torch.randn(pages, hk, page, generator=gen, device=dev))
        s["weights"] = w * (torch.rand(w.shape, generator=gen, device=dev) >= 0.1)
        s["first_out"] = sum(need)
        order = torch.randperm(extra, generator=gen, device=dev).int() + sum(need)
        s["out_table"] = order.view(b, -1)
        s["kept"] = torch.empty(b, hk, case["budget"], dtype=torch.int32, device=dev)
        s["new_lens"] = torch.empty(b, dtype=torch.int32, device=dev)
        return s
    s["q"] = normal(b, case["q_len"], case["heads"], d)
    s["out"] = torch.empty_like(s["q"])
    s["q_lens"] = ints(_q_lens(case)) if case["ragged_q"] else None
    h = torch.arange(1, case["heads"] + 1, dtype=torch.float64)
    s["slopes"] = torch.pow(2.0, -8.0 * h / case["heads"]).float().to(dev) if case["alibi"] else None
    s["weights"] = torch.zeros(pages, hk, page, device=dev) if case["weights"] else None
    return s


def _places(s, table, n):
    """Page and place in it of tokens 0 .. n - 1 of each sequence: [batch, n] each."""
    j = torch.arange(n, device=table.device)
    page = s["case"]["page"]
    return table.long()[:, j // page], (j % page).expand(table.shape[0], n)


def _plain_attend(s):
    case = s["case"]
    b, ql, h, d = s["q"].shape
    hk = case["kv_heads"]
    n = max(case["kv_max"], 1)
    at, place = _places(s, s["table"], n)
    j = torch.arange(n, device=s["q"].device)
    q_lens = s["q_lens"] if s["q_lens"] is not None else torch.full_like(s["lens"], ql)
    row = torch.arange(ql, device=j.device)[None, :, None]
    diag = row + (s["lens"] - q_lens)[:, None, None]
    seen = (j < s["lens"][:, None, None]) & (j <= diag) & (row < q_lens[:, None, None])
    if case["window"] >= 0:
        seen = seen & (diag - j <= case["window"])
    seen = seen[:, None, None]  # [batch, kv_head, group, row, token]
    q = s["q"].unflatten(2, (hk, -1)).permute(0, 2, 3, 1, 4)
    out = torch.empty(q.shape, dtype=s["q"].dtype, device=j.device)
    step = max(1, int(3e8) // (b * (h // hk) * ql * n))  # kv heads at a time, by the scores' size
    for lo in range(0, hk, step):
        hs = slice(lo, lo + step)
        k, v = (c[:, hs][at, :, place].transpose(1, 2).float() for c in (s["k_cache"], s["v_cache"]))
        x = (q[:, hs].float().flatten(2, 3) @ k.transpose(2, 3)).unflatten(2, q.shape[2:4]) / math.sqrt(d)
        if case["cap"] > 0:
            x = torch.tanh(x / case["cap"]) * case["cap"]
        if s["slopes"] is not None:  # the distance from the row's own token: the softmax is the same
            x = x + s["slopes"].view(hk, -1, 1, 1)[hs] * (j - diag)[:, None, None].float()
        x = x.masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True)
        x = torch.exp(x - top.masked_fill(top == -math.inf, 0.0))
        x = x / x.sum(-1, keepdim=True).clamp_min(1e-30)
        out[:, hs] = (x.flatten(2, 3) @ v).unflatten(2, q.shape[2:4]).to(out.dtype)
        if s["weights"] is not None:
            w = x.sum((2, 3))  # [batch, kv_head, token]
            bi, ti = (j < s["lens"][:, None]).nonzero(as_tuple=True)
            s["weights"][:, hs][at[bi, ti], :, place[bi, ti]] = w.transpose(1, 2)[bi, ti]
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)


def _plain_evict(s):
    case = s["case"]
    b, hk, budget = s["kept"].shape
    n = max(case["kv_max"], budget)
    j = torch.arange(n, device=s["lens"].device)
    table = s["table"]
    if table.shape[1] * case["page"] < n:
        table = torch.nn.functional.pad(table, (0, -(-n // case["page"]) - table.shape[1]))
    at, place = _places(s, table, n)
    lens = s["lens"][:, None]
    w = s["weights"][at, :, place].transpose(1, 2)  # [batch, kv_head, token]
    w = torch.where(w.isnan(), -math.inf, w) + 0.0
    order = w.argsort(dim=-1, descending=True, stable=True)  # of equal weights the earliest first
    kind = torch.ones_like(at).masked_fill((j < case["sinks"]) | (j >= lens - case["recent"]), 0).masked_fill(j >= lens, 2)
    kind = kind[:, None].expand(b, hk, n).gather(2, order)
    order = order.gather(2, kind.argsort(dim=-1, stable=True))[..., :budget]
    new_lens = s["lens"].clamp_max(budget)
    r = torch.arange(budget, device=j.device)
    held = (r < new_lens[:, None])[:, None]
    kept = order.masked_fill(~held, n).sort(-1).values
    kept = kept.masked_fill(~held, -1)
    s["kept"].copy_(kept)
    s["new_lens"].copy_(new_lens)
    bi, hi, ri = held.expand(b, hk, budget).nonzero(as_tuple=True)
    src = kept[bi, hi, ri]
    to, to_place = _places(s, s["out_table"], budget)
    for c in (s["k_cache"], s["v_cache"], s["weights"]):
        c[to[bi, ri], hi, to_place[bi, ri]] = c[at[bi, src], hi, place[bi, src]]


def _plain_store(s):
    page = s["case"]["page"]
    b, rows = s["k"].shape[:2]
    i = torch.arange(rows, device=s["k"].device)
    bi, ri = (i < s["lens"][:, None]).nonzero(as_tuple=True)
    j = s["start"].long()[bi] + ri
    at = s["table"].long()[bi, j // page]
    s["k_cache"][at, :, j % page] = s["k"][bi, ri]
    s["v_cache"][at, :, j % page] = s["v"][bi, ri]


def run(s):
    case = s["case"]
    if own:
        import llmx_b200
    if case["kind"] == "store":
        if own:
            llmx_b200.paged_store(s["k_cache"], s["v_cache"], s["k"], s["v"], start=s["start"], lens=s["lens"],
                                  block_table=s["table"])
        else:
            _plain_store(s)
        return s["k_cache"], s["v_cache"]
    if case["kind"] == "evict":
        if own:
            llmx_b200.paged_evict(s["k_cache"], s["v_cache"], s["weights"], case["budget"], kv_lens=s["lens"],
                                  block_table=s["table"], recent=case["recent"], sinks=case["sinks"],
                                  out_table=s["out_table"], kept=s["kept"], new_lens=s["new_lens"])
        else:
            _plain_evict(s)
        first = s["first_out"]  # the pages that the kept rows move to are the last ones
        return s["kept"], s["new_lens"], s["k_cache"][first:], s["v_cache"][first:], s["weights"][first:]
    if own:
        llmx_b200.paged_attention(s["out"], s["q"], s["k_cache"], s["v_cache"], case["head_dim"] ** -0.5, case["window"],
                                  case["cap"], kv_lens=s["lens"], block_table=s["table"], q_lens=s["q_lens"],
                                  alibi_slopes=s["slopes"], key_weights=s["weights"], decay=0.0)
        out = s["out"]
    else:
        out = _plain_attend(s)
    return out if s["weights"] is None else (out, s["weights"])


def _seen(case):
    """Pairs of a query row and a token that it sees, and tokens that some row sees, over all sequences."""
    pairs = tokens = 0
    for n, ql in zip(_kv_lens(case), _q_lens(case)):
        first = n
        for i in range(ql):
            hi = min(n, i + n - ql + 1)
            lo = max(0, i + n - ql - case["window"]) if case["window"] >= 0 else 0
            if hi > lo:
                pairs += hi - lo
                first = min(first, lo)
        tokens += n - first
    return pairs, tokens


def work(case):
    d, hk = case["head_dim"], case["kv_heads"]
    row = 2 * 2 * hk * d  # bytes of a token's K and V
    if case["kind"] == "store":
        n = sum(_rows(case)[1])
        return {"bytes": 2 * n * row, "flops": 0}
    if case["kind"] == "evict":
        lens = _kv_lens(case)
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": 4 * hk * sum(lens) + 2 * kept * row + kept * hk * (4 + 4), "flops": hk * sum(lens)}
    pairs, tokens = _seen(case)
    qo = 2 * 2 * sum(_q_lens(case)) * case["heads"] * d
    noted = 4 * hk * sum(_kv_lens(case)) if case["weights"] else 0
    return {"bytes": tokens * row + qo + noted, "flops": 4 * d * case["heads"] * pairs}


def exact(case, seed):
    """From the definitions, in 64 bits, one sequence (and kv head) after the other."""
    s = prepare(case, seed)
    page, table = case["page"], s["table"].tolist()
    if case["kind"] == "store":
        k, v = s["k_cache"].double(), s["v_cache"].double()
        first, count = _rows(case)
        for b in range(case["batch"]):
            i = 0
            while i < count[b]:  # up to the end of the page
                p, o = divmod(first[b] + i, page)
                m = min(page - o, count[b] - i)
                k[table[b][p], :, o:o + m] = s["k"][b, i:i + m].transpose(0, 1).double()
                v[table[b][p], :, o:o + m] = s["v"][b, i:i + m].transpose(0, 1).double()
                i += m
        return k, v
    lens = _kv_lens(case)

    def rows(c, b, n):  # [kv_heads, n, ...] of the first n tokens
        parts = [c[p] for p in table[b][:-(-n // page)]]
        return torch.cat(parts, 1)[:, :n] if parts else c[:0].transpose(0, 1).flatten(1, 2)

    if case["kind"] == "evict":
        first = s["first_out"]
        outs = [s[c][first:].double() for c in ("k_cache", "v_cache", "weights")]
        kept = torch.full_like(s["kept"], -1)
        to = s["out_table"].tolist()
        for b, n in enumerate(lens):
            m = min(n, case["budget"])
            sets = [rows(s[c], b, n) for c in ("k_cache", "v_cache", "weights")]
            for h in range(case["kv_heads"]):
                if n <= case["budget"]:
                    pick = torch.arange(n, device="cuda")
                else:
                    sinks, recent = case["sinks"], case["recent"]
                    mid = sets[2][h, sinks:n - recent].tolist()
                    best = sorted(range(len(mid)), key=lambda i: (-mid[i], i))[:m - sinks - recent]
                    pick = list(range(sinks)) + sorted(sinks + i for i in best) + list(range(n - recent, n))
                    pick = torch.tensor(pick, device="cuda")
                kept[b, h, :m] = pick
                for i in range(0, m, page):
                    c = min(page, m - i)
                    for o, x in zip(outs, sets):
                        o[to[b][i // page] - first, h, :c] = x[h, pick[i:i + c]].double()
        return (kept, torch.tensor([min(n, case["budget"]) for n in lens], device="cuda"), *outs)
    d, group = case["head_dim"], case["heads"] // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    noted = torch.zeros(s["k_cache"].shape[:3], dtype=torch.float64, device="cuda")
    ar = torch.arange(1, case["heads"] + 1, dtype=torch.float64)
    slopes = torch.pow(2.0, -8.0 * ar / case["heads"]).float().double().cuda()
    for b, (n, ql) in enumerate(zip(lens, _q_lens(case))):
        if n == 0:
            continue
        keys, values = rows(s["k_cache"], b, n), rows(s["v_cache"], b, n)
        pos = torch.arange(n, device="cuda")
        last = torch.arange(ql, device="cuda")[:, None] + (n - ql)
        hidden = (pos > last) | ((last - pos > case["window"]) if case["window"] >= 0 else False)
        for h in range(case["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            x = torch.einsum("rgd,nd->grn", s["q"][b, :ql, heads].double(), keys[h].double()) * d ** -0.5
            if case["cap"] > 0:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["alibi"]:
                x = x + slopes[heads, None, None] * pos
            p = torch.softmax(x.masked_fill_(hidden, -math.inf), -1).nan_to_num_(0.0)
            out[b, :ql, heads] = torch.einsum("grn,nd->rgd", p, values[h].double())
            w = torch.nn.functional.pad(p.sum((0, 1)), (0, -n % page)).view(-1, page)
            noted[torch.tensor(table[b][:w.shape[0]], device="cuda"), h] = w
    return (out, noted) if case["weights"] else out

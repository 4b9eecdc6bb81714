"""Cases of the operators on a key/value cache held in 4 bits: writing rows into
it (and reading them back), reading it as dense rows, and attention over it.

The cache is a uint8 tensor [pages, kv_heads, page_size / 16, 18 * head_dim]:
tiles of 16 tokens, each with the K codes, the V codes and the parameters of
its tokens.  Channels are quantised in groups of 64 with a step s and a
minimum m, both of the type of K and V:

    m = min x,  r = fl32(fl32(max x - m) / 15),  s = the smallest s >= r
    n = min(15, round_half_even(fl32(fl32(x - m) / s)))  (0 where s = 0)
    value = n * s + m

Codes of a tile lie in 32-bit words of 8 consecutive channels, channel c of
the word in bits 4c .. 4c + 3, and the words in the order [word / 4][8][4][word % 4]:

    K: word (r, h, w) of [g][t]: token 8 r + g, channels 64 h + 16 t + 8 w ..
    V: word (a, c, h) of [g][t]: token 8 a + 2 t + c, channels 64 h + 8 g ..

The parameters follow as [token][K, V][group][s, m].
"""
import math
import random

import torch

own = False

GROUP = 64
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _attend(name, dtype, batch, heads, kv_heads, head_dim, kv_min, kv_max, page, q_len=1, alibi=False, window=-1, cap=0.0,
            ragged_q=False):
    return {"name": name, "kind": "attend", "dtype": dtype, "batch": batch, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "kv_min": kv_min, "kv_max": kv_max, "page": page, "q_len": q_len, "alibi": alibi,
            "window": window, "cap": cap, "ragged_q": ragged_q}


def _rows(name, kind, dtype, batch, rows, kv_heads, head_dim, page, start_min=0, start_max=0, ragged=False):
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "rows": rows, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "start_min": start_min, "start_max": start_max, "ragged": ragged}


def listed():
    return [
        # one short sequence, the first tokens of an answer: latency
        _attend("attend_one_short", "fp16", 1, 8, 2, 64, 77, 77, 16),
        # the benchmark's batched ALiBi decode with its lengths, over a 4-bit cache
        _attend("attend_batch_alibi", "bf16", 64, 32, 32, 128, 256, 4096, 64, alibi=True),
        # a serving batch of grouped-query heads, mixed lengths
        _attend("attend_batch_gqa", "bf16", 32, 32, 8, 128, 1001, 8191, 64),
        # one long document, a single sequence
        _attend("attend_one_long", "fp16", 1, 32, 8, 128, 131071, 131071, 128),
        # wide heads with a sliding window and soft-capped scores
        _attend("attend_window_cap", "bf16", 8, 16, 8, 256, 900, 4097, 32, window=1023, cap=50.0),
        # several proposed tokens a sequence checked at once, ragged, some sequences new
        _attend("attend_verify", "bf16", 16, 32, 8, 128, 0, 4096, 64, q_len=5, ragged_q=True),
        # one kv head for all query heads
        _attend("attend_mqa", "fp16", 16, 32, 1, 128, 500, 8192, 128),
        # the new token's keys and values of a decode step
        _rows("write_token", "write", "bf16", 64, 1, 32, 128, 64, 255, 4095),
        # the prompts of a prefill (the benchmark's causal prefill shape)
        _rows("write_prompt", "write", "bf16", 8, 2048, 32, 128, 64),
        # chunks of prompts that begin and end inside tiles
        _rows("write_ragged", "write", "fp16", 5, 333, 16, 64, 16, 1, 100, ragged=True),
        # a cached prefix expanded for a prefill over it
        _rows("load_prefix", "load", "bf16", 16, 4096, 8, 128, 64, ragged=True),
        # a few rows of wide heads
        _rows("load_few", "load", "fp16", 3, 65, 2, 256, 32, 3, 40, ragged=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "load"])
    dtype = rng.choice(["fp16", "bf16"])
    d = rng.choice([64, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
    if kind == "attend":
        group = rng.choice([1, 2, 3, 4, 7, 8]) if kv_heads <= 8 else 1
        batch = _log(rng, 1, 64)
        kv_max = _log(rng, 16, max(17, min(131072, int(3e8) // (batch * kv_heads * d))))
        kv_min = rng.choice([0, kv_max // 2, kv_max])
        q_len = rng.choice([1, 1, 1, rng.randint(2, 8)])
        window = rng.choice([-1, -1, rng.randint(1, kv_max)])
        c = _attend("", dtype, batch, kv_heads * group, kv_heads, d, kv_min, kv_max, page, q_len,
                    rng.random() < 0.25, window, rng.choice([0.0, 0.0, 30.0]), q_len > 1 and rng.random() < 0.5)
    else:
        batch = _log(rng, 1, 64)
        rows = _log(rng, 1, max(2, min(8192, int(6e7) // (batch * kv_heads * d))))
        start = rng.choice([0, rng.randint(0, 2000)])
        c = _rows("", kind, dtype, batch, rows, kv_heads, d, page, start // 2, start, rng.random() < 0.5)
    del c["name"]
    return c


def _spread(lo, hi, n):
    """n whole numbers evenly from lo to hi, in an order that only n gives."""
    v = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n).shuffle(v)
    return v


def _spans(case):
    """Of each sequence: where its tokens in the cache begin, and how many there are."""
    b = case["batch"]
    if case["kind"] == "attend":
        return [0] * b, _spread(case["kv_min"], case["kv_max"], b)
    n = _spread(case["rows"] // 2, case["rows"], b) if case["ragged"] else [case["rows"]] * b
    return _spread(case["start_min"], case["start_max"], b), n


def _q_lens(case):
    return [1 + i % case["q_len"] if case["ragged_q"] else case["q_len"] for i in range(case["batch"])]


def _rows_of(gen, case, n):
    """Keys and values of n tokens, [n, kv_heads, head_dim]: normal, as in the repository's workloads."""
    shape = (n, case["kv_heads"], case["head_dim"])
    return [torch.randn(shape, generator=gen, device="cuda").mul_(spread).to(DTYPES[case["dtype"]]) for spread in (1.0, 0.7)]


def _quantised(x):
    """Codes, steps and minima of the groups of x [..., head_dim], in 32 bits."""
    g = x.unflatten(-1, (-1, GROUP))
    m = g.amin(-1, keepdim=True)
    r = (g.amax(-1, keepdim=True).float() - m.float()).div(torch.full_like(m, 15.0, dtype=torch.float32))  # a true division: by a plain number it is a product with a rounded 1 / 15
    s = r.to(x.dtype)
    s = torch.where(s.float() < r, (s.view(torch.int16) + 1).view(x.dtype), s)
    n = torch.where(s > 0, (g.float() - m.float()) / s.float(), 0.0).round().clamp(0, 15)
    return n, s, m


def _tiles(k, v):
    """Tiles [tiles, kv_heads, 18 head_dim] of whole tiles of tokens k, v [16 tiles, kv_heads, head_dim]."""
    groups = k.shape[-1] // GROUP
    (nk, sk, mk), (nv, sv, mv) = _quantised(k), _quantised(v)

    def words(n):  # [tile, kv_head, slot (word, 4 groups), 8, 4, channel] to bytes in the order of the tile
        b = n.to(torch.uint8)
        b = b[..., 0::2] | (b[..., 1::2] << 4)
        return b.unflatten(2, (groups, 4)).permute(0, 1, 2, 4, 5, 3, 6).flatten(2)

    tiles, heads = k.shape[0] // 16, k.shape[1]
    nk = nk.reshape(tiles, 2, 8, heads, groups, 4, 2, 8).permute(0, 3, 1, 4, 6, 2, 5, 7).flatten(2, 4)
    nv = nv.reshape(tiles, 2, 4, 2, heads, groups, 8, 8).permute(0, 4, 1, 3, 5, 6, 2, 7).flatten(2, 4)
    p = torch.stack([torch.cat([sk, mk], -1), torch.cat([sv, mv], -1)], 2)  # [token, head, K V, group, s m]
    p = p.unflatten(0, (tiles, 16)).permute(0, 2, 1, 3, 4, 5).flatten(2).contiguous().view(torch.uint8)
    return torch.cat([words(nk), words(nv), p], -1)


def prepare(case, seed):
    dev, t = "cuda", DTYPES[case["dtype"]]
    gen = torch.Generator(device=dev).manual_seed(seed)
    first, count = _spans(case)
    b, page, d = case["batch"], case["page"], case["head_dim"]
    need = [-(-(f + n) // page) for f, n in zip(first, count)]
    order = torch.randperm(sum(need) + 3, generator=gen, device=dev).int()
    table = torch.zeros(b, max(max(need), 1), dtype=torch.int32, device=dev)
    cache = torch.zeros(sum(need) + 3, case["kv_heads"], page // 16, 18 * d, dtype=torch.uint8, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s = {"case": case, "cache": cache, "table": table, "start": torch.tensor(first, dtype=torch.int32, device=dev),
         "lens": torch.tensor(count, dtype=torch.int32, device=dev)}
    if case["kind"] == "write":
        s["k"] = torch.zeros(b, case["rows"], case["kv_heads"], d, dtype=t, device=dev)
        s["v"] = torch.zeros_like(s["k"])
        for i in range(b):
            s["k"][i, :count[i]], s["v"][i, :count[i]] = _rows_of(gen, case, count[i])
    else:
        for i in range(b):  # the tokens before `start` are never read here: zeros
            k, v = (torch.nn.functional.pad(x, (0, 0, 0, 0, first[i], need[i] * page - first[i] - count[i]))
                    for x in _rows_of(gen, case, count[i]))
            if need[i]:
                cache[table[i, :need[i]].long()] = _tiles(k, v).unflatten(0, (need[i], page // 16)).transpose(1, 2)
    if case["kind"] == "attend":
        s["q"] = torch.randn(b, case["q_len"], case["heads"], d, generator=gen, device=dev).to(t)
        s["out"] = torch.empty_like(s["q"])
        s["q_lens"] = torch.tensor(_q_lens(case), dtype=torch.int32, device=dev) if case["ragged_q"] else None
        h = torch.arange(1, case["heads"] + 1, dtype=torch.float64)
        s["slopes"] = torch.pow(2.0, -8.0 * h / case["heads"]).float().to(dev) if case["alibi"] else None
    else:
        s["k_out"] = torch.empty(b, case["rows"], case["kv_heads"], d, dtype=t, device=dev)
        s["v_out"] = torch.empty_like(s["k_out"])
    return s


def _unpacked(s):
    """Keys and values in 32 bits, [batch, tokens, kv_heads, head_dim], of all pages of the table."""
    case = s["case"]
    d, t = case["head_dim"], DTYPES[case["dtype"]]
    groups = d // GROUP
    pages = s["cache"][s["table"].long()].transpose(2, 3).flatten(1, 2)  # [batch, tile, kv_head, bytes]
    k, v, p = pages[..., :8 * d], pages[..., 8 * d:16 * d], pages[..., 16 * d:].contiguous().view(t)

    def codes(x):  # [batch, tile, kv_head, slot, 8, 4, channel of the word]
        x = x.unflatten(-1, (groups, 8, 4, 4, 4)).permute(0, 1, 2, 3, 6, 4, 5, 7).flatten(3, 4)
        return torch.stack([x & 15, x >> 4], -1).flatten(-2)

    k = codes(k).unflatten(3, (2, groups, 2)).permute(0, 1, 3, 6, 2, 4, 7, 5, 8)
    v = codes(v).unflatten(3, (2, 2, groups)).permute(0, 1, 3, 7, 4, 2, 5, 6, 8)
    p = p.float().unflatten(-1, (16, 2, groups, 2)).permute(0, 1, 3, 4, 2, 5, 6).flatten(1, 2)  # [batch, token, K V, kv_head, group, s m]
    shape = (p.shape[0], p.shape[1], case["kv_heads"], groups, GROUP)
    return [(c.reshape(shape).float() * p[:, :, i, ..., 0:1] + p[:, :, i, ..., 1:2]).flatten(3) for i, c in enumerate((k, v))]


def _plain_attend(s):
    case = s["case"]
    k, v = _unpacked(s)
    b, n, hk, d = k.shape
    q = s["q"].float().unflatten(2, (hk, -1)).permute(0, 2, 3, 1, 4)  # [batch, kv_head, group, row, d]
    scores = (q.flatten(2, 3) @ k.permute(0, 2, 3, 1)).unflatten(2, (q.shape[2], q.shape[3])) / math.sqrt(d)
    if case["cap"] > 0:
        scores = torch.tanh(scores / case["cap"]) * case["cap"]
    j = torch.arange(n, device=k.device)
    if s["slopes"] is not None:
        scores = scores + s["slopes"].view(hk, -1, 1, 1) * j.float()
    q_lens = s["q_lens"] if s["q_lens"] is not None else torch.full_like(s["lens"], case["q_len"])
    row = torch.arange(case["q_len"], device=k.device)[None, :, None]
    diag = row + (s["lens"] - q_lens)[:, None, None]
    seen = (j < s["lens"][:, None, None]) & (j <= diag) & (row < q_lens[:, None, None])
    if case["window"] >= 0:
        seen = seen & (diag - j <= case["window"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    o = (e.flatten(2, 3) @ v.transpose(1, 2)) / e.sum(-1).flatten(2, 3)[..., None].clamp_min(1e-30)
    return o.unflatten(2, (q.shape[2], q.shape[3])).permute(0, 3, 1, 2, 4).flatten(2, 3).to(s["q"].dtype)


def _plain_rows(s, k, v):
    """The rows of `rows` behind each sequence's length as 0, in the type of the cache."""
    r = torch.arange(s["k_out"].shape[1], device=k.device)
    kept = (r < s["lens"][:, None])[..., None, None]
    return [x.masked_fill(~kept, 0.0).to(s["k_out"].dtype) for x in (k, v)]


def run(s):
    case = s["case"]
    if own:
        import llmx_b200

        if case["kind"] == "attend":
            llmx_b200.kv4_attention(s["out"], s["q"], s["cache"], case["head_dim"] ** -0.5, case["window"], case["cap"],
                                    alibi_slopes=s["slopes"], q_lens=s["q_lens"], kv_lens=s["lens"], block_table=s["table"])
            return s["out"]
        if case["kind"] == "write":
            llmx_b200.kv4_store(s["cache"], s["k"], s["v"], start=s["start"], lens=s["lens"], block_table=s["table"])
        llmx_b200.kv4_load(s["cache"], s["k_out"], s["v_out"], start=s["start"], lens=s["lens"], block_table=s["table"])
        return s["k_out"], s["v_out"]
    if case["kind"] == "attend":
        return _plain_attend(s)
    if case["kind"] == "write":
        k, v = ((n * st.float() + m.float()).flatten(-2) for n, st, m in (_quantised(s["k"]), _quantised(s["v"])))
        return tuple(_plain_rows(s, k, v))
    k, v = _unpacked(s)
    at = s["start"].long()[:, None] + torch.arange(case["rows"], device=k.device)
    at = at.clamp_max(k.shape[1] - 1)[..., None, None].expand(-1, -1, *k.shape[2:])
    return tuple(_plain_rows(s, k.gather(1, at), v.gather(1, at)))


def _seen(case):
    """Pairs of a query row and a key that it sees, and tokens that some row sees, over all sequences."""
    pairs = tokens = 0
    for n, ql in zip(_spans(case)[1], _q_lens(case)):
        lo_all = n
        for i in range(ql):
            hi = min(n, i + n - ql + 1)
            lo = max(0, i + n - ql - case["window"]) if case["window"] >= 0 else 0
            if hi > lo:
                pairs += hi - lo
                lo_all = min(lo_all, lo)
        tokens += n - lo_all
    return pairs, tokens


def work(case):
    d, hk = case["head_dim"], case["kv_heads"]
    held = 2 * hk * (d // 2 + 4 * (d // GROUP))  # bytes of a token in the cache
    if case["kind"] == "attend":
        pairs, tokens = _seen(case)
        qo = 2 * 2 * sum(_q_lens(case)) * case["heads"] * d
        return {"bytes": tokens * held + qo, "flops": 4 * d * case["heads"] * pairs}
    n = sum(_spans(case)[1])
    dense = 2 * 2 * n * hk * d
    return {"bytes": n * held + dense * (2 if case["kind"] == "write" else 1), "flops": 4 * n * hk * d}


def exact(case, seed):
    """From the definition in 64 bits, on the drawn rows themselves: no cache, and one sequence at a time."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    first, count = _spans(case)
    need = [-(-(f + n) // case["page"]) for f, n in zip(first, count)]
    torch.randperm(sum(need) + 3, generator=gen, device="cuda")
    d = case["head_dim"]

    def held(x):
        y = x.double().reshape(*x.shape[:-1], d // GROUP, GROUP)
        lo, hi = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
        step = ((hi - lo).float().double() / torch.full_like(lo, 15.0)).float().double()
        near = step.to(x.dtype)
        bits = near.view(torch.int16)
        s = torch.where(near.double() < step, bits + 1, bits).view(x.dtype).double()
        place = ((y - lo).float().double() / torch.where(s == 0, 1.0, s)).float().double()
        return (torch.clamp(torch.round(place), max=15) * s + lo).reshape(x.shape)

    values = []
    for i in range(case["batch"]):
        k, v = _rows_of(gen, case, count[i])
        values.append((k, v))
    if case["kind"] != "attend":
        out = [torch.zeros(case["batch"], case["rows"], case["kv_heads"], d, dtype=torch.float64, device="cuda") for _ in range(2)]
        for i, kv in enumerate(values):
            for o, x in zip(out, kv):
                if count[i]:
                    o[i, :count[i]] = held(x)
        return tuple(out)
    q = torch.randn(case["batch"], case["q_len"], case["heads"], d, generator=gen, device="cuda").to(DTYPES[case["dtype"]])
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    group = case["heads"] // case["kv_heads"]
    h = torch.arange(1, case["heads"] + 1, dtype=torch.float64)
    slopes = torch.pow(2.0, -8.0 * h / case["heads"]).float().double().cuda()
    for i, (k, v) in enumerate(values):
        n, ql = count[i], _q_lens(case)[i]
        if n == 0:
            continue
        pos = torch.arange(n, device="cuda")
        rows = torch.arange(ql, device="cuda")[:, None] + (n - ql)
        hidden = (pos > rows) | ((rows - pos > case["window"]) if case["window"] >= 0 else False)
        for kh in range(case["kv_heads"]):
            kd, vd = held(k[:, kh]), held(v[:, kh])
            heads = slice(kh * group, (kh + 1) * group)
            x = torch.einsum("rhd,nd->hrn", q[i, :ql, heads].double(), kd) * d ** -0.5
            if case["cap"] > 0:
                x = case["cap"] * torch.tanh(x / case["cap"])
            if case["alibi"]:
                x = x + slopes[heads, None, None] * pos
            x = x.masked_fill(hidden, -math.inf)
            p = torch.softmax(x, -1).nan_to_num(0.0)
            out[i, :ql, heads] = torch.einsum("hrn,nd->rhd", p, vd)
    return out

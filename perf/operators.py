"""Operators of speculative and batched serving over a paged key/value cache, as cases to measure.

- append: new rows of K and V are written into the pages of their sequences (F16, or 8 bits with one F32 scale per position and head);
- gather: a sequence's last rows are read back out of its pages;
- attention: each new row attends to its sequence's cached rows, causal, optionally with a sliding window and a softcap;
- verify: drafted tokens are accepted or replaced against the target's probabilities, from given random numbers.

`run` computes an operator in its plain form, or, where `own` is true, by the framework's own calls.
"""
import math
import random

import torch

own = False

DEV = "cuda"
ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
KV = {"f16": torch.float16, "q8": torch.int8, "f8": torch.float8_e4m3fn}


# ── cases ───────────────────────────────────────────────────────────────────
# rows_lo..rows_hi: new rows of a sequence; len_lo..len_hi: its length with them; `mix` fixes which sequence has how many.
def listed():
    return [
        # one decode step of 32 sequences: what each layer writes
        dict(name="append_f16_decode", op="append", kv="f16", act="f32", hd=128, n_kv=8, page=16, seqs=32,
             rows_lo=1, rows_hi=1, len_lo=1, len_hi=40, mix=1),
        # the same into 8 bits, and the rows read back as the next call's reader sees them
        dict(name="append_gather_q8_decode", op="append_gather", kv="q8", act="bf16", hd=128, n_kv=8, page=16, seqs=32,
             rows_lo=1, rows_hi=1, len_lo=1, len_hi=512, mix=2),
        # prompt chunks of eight requests, ragged
        dict(name="append_gather_f8_chunks", op="append_gather", kv="f8", act="bf16", hd=128, n_kv=8, page=64, seqs=8,
             rows_lo=1, rows_hi=2047, len_lo=2047, len_hi=4095, mix=3),
        # whole sequences out of the cache, as when they are moved or stored
        dict(name="gather_q8_long", op="gather", kv="q8", act="f32", hd=128, n_kv=8, page=32, seqs=4,
             rows_lo=4096, rows_hi=8192, len_lo=8192, len_hi=8192, mix=4),
        # one request's decode step, 8B model: 32 heads on 8, latency counts
        dict(name="attention_decode_one", op="attention", kv="q8", act="f32", hd=128, n_kv=8, group=4, page=16, seqs=1,
             rows_lo=1, rows_hi=1, len_lo=2049, len_hi=2049, window=0, softcap=0.0, mix=5),
        # a batch of 32 requests of very different lengths, sliding window of 4096
        dict(name="attention_decode_batch", op="attention", kv="f16", act="f16", hd=128, n_kv=8, group=4, page=16, seqs=32,
             rows_lo=1, rows_hi=1, len_lo=17, len_hi=8192, window=4096, softcap=0.0, mix=6),
        # four drafted tokens and the one before them, for 16 requests
        dict(name="attention_verify_batch", op="attention", kv="q8", act="bf16", hd=128, n_kv=8, group=4, page=32, seqs=16,
             rows_lo=1, rows_hi=5, len_lo=100, len_hi=8192, window=0, softcap=0.0, mix=7),
        # prompt chunks with heads of 256, softcap and window
        dict(name="attention_chunk_softcap", op="attention", kv="f8", act="bf16", hd=256, n_kv=8, group=2, page=64, seqs=3,
             rows_lo=200, rows_hi=511, len_lo=1000, len_hi=5000, window=4096, softcap=50.0, mix=8),
        # a prompt chunk in 32-bit activations over an F16 cache
        dict(name="attention_chunk_f32", op="attention", kv="f16", act="f32", hd=64, n_kv=2, group=4, page=16, seqs=2,
             rows_lo=300, rows_hi=512, len_lo=512, len_hi=2047, window=0, softcap=0.0, mix=9),
        # the last chunk of a long prompt: the largest
        dict(name="attention_chunk_long", op="attention", kv="q8", act="bf16", hd=128, n_kv=8, group=4, page=64, seqs=1,
             rows_lo=2048, rows_hi=2048, len_lo=16384, len_hi=16384, window=0, softcap=0.0, mix=10),
        # one request with four drafted tokens, drafted without probabilities (by lookup)
        dict(name="verify_one", op="verify", act="f32", vocab=32000, seqs=1, rows_lo=5, rows_hi=5, probs=False, mix=11),
        # 64 requests, up to seven drafted tokens of a draft model each, some greedy
        dict(name="verify_batch", op="verify", act="bf16", vocab=128256, seqs=64, rows_lo=1, rows_hi=8, probs=True, mix=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    mix = rng.randrange(1 << 30)
    op = rng.choice(["append", "append_gather", "gather", "attention", "attention", "attention", "verify", "verify"])
    act = rng.choice(["f32", "f16", "bf16"])
    if op == "verify":
        case = dict(op=op, act=act, vocab=_log_int(rng, 1000, 256000), seqs=_log_int(rng, 1, 96), rows_lo=1,
                    rows_hi=_log_int(rng, 1, 9), probs=rng.random() < 0.5, mix=mix)
        while case["seqs"] * case["rows_hi"] * case["vocab"] > 66_000_000:
            case["seqs"] = max(1, case["seqs"] // 2)
        return case
    kv, hd, page = rng.choice(["f16", "q8", "f8"]), rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
    if op in ("append", "append_gather", "gather"):
        if op == "append":
            kv = "f16"
        hi = _log_int(rng, 1, 4096)
        case = dict(op=op, kv=kv, act=act, hd=hd, n_kv=rng.choice([1, 2, 4, 8]), page=page, seqs=_log_int(rng, 1, 64),
                    rows_lo=rng.randint(0, hi), rows_hi=hi, len_lo=hi, len_hi=_log_int(rng, hi, 2 * hi + 100), mix=mix)
        while case["seqs"] * case["len_hi"] * case["n_kv"] * hd > 32_000_000:
            case["seqs"], case["len_hi"] = max(1, case["seqs"] // 2), max(hi, case["len_hi"] // 2)
            if case["seqs"] == 1 and case["len_hi"] == hi:
                break
        return case
    kind = rng.choice(["decode", "verify", "chunk"])
    rows = {"decode": 1, "verify": rng.randint(2, 8), "chunk": _log_int(rng, 9, 2048)}[kind]
    seqs = _log_int(rng, 1, 4) if kind == "chunk" else _log_int(rng, 1, 64)
    length = _log_int(rng, max(2, rows), 16384)
    group, n_kv = rng.choice([1, 2, 4, 4, 7, 8]), rng.choice([1, 2, 4, 8])
    case = dict(op=op, kv=kv, act=act, hd=hd, n_kv=n_kv, group=group, page=page, seqs=seqs, rows_lo=max(1, rows // 2), rows_hi=rows,
                len_lo=max(1, rows, length // rng.choice([1, 2, 16])), len_hi=length,
                window=rng.choice([0, 0, 0, rng.randint(1, 4096)]), softcap=rng.choice([0.0, 0.0, 50.0]), mix=mix)
    while max(rows * n_kv * group * hd / 128, 128) * case["seqs"] * case["len_hi"] > 32 * 2048 * 16384:
        if case["seqs"] > 1:
            case["seqs"] //= 2
        else:
            case["len_hi"] = max(rows, case["len_hi"] // 2)
            case["len_lo"] = min(case["len_lo"], case["len_hi"])
            if case["len_hi"] == rows:
                break
    return case


def _sizes(case):
    """New rows and length of each sequence (fixed by the case); the first has the most rows and the greatest length."""
    r = random.Random(case["mix"])
    n = [r.randint(case["rows_lo"], case["rows_hi"]) for _ in range(case["seqs"])]
    n[0] = case["rows_hi"]
    if "len_lo" not in case:
        return n, None
    length = [max(a, _log_int(r, max(1, case["len_lo"]), max(1, case["len_hi"]))) for a in n]
    length[0] = max(n[0], case["len_hi"])
    return n, length


def work(case):
    n, length = _sizes(case)
    rows, act = sum(n), {"f32": 4, "f16": 2, "bf16": 2}[case["act"]]
    if case["op"] == "verify":
        values = rows * case["vocab"]
        return {"bytes": values * act + (case["seqs"] * case["vocab"] * 4 if case["probs"] else 0), "flops": 4 * values}
    es = 2 if case["kv"] == "f16" else 1
    row = case["n_kv"] * (case["hd"] * es + (4 if es == 1 else 0))  # one position of K, or of V
    io = rows * case["n_kv"] * case["hd"] * act                    # the same in activations
    if case["op"] == "append":
        return {"bytes": 2 * (row * rows + io), "flops": 2 * rows * case["n_kv"] * case["hd"]}
    if case["op"] == "gather":
        return {"bytes": 2 * (row * rows + io), "flops": 2 * rows * case["n_kv"] * case["hd"]}
    if case["op"] == "append_gather":
        return {"bytes": 2 * (row * rows + 2 * io), "flops": 8 * rows * case["n_kv"] * case["hd"]}
    w = case["window"] or 1 << 40
    pairs = sum(sum(min(p + 1, w) for p in range(L - a, L)) for a, L in zip(n, length))
    keys = sum(L - max(0, L - a - w + 1) for a, L in zip(n, length))  # those that some row sees
    heads = case["n_kv"] * case["group"]
    return {"bytes": 2 * row * keys + 2 * rows * heads * case["hd"] * act, "flops": 4 * pairs * heads * case["hd"]}


# ── inputs ──────────────────────────────────────────────────────────────────
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 7919 + 17)
    return g


def _starts(n):
    s = [0]
    for a in n:
        s.append(s[-1] + a)
    return s


def prepare(case, seed):
    g = _generator(seed)
    n, length = _sizes(case)
    rows, act = sum(n), ACT[case["act"]]
    s = {"case": case, "rows": rows, "max_rows": max(n), "row_start": torch.tensor(_starts(n), dtype=torch.int32, device=DEV)}
    if case["op"] == "verify":
        V, S = case["vocab"], case["seqs"]
        # a peaked target; the draft model's distribution is near it, and its tokens are drawn from its own distribution
        base = torch.randn(rows, V, generator=g, device=DEV) * 2.0
        base.scatter_add_(1, torch.randint(0, V, (rows, 4), generator=g, device=DEV), torch.rand(rows, 4, generator=g, device=DEV) * 6 + 6)
        draft = torch.softmax(base + 0.3 * torch.randn(rows, V, generator=g, device=DEV), -1)
        s["logits"] = base.to(act)
        s["draft"] = torch.multinomial(draft, 1, generator=g).squeeze(1).to(torch.int32)
        s["draft_probs"] = draft if case["probs"] else None
        t = torch.rand(S, generator=g, device=DEV) * 0.8 + 0.4
        s["temperature"] = torch.where(torch.arange(S, device=DEV) % 4 == 3, torch.zeros_like(t), t)
        s["u_accept"] = torch.rand(rows, generator=g, device=DEV)
        s["u_sample"] = torch.rand(S, generator=g, device=DEV)
        return s
    hd, n_kv, page, S = case["hd"], case["n_kv"], case["page"], case["seqs"]
    per_seq = [-(-L // page) for L in length]
    cols, used = max(per_seq), sum(per_seq)
    n_pages = used + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    at = torch.arange(cols, device=DEV)[None, :]
    first = torch.tensor(_starts(per_seq)[:-1], device=DEV)[:, None]
    mapped = at < torch.tensor(per_seq, device=DEV)[:, None]
    s["page_table"] = torch.where(mapped, order[(first + at).clamp(max=n_pages - 1)], torch.full_like(order[:1], -1))
    s["seq_len"] = torch.tensor(length, dtype=torch.int32, device=DEV)
    s["max_len"] = max(length)
    shape = (n_pages, n_kv, page, hd)
    # what the cache holds: keys with a few strong channels, values of about one; in 8 bits the largest of a row is the type's largest
    for name, strength in (("k", 4.0), ("v", 1.0)):
        x = torch.randn(shape, generator=g, device=DEV)
        x[..., 3] *= strength
        if case["kv"] == "f16":
            s[name], s[name + "_scale"] = x.to(torch.float16), None
        else:
            top = 127.0 if case["kv"] == "q8" else 448.0
            scale = x.abs().amax(-1) / top
            x = x / scale[..., None]
            s[name] = x.round().to(torch.int8) if case["kv"] == "q8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)
            s[name + "_scale"] = scale
    if case["op"] in ("append", "append_gather"):
        # K and V as they leave the projection: two column ranges of one packed matrix
        s["kv_rows"] = torch.randn(rows, 2 * n_kv, hd, generator=g, device=DEV).to(act)
    if case["op"] == "attention":
        s["q"] = (1.5 * torch.randn(rows, n_kv * case["group"], hd, generator=g, device=DEV)).to(act)
    if own:  # the handles that a program keeps beside its cache and for its batch
        from dotnetfoundryllm_b200 import paged
        s["cache"] = paged.PagedKvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["batch"] = paged.PagedBatch(s["page_table"], s["seq_len"], s["row_start"], max_rows=s["max_rows"])
    return s


# ── plain forms ─────────────────────────────────────────────────────────────
def _row_places(s):
    """(sequence, position, page, offset in the page) of each new row."""
    start = s["row_start"].long()
    row = torch.arange(s["rows"], device=DEV)
    seq = torch.bucketize(row, start[1:], right=True)
    pos = s["seq_len"].long()[seq] - (start[seq + 1] - row)
    page = s["case"]["page"]
    return seq, pos, s["page_table"].long()[seq, pos // page], pos % page


def _quantise(x, kv):
    """Values of the type and F32 scales: 64 bits decide the rounding, because quotients lie next to its borders."""
    if kv == "f16":
        return x.float().clamp(-65504.0, 65504.0).to(torch.float16), None
    x = x.double()
    top = torch.full((), 127.0 if kv == "q8" else 448.0, dtype=torch.float64, device=DEV)
    scale = (x.abs().amax(-1) / top).float()
    y = torch.where(scale[..., None] > 0, x / scale.double()[..., None], torch.zeros_like(x))
    if kv == "q8":
        return y.round().clamp(-127, 127).to(torch.int8), scale
    step = torch.ldexp(torch.ones_like(y), torch.frexp(y.abs()).exponent.clamp(min=-5) - 4)  # e4m3: three bits after the first
    return ((y / step).round() * step).clamp(-448, 448).float().to(torch.float8_e4m3fn), scale


def _write(s):
    n_kv, kv = s["case"]["n_kv"], s["case"]["kv"]
    _, _, page, at = _row_places(s)
    k, ks = _quantise(s["kv_rows"][:, :n_kv], kv)
    v, vs = _quantise(s["kv_rows"][:, n_kv:], kv)
    if kv == "f16":
        s["k"][page, :, at] = k
        s["v"][page, :, at] = v
    else:
        s["k"].view(torch.uint8)[page, :, at] = k.view(torch.uint8)
        s["v"].view(torch.uint8)[page, :, at] = v.view(torch.uint8)
        s["k_scale"][page, :, at] = ks
        s["v_scale"][page, :, at] = vs


def _bits(x):
    return x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x


def _read_rows(s):
    _, _, page, at = _row_places(s)
    k, v = (_bits(s[n])[page, :, at].view(s[n].dtype).float() for n in "kv")
    if s["k_scale"] is not None:
        k, v = k * s["k_scale"][page, :, at][..., None], v * s["v_scale"][page, :, at][..., None]
    act = ACT[s["case"]["act"]]
    return k.to(act), v.to(act)


def _attend(s):
    case = s["case"]
    n_kv, grp, hd, S, R = case["n_kv"], case["group"], case["hd"], case["seqs"], s["max_rows"]
    table = s["page_table"].long().clamp(min=0)

    def cached(name):  # [S, n_kv, keys, hd]
        x = _bits(s[name])[table].view(s[name].dtype).float()
        if s[name + "_scale"] is not None:
            x = x * s[name + "_scale"][table][..., None]
        return x.transpose(1, 2).reshape(S, n_kv, -1, hd)

    seq, pos, _, _ = _row_places(s)
    i = torch.arange(s["rows"], device=DEV) - s["row_start"].long()[seq]  # a row's place in its sequence's chunk
    q = torch.zeros(S, R, n_kv * grp, hd, device=DEV)
    q[seq, i] = s["q"].float()
    at = torch.full((S, R), -1, device=DEV)
    at[seq, i] = pos
    k = cached("k")
    x = q.view(S, R, n_kv, grp, hd).permute(0, 2, 1, 3, 4).reshape(S, n_kv, R * grp, hd) @ k.transpose(-1, -2) * (1.0 / math.sqrt(hd))
    del k
    if case["softcap"] > 0:
        x = case["softcap"] * torch.tanh(x / case["softcap"])
    key = torch.arange(x.shape[-1], device=DEV)
    seen = key <= at[..., None]
    if case["window"] > 0:
        seen &= key > at[..., None] - case["window"]
    x = x.view(S, n_kv, R, grp, -1).masked_fill_(~seen[:, None, :, None, :], -math.inf)
    m = x.amax(-1, keepdim=True)
    x = (x - torch.where(m > -math.inf, m, torch.zeros_like(m))).exp_()
    total = x.sum(-1, keepdim=True)
    o = x.view(S, n_kv, R * grp, -1) @ cached("v")
    o = o.view(S, n_kv, R, grp, hd) / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 2, 1, 3, 4).reshape(S, R, n_kv * grp, hd)[seq, i].to(ACT[case["act"]])


def _verify(s):
    rows, S, start = s["rows"], s["case"]["seqs"], s["row_start"].long()
    row = torch.arange(rows, device=DEV)
    seq = torch.bucketize(row, start[1:], right=True)
    temp = s["temperature"].double()
    greedy = temp <= 0
    logits = s["logits"].double()  # 64 bits: draws lie next to the borders of the cumulative sums
    m, best = logits.max(-1)
    e = ((logits - m[:, None]) / torch.where(greedy, torch.ones_like(temp), temp)[seq][:, None]).exp()
    z = e.sum(-1)
    d = s["draft"].long()
    q = torch.ones(rows, dtype=torch.float64, device=DEV) if s["draft_probs"] is None else s["draft_probs"][row, d].double()
    accept = torch.where(greedy[seq], best == d, s["u_accept"].double() * q * z < e[row, d])
    last = row == start[seq + 1] - 1
    stop = torch.full((S,), rows, device=DEV).scatter_reduce(0, seq, torch.where(last | ~accept, row, rows), "amin")
    r = stop.clamp(max=rows - 1)
    w = e[r]
    if s["draft_probs"] is None:
        rest = w.clone()
        rest[torch.arange(S, device=DEV), d[r]] = 0.0
    else:
        rest = (w - s["draft_probs"][r].double() * z[r][:, None]).clamp(min=0.0)
    w = torch.where((~last[r] & (rest.sum(-1) > 0))[:, None], rest, w)
    c = w.cumsum(-1)
    drawn = (c <= s["u_sample"].double()[:, None] * c[:, -1:]).sum(-1)
    token = torch.where(greedy, best[r], drawn)
    out = torch.where(row < stop[seq], d, torch.where(row == stop[seq], token[seq], torch.full_like(d, -1)))
    return {"tokens": out.to(torch.int32), "accepted": (stop - start[:-1]).to(torch.int32)}


# ── one pass ────────────────────────────────────────────────────────────────
def run(s):
    case = s["case"]
    op = case["op"]
    if own:
        if op == "verify":
            from dotnetfoundryllm_b200 import speculate
            tokens, accepted = speculate.verify_drafts(s["logits"], s["row_start"], s["draft"], s["temperature"], s["u_accept"],
                                                       s["u_sample"], draft_probs=s["draft_probs"])
            return {"tokens": tokens, "accepted": accepted}
        cache, batch = s["cache"], s["batch"]
        if op == "attention":
            return cache.attention(batch, s["q"], scale=1.0 / math.sqrt(case["hd"]), window=case["window"], softcap=case["softcap"])
        if op != "gather":
            cache.append(batch, s["kv_rows"][:, :case["n_kv"]], s["kv_rows"][:, case["n_kv"]:])
        if op == "append":
            return {"k": s["k"], "v": s["v"]}
        k, v = cache.gather(batch, s["rows"], ACT[case["act"]])
        return {"k": k, "v": v}
    if op == "verify":
        return _verify(s)
    if op == "attention":
        return _attend(s)
    if op != "gather":
        _write(s)
    if op == "append":
        return {"k": s["k"], "v": s["v"]}
    k, v = _read_rows(s)
    return {"k": k, "v": v}


# ── the definitions in 64 bits ──────────────────────────────────────────────
def exact(case, seed):
    if case["op"] == "verify":
        return None  # whole numbers: equal or wrong
    s = prepare(case, seed)
    n, length = _sizes(case)
    page, kv, n_kv, hd = case["page"], case["kv"], case["n_kv"], case["hd"]

    def sequence(name, b, count):  # [count, n_kv, hd], positions 0.. of sequence b
        pages = s["page_table"][b].tolist()[:-(-count // page)]
        x = torch.cat([s[name][p].double() for p in pages], dim=1)[:, :count]
        if s[name + "_scale"] is not None:
            x = x * torch.cat([s[name + "_scale"][p].double() for p in pages], dim=1)[:, :count, None]
        return x.transpose(0, 1)

    if case["op"] in ("append", "append_gather"):
        def stored(x):  # the value that a written element stands for
            x = x.double()
            if kv == "f16":
                return x.clamp(-65504, 65504).half().double()
            a = x.abs().max(-1, keepdim=True).values
            scale = (a / torch.tensor(127.0 if kv == "q8" else 448.0, dtype=torch.float64, device=DEV)).float().double()
            y = x / torch.where(scale == 0, torch.ones_like(scale), scale)
            if kv == "q8":
                return y.round().clamp(-127, 127) * scale
            e = torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -30))).clamp(min=-6)
            e = torch.where(torch.exp2(e) > y.abs().clamp(min=2.0 ** -6), e - 1, e)
            e = torch.where(torch.exp2(e + 1) <= y.abs(), e + 1, e).clamp(min=-6)
            return (y * torch.exp2(3 - e)).round().mul(torch.exp2(e - 3)).clamp(-448, 448) * scale
        k, v = stored(s["kv_rows"][:, :n_kv]), stored(s["kv_rows"][:, n_kv:])
        if case["op"] == "append_gather":
            return {"k": k, "v": v}
        out, row = {"k": s["k"].double(), "v": s["v"].double()}, 0
        for b in range(case["seqs"]):
            pages = s["page_table"][b].tolist()
            for p in range(length[b] - n[b], length[b]):
                out["k"][pages[p // page], :, p % page] = k[row]
                out["v"][pages[p // page], :, p % page] = v[row]
                row += 1
        return out
    if case["op"] == "gather":
        k = [sequence("k", b, length[b])[length[b] - n[b]:] for b in range(case["seqs"])]
        v = [sequence("v", b, length[b])[length[b] - n[b]:] for b in range(case["seqs"])]
        return {"k": torch.cat(k), "v": torch.cat(v)}
    out, row = torch.zeros(sum(n), n_kv * case["group"], hd, dtype=torch.float64, device=DEV), 0
    for b in range(case["seqs"]):
        L, a = length[b], n[b]
        K, V = sequence("k", b, L), sequence("v", b, L)
        p = torch.arange(L - a, L, device=DEV)[:, None]
        j = torch.arange(L, device=DEV)[None, :]
        hidden = (j > p) | (j <= p - (case["window"] or L + 1))
        for h in range(n_kv * case["group"]):
            x = s["q"][row:row + a, h].double() @ K[:, h // case["group"]].T / math.sqrt(hd)
            if case["softcap"] > 0:
                x = torch.tanh(x / case["softcap"]) * case["softcap"]
            out[row:row + a, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ V[:, h // case["group"]]
        row += a
    return out

"""Performance cases of the paged key and value cache on one GPU: rotating and appending rows, and attention over it.

Kinds of case (field "kind"):
  append  rows of queries, keys and values as a projection leaves them: queries and keys rotated by their
          positions, keys and values put into the pages of their sequences (bf16, or 8 bits with a scale for every
          16 tokens and head); of an 8-bit cache the touched blocks are read back, as a program does that moves them.
  attend  attention of query rows over the pages of their sequences (causal, with or without a sliding window and
          first tokens that stay visible), prompts, chunks and single tokens.

8 heads of 128 and chunks of 1 to 14 rows for up to 64 streams are the 0.6B FastConformer's; the other head counts
and widths are generic.
"""
import math
import os
import random
import sys

import torch

own = False

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"f32": (0, torch.float32), "bf16": (1, torch.bfloat16), "e4m3": (2, torch.uint8)}
BLOCK = 16  # tokens that share a scale
BASE, OLD_LEN, STRETCH, TURNS = 10000.0, 4096, 8.0, (1.0, 4.0)  # of the rotation, and of its scaled form


def listed():
    def append(name, rows_type, cache, **more):
        return {"name": name, "kind": "append", "rows_type": rows_type, "cache": cache, "streams": 1, "rows": 1, "len": 0,
                "ragged": False, "heads": 32, "kv_heads": 8, "dh": 128, "rot": 128, "inter": False, "scaled": False,
                "page": 64, **more}

    def attend(name, rows_type, cache, **more):
        return {"name": name, "kind": "attend", "rows_type": rows_type, "cache": cache, "streams": 1, "rows": 1, "len": 0,
                "ragged": False, "heads": 32, "kv_heads": 8, "dh": 128, "window": 0, "sinks": 0, "page": 64, **more}

    return [
        # one token of one stream: the smallest call
        append("append_token_1", "bf16", "bf16", len=1000, heads=8),
        # a server's step: one token of each of 64 streams, far along, the earlier pages dropped
        append("append_step_64", "bf16", "e4m3", streams=64, len=100000, ragged=True, scaled=True),
        # one long prompt into an 8-bit cache
        append("append_prompt_8192", "bf16", "e4m3", rows=8192),
        # f32 rows of mixed prompts, some continued, an odd width rotated in part, pairs side by side
        append("append_prompts", "f32", "bf16", streams=24, rows=1500, len=700, ragged=True, heads=12, kv_heads=4, dh=96, rot=48,
               inter=True, page=16),
        # one token of one stream
        attend("attend_token_1", "bf16", "bf16", len=1000, heads=8),
        # a server's step over mixed lengths, 8-bit cache
        attend("attend_step_64", "bf16", "e4m3", streams=64, len=16384, ragged=True),
        # one token behind a very long context
        attend("attend_long_131071", "bf16", "bf16", len=131071),
        # an encoder-like step: 560 ms chunks of f32 rows, a window of cached frames
        attend("attend_chunks_f32", "f32", "bf16", streams=16, rows=7, len=4000, ragged=True, heads=8, window=1024, page=16),
        # one long prompt: the most products
        attend("attend_prompt_8192", "bf16", "bf16", rows=8192),
        # prompts of mixed lengths behind what is cached, a window and first tokens that stay, 8-bit cache
        attend("attend_prompts_window", "bf16", "e4m3", streams=12, rows=1500, len=2500, ragged=True, heads=16, kv_heads=4, dh=64,
               window=512, sinks=4),
        # f32 rows of an odd width, three heads to a pair of keys and values
        attend("attend_prompt_f32", "f32", "e4m3", rows=1000, len=500, heads=12, kv_heads=4, dh=80, page=32),
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))

    kind = rng.choice(["append", "attend", "attend"])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    group = rng.choice([1, 1, 2, 3, 4, 4, 6, 8])
    heads = kv_heads * group if kv_heads * group <= 32 else 32
    dh = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    streams = log_int(1, 64)
    case = {"kind": kind, "rows_type": rng.choice(["bf16", "bf16", "f32"]), "cache": rng.choice(["bf16", "e4m3"]), "streams": streams,
            "ragged": rng.random() < 0.7, "heads": heads, "kv_heads": kv_heads, "dh": dh, "page": rng.choice([16, 32, 64, 128])}
    stage = rng.choice(["step", "step", "chunk", "prompt", "prompt"])
    rows = 1 if stage == "step" else log_int(2, 16) if stage == "chunk" else log_int(17, max(17, 8192 // streams))
    if kind == "append":
        rot = rng.choice([dh, dh, dh // 2, dh // 4])
        return dict(case, rows=rows, len=rng.choice([0, log_int(1, 2000), log_int(1000, 500000)]), rot=rot,
                    inter=rng.random() < 0.4, scaled=rng.random() < 0.4)
    # what is cached: as many tokens and scores as the largest listed cases have, at the most
    most = min((1 << 20) * 1024 // (streams * kv_heads * dh), (1 << 31) // (streams * rows * heads) - rows, 131071)
    window = rng.choice([0, 0, log_int(16, 4096)])
    return dict(case, rows=rows, len=0 if stage == "prompt" and rng.random() < 0.5 else log_int(1, max(1, most)), window=window,
                sinks=rng.choice([0, 4, 1, 40]) if window else 0)


# ---- shapes ----------------------------------------------------------------------------------------


def table(case):
    """A sequence's first row, its rows, the tokens cached before them and its row of the page table."""
    out, first = [], 0
    for s in range(case["streams"]):
        rows, start = case["rows"], case["len"]
        if case["ragged"]:
            start = max(0, start - start * ((37 * s + 11) % 53) // 60)
            rows = 0 if s % 11 == 5 else 1 + (rows - 1) * ((29 * s + 50) % 51) // 50
        out.append((first, rows, start, (5 * s + 3) % case["streams"] if case["streams"] % 5 else s))
        first += rows
    return out


def rows_of(case):
    """Rows of the operands: a ragged batch has a few behind the last sequence."""
    return max(1, sum(t[1] for t in table(case)) + (3 if case["ragged"] else 0))


def spans(case):
    """Per sequence its rows, the first and one past the last token that any of them sees behind the sinks."""
    out = []
    for _, rows, start, _ in table(case):
        lo = max(0, start + 1 - case["window"]) if case["window"] else 0
        out.append((rows, lo, start + rows))
    return out


def seen(case):
    """Pairs of a row and a token that it sees."""
    total = 0
    for _, rows, start, _ in table(case):
        for i in range(rows):
            p = start + i
            lo = max(0, p + 1 - case["window"]) if case["window"] else 0
            total += p + 1 - lo + min(lo, case["sinks"] if case["window"] else 0)
    return total


def work(case):
    size = 4 if case["rows_type"] == "f32" else 2
    per = 2 * case["kv_heads"] * case["dh"] * (1 if case["cache"] == "e4m3" else 2)  # bytes of a token's keys and values
    per += 2 * case["kv_heads"] / BLOCK if case["cache"] == "e4m3" else 0
    m = sum(t[1] for t in table(case))
    q = case["heads"] * case["dh"]
    if case["kind"] == "append":
        kv = 2 * case["kv_heads"] * case["dh"]
        back = sum(t[1] + t[2] % BLOCK for t in table(case) if t[1]) if case["cache"] == "e4m3" else 0
        return {"bytes": m * (size * (2.0 * q + kv) + per) + 2.0 * back * kv, "flops": 3.0 * m * case["rot"] * (case["heads"] + case["kv_heads"])}
    tokens = sum(hi - lo + min(lo, case["sinks"]) for rows, lo, hi in spans(case) if rows)
    return {"bytes": 2.0 * size * m * q + tokens * per, "flops": 4.0 * seen(case) * q}


# ---- inputs ----------------------------------------------------------------------------------------


class _Rand:
    def __init__(self, seed, tag):
        self.g = torch.Generator(device="cuda").manual_seed(1000003 * tag + seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda")


def frequencies(case):
    """Radians per position of every rotated pair; scaled: those that turn seldom within the old length are slowed
    down, those that turn often kept, what lies between blended."""
    half = case["rot"] // 2
    f = [BASE ** (-2.0 * i / case["rot"]) for i in range(half)]
    if case["scaled"]:
        lo, hi = TURNS
        keep = [min(1.0, max(0.0, (OLD_LEN * v / (2 * math.pi) - lo) / (hi - lo))) for v in f]
        f = [v * (k + (1 - k) / STRETCH) for v, k in zip(f, keep)]
    return f


def prepare(case, seed):
    r, dev = _Rand(seed, 7), "cuda"
    seqs, page, hk, dh = table(case), case["page"], case["kv_heads"], case["dh"]
    m, dt = rows_of(case), TYPES[case["rows_type"]][1]
    st = {"case": case, "m": m, "max_rows": max(t[1] for t in seqs), "max_len": max(t[1] + t[2] for t in seqs)}
    # the pages that a sequence still has: an append needs those of the open block on, a window those it reaches
    width = max(1, max(-(-(t[1] + t[2]) // page) for t in seqs))
    need = [[] for _ in seqs]
    for (_, rows, start, row) in seqs:
        for j in range(-(-(rows + start) // page)):
            lo, hi = j * page, (j + 1) * page
            if case["kind"] == "append":
                kept = hi > start // BLOCK * BLOCK
            else:
                kept = not case["window"] or hi > start + 1 - case["window"] or lo < case["sinks"]
            if kept:
                need[row].append(j)
    pages = sum(len(n) for n in need) + 3
    order = list(range(pages))
    random.Random(seed).shuffle(order)
    places = torch.full((len(seqs), width), -1, dtype=torch.int32)
    at = 0
    for row, n in enumerate(need):
        places[row, n] = torch.tensor(order[at:at + len(n)], dtype=torch.int32)
        at += len(n)
    st["places"] = places.to(dev)
    st["seqs"] = torch.tensor(seqs, dtype=torch.int32, device=dev)
    shape = (pages, hk, page, dh)
    for n in ("k", "v"):
        if case["cache"] == "bf16":
            st[n + "c"], st[n + "s"] = r.normal(*shape).to(torch.bfloat16), None
        else:  # codes and the powers of two that their blocks have
            st[n + "c"] = r.normal(*shape, std=64.0).to(torch.float8_e4m3fn).view(torch.uint8)
            st[n + "s"] = r.ints(119, 123, pages, hk, page // BLOCK).to(torch.uint8)
    nq, nk = case["heads"] * dh, hk * dh
    if case["kind"] == "append":
        st["qkv"] = (r.normal(m, nq + 2 * nk) * torch.exp(0.3 * r.normal(m, 1))).to(dt)  # one projection's rows
        st["freq"] = torch.tensor(frequencies(case), dtype=torch.float32, device=dev)
        st["out"] = torch.zeros(m, nq, dtype=dt, device=dev)
        if case["cache"] == "e4m3":  # what is read back: from the open block on
            back, first = [], 0
            for (_, rows, start, row) in seqs:
                n = rows + start % BLOCK if rows else 0
                back.append((first, n, start // BLOCK * BLOCK, row))
                first += n
            st["back"] = torch.tensor(back, dtype=torch.int32, device=dev)
            st["mb"] = max(1, first)
            st["max_back"] = max(b[1] for b in back)
            st["kr"] = torch.zeros(st["mb"], nk, dtype=torch.bfloat16, device=dev)
            st["vr"] = torch.zeros(st["mb"], nk, dtype=torch.bfloat16, device=dev)
    else:
        st["q"] = r.normal(m, nq, std=2.0).to(dt)
        st["out"] = torch.zeros(m, nq, dtype=dt, device=dev)
    return st


# ---- one pass --------------------------------------------------------------------------------------


def run(state):
    return _own(state) if own else _plain(state)


def _gpu():
    if not hasattr(_gpu, "g"):
        if os.path.join(REPO, "nemo-c_amd") not in sys.path:
            sys.path.insert(0, os.path.join(REPO, "nemo-c_amd"))
        import nemoasr
        _gpu.g, _gpu.api = nemoasr.Gpu(), nemoasr
    return _gpu.g, _gpu.api


def _own(st):
    g, api = _gpu()
    L, case = api.lib(), st["case"]
    p = {k: v.data_ptr() if torch.is_tensor(v) else None for k, v in st.items()}
    dh, hk, hq, rows_type = case["dh"], case["kv_heads"], case["heads"], TYPES[case["rows_type"]][0]
    kv = api.Kv(type=TYPES[case["cache"]][0], heads=hk, dh=dh, page=case["page"], pages=st["kc"].shape[0], k=p["kc"], v=p["vc"],
                ks=p["ks"], vs=p["vs"], table=p["places"], ldt=st["places"].shape[1], tables=st["places"].shape[0])
    n = case["streams"]
    g.begin()
    if case["kind"] == "attend":
        a = api.Attend(type=rows_type, q=p["q"], ldq=hq * dh, o=p["out"], ldo=hq * dh, heads=hq, window=case["window"],
                       sinks=case["sinks"], scale=1 / math.sqrt(dh), seqs=p["seqs"], nseq=n, max_rows=st["max_rows"],
                       max_len=st["max_len"], M=st["m"])
        g.check(L.nk_attention_kv(g.h, api.C.byref(kv), api.C.byref(a)))
        g.end()
        return st["out"]
    size, ld = st["qkv"].element_size(), (hq + 2 * hk) * dh
    a = api.Append(type=rows_type, q=p["qkv"], ldq=ld, k=p["qkv"] + size * hq * dh, ldk=ld, v=p["qkv"] + size * (hq + hk) * dh,
                   ldv=ld, qo=p["out"], ldqo=hq * dh, heads=hq, rot=case["rot"], inter=int(case["inter"]), freq=p["freq"], amp=1.0,
                   seqs=p["seqs"], nseq=n, max_rows=st["max_rows"], M=st["m"])
    g.check(L.nk_kv_append(g.h, api.C.byref(kv), api.C.byref(a)))
    if case["cache"] == "bf16":
        g.end()
        return {"q": st["out"], "k": st["kc"], "v": st["vc"]}
    g.check(L.nk_kv_read(g.h, api.C.byref(kv), p["kr"], hk * dh, p["vr"], hk * dh, TYPES["bf16"][0], p["back"], n, st["max_back"],
                         st["mb"]))
    g.end()
    return {"q": st["out"], "k": st["kr"], "v": st["vr"]}


# ---- the plain forms -------------------------------------------------------------------------------


def _values8(codes):
    """The values of 8-bit codes: a sign, four bits of an exponent and three of a fraction."""
    i = torch.arange(256, device=codes.device)
    e, f = (i >> 3) & 15, (i & 7).float()
    v = torch.where(e == 0, f / 8 * 2.0 ** -6, (1 + f / 8) * torch.exp2(e.float() - 7))
    v = torch.where(i >= 128, -v, v)
    v[127] = v[255] = math.nan
    return v[codes.long()]


def _round8(x):
    """64-bit values to the nearest that 8 bits stand for, ties to the even one, those beyond the largest to that."""
    e = torch.clamp(torch.frexp(x)[1] - 1, min=-6)
    step = torch.exp2((e - 3).double())
    return torch.clamp(torch.round(x / step) * step, -448.0, 448.0)


def _places_of(seqs, total):
    """Per row in order of the sequences: its sequence, its row in the operands and its position."""
    first, count, start = (seqs[:, i].long() for i in range(3))
    seq = torch.repeat_interleave(torch.arange(len(first), device=first.device), count, output_size=total)
    i = torch.arange(total, device=first.device) - (torch.cumsum(count, 0) - count)[seq]
    return seq, first[seq] + i, start[seq] + i


def _rotate(x, angle, rot, inter):
    """x [rows][heads][dh] with its first `rot` values of every head turned by angle [rows][rot / 2], in 64 bits."""
    x = x.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = (x[:, :, 0:rot:2], x[:, :, 1:rot:2]) if inter else (x[:, :, :rot // 2], x[:, :, rot // 2:rot])
    u, v = a * c - b * s, b * c + a * s
    y = torch.stack((u, v), -1).flatten(2) if inter else torch.cat((u, v), 2)
    return torch.cat((y, x[:, :, rot:]), 2)


def _plain(st):
    return _plain_append(st) if st["case"]["kind"] == "append" else _plain_attend(st)


def _plain_append(st):
    case = st["case"]
    hq, hk, dh, page = case["heads"], case["kv_heads"], case["dh"], case["page"]
    seq, row, pos = _places_of(st["seqs"], sum(t[1] for t in table(case)))
    angle = pos[:, None].double() * st["freq"].double()
    x = st["qkv"][row]
    q = _rotate(x[:, :hq * dh].view(-1, hq, dh), angle, case["rot"], case["inter"])
    st["out"][row] = q.flatten(1).to(st["out"].dtype)
    k = _rotate(x[:, hq * dh:(hq + hk) * dh].view(-1, hk, dh), angle, case["rot"], case["inter"])
    v = x[:, (hq + hk) * dh:].view(-1, hk, dh).double()
    table_row = st["seqs"][:, 3].long()
    at = st["places"][table_row[seq], pos // page].long()
    if case["cache"] == "bf16":
        st["kc"][at, :, pos % page] = k.to(torch.bfloat16)
        st["vc"][at, :, pos % page] = v.to(torch.bfloat16)
        return {"q": st["out"], "k": st["kc"], "v": st["vc"]}
    out = {"q": st["out"]}
    # a sequence's touched blocks, one behind another; the first may hold tokens from before
    bseq, brow, bpos = _places_of(st["back"], st["mb"])
    start = st["seqs"][:, 2].long()
    count = torch.where(st["back"][:, 1] > 0, (st["back"][:, 1].long() + BLOCK - 1) // BLOCK, 0)
    first_block = torch.cumsum(count, 0) - count
    blocks = -(-st["mb"] // BLOCK) + len(count)
    of_new = first_block[seq] + pos // BLOCK - start[seq] // BLOCK
    of_back = first_block[bseq] + bpos // BLOCK - start[bseq] // BLOCK
    page_back = st["places"][table_row[bseq], bpos // page].long()
    old = bpos < start[bseq]
    for name, new in (("k", k), ("v", v)):
        codes, scales = st[name + "c"][page_back, :, bpos % page], st[name + "s"][page_back, :, bpos % page // BLOCK]
        top = torch.zeros(blocks, hk, dtype=torch.float64, device=new.device)
        top.index_reduce_(0, of_new, new.abs().amax(-1), "amax")
        frac, e = torch.frexp(top)  # the least power of two of which 448 times reach the largest
        e = torch.clamp(torch.where(frac > 0.875, e - 8, e - 9), min=-117)
        was = torch.where(old[:, None], scales.long() - 127, -117)
        e = e.long().index_reduce(0, of_back, was, "amax")
        step = torch.exp2(e.double())
        kept = _values8(codes).double() * torch.exp2(scales.double() - 127)[:, :, None]
        whole = torch.where(old[:, None, None], kept, 0.0)
        whole[~old] = new
        whole = _round8(whole / step[of_back][:, :, None]) * step[of_back][:, :, None]
        rows = torch.zeros(st["mb"], hk * dh, dtype=torch.bfloat16, device=new.device)
        rows[brow] = whole.flatten(1).to(torch.bfloat16)
        out[name] = rows
    return out


def _plain_attend(st):
    case = st["case"]
    hq, hk, dh, page, n = case["heads"], case["kv_heads"], case["dh"], case["page"], case["streams"]
    group, R, T = hq // hk, st["max_rows"], st["max_len"]
    seq, row, pos = _places_of(st["seqs"], sum(t[1] for t in table(case)))
    start, count = st["seqs"][:, 2].long(), st["seqs"][:, 1].long()
    q = torch.zeros(n, R, hq * dh, device=row.device)
    q[seq, pos - start[seq]] = st["q"][row].float()
    q = q.view(n, R, hk, group, dh).permute(0, 2, 3, 1, 4).reshape(n, hk, group * R, dh)
    j = torch.arange(T, device=row.device)
    at = st["places"][st["seqs"][:, 3].long()][:, j // page].long()  # [n][T]
    there = at >= 0
    at = at.clamp(min=0)

    def cached(name):
        c = st[name + "c"][at, :, j % page]  # [n][T][heads][dh]
        if case["cache"] == "e4m3":
            c = _values8(c) * torch.exp2(st[name + "s"][at, :, j % page // BLOCK].float() - 127)[..., None]
        return c.float().permute(0, 2, 1, 3).contiguous()

    s = torch.matmul(q, cached("k").transpose(2, 3).contiguous()) * (1 / math.sqrt(dh))
    i = start[:, None] + torch.arange(R, device=row.device)  # positions [n][R]
    see = (j <= i[:, :, None]) & there[:, None]
    if case["window"]:
        see &= (j > i[:, :, None] - case["window"]) | (j < case["sinks"])
    s = s.view(n, hk, group, R, T)
    s.masked_fill_(~see[:, None, None], -math.inf)
    s -= s.amax(-1, keepdim=True).clamp(min=-3e38)
    s.exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(n, hk, group * R, T), cached("v")).view(n, hk, group, R, dh) / torch.where(total > 0, total, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, R, hq * dh)
    out = torch.zeros_like(st["out"])
    out[row] = o[seq, pos - start[seq]].to(out.dtype)
    return out


# ---- the same results in 64 bits -------------------------------------------------------------------


def _kept64(block):
    """A block's values in 8 bits, by the distances to all that its codes stand for, with the least sufficient scale of at
    least `floor`: block [tokens][heads][dh] and the exponents [heads]."""
    e, x = block
    mags = torch.tensor(sorted([f / 8 * 2.0 ** -6 for f in range(8)] +
                               [(1 + f / 8) * 2.0 ** (p - 7) for p in range(1, 16) for f in range(8) if (p, f) != (15, 7)]),
                        dtype=torch.float64, device=x.device)
    step = torch.exp2(e.double())[:, None]
    a = (x / step).abs()
    hi = torch.searchsorted(mags, a).clamp(max=len(mags) - 1)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - mags[lo], mags[hi] - a
    up = (dh < dl) | ((dh == dl) & (hi % 2 == 0))
    return torch.where(x < 0, -1.0, 1.0) * torch.where(up, mags[hi], mags[lo]) * step


def _exact_append(case, st):
    hq, hk, dh, page, rot = case["heads"], case["kv_heads"], case["dh"], case["page"], case["rot"]
    out = {"q": torch.zeros(st["m"], hq * dh, dtype=torch.float64, device="cuda")}
    whole = {n: st[n + "c"].double() for n in "kv"} if case["cache"] == "bf16" else \
        {n: torch.zeros(st["mb"], hk * dh, dtype=torch.float64, device="cuda") for n in "kv"}
    freq, back = st["freq"].double(), 0
    pairs = torch.arange(rot // 2, device="cuda")
    a, b = (2 * pairs, 2 * pairs + 1) if case["inter"] else (pairs, pairs + rot // 2)
    for first, rows, start, row in table(case):
        if not rows:
            continue
        pos = torch.arange(start, start + rows, device="cuda")
        turn = torch.polar(torch.ones(rows, rot // 2, dtype=torch.float64, device="cuda"), pos[:, None].double() * freq)[:, None]
        x = st["qkv"][first:first + rows].double().view(rows, hq + 2 * hk, dh)
        z = torch.complex(x[:, :hq + hk][:, :, a], x[:, :hq + hk][:, :, b]) * turn
        y = x.clone()
        y[:, :hq + hk, a], y[:, :hq + hk, b] = z.real, z.imag
        out["q"][first:first + rows] = y[:, :hq].reshape(rows, -1)
        new = {"k": y[:, hq:hq + hk], "v": y[:, hq + hk:]}
        places = st["places"][row].long()
        for n in "kv":
            if case["cache"] == "bf16":
                whole[n][places[pos // page], :, pos % page] = new[n]
                continue
            begin, end, got = start // BLOCK * BLOCK, start + rows, []
            before = torch.arange(begin, start, device="cuda")
            p = places[before // page]
            old_e = st[n + "s"][p, :, before % page // BLOCK].long() - 127
            old = st[n + "c"][p, :, before % page].view(torch.float8_e4m3fn).double() * torch.exp2(old_e.double())[..., None]
            # the open block, then all whole and last ones side by side
            head = new[n][:max(0, min(rows, begin + BLOCK - start))]
            tail = new[n][len(head):]
            for fresh, kept, floor in ((head, old, old_e), (tail, old[:0], old_e[:0])):
                if not len(fresh):
                    continue
                blocks = -(-(len(fresh) + len(kept)) // BLOCK)
                top = torch.zeros(blocks * BLOCK, hk, dtype=torch.float64, device="cuda")
                top[len(kept):len(kept) + len(fresh)] = fresh.abs().amax(-1)
                top = top.view(blocks, BLOCK, hk).amax(1)
                e = torch.ceil(torch.log2(top / 448))
                e = torch.where(448 * torch.exp2(e - 1) >= top, e - 1, torch.where(448 * torch.exp2(e) < top, e + 1, e))
                e = e.clamp(min=-117.0)
                if len(kept):
                    e[0] = torch.maximum(e[0], floor.amax(0).double())
                e = e.repeat_interleave(BLOCK, 0)[:len(kept) + len(fresh)]
                got.append(_kept64((e.flatten(), torch.cat((kept, fresh)).flatten(0, 1))).view(-1, hk * dh))
            got = torch.cat(got)
            whole[n][back:back + len(got)] = got
        back += rows + start % BLOCK
    return {**out, **whole}


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, st)
    hq, hk, dh, page = case["heads"], case["kv_heads"], case["dh"], case["page"]
    out = torch.zeros(st["m"], hq, dh, dtype=torch.float64, device="cuda")
    for first, rows, start, row in table(case):
        j = torch.arange(start + rows, device="cuda")
        p = st["places"][row].long()[j // page]
        i = start + torch.arange(rows, device="cuda")[:, None]
        hidden = (j > i) | (p < 0)
        if case["window"]:
            hidden |= (i - j >= case["window"]) & (j >= case["sinks"])
        p = p.clamp(min=0)
        for h in range(hk if rows else 0):
            k, v = st["kc"][p, h, j % page], st["vc"][p, h, j % page]
            if case["cache"] == "e4m3":
                k, v = k.view(torch.float8_e4m3fn).double(), v.view(torch.float8_e4m3fn).double()
                k = torch.ldexp(k, st["ks"][p, h, j % page // BLOCK].long()[:, None] - 127)
                v = torch.ldexp(v, st["vs"][p, h, j % page // BLOCK].long()[:, None] - 127)
            k, v = k.double(), v.double()
            for u in range(h * hq // hk, (h + 1) * hq // hk):
                s = st["q"][first:first + rows, u * dh:(u + 1) * dh].double() @ k.t() / math.sqrt(dh)
                s[hidden] = -math.inf
                out[first:first + rows, u] = torch.exp(s - torch.logsumexp(s, 1, keepdim=True)) @ v
    return out.flatten(1)

"""What is measured of the paged-cache operators: cases, inputs, plain forms and exact values.

The operators serve a continuous batch: every sequence keeps its keys and values in pages of a shared pool,
`block_table[b]` lists a sequence's pages in order and `lens[b]` says how many rows it holds, both on the device.

* append   rotates the q and k heads of a stacked projection [tokens, (hq + 2 hkv) d] by the tokens' positions (one
           axis, or several axes that share the frequencies) and stores the k and v heads as the last rows of their
           sequences; pages hold bf16 or NVFP4 rows.
* decode   attention of the last (one or few) tokens of every sequence over its pages.
* prompt   the same for ragged runs of query tokens (`cu_q`), fresh prompts and chunks over an earlier part alike.

A query at position p sees the rows k < len with k <= p and, where there is a window, p - k < window; rows
k < prefix[b] are seen by every query of the sequence. The score is cap * tanh(s / cap) (s = scale * q.k; s itself
without a cap) minus slope[head] * |p - k|.

With `own` false the operators run in elementary torch operations, with `own` true through maryml_b200.paged.
"""
import math
import random

import numpy as np
import torch

own = False

THETA = 1.0e6            # the rotary base of the repository's decoder layer
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _append(name, **kw):
    c = {"name": name, "op": "append", "batch": 1, "q_lo": 1, "q_hi": 1, "past_lo": 0, "past_hi": 0, "heads": 32,
         "kv_heads": 8, "d": 128, "page": 64, "elem": "bf16", "axes": 1, "shape_seed": 1}
    c.update(kw)
    return c


def _attn(name, op, **kw):
    c = {"name": name, "op": op, "batch": 1, "q_lo": 1, "q_hi": 1, "past_lo": 0, "past_hi": 0, "heads": 32, "kv_heads": 8,
         "d": 128, "page": 64, "elem": "bf16", "softcap": 0.0, "window": 0, "slopes": False, "prefix": 0, "q_gain": 1.0,
         "shape_seed": 1}
    c.update(kw)
    return c


def listed():
    """Sizes of the repository's decoder layer (32 query heads, 8 KV heads of 128; 64 sequences over 4096 rows; 32 over
    32768; prompts of 8192 tokens) and smaller ones around them."""
    return [
        # one user's next token: launch latency is all there is
        _append("append 1 token", past_lo=776, past_hi=776, page=16),
        # a serving step of 64 sequences
        _append("append 64 sequences", batch=64, past_lo=3500, past_hi=4500),
        # ragged prompts joining the batch in one pass
        _append("append 8192 prompt tokens", batch=5, q_lo=700, q_hi=2577, page=128, shape_seed=2),
        # image and video tokens (time, height, width) into a cache of four-bit rows
        _append("append 3 axes nvfp4", batch=3, q_lo=901, q_hi=2115, past_lo=5, past_hi=77, page=32, elem="nvfp4", axes=3),
        # one user's next token
        _attn("decode 1 x 777", "decode", past_lo=776, past_hi=776, page=16),
        # a serving step, lengths spread as they are in a running batch
        _attn("decode 64 x 4096", "decode", batch=64, past_lo=1500, past_hi=6700),
        # long contexts
        _attn("decode 32 x 32768", "decode", batch=32, past_lo=32767, past_hi=32767, page=256),
        # capped scores over four-bit rows, first rows and a window of the last ones visible, two draft tokens to check
        _attn("decode 32 nvfp4 cap window", "decode", batch=32, q_lo=2, q_hi=2, past_lo=9000, past_hi=18000, page=48,
              elem="nvfp4", softcap=30.0, window=8000, prefix=64, q_gain=4.0),
        # short ragged prompts of a chat front end, small heads
        _attn("prompt short ragged", "prompt", batch=7, q_lo=5, q_hi=311, heads=16, kv_heads=4, d=64, page=16),
        # a fresh long prompt
        _attn("prompt 8192", "prompt", q_lo=8192, q_hi=8192),
        # chunks of prompts over what earlier chunks left in the cache, capped scores
        _attn("prompt chunks cap", "prompt", batch=2, q_lo=500, q_hi=530, past_lo=11000, past_hi=13000, page=128,
              softcap=50.0, q_gain=4.0),
        # distance bias and a two-way prefix (an image before its text) over four-bit rows
        _attn("prompt slopes prefix nvfp4", "prompt", batch=3, q_lo=1200, q_hi=2000, past_lo=0, past_hi=300, page=32,
              elem="nvfp4", slopes=True, prefix=577),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "prompt"])
    d = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "d": d, "page": rng.choice([16, 32, 48, 64, 128, 256]),
         "elem": rng.choice(["bf16", "bf16", "nvfp4"]), "shape_seed": rng.randrange(1 << 20)}
    if op == "append":
        tokens = _log(rng, 1, 8192)
        c["batch"] = _log(rng, 1, min(tokens, 64))
        c["q_lo"] = max(1, tokens // (2 * c["batch"]))
        c["q_hi"] = max(c["q_lo"], (3 * tokens) // (2 * c["batch"]))
        c["past_lo"] = rng.choice([0, rng.randrange(1, 100)])
        c["past_hi"] = c["past_lo"] + _log(rng, 1, 2000)
        c["axes"] = rng.choice([1, 3])
        return c
    c["softcap"] = rng.choice([0.0, 0.0, 20.0, 50.0])
    c["q_gain"] = rng.choice([1.0, 4.0])
    c["slopes"] = rng.random() < 0.3
    if op == "decode":
        c["batch"] = _log(rng, 1, 64)
        top = min(32768, 700000 // c["batch"])
        mean = _log(rng, 1, top)
        c["q_lo"] = c["q_hi"] = rng.choice([1, 1, 1, 3])
    else:
        c["batch"] = _log(rng, 1, 6)
        q = _log(rng, 2, 3500)
        c["q_lo"], c["q_hi"] = max(1, q // 2), q
        mean = _log(rng, 1, max(2, int(1.2e9 / (c["batch"] * heads * q))) if q < 900 else 600)
        mean = min(mean, 20000)
    c["past_lo"], c["past_hi"] = mean // 2, mean
    c["window"] = rng.choice([0, 0, _log(rng, 1, 4 * mean + 16)])
    c["prefix"] = rng.choice([0, 0, _log(rng, 1, mean + c["q_hi"])])
    return c


def _lengths(case):
    """Query tokens and lengths (query tokens included) of the sequences of a case: part of the case, not of the seed."""
    r = np.random.RandomState(case["shape_seed"])
    q = r.randint(case["q_lo"], case["q_hi"] + 1, case["batch"]).astype(np.int64)
    past = r.randint(case["past_lo"], case["past_hi"] + 1, case["batch"]).astype(np.int64)
    return q, past + q


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    q_len, lens = _lengths(case)
    batch, page, kvh, d = case["batch"], case["page"], case["kv_heads"], case["d"]
    per_seq = -(-lens // page)
    pages = int(per_seq.sum()) + 3
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).cpu().numpy()
    table = np.full((batch, int(per_seq.max()) + 1), -1, dtype=np.int32)
    at = 0
    for b in range(batch):                       # the pages of a sequence lie anywhere in the pool
        table[b, :per_seq[b]] = order[at:at + per_seq[b]]
        at += int(per_seq[b])
    s = {"case": dict(case), "table": torch.from_numpy(table).to(dev), "lens": torch.from_numpy(lens.astype(np.int32)).to(dev),
         "cu_q": torch.from_numpy(np.concatenate([[0], np.cumsum(q_len)]).astype(np.int32)).to(dev)}
    for name in ("k", "v"):
        if case["elem"] == "bf16":
            s[name] = torch.empty((pages, page, kvh, d), dtype=torch.bfloat16, device=dev).normal_(generator=g)
            s[name + "_scales"] = None
        else:
            # codes of all sixteen values under scales of a quarter to a half: rows of unit size
            s[name] = torch.randint(0, 256, (pages, page, kvh * d // 2), dtype=torch.uint8, device=dev, generator=g)
            s[name + "_scales"] = torch.randint(0x28, 0x31, (pages, page, kvh * d // 16), dtype=torch.uint8, device=dev,
                                                generator=g)
    total = int(q_len.sum())
    if case["op"] == "append":
        s["qkv"] = torch.empty((total, (case["heads"] + 2 * kvh) * d), dtype=torch.bfloat16, device=dev).normal_(generator=g)
        f = np.arange(d // 2, dtype=np.float64)
        s["inv_freq"] = torch.from_numpy((1.0 / THETA ** (2.0 * f / d)).astype(np.float32)).to(dev)
        if case["axes"] > 1:
            s["positions"] = torch.randint(0, 5000, (case["axes"], total), dtype=torch.int32, device=dev, generator=g)
            s["sections"] = (d // 8, d // 2 - d // 8 - 3 * d // 16, 3 * d // 16)
        else:
            s["positions"] = s["sections"] = None
        return s
    shape = (batch, case["q_hi"], case["heads"], d) if case["op"] == "decode" else (total, case["heads"], d)
    s["q"] = (torch.empty(shape, device=dev).normal_(generator=g) * case["q_gain"]).to(torch.bfloat16)
    s["scale"] = 1.0 / math.sqrt(d)
    s["slopes"] = None
    if case["slopes"]:
        h = torch.arange(1, case["heads"] + 1, device=dev, dtype=torch.float32)
        s["slopes"] = torch.exp2(-8.0 * h / case["heads"])
    s["prefix"] = None
    if case["prefix"]:
        s["prefix"] = torch.randint(case["prefix"] // 2, case["prefix"] + 1, (batch,), dtype=torch.int32, device=dev, generator=g)
    return s


# ---- the operators through the framework ------------------------------------------------
def _own(s):
    from maryml_b200 import nvfp4
    from maryml_b200.paged import PagedCache, paged_append, paged_attention_decode, paged_attention_prompt
    c = s["case"]
    cache = PagedCache(s["k"], s["v"], s["k_scales"], s["v_scales"], head_dim=c["d"])
    if c["op"] == "append":
        q = paged_append(s["qkv"], cache, s["table"], s["lens"], s["inv_freq"], cu_q=s["cu_q"], positions=s["positions"],
                         sections=s["sections"])
        if c["elem"] == "bf16":
            return {"q": q, "k": s["k"], "v": s["v"]}
        rows, width = s["k"].shape[0] * c["page"], c["kv_heads"] * c["d"]
        values = lambda name: nvfp4.dequantize(s[name].view(rows, -1), s[name + "_scales"].view(rows, -1), 1.0, rows, width,
                                               torch.bfloat16)
        return {"q": q, "k": values("k"), "v": values("v")}
    terms = {"scale": s["scale"], "softcap": c["softcap"], "window": c["window"], "slopes": s["slopes"], "prefix": s["prefix"]}
    if c["op"] == "decode":
        return paged_attention_decode(s["q"], cache, s["table"], s["lens"], **terms)
    return paged_attention_prompt(s["q"], s["cu_q"], cache, s["table"], s["lens"], **terms)


# ---- plain forms --------------------------------------------------------------------------
def _values(codes, scales):
    """NVFP4 rows [.., width / 2] and [.., width / 16] -> f32 [.., width]."""
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float32, device=codes.device)
    pair = torch.stack((codes & 15, codes >> 4), dim=-1).int()
    v = table[pair].view(*codes.shape[:-1], -1, 16)
    return (v * scales.view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def _quantize(rows):
    """bf16 rows [n, width] -> (codes, scales): per 16 values the scale e4m3(min(amax / 6, 448)), the codes
    e2m1(x * (1 / scale)) with ties to the even code, both in 32 bits."""
    x = rows.float().view(rows.shape[0], -1, 16)
    scales = (x.abs().amax(-1) / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
    back = scales.float()
    y = x * torch.where(back > 0, 1.0 / back, torch.zeros_like(back)).unsqueeze(-1)
    a = y.abs()
    code = ((a > 0.25).int() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * torch.signbit(y)).to(torch.uint8).view(rows.shape[0], -1, 2)
    return code[..., 0] | (code[..., 1] << 4), scales.view(torch.uint8)


def _tokens(s):
    """Per query token: its sequence and its row there."""
    cu = s["cu_q"].long()
    q_len = cu[1:] - cu[:-1]
    total = s["qkv"].shape[0] if "qkv" in s else s["q"].shape[0]
    seq = torch.repeat_interleave(torch.arange(cu.numel() - 1, device=cu.device), q_len, output_size=total)
    row = s["lens"].long()[seq] - q_len[seq] + torch.arange(total, device=cu.device) - cu[seq]
    return seq, row


def _plain_append(s):
    c = s["case"]
    hq, kvh, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    seq, row = _tokens(s)
    total = seq.numel()
    if s["positions"] is None:
        pos = row.double().unsqueeze(1)
    else:
        axis = torch.repeat_interleave(torch.arange(c["axes"], device=row.device),
                                       torch.tensor(s["sections"], device=row.device), output_size=d // 2)
        pos = s["positions"].double().t()[:, axis]
    angle = pos * s["inv_freq"].double()                   # far positions lose their fraction in 32 bits
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    x = s["qkv"].view(total, hq + 2 * kvh, d)
    lo, hi = x[:, :hq + kvh, :d // 2].float(), x[:, :hq + kvh, d // 2:].float()
    rot = torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), dim=-1).to(torch.bfloat16)
    at = s["table"][seq, row // page].long() * page + row % page
    for name, new in (("k", rot[:, hq:]), ("v", x[:, hq + kvh:])):
        if c["elem"] == "bf16":
            s[name].view(-1, kvh, d)[at] = new
        else:
            codes, scales = _quantize(new.reshape(total, -1))
            s[name].view(-1, kvh * d // 2)[at] = codes
            s[name + "_scales"].view(-1, kvh * d // 16)[at] = scales
    out = {"q": rot[:, :hq].contiguous(), "k": s["k"], "v": s["v"]}
    if c["elem"] != "bf16":
        rows = s["k"].shape[0] * page
        out["k"] = _values(s["k"], s["k_scales"]).view(rows, -1).to(torch.bfloat16)
        out["v"] = _values(s["v"], s["v_scales"]).view(rows, -1).to(torch.bfloat16)
    return out


def _gather(s, name):
    """The rows of all sequences, padded to the longest: f32 [batch, kv_heads, rows, d]."""
    c = s["case"]
    pages = s["table"].clamp(min=0).long()
    x = s[name][pages]
    x = x.float() if c["elem"] == "bf16" else _values(x, s[name + "_scales"][pages])
    return x.view(c["batch"], -1, c["kv_heads"], c["d"]).transpose(1, 2)


def _plain_attention(s):
    c = s["case"]
    batch, heads, kvh, d = c["batch"], c["heads"], c["kv_heads"], c["d"]
    group = heads // kvh
    if c["op"] == "decode":
        q, nq = s["q"], s["q"].shape[1]
        pos = s["lens"].long().unsqueeze(1) - nq + torch.arange(nq, device=q.device)
    else:
        seq, row = _tokens(s)
        slot = torch.arange(seq.numel(), device=row.device) - s["cu_q"].long()[seq]
        nq = int(_lengths(c)[0].max())
        q = s["q"].new_zeros((batch, nq, heads, d))
        q[seq, slot] = s["q"]
        pos = torch.zeros((batch, nq), dtype=torch.long, device=row.device)
        pos[seq, slot] = row
    k, v = _gather(s, "k"), _gather(s, "v")
    rows = k.shape[2]
    qg = q.float().view(batch, nq, kvh, group, d).permute(0, 2, 3, 1, 4).reshape(batch, kvh, group * nq, d)
    x = torch.matmul(qg, k.transpose(2, 3)).mul_(s["scale"]).view(batch, kvh, group, nq, rows)
    if c["softcap"]:
        x = torch.tanh_(x.div_(c["softcap"])).mul_(c["softcap"])
    kpos = torch.arange(rows, device=q.device)
    away = pos.unsqueeze(2) - kpos                          # [batch, nq, rows]
    if s["slopes"] is not None:
        x -= s["slopes"].view(1, kvh, group, 1, 1) * away.abs().float().view(batch, 1, 1, nq, rows)
    seen = away >= 0
    if c["window"]:
        seen &= away < c["window"]
    if s["prefix"] is not None:
        seen |= kpos < s["prefix"].view(batch, 1, 1)
    seen &= kpos < s["lens"].view(batch, 1, 1)
    x.masked_fill_(~seen.view(batch, 1, 1, nq, rows), float("-inf"))
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(batch, kvh, group * nq, rows), v).view(batch, kvh, group, nq, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    o = o.permute(0, 3, 1, 2, 4).reshape(batch, nq, heads, d).to(torch.bfloat16)
    return o if c["op"] == "decode" else o[seq, slot]


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attention(state)


# ---- what a pass cannot do without ----------------------------------------------------------
def _seen_rows(case):
    """Per sequence: (rows of keys and values some query sees, query-key pairs in all), the prefix at its mean."""
    q_len, lens = _lengths(case)
    pre = np.minimum(int(case["prefix"] * 0.75), lens)
    rows, pairs = 0.0, 0.0
    for b in range(case["batch"]):
        p = np.arange(lens[b] - q_len[b], lens[b], dtype=np.float64)
        first = np.maximum(0, p + 1 - case["window"]) if case["window"] else np.zeros_like(p)
        pairs += float(np.sum(np.maximum(pre[b], p + 1) - first + np.minimum(first, pre[b])))
        lo = max(int(first[0]), int(pre[b])) if len(p) else 0
        rows += float(lens[b] - lo + pre[b])
    return rows, pairs


def work(case):
    q_len, lens = _lengths(case)
    total, width = int(q_len.sum()), case["kv_heads"] * case["d"]
    per_value = 2.0 if case["elem"] == "bf16" else 0.5625
    q_bytes = total * case["heads"] * case["d"] * 2.0
    if case["op"] == "append":
        # read the projection, write the rotated queries and the rows; 3 operations per rotated value
        return {"bytes": 2 * q_bytes + 2 * total * width * (2.0 + per_value),
                "flops": 3.0 * total * (case["heads"] * case["d"] + width)}
    rows, pairs = _seen_rows(case)
    return {"bytes": 2 * q_bytes + 2 * rows * width * per_value, "flops": 4.0 * pairs * case["heads"] * case["d"]}


# ---- exact values -------------------------------------------------------------------------------
def _e_rows(s, name):
    """All rows of a pool in 64 bits: [pages * page, kv_heads, d]."""
    c = s["case"]
    if c["elem"] == "bf16":
        return s[name].double().reshape(-1, c["kv_heads"], c["d"])
    b, sc = s[name].reshape(-1, c["kv_heads"], c["d"] // 2).long(), s[name + "_scales"].reshape(-1, c["kv_heads"], c["d"] // 16).long()

    def e2m1(n):
        e, m = (n >> 1) & 3, (n & 1).double()
        mag = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.double() - 1))
        return torch.where(n >= 8, -mag, mag)

    e, m = (sc >> 3) & 15, (sc & 7).double()
    scale = torch.where(e == 0, m / 512, (1 + m / 8) * torch.exp2(e.double() - 7))
    v = torch.empty((*b.shape[:2], c["d"]), dtype=torch.float64, device=b.device)
    v[..., 0::2], v[..., 1::2] = e2m1(b & 15), e2m1(b >> 4)
    return v * scale.repeat_interleave(16, dim=-1)


def _e_nvfp4(rows):
    """What a bf16 row, given in 64 bits, is after four-bit storage: nearest of the sixteen values, even code on a tie,
    of x times the 32-bit reciprocal of the block's e4m3 scale."""
    x = rows.reshape(rows.shape[0], -1, 16)
    want = (x.abs().amax(-1) / 6.0).clamp(max=448.0)
    e = torch.floor(torch.log2(want.clamp(min=2.0 ** -20))).clamp(min=-6.0)
    scale = torch.round(want / torch.exp2(e - 3)) * torch.exp2(e - 3)         # torch.round: ties to even
    r = torch.where(scale > 0, 1.0 / scale.clamp(min=2.0 ** -9), torch.zeros_like(scale)).float().double()
    y = (x * r.unsqueeze(-1)).float().double()
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2.0, 0.5, torch.where(a < 4.0, 1.0, 2.0)).double()
    near = torch.round(a / step) * step
    near = torch.where((a == 5.0), torch.full_like(a, 4.0), near)
    return (torch.sign(y) * near * scale.unsqueeze(-1)).reshape(rows.shape)


def _e_append(s):
    c = s["case"]
    hq, kvh, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    q_len, lens = _lengths(c)
    k, v = _e_rows(s, "k"), _e_rows(s, "v")
    x = s["qkv"].double().reshape(-1, hq + 2 * kvh, d)
    freq = s["inv_freq"].double()
    q = torch.empty((x.shape[0], hq, d), dtype=torch.float64, device=x.device)
    t0 = 0
    for b in range(c["batch"]):
        n = int(q_len[b])
        row = torch.arange(int(lens[b]) - n, int(lens[b]), device=x.device)
        if s["positions"] is None:
            angle = row.double()[:, None] * freq
        else:
            parts, f0 = [], 0
            for ax, size in enumerate(s["sections"]):
                parts.append(s["positions"][ax, t0:t0 + n].double()[:, None] * freq[f0:f0 + size])
                f0 += size
            angle = torch.cat(parts, dim=1)
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        z = torch.complex(x[t0:t0 + n, :hq + kvh, :d // 2], x[t0:t0 + n, :hq + kvh, d // 2:]) * turn
        rot = torch.cat((z.real, z.imag), dim=-1)
        q[t0:t0 + n] = rot[:, :hq]
        new_k, new_v = rot[:, hq:], x[t0:t0 + n, hq + kvh:]
        if c["elem"] != "bf16":                            # four-bit rows store the bf16 row
            new_k = _e_nvfp4(new_k.to(torch.bfloat16).double().reshape(n, -1)).view(n, kvh, d)
            new_v = _e_nvfp4(new_v.reshape(n, -1)).view(n, kvh, d)
        at = s["table"][b].long()[row // page] * page + row % page
        k[at], v[at] = new_k, new_v
        t0 += n
    shape = s["k"].shape if c["elem"] == "bf16" else (s["k"].shape[0] * page, kvh * d)
    return {"q": q, "k": k.view(shape), "v": v.view(shape)}


def _e_attention(s):
    c = s["case"]
    heads, kvh, d, page = c["heads"], c["kv_heads"], c["d"], c["page"]
    group = heads // kvh
    q_len, lens = _lengths(c)
    flat = s["q"].reshape(-1, heads, d)
    out = torch.zeros(flat.shape, dtype=torch.float64, device=flat.device)
    wide = {"case": c, "k_scales": None, "v_scales": None}
    t0 = 0
    for b in range(c["batch"]):
        n, length = int(q_len[b]), int(lens[b])
        used = s["table"][b, :-(-length // page)].long()
        for name in ("k", "v"):
            wide[name] = s[name][used]
            if c["elem"] != "bf16":
                wide[name + "_scales"] = s[name + "_scales"][used]
        k, v = _e_rows(wide, "k")[:length], _e_rows(wide, "v")[:length]
        kpos = torch.arange(length, device=flat.device)
        for i0 in range(0, n, 1024):
            i1 = min(n, i0 + 1024)
            p = torch.arange(length - n + i0, length - n + i1, device=flat.device)[:, None]
            seen = kpos <= p
            if c["window"]:
                seen = seen & (kpos > p - c["window"])
            if s["prefix"] is not None:
                seen = seen | (kpos < s["prefix"][b])
            for h in range(heads):
                x = flat[t0 + i0:t0 + i1, h].double() @ k[:, h // group].t() * s["scale"]
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                if s["slopes"] is not None:
                    x = x - s["slopes"][h].double() * (p - kpos).abs()
                x = torch.where(seen, x, torch.full_like(x, float("-inf")))
                out[t0 + i0:t0 + i1, h] = torch.nan_to_num(torch.softmax(x, dim=-1), nan=0.0) @ v[:, h // group]
        t0 += n
    return out.view(s["q"].shape)


def exact(case, seed):
    s = prepare(case, seed)
    return _e_append(s) if case["op"] == "append" else _e_attention(s)

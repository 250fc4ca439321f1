"""Cases for the paged-cache serving operators: the rotating append
(``fmha_rope_append``), single-token attention over the paged cache
(``fmha_paged_decode``) and attention over packed prompts (``fmha_prompt``).

With ``own`` false, ``run`` computes an operator in its plain form with
elementary torch operations in fp32; with ``own`` true it calls fmha_b200.
Sequence lengths belong to the case (drawn from its ``lens`` number), values
and page numbers to the seed.
"""
import math
import random

import torch

own = False

F8_MAX = 448.0  # largest e4m3 value
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": torch.float8_e4m3fn}


def listed():
    return [
        # One user's next token: the smallest call of a decode step, all latency.
        dict(name="append 1 token", op="append", batch=1, lo=1, hi=1, past=700, hq=32, hkv=8, d=128,
             page=16, order="hnd", rot=128, inter=False, dtype="bf16", cache="bf16", keep=False, lens=1),
        # A decode step of a full server: one token each of many sequences, 8-bit cache,
        # a partly rotated head in interleaved pairs, pages stored token by token.
        dict(name="append 509 tokens e4m3", op="append", batch=509, lo=1, hi=1, past=300, hq=32, hkv=16,
             d=256, page=32, order="nhd", rot=64, inter=True, dtype="bf16", cache="e4m3", keep=False, lens=2),
        # A batch of prompts of all lengths, packed; the rotated keys are also kept for the prompt's attention.
        dict(name="append prompts 18k tokens", op="append", batch=23, lo=31, hi=4096, past=0, hq=32, hkv=8,
             d=128, page=64, order="hnd", rot=128, inter=False, dtype="bf16", cache="bf16", keep=True, lens=3),
        # The shortest conversation: one sequence of about a hundred tokens.
        dict(name="decode 1x137", op="decode", batch=1, lo=137, hi=137, hq=16, hkv=16, d=128,
             page=16, order="hnd", dtype="bf16", cache="bf16", out="fp16", lens=4),
        # A busy server: ragged conversations, four query heads to each cached head.
        dict(name="decode 131 ragged to 8k", op="decode", batch=131, lo=16, hi=8192, hq=32, hkv=8, d=128,
             page=16, order="hnd", dtype="bf16", cache="bf16", out="bf16", lens=5),
        # One long document: only splitting its length fills the card.
        dict(name="decode 1x131071", op="decode", batch=1, lo=131071, hi=131071, hq=32, hkv=4, d=128,
             page=64, order="nhd", dtype="fp16", cache="fp16", out="fp16", lens=6),
        # Wide heads on an 8-bit cache, two query heads to each cached head.
        dict(name="decode 61 e4m3 wide heads", op="decode", batch=61, lo=200, hi=8192, hq=32, hkv=16, d=256,
             page=32, order="hnd", dtype="bf16", cache="e4m3", out="bf16", lens=7),
        # No grouping (each query head has its own cached head), fp16, medium lengths.
        dict(name="decode 48 ungrouped", op="decode", batch=48, lo=100, hi=2048, hq=32, hkv=32, d=128,
             page=16, order="hnd", dtype="fp16", cache="fp16", out="fp16", lens=8),
        # A single short question.
        dict(name="prompt 1x100", op="prompt", batch=1, lo=100, hi=100, past=0, hq=16, hkv=16, d=128,
             causal=True, dtype="bf16", out="fp16", lens=9),
        # Prompts of all lengths packed together, four query heads to each key head.
        dict(name="prompt 29 ragged to 1.5k", op="prompt", batch=29, lo=9, hi=1537, past=0, hq=32, hkv=8, d=128,
             causal=True, dtype="bf16", out="bf16", lens=10),
        # A long document: the tensor cores' case.
        dict(name="prompt 1x16384", op="prompt", batch=1, lo=16384, hi=16384, past=0, hq=16, hkv=4, d=128,
             causal=True, dtype="bf16", out="bf16", lens=11),
        # Wide heads in fp16, prompts that follow on earlier turns (more keys than queries).
        dict(name="prompt 5 after a prefix wide", op="prompt", batch=5, lo=500, hi=2500, past=1111, hq=16, hkv=2,
             d=256, causal=True, dtype="fp16", out="fp16", lens=12),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _lengths(case):
    """(new tokens, cached tokens before them) of each sequence; for decode (1, length - 1)."""
    rng = random.Random(case["lens"])
    new = [_log_int(rng, case["lo"], case["hi"]) for _ in range(case["batch"])]
    if case["op"] == "decode":
        return [1] * len(new), [n - 1 for n in new]
    return new, [rng.randint(case["past"] // 2, case["past"]) for _ in new]


def _draw_once(rng):
    op = rng.choice(("append", "decode", "prompt"))
    hkv = rng.choice((1, 2, 3, 4, 5, 8, 16))
    g = rng.choice((1, 2, 3, 4, 5, 6, 7, 8, 16))
    while hkv * g > 64:
        g = rng.choice((1, 2, 3, 4))
    d = rng.choice((128, 128, 256))
    c = dict(op=op, hq=hkv * g, hkv=hkv, d=d, dtype=rng.choice(("bf16", "bf16", "fp16")),
             lens=rng.randrange(1 << 20))
    if op != "prompt":
        c.update(page=rng.choice((1, 8, 16, 32, 48, 64, 128, 256)), order=rng.choice(("hnd", "nhd")),
                 cache=rng.choice((c["dtype"], c["dtype"], "e4m3")))
    if op == "append":
        step = rng.random() < 0.5
        hi = 1 if step else _log_int(rng, 2, 4096)
        c.update(batch=_log_int(rng, 1, 512 if step else 24), lo=1, hi=hi, past=rng.choice((0, 100, 2000)),
                 rot=rng.choice((d, d, d // 2, 48)), inter=rng.random() < 0.3, keep=rng.random() < 0.5)
    elif op == "decode":
        hi = _log_int(rng, 1, 131072)
        c.update(batch=_log_int(rng, 1, 256), lo=max(1, hi // rng.choice((1, 2, 50))), hi=hi,
                 out=rng.choice(("fp16", "bf16")))
    else:
        hi = _log_int(rng, 1, 8192)
        c.update(batch=_log_int(rng, 1, 32), lo=max(1, hi // rng.choice((1, 2, 50))), hi=hi,
                 past=rng.choice((0, 0, 77, 1024)), causal=rng.random() < 0.8, out=rng.choice(("fp16", "bf16")))
    return c


# The largest listed cases, and what the plain forms have room for.
_MOST_BYTES, _MOST_FLOPS, _MOST_PAIRS, _MOST_POOL = 0.8e9, 1.0e12, 4.0e9, 6.0e8


def draw(rng):
    while True:
        c = _draw_once(rng)
        new, past = _lengths(c)
        longest = max(n + p for n, p in zip(new, past))
        w = work(c)
        # Values of one pool (decode: of the padded cache that the plain form makes), and its scores.
        pool = c["hkv"] * c["d"] * (sum(new) + sum(past) if c["op"] == "append" else c["batch"] * longest)
        pairs = c["batch"] * c["hq"] * max(new) * longest if c["op"] == "prompt" else 0
        if (w["bytes"] <= _MOST_BYTES and w["flops"] <= _MOST_FLOPS and pairs <= _MOST_PAIRS
                and pool <= (_MOST_POOL if c["op"] == "append" else 4 * _MOST_POOL)):
            return c


def _pages(case):
    new, past = _lengths(case)
    return [-(-(n + p) // case["page"]) for n, p in zip(new, past)]


def _pool(case, pages, gen):
    """One pool of pages as [page, head, token, d], stored head by head or token by token."""
    shape = (pages, case["hkv"], case["page"], case["d"])
    if case["order"] == "nhd":
        shape = (pages, case["page"], case["hkv"], case["d"])
    pool = torch.randn(shape, device="cuda", generator=gen, dtype=torch.float16)
    if case["cache"] == "e4m3":
        pool *= 25.0  # with the scales in prepare, values of about one
    pool = pool.to(TYPES[case["cache"]])
    return pool.transpose(1, 2) if case["order"] == "nhd" else pool


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, past = _lengths(case)
    dt, hq, hkv, d = TYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    total = cu[-1]
    s = dict(case=case)
    i32 = dict(dtype=torch.int32, device="cuda")
    s["cu"] = torch.tensor(cu, **i32)
    s["seqlens"] = torch.tensor([n + p for n, p in zip(new, past)], **i32)
    s["longest_q"], s["longest"] = max(new), max(n + p for n, p in zip(new, past))

    if case["op"] == "prompt":
        # Queries, keys and values as a fused projection leaves them, one row a token, when
        # there is no prefix; else keys and values of prefix and prompt together.
        if case["past"]:
            kv_rows = sum(n + p for n, p in zip(new, past))
            s["q"] = torch.randn((total, hq, d), device="cuda", generator=gen).to(dt)
            kv = torch.randn((kv_rows, 2 * hkv, d), device="cuda", generator=gen).to(dt)
            s["k"], s["v"] = kv[:, :hkv], kv[:, hkv:]
            s["cu_kv"] = torch.cat([s["cu"][:1], torch.cumsum(s["seqlens"], 0).to(torch.int32)])
        else:
            qkv = torch.randn((total, hq + 2 * hkv, d), device="cuda", generator=gen).to(dt)
            s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
            s["cu_kv"] = s["cu"]
        return s

    counts = _pages(case)
    spare = 3
    s["pool_k"] = _pool(case, sum(counts) + spare, gen)
    s["pool_v"] = _pool(case, sum(counts) + spare, gen)
    order = torch.randperm(sum(counts) + spare, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros((len(counts), max(counts)), **i32)
    columns = torch.arange(max(counts), device="cuda")
    held = columns[None, :] < torch.tensor(counts, device="cuda")[:, None]
    table[held] = order[: sum(counts)]
    s["table"] = table
    s["k_scale"], s["v_scale"] = (0.04, 0.03) if case["cache"] == "e4m3" else (1.0, 1.0)
    if case["op"] == "decode":
        # Scores spread like a trained model's: some heads attend sharply.
        s["q"] = (torch.randn((total, hq, d), device="cuda", generator=gen)
                  * torch.rand((1, hq, 1), device="cuda", generator=gen) * 3).to(dt)
        return s
    qkv = torch.randn((total, hq + 2 * hkv, d), device="cuda", generator=gen).to(dt)
    s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    inv = 10000.0 ** (-torch.arange(0, case["rot"], 2, device="cuda", dtype=torch.float64) / case["rot"])
    angle = torch.arange(s["longest"], device="cuda", dtype=torch.float64)[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    return s


# ------------------------------------------------------------ plain forms


def _places(s):
    """Sequence, position and (page, row) of every new token."""
    t = torch.arange(s["q"].shape[0], device="cuda")
    seq = (t[:, None] >= s["cu"][1:][None, :]).sum(1)
    pos = (s["seqlens"][seq] - s["cu"][seq + 1] + t).long()
    page = s["table"][seq, pos // s["case"]["page"]].long()
    return pos, page, pos % s["case"]["page"]


def _rotate(x, cos, sin, rot, inter):
    x = x.float()
    y = x.clone()
    if inter:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        y[..., : rot // 2], y[..., rot // 2: rot] = a * cos - b * sin, b * cos + a * sin
    return y


def _store(pool, page, row, x, scale):
    if pool.dtype == torch.float8_e4m3fn:
        x = (x / scale).clamp(-F8_MAX, F8_MAX).to(pool.dtype).view(torch.uint8)
        pool = pool.view(torch.uint8)
    else:
        x = x.to(pool.dtype)
    pool[page, :, row] = x


def _plain_append(s):
    case = s["case"]
    pos, page, row = _places(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    q = _rotate(s["q"], cos, sin, case["rot"], case["inter"]).to(s["q"].dtype)
    k = _rotate(s["k"], cos, sin, case["rot"], case["inter"])
    _store(s["pool_k"], page, row, k, s["k_scale"])
    _store(s["pool_v"], page, row, s["v"].float(), s["v_scale"])
    out = {"q": q, "pool_k": s["pool_k"], "pool_v": s["pool_v"]}
    if case["keep"]:
        out["k"] = k.to(s["k"].dtype)
    return out


def _gathered(pool, table, scale):
    """The cached rows of every sequence as fp32 [batch, head, token, d]."""
    x = pool[table.long()] if pool.dtype != torch.float8_e4m3fn else pool.view(torch.uint8)[table.long()].view(pool.dtype)
    x = x.transpose(1, 2).float()
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1]).mul_(scale)


def _attend(q, k, v, seen):
    """softmax(q k^T / sqrt(d)) v over the places that `seen` allows, zero where it allows none;
    q [b, hkv, rows, d], k and v [b, hkv, keys, d]."""
    p = torch.matmul(q * (1.0 / math.sqrt(q.shape[-1])), k.transpose(-1, -2))
    p = p.masked_fill_(~seen, -math.inf)
    top = p.amax(-1, keepdim=True)
    p = p.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v)
    return torch.where(total > 0, o / total, torch.zeros_like(o))


def _plain_decode(s):
    case = s["case"]
    k = _gathered(s["pool_k"], s["table"], s["k_scale"])
    v = _gathered(s["pool_v"], s["table"], s["v_scale"])
    seen = torch.arange(k.shape[2], device="cuda")[None, :] < s["seqlens"][:, None]
    v = v.masked_fill_(~seen[:, None, :, None], 0.0)
    q = s["q"].float().reshape(case["batch"], case["hkv"], -1, case["d"])
    o = _attend(q, k, v, seen[:, None, None, :])
    return o.reshape(case["batch"], case["hq"], case["d"]).to(TYPES[case["out"]])


def _padded(x, cu, longest):
    """Packed rows as fp32 [batch, longest, heads, d], zero behind each sequence's end."""
    at = cu[:-1, None] + torch.arange(longest, device="cuda")[None, :]
    held = at < cu[1:, None]
    return x[at.clamp(max=x.shape[0] - 1).long()].float() * held[:, :, None, None], held


def _plain_prompt(s):
    case = s["case"]
    q, held = _padded(s["q"], s["cu"], s["longest_q"])
    k, held_k = _padded(s["k"], s["cu_kv"], s["longest"])
    v, _ = _padded(s["v"], s["cu_kv"], s["longest"])
    b, g = case["batch"], case["hq"] // case["hkv"]
    q = q.reshape(b, s["longest_q"], case["hkv"], g, case["d"]).permute(0, 2, 3, 1, 4)
    k, v = k.transpose(1, 2).unsqueeze(2), v.transpose(1, 2).unsqueeze(2)
    seen = held_k[:, None, :]
    if case["causal"]:
        i = torch.arange(s["longest_q"], device="cuda")[None, :, None]
        j = torch.arange(s["longest"], device="cuda")[None, None, :]
        ahead = (s["seqlens"] - (s["cu"][1:] - s["cu"][:-1]))[:, None, None]
        seen = seen & (j <= i + ahead)
    o = _attend(q, k, v, seen[:, None, None])
    return o.permute(0, 3, 1, 2, 4).reshape(b, s["longest_q"], case["hq"], case["d"])[held].to(TYPES[case["out"]])


# ------------------------------------------------------------ the framework's kernels


def _own_append(s):
    import fmha_b200
    case = s["case"]
    got = fmha_b200.fmha_rope_append(
        s["q"], s["k"], s["v"], s["pool_k"], s["pool_v"], s["table"], s["seqlens"], s["cos"], s["sin"],
        cu_seqlens_q=None if case["hi"] == 1 else s["cu"], interleaved=case["inter"],
        k_scale=s["k_scale"], v_scale=s["v_scale"], return_k=case["keep"])
    out = {"q": got[0] if case["keep"] else got, "pool_k": s["pool_k"], "pool_v": s["pool_v"]}
    if case["keep"]:
        out["k"] = got[1]
    return out


def _own_decode(s):
    import fmha_b200
    return fmha_b200.fmha_paged_decode(
        s["q"], s["pool_k"], s["pool_v"], s["table"], s["seqlens"], k_scale=s["k_scale"],
        v_scale=s["v_scale"], out_dtype=TYPES[s["case"]["out"]])


def _own_prompt(s):
    import fmha_b200
    return fmha_b200.fmha_prompt(
        s["q"], s["k"], s["v"], s["cu"], None if s["cu_kv"] is s["cu"] else s["cu_kv"],
        causal=s["case"]["causal"], out_dtype=TYPES[s["case"]["out"]])


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "prompt": _own_prompt}[op](state)
    return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt}[op](state)


# ------------------------------------------------------------ what a pass cannot do without


def work(case):
    new, past = _lengths(case)
    total, hq, hkv, d = sum(new), case["hq"], case["hkv"], case["d"]
    keys = sum(n + p for n, p in zip(new, past))
    if case["op"] == "append":
        held = 1 if case["cache"] == "e4m3" else 2
        positions = len({p + i for n, p in zip(new, past) for i in range(n)})
        moved = total * d * (2 * hq * 2 + 2 * hkv * (2 + held) + (2 * hkv if case["keep"] else 0))
        return {"bytes": moved + positions * case["rot"] * 4 + 4 * total, "flops": 3 * total * (hq + hkv) * case["rot"]}
    if case["op"] == "decode":
        held = 1 if case["cache"] == "e4m3" else 2
        return {"bytes": keys * hkv * d * 2 * held + 2 * total * hq * d * 2 + 4 * sum(_pages(case)),
                "flops": 4 * keys * hq * d}
    # A causal row i of n sees past + i + 1 keys.
    pairs = sum(n * p + n * (n + 1) // 2 if case["causal"] else n * (n + p) for n, p in zip(new, past))
    return {"bytes": 2 * d * (2 * total * hq + 2 * keys * hkv), "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------ 64 bits, from the definitions


def exact(case, seed):
    s = prepare(case, seed)
    d, g = case["d"], case["hq"] // case["hkv"]
    new, past = _lengths(case)
    if case["op"] == "append":
        out = {"q": s["q"].double(), "pool_k": s["pool_k"].double() if case["cache"] != "e4m3" else s["pool_k"].float().double(),
               "pool_v": s["pool_v"].double() if case["cache"] != "e4m3" else s["pool_v"].float().double()}
        k64, half = s["k"].double(), case["rot"] // 2
        index = torch.arange(half, device="cuda")
        first, second = (2 * index, 2 * index + 1) if case["inter"] else (index, index + half)
        table, at = s["table"].tolist(), 0
        for b, (n, p) in enumerate(zip(new, past)):
            places = torch.arange(p, p + n, device="cuda")
            c, w = s["cos"][places].double()[:, None], s["sin"][places].double()[:, None]
            for x in (out["q"], k64):
                # (first + i second) turned by the angle
                turned = torch.complex(x[at:at + n][..., first], x[at:at + n][..., second]) * torch.complex(c, w)
                x[at:at + n, :, first], x[at:at + n, :, second] = turned.real, turned.imag
            for lo in range(0, p + n, case["page"]):
                a, z = max(lo, p), min(lo + case["page"], p + n)
                if a < z:
                    page = table[b][lo // case["page"]]
                    rows = slice(at + a - p, at + z - p)
                    out["pool_k"][page, :, a - lo:z - lo] = k64[rows].transpose(0, 1) / s["k_scale"]
                    out["pool_v"][page, :, a - lo:z - lo] = s["v"][rows].double().transpose(0, 1) / s["v_scale"]
            at += n
        if case["keep"]:
            out["k"] = k64
        return out

    o = torch.zeros((sum(new), case["hq"], d), dtype=torch.float64, device="cuda")
    at = at_k = 0
    for b, (n, p) in enumerate(zip(new, past)):
        keys = n + p
        if case["op"] == "decode":
            pages = s["table"][b, : -(-keys // case["page"])].tolist()
        for h in range(case["hkv"]):
            if case["op"] == "decode":
                if case["cache"] == "e4m3":
                    kh = s["pool_k"].view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).float()
                    vh = s["pool_v"].view(torch.uint8)[pages, h].view(torch.float8_e4m3fn).float()
                else:
                    kh, vh = s["pool_k"][pages, h], s["pool_v"][pages, h]
                kh = kh.reshape(-1, d)[:keys].double() * s["k_scale"]
                vh = vh.reshape(-1, d)[:keys].double() * s["v_scale"]
            else:
                kh, vh = s["k"][at_k:at_k + keys, h].double(), s["v"][at_k:at_k + keys, h].double()
            qh = s["q"][at:at + n, h * g:(h + 1) * g].double()  # [n, g, d]
            for r in range(0, n, 4096):
                z = torch.einsum("ngd,kd->gnk", qh[r:r + 4096], kh) / math.sqrt(d)
                if case["op"] == "prompt" and case["causal"]:
                    rows = torch.arange(r, min(n, r + 4096), device="cuda") + p
                    z.masked_fill_(torch.arange(keys, device="cuda")[None] > rows[:, None], -math.inf)
                o[at + r:at + min(n, r + 4096), h * g:(h + 1) * g] = torch.einsum("gnk,kd->ngd", torch.softmax(z, -1), vh)
        at += n
        at_k += keys
    return o

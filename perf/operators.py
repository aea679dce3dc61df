"""What the paged key-value cache and the attention that reads it are measured on.

Three paths of a decoder that runs next to the MonarchAttention encoder:

  * ``store``   new tokens' keys and values are written into a paged cache (rounded to the
                cache's type, with one scale a token and head for e4m3 and int8), and the
                sequences are read back as dense (E, Hk, N, D) tensors with their mask;
  * ``attend``  one new token a sequence attends to the keys and values of its pages;
  * ``step``    one decoder step: the new token's keys and values are written, then it attends.

``own`` false: elementary torch operations in 32 bits.  ``own`` true: the package's entry points.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "int8": 1}
QMAX = {"e4m3": 448.0, "int8": 127.0}  # the largest code of a quantised cache
AMAX_MIN = 1e-12  # a token whose values are all zero gets this over the largest code as its scale


def listed():
    return [
        # the first tokens of a decoder's own cache, BART-base heads: latency alone
        dict(name="attend_first_tokens", op="attend", cache="bf16", x="bf16", E=1, H=12, Hk=12, D=64,
             page=16, min_len=1, max_len=24, mask=False),
        # cross attention to an encoder of 1024 tokens with its key-padding mask (BART-base, batch 4)
        dict(name="attend_cross_1k_mask", op="attend", cache="bf16", x="bf16", E=4, H=12, Hk=12, D=64,
             page=16, min_len=512, max_len=1024, mask=True),
        # cross attention to the longest BART encoder, fp16 pipeline, ragged lengths
        dict(name="attend_cross_8k_f16", op="attend", cache="f16", x="f16", E=4, H=12, Hk=12, D=64,
             page=64, min_len=4096, max_len=8192, mask=False),
        # a served batch with shared heads and an e4m3 cache, lengths far apart
        dict(name="attend_batch64_e4m3", op="attend", cache="e4m3", x="bf16", E=64, H=32, Hk=8, D=128,
             page=64, min_len=256, max_len=4096, mask=False),
        # the long-sequence sweep's heads and largest length
        dict(name="attend_long_64k", op="attend", cache="bf16", x="bf16", E=4, H=16, Hk=16, D=128,
             page=128, min_len=65536, max_len=65536, mask=False),
        # few rows over a long axis: every query head shares one int8 head of an odd size
        dict(name="attend_one_head_int8", op="attend", cache="int8", x="f16", E=3, H=24, Hk=1, D=80,
             page=48, min_len=30001, max_len=50001, mask=False),
        # the 32-bit pipelines' precision
        dict(name="attend_f32", op="attend", cache="f32", x="f32", E=8, H=12, Hk=12, D=64,
             page=16, min_len=100, max_len=2000, mask=False),
        # a batch of single new tokens, and the context read back for re-encoding (RoBERTa lengths)
        dict(name="store_token_e4m3", op="store", cache="e4m3", x="bf16", E=32, Hk=12, D=64,
             page=16, T=1, min_start=128, max_start=511, ragged=False),
        # a long prompt of the long-sequence heads quantised as it is written
        dict(name="store_prompt_16k_e4m3", op="store", cache="e4m3", x="bf16", E=4, Hk=16, D=128,
             page=64, T=16384, min_start=0, max_start=0, ragged=False),
        # a chunk of a ragged batch with the odd head size of DiT, behind what is there already
        dict(name="store_chunk_int8_odd", op="store", cache="int8", x="f16", E=5, Hk=6, D=72,
             page=24, T=333, min_start=0, max_start=100, ragged=True),
        # one step of a served batch with shared heads
        dict(name="step_batch8", op="step", cache="bf16", x="bf16", E=8, H=32, Hk=8, D=128,
             page=32, min_len=1000, max_len=2000),
        # one step of a BART decoder's own attention
        dict(name="step_bart_f16", op="step", cache="f16", x="f16", E=4, H=12, Hk=12, D=64,
             page=16, min_len=1, max_len=1023),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "store", "step"])
    D = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 256])
    page = rng.choice([8, 16, 16, 24, 32, 48, 64, 128])
    most = max(work(c)["bytes"] for c in listed())
    while True:
        E = _log_int(rng, 1, 64)
        if op == "store":
            cache = rng.choice(["f16", "bf16", "e4m3", "e4m3", "int8", "f32"])
            x = cache if cache in ("f32", "f16", "bf16") else rng.choice(["f16", "bf16", "f32"])
            start = _log_int(rng, 1, 1024)
            case = dict(op=op, cache=cache, x=x, E=E, Hk=rng.randint(1, 16), D=D, page=page,
                        T=_log_int(rng, 1, 16384), min_start=rng.randint(0, start), max_start=start,
                        ragged=rng.random() < 0.5)
        else:
            Hk, group = rng.choice([(12, 1), (16, 1), (8, 4), (4, 8), (2, 5), (1, 16), (1, 24), (3, 2)])
            if op == "attend":
                cache = rng.choice(["f16", "bf16", "bf16", "e4m3", "int8", "f32"])
            else:
                cache = rng.choice(["f16", "bf16", "f32"])
            x = cache if cache in ("f32", "f16", "bf16") else rng.choice(["f16", "bf16"])
            hi = _log_int(rng, 2, 65536 if op == "attend" else 8192)
            case = dict(op=op, cache=cache, x=x, E=E, H=Hk * group, Hk=Hk, D=D, page=page,
                        min_len=rng.randint(0, hi), max_len=hi)
            if op == "attend":
                case["mask"] = rng.random() < 0.3
        # a pass reads or writes no more than half of what the largest listed one does
        if work(case)["bytes"] <= most / 2:
            return case


def _rows(case):
    """The longest sequence that the case's pages hold."""
    if case["op"] == "store":
        return case["max_start"] + case["T"]
    return case["max_len"] + (1 if case["op"] == "step" else 0)


def _codes(g, shape, cache):
    """Random pages in the cache's type, with the scales of tokens whose sizes differ."""
    x = torch.randn(shape, generator=g, device="cuda")
    if cache not in QMAX:
        return x.to(TYPES[cache]), None
    size = torch.exp(0.5 * torch.randn(shape[:3], generator=g, device="cuda"))
    amax = x.abs().amax(-1)
    y = x / (amax / QMAX[cache])[..., None]
    y = y.round().to(torch.int8) if cache == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return y, amax * size / QMAX[cache]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    E, Hk, D, page = case["E"], case["Hk"], case["D"], case["page"]
    per = -(-_rows(case) // page)
    # every sequence has its pages, in no order, among a few that belong to nobody
    table = torch.randperm(E * per + 3, generator=g, device="cuda")[: E * per].view(E, per).int()
    shape = (E * per + 3, Hk, page, D)
    k_pages, k_scale = _codes(g, shape, case["cache"])
    v_pages, v_scale = _codes(g, shape, case["cache"])
    s = dict(case=case, k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale,
             page_table=table, mask=None, count=None)
    dt = TYPES[case["x"]]

    def fresh(T):  # the projections' output, seen as heads, as the attention hooks pass it
        return torch.randn((E, T, Hk * D), generator=g, device="cuda").to(dt).view(E, T, Hk, D).permute(0, 2, 1, 3)

    if case["op"] == "store":
        T = case["T"]
        s["k"], s["v"] = fresh(T), fresh(T)
        s["start"] = torch.randint(case["min_start"], case["max_start"] + 1, (E,), generator=g,
                                   device="cuda", dtype=torch.int32)
        if case["ragged"]:
            s["count"] = torch.randint(0, T + 1, (E,), generator=g, device="cuda", dtype=torch.int32)
        s["lengths"] = s["start"] + (s["count"] if case["ragged"] else T)
        s["N"] = _rows(case)
        return s
    q = torch.randn((E, 1, case["H"] * D), generator=g, device="cuda").to(dt)
    s["q"] = q.view(E, 1, case["H"], D).permute(0, 2, 1, 3)
    lens = torch.randint(case["min_len"], case["max_len"] + 1, (E,), generator=g, device="cuda", dtype=torch.int32)
    if case["op"] == "step":
        s["k"], s["v"] = fresh(1), fresh(1)
        s["start"], s["lengths"] = lens, lens + 1
        return s
    s["lengths"] = lens
    if case["mask"]:  # key padding inside the cached length, as an encoder's batch leaves it
        valid = torch.randint(max(1, case["max_len"] // 2), case["max_len"] + 1, (E,), generator=g, device="cuda")
        s["mask"] = torch.arange(case["max_len"], device="cuda")[None, :] < valid[:, None]
    return s


def work(case):
    E, Hk, D = case["E"], case["Hk"], case["D"]
    cb, xb = BYTES[case["cache"]], BYTES[case["x"]]
    sc = 4 if case["cache"] in QMAX else 0
    row = 2 * Hk * (D * cb + sc)  # a token's keys and values in the cache
    if case["op"] == "store":
        T = case["T"] * (0.5 if case["ragged"] else 1.0)
        mean = (case["min_start"] + case["max_start"]) / 2 + T
        new = E * T * (2 * Hk * D * xb + row)
        back = E * mean * row + E * _rows(case) * (2 * Hk * D * xb + 1)
        return {"bytes": new + back, "flops": E * T * 2 * Hk * D * 2 + E * mean * 2 * Hk * D}
    H = case["H"]
    keys = (case["min_len"] + case["max_len"]) / 2
    if case.get("mask"):
        keys = min(keys, 0.75 * case["max_len"])
    got = E * keys * row + E * H * D * xb * 2 + E * H * 4
    flops = E * H * keys * (4 * D + 4)
    if case["op"] == "step":
        got += E * 2 * Hk * D * xb + E * row
    return {"bytes": got, "flops": flops}


# ---- the plain forms -----------------------------------------------------------------------

def _gather(pages, scale, table):
    """(E, Hk, tokens, D) in 32 bits: the pages of each sequence one behind the other."""
    E, per = table.shape
    _, Hk, page, D = pages.shape
    at = table.long()
    raw = pages.view(torch.uint8)[at].view(pages.dtype) if pages.dtype.itemsize == 1 else pages[at]
    x = raw.float()
    if scale is not None:
        x = x * scale[at][..., None]
    return x.permute(0, 2, 1, 3, 4).reshape(E, Hk, per * page, D)


def _quantise(x, dtype):
    """Codes and scales of rows of 32-bit values: the largest value over the largest code."""
    top = 127.0 if dtype == torch.int8 else 448.0
    scale = x.abs().amax(-1).clamp_min(AMAX_MIN) / top
    y = x / scale[..., None]
    if dtype == torch.int8:
        return y.round().clamp(-127, 127).to(torch.int8), scale
    return y.clamp(-448, 448).to(dtype), scale


def _plain_write(x, pages, scales, table, start, count):
    E, Hk, T, D = x.shape
    page = pages.shape[2]
    pos = start.long()[:, None] + torch.arange(T, device=x.device)[None, :]
    row, slot = table.long().gather(1, pos // page), pos % page  # (E, T)
    new, scale = x.float().permute(0, 2, 1, 3), None
    if scales is not None:
        new, scale = _quantise(new, pages.dtype)
    else:
        new = new.to(pages.dtype)
    to = pages.view(torch.uint8) if pages.dtype.itemsize == 1 else pages
    new = new.view(torch.uint8) if pages.dtype.itemsize == 1 else new
    if count is not None:  # what lies behind a sequence's count stays
        ok = (torch.arange(T, device=x.device)[None, :] < count[:, None])[..., None]
        new = torch.where(ok[..., None], new, to[row, :, slot])
        if scale is not None:
            scale = torch.where(ok, scale, scales[row, :, slot])
    to[row, :, slot] = new
    if scale is not None:
        scales[row, :, slot] = scale


def _plain_read(s, pages, scales):
    N = s["N"]
    ok = torch.arange(N, device=pages.device)[None, :] < s["lengths"][:, None]
    x = _gather(pages, scales, s["page_table"])[:, :, :N]
    return torch.where(ok[:, None, :, None], x, 0.0).to(TYPES[s["case"]["x"]]), ok


def _plain_attend(s):
    q = s["q"]
    E, H, _, D = q.shape
    k = _gather(s["k_pages"], s["k_scale"], s["page_table"])
    Hk, N = k.shape[1:3]
    ok = torch.arange(N, device=q.device)[None, :] < s["lengths"][:, None]
    if s["mask"] is not None:
        ok[:, : s["mask"].shape[1]] &= s["mask"]
    a = torch.matmul(q.float().reshape(E, Hk, H // Hk, D), k.transpose(2, 3)) * (1.0 / math.sqrt(D))
    del k
    a = a.masked_fill(~ok[:, None, None, :], -math.inf)
    top = a.amax(-1, keepdim=True)
    p = torch.exp(a - top.clamp_min(-3e38))
    total = p.sum(-1, keepdim=True)
    v = _gather(s["v_pages"], s["v_scale"], s["page_table"])
    v = torch.where(ok[:, None, :, None], v, 0.0)
    o = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).reshape(E, H)
    return o.reshape(E, H, 1, D).to(q.dtype), lse


def _run_plain(s):
    op = s["case"]["op"]
    if op in ("store", "step"):
        _plain_write(s["k"], s["k_pages"], s["k_scale"], s["page_table"], s["start"], s["count"])
        _plain_write(s["v"], s["v_pages"], s["v_scale"], s["page_table"], s["start"], s["count"])
    if op == "store":
        k, mask = _plain_read(s, s["k_pages"], s["k_scale"])
        v, _ = _plain_read(s, s["v_pages"], s["v_scale"])
        return {"k": k, "v": v, "mask": mask, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    out, lse = _plain_attend(s)
    if op == "step":
        return {"out": out, "lse": lse, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return {"out": out, "lse": lse}


def _run_own(s):
    import monarch_attention_b200 as mab
    op = s["case"]["op"]
    cache = (s["k_pages"], s["v_pages"], s["page_table"])
    scales = None if s["k_scale"] is None else (s["k_scale"], s["v_scale"])
    if op in ("store", "step"):
        mab.kv_cache_write(s["k"], s["v"], *cache, s["start"], scales=scales, count=s["count"])
    if op == "store":
        k, v, mask = mab.kv_cache_read(*cache, s["lengths"], s["N"], scales=scales, dtype=TYPES[s["case"]["x"]])
        return {"k": k, "v": v, "mask": mask, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    out, lse = mab.decode_attention(s["q"], *cache, s["lengths"], s["mask"], scales=scales, return_lse=True)
    if op == "step":
        return {"out": out, "lse": lse, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    return {"out": out, "lse": lse}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definition in 64 bits ---------------------------------------------------------------

def _round_codes(y, cache):
    """The nearest code, ties to even, in 64 bits."""
    if cache == "int8":
        return torch.round(y).clamp(-127, 127)
    _, e = torch.frexp(y.abs())
    step = torch.ldexp(torch.ones_like(y), e.clamp_min(-5) - 4)  # 3 bits behind the first; 2**-9 below 2**-6
    return (torch.round(y / step) * step).clamp(-448, 448)


def exact(case, seed):
    s = prepare(case, seed)
    op, cache, page, D = case["op"], case["cache"], case["page"], case["D"]
    table, lens = s["page_table"].tolist(), s["lengths"].tolist()
    quant = cache in QMAX
    dense = {}
    for n in ("k", "v"):
        pages, scale = s[n + "_pages"], s[n + "_scale"]
        scale64 = scale.double() if quant else None
        if op in ("store", "step"):
            codes = pages.double() if op == "store" or not quant else None
            start = s["start"].tolist()
            count = s["count"].tolist() if s["count"] is not None else [s[n].shape[2]] * case["E"]
            for e in range(case["E"]):
                pos = torch.arange(start[e], start[e] + count[e], device="cuda")
                at = s["page_table"][e].long()[pos // page]
                x = s[n][e, :, : count[e]].double().transpose(0, 1)  # (tokens, Hk, D)
                if quant:
                    sc = x.abs().amax(-1).clamp_min(AMAX_MIN) / QMAX[cache]
                    scale64[at, :, pos % page] = sc
                    x = _round_codes(x / sc[..., None], cache)
                codes[at, :, pos % page] = x
        else:
            codes = pages
        dense[n] = (codes, scale64)

    def rows(n, e, length):
        codes, scale = dense[n]
        at = torch.tensor(table[e][: -(-length // page)], device="cuda", dtype=torch.long)
        x = torch.stack([codes[i] for i in at.tolist()]).double() if codes.dtype.itemsize == 1 else codes[at].double()
        if scale is not None:
            x = x * scale[at][..., None]
        return x.transpose(0, 1).reshape(case["Hk"], -1, D)[:, :length]

    if op == "store":
        out = {}
        for n in ("k", "v"):
            x = torch.zeros(case["E"], case["Hk"], s["N"], D, dtype=torch.float64, device="cuda")
            for e in range(case["E"]):
                if lens[e]:
                    x[e, :, : lens[e]] = rows(n, e, lens[e])
            out[n], out[n + "_scale"] = x, dense[n][1]
        return {"k": out["k"], "v": out["v"], "mask": None, "k_scale": out["k_scale"], "v_scale": out["v_scale"]}
    E, H, Hk = case["E"], case["H"], case["Hk"]
    out = torch.zeros(E, H, 1, D, dtype=torch.float64, device="cuda")
    lse = torch.full((E, H), -math.inf, dtype=torch.float64, device="cuda")
    for e in range(E):
        if lens[e] == 0:
            continue
        k, v = rows("k", e, lens[e]), rows("v", e, lens[e])
        if s["mask"] is not None:
            keep = s["mask"][e, : lens[e]].nonzero()[:, 0]
            k, v = k[:, keep], v[:, keep]
        if k.shape[1] == 0:
            continue
        for h in range(H):
            z = (k[h // (H // Hk)] @ s["q"][e, h, 0].double()) / math.sqrt(D)
            lse[e, h] = torch.logsumexp(z, 0)
            out[e, h, 0] = torch.softmax(z, 0) @ v[h // (H // Hk)]
    if op == "step":
        return {"out": out, "lse": lse, "k_pages": dense["k"][0], "v_pages": dense["v"][0]}
    return {"out": out, "lse": lse}

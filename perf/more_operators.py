"""Serving operators over a cache held in 8 bits, over its pages, and over logits, as cases to be timed and compared.

Kinds (head layouts and vocabularies are those of the framework's own model configurations):

  store   RoPE (with optional QK RMSNorm) of new tokens' q and k rows, their K and V rounded to 8 bits
          with a scale for each block of 16 positions and KV head (camelid_hip_paged8_rope_kv), and the
          sequences' K and V read back as 16-bit rows (camelid_hip_paged8_read), which is how a session
          is saved or moved to a 16-bit cache
  attend  attention of new tokens over such a cache, from one token to whole prompts
          (camelid_hip_paged8_attention)
  branch  sequences forked (camelid_hip_pages_fork), room made for the next tokens of parents and
          children, pages that they share and would write replaced (camelid_hip_pages_reserve) and copied
          in all layers' buffers (camelid_hip_pages_copy), then the children let go
  compact the pages in use moved to the front of the pool (camelid_hip_pages_compact and _copy)
  logits  penalties for repeated tokens, biases and grammar masks on a step's logits
          (camelid_hip_adjust_logits)

An 8-bit cache is n_pages pages of page_size positions.  K of one page: [n_kv][hd / 16][page_size][16] bytes, V:
[n_kv][page_size / 16][hd][16]; exponents of either: [n_pages][n_kv][page_size / 16], byte b for 2^(b - 127).  An
element stands for its byte (int8 or e4m3) times that.  Position p of sequence s lies in page table[s][p / page_size].
"""
from __future__ import annotations

import ctypes
import math

import numpy as np
import torch

own = False

# (n_heads, n_kv, head_dim) of the framework's configurations, and their vocabularies
HEADS = {"tinyllama": (32, 4, 64), "llama3b": (24, 8, 128), "mistral": (32, 8, 128), "qwen": (32, 8, 128)}
VOCAB = {"tinyllama": 32000, "llama3b": 128256, "mistral": 32768, "qwen": 151936}
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}
KV8 = {"i8": 3, "e4m3": 4}
LARGEST = {"i8": 127.0, "e4m3": 448.0}
TOP_EXP = {"i8": 121, "e4m3": 119}
BLOCK = 16


def listed():
    return [
        # the smallest call: one token of one sequence, where only latency counts
        {"name": "store tinyllama 1x1", "kind": "store", "heads": "tinyllama", "seqs": 1, "new": 1, "ragged": False,
         "history": 127, "page": 16, "norm": False, "split_half": False, "q": "f32", "kv": "i8"},
        # the prompts of a small batch behind a shared system prompt that ends inside a block
        {"name": "store qwen 4x2047", "kind": "store", "heads": "qwen", "seqs": 4, "new": 2047, "ragged": True,
         "history": 200, "page": 64, "norm": True, "split_half": True, "q": "bf16", "kv": "e4m3"},
        # chat with one user on the smallest model: latency
        {"name": "attend tinyllama 1x127", "kind": "attend", "heads": "tinyllama", "seqs": 1, "new": 1, "len": 127,
         "ragged": False, "page": 16, "q": "f32", "kv": "i8"},
        # one user far into long documents, what an 8-bit cache is for: the split over the length has to fill the GPU
        {"name": "attend mistral 1x32775", "kind": "attend", "heads": "mistral", "seqs": 1, "new": 1, "len": 32775,
         "ragged": False, "page": 64, "q": "f32", "kv": "e4m3"},
        # a serving batch of every age, 16-bit activations
        {"name": "attend llama3b 64x4001", "kind": "attend", "heads": "llama3b", "seqs": 64, "new": 1, "len": 4001,
         "ragged": True, "page": 32, "q": "bf16", "kv": "i8"},
        # drafts verified over a batch's caches
        {"name": "attend qwen 16x1100 d5", "kind": "attend", "heads": "qwen", "seqs": 16, "new": 5, "len": 1100,
         "ragged": True, "page": 32, "q": "f16", "kv": "e4m3"},
        # prompts of a few requests at once, f32 activations as the engine's own
        {"name": "prompt llama3b 3x1023", "kind": "attend", "heads": "llama3b", "seqs": 3, "new": 1023, "len": 1023,
         "ragged": True, "page": 64, "q": "f32", "kv": "i8"},
        # the largest: the last piece of a long prompt over what was stored before
        {"name": "prompt mistral 1x4096 at 12288", "kind": "attend", "heads": "mistral", "seqs": 1, "new": 4096,
         "len": 16384, "ragged": False, "page": 128, "q": "bf16", "kv": "i8"},
        # four answers from each of 16 prompts: one page each is shared and written
        {"name": "branch llama3b 16x3", "kind": "branch", "heads": "llama3b", "seqs": 16, "children": 3, "len": 1000,
         "new": 2, "page": 32, "layers": 8, "spare": 64},
        # a pool after a busy hour, half of it free: the rest moves to its front
        {"name": "compact mistral 2048", "kind": "compact", "heads": "mistral", "pages": 2048, "seqs": 40, "used": 0.5,
         "page": 16, "layers": 8},
        # one user, penalties over a short history
        {"name": "logits tinyllama 1x1", "kind": "logits", "vocab": "tinyllama", "seqs": 1, "rows": 1, "history": 300,
         "bias": 0, "mask": False, "in_place": True, "type": "f32"},
        # a serving batch with drafts: penalties, a few biases, grammars for some
        {"name": "logits qwen 32x6", "kind": "logits", "vocab": "qwen", "seqs": 32, "rows": 6, "history": 2000,
         "bias": 40, "mask": True, "in_place": False, "type": "bf16"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "prompt", "branch", "compact", "logits"])
    if kind == "logits":
        rows = rng.choice([1, 1, rng.randint(2, 8)])
        seqs = _log_int(rng, 1, 48 if rows == 1 else 24)
        return {"kind": kind, "vocab": rng.choice(sorted(VOCAB)), "seqs": seqs, "rows": rows,
                "history": _log_int(rng, 1, 16000), "bias": rng.choice([0, _log_int(rng, 1, 300)]),
                "mask": rng.random() < 0.5, "in_place": rng.random() < 0.5, "type": rng.choice(sorted(TYPES))}
    c = {"kind": kind, "heads": rng.choice(sorted(HEADS)), "page": rng.choice([16, 32, 64, 128, 256])}
    if kind == "branch":
        c.update(seqs=_log_int(rng, 1, 32), children=rng.randint(1, 7), len=_log_int(rng, 1, 3000),
                 new=rng.randint(1, 8), layers=rng.randint(1, 8), spare=rng.randint(0, 100))
        return c
    if kind == "compact":
        c.update(pages=_log_int(rng, 16, 32768 // c["page"]), seqs=_log_int(rng, 1, 64), used=rng.uniform(0.05, 0.95),
                 layers=rng.randint(1, 8))
        return c
    c.update(kv=rng.choice(sorted(KV8)), ragged=rng.random() < 0.6, q=rng.choice(sorted(TYPES)))
    if kind == "store":
        c.update(seqs=_log_int(rng, 1, 64), new=_log_int(rng, 1, 2048), history=_log_int(rng, 1, 1024),
                 norm=rng.random() < 0.5, split_half=rng.random() < 0.5)
        c["new"] = min(c["new"], 8192 // c["seqs"])
        return c
    c["kind"] = "attend"
    if kind == "attend":
        c.update(seqs=_log_int(rng, 1, 128), new=rng.choice([1, 1, rng.randint(2, 8)]))
        c["len"] = min(_log_int(rng, 8, 65536), 250000 // c["seqs"])
        return c
    c.update(seqs=_log_int(rng, 1, 8), new=_log_int(rng, 9, 4096))
    c["new"] = min(c["new"], 4096 // c["seqs"])
    c["len"] = c["new"] + rng.choice([0, _log_int(rng, 1, 12000 // c["seqs"])])
    return c


# ---------------------------------------------------------------------------------------- inputs
def _spread(n, top, ragged):
    """Lengths 1 ... top of n sequences, spread evenly without order (the first one is `top`)."""
    return [top if not ragged or i == 0 else 1 + int(top * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lens(case):
    """(positions in the cache with the new tokens, new tokens) of each sequence."""
    n = case["seqs"]
    new = _spread(n, case["new"], case["ragged"])
    if case["kind"] == "store":
        return [case["history"] + t for t in new], new
    return [max(x, t) for x, t in zip(_spread(n, max(case["len"], case["new"]), case["ragged"]), new)], new


def _u32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache(case, gen):
    """Pages in an order of their own, some of them nobody's, filled with a model's k and v rows."""
    _, n_kv, hd = HEADS[case["heads"]]
    ps, lens = case["page"], _lens(case)[0]
    stride = -(-max(lens) // ps)
    used = case["seqs"] * stride
    pages = used + 3
    st = {"pages": pages, "stride": stride, "lens": _u32(lens)}
    for name in ("k", "v"):
        x = torch.empty(pages, n_kv, hd * ps, device="cuda").normal_(generator=gen)
        if case["kv"] == "i8":
            x = x.mul_(36).round_().clamp_(-127, 127).to(torch.int8)
        else:
            x = x.mul_(120).clamp_(-448, 448).to(torch.float8_e4m3fn)
        st[name] = x.view(torch.uint8)
        near = 127 - (5 if case["kv"] == "i8" else 7)
        st[name + "_exp"] = torch.randint(near - 1, near + 2, (pages, n_kv, ps // BLOCK), generator=gen, device="cuda",
                                          dtype=torch.uint8)
    table = torch.randperm(pages, generator=gen, device="cuda")[:used].to(torch.int32).view(case["seqs"], stride)
    return {**st, "table": table.contiguous()}


def _rope(case, rows, hd, lens, new):
    """cos and sin rows [rows][hd / 2] of each row's position."""
    n = case["new"]
    pos = torch.tensor([[x - t + i for i in range(n)] for x, t in zip(lens, new)], device="cuda").double().view(rows, 1)
    f = 500000.0 ** (-2.0 * torch.arange(hd // 2, device="cuda").double() / hd)
    return (pos * f).cos().float(), (pos * f).sin().float()


def _buffers(case, pages, gen):
    """K and V bytes and exponents of all layers: [2 layers][pages][bytes]."""
    _, n_kv, hd = HEADS[case["heads"]]
    size = (2 * case["layers"], pages, n_kv * hd * case["page"])
    return (torch.randint(256, size, generator=gen, device="cuda", dtype=torch.uint8),
            torch.randint(256, (*size[:2], n_kv * case["page"] // BLOCK), generator=gen, device="cuda",
                          dtype=torch.uint8))


def _prepare_branch(case, gen):
    n, c, ps = case["seqs"], case["children"], case["page"]
    lens = _spread(n, case["len"], True)
    held = [-(-x // ps) for x in lens]
    rows = n * (1 + c)
    # what parents and children write: the last page where it is not full, and what the new tokens add
    writes = [-(-(x + case["new"]) // ps) - x // ps for x in lens]
    stride = -(-(case["len"] + case["new"]) // ps)
    pages = sum(held) + (1 + c) * sum(writes) + case["spare"]
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(rows, stride, dtype=torch.int32, device="cuda")
    at = _u32(held).cumsum(0)[:, None] - _u32(held)[:, None] + torch.arange(stride, device="cuda")[None]
    mine = torch.arange(stride, device="cuda")[None] < _u32(held)[:, None]
    table[:n] = torch.where(mine, order[at.clamp_max(pages - 1)], 0)
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:sum(held)].long()] = 1
    kv, exps = _buffers(case, pages, gen)
    first = lens + [x for x in lens for _ in range(c)]
    return {"table": table, "refs": refs, "held": _u32(held + [0] * (n * c)), "kv": kv, "exps": exps,
            "pages": pages, "stride": stride, "lens": _u32(lens + [0] * (n * c)), "first": _u32(first),
            "grown": _u32([x + case["new"] for x in first]),
            "parents": _u32([i for i in range(n) for _ in range(c)]), "children": _u32(list(range(n, rows))),
            "max_pairs": rows, "pairs": torch.zeros(rows, 2, dtype=torch.int32, device="cuda"),
            "n_pairs": torch.zeros(1, dtype=torch.int32, device="cuda"),
            "granted": torch.zeros(rows, dtype=torch.int32, device="cuda")}


def _prepare_compact(case, gen):
    """Sequences of different lengths, neighbours in the list sharing their first page."""
    n, pages = case["seqs"], case["pages"]
    used = max(1, min(pages, int(pages * case["used"])))
    n = min(n, used)
    share = [used // n + (i < used % n) for i in range(n)]
    stride = max(share) + 1
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.zeros(n, stride, dtype=torch.int32, device="cuda")
    ends = _u32(share).cumsum(0)
    j = torch.arange(stride, device="cuda")[None]
    owned = order[(ends[:, None] - _u32(share)[:, None] + j).clamp_max(pages - 1)]
    table[:] = torch.where(j < _u32(share)[:, None], owned, 0)
    held, refs = share[:], torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:used].long()] = 1
    for i in range(1, n, 2):  # every second one has the first page of the one before it behind its own
        table[i, share[i]] = table[i - 1, 0]
        refs[table[i - 1, 0].long()] += 1
        held[i] += 1
    kv, exps = _buffers(case, pages, gen)
    return {"table": table, "refs": refs, "held": _u32(held), "kv": kv, "exps": exps, "pages": pages, "stride": stride,
            "n": n, "table_out": torch.zeros_like(table), "refs_out": torch.zeros_like(refs),
            "max_pairs": pages // 2 + 1, "pairs": torch.zeros(pages // 2 + 1, 2, dtype=torch.int32, device="cuda"),
            "n_pairs": torch.zeros(1, dtype=torch.int32, device="cuda"),
            "extent": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _prepare_logits(case, gen):
    n, rows, v = case["seqs"], case["rows"], VOCAB[case["vocab"]]
    x = torch.empty(n, rows, v, device="cuda").normal_(0, 2.5, generator=gen).to(TYPES[case["type"]][0])

    def tokens(*shape):  # a few tokens come up again and again
        return (torch.rand(*shape, generator=gen, device="cuda").pow(4) * v).to(torch.int32)

    lens = _spread(n, case["history"], True)
    b = max(case["bias"], 1)
    mask = None
    if case["mask"]:  # a grammar allows few tokens; sequences without one allow all
        words = -(-v // 32)
        some = torch.rand(n, rows, words, 32, generator=gen, device="cuda") < 0.03
        bits = (some.long() << torch.arange(32, device="cuda")).sum(-1)
        free = (torch.arange(n, device="cuda") % 3 == 2)[:, None, None]
        bits = torch.where(free, torch.full_like(bits, 0xffffffff), bits)
        mask = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    pick = [i % 4 for i in range(n)]
    return {"logits": x, "out": x if case["in_place"] else torch.zeros_like(x), "history": tokens(n, case["history"]),
            "history_lens": _u32(lens), "prompt_lens": _u32([t // 3 for t in lens]),
            "draft": tokens(n, max(rows - 1, 1)), "draft_lens": _u32([min(t, rows) - 1 for t in _spread(n, rows, True)]),
            "repetition": torch.tensor([[1.1, 1.0, 1.3, 1.05][i] for i in pick], device="cuda"),
            "frequency": torch.tensor([[0.0, 0.2, 0.1, 0.5][i] for i in pick], device="cuda"),
            "presence": torch.tensor([[0.0, 0.6, 0.0, -0.3][i] for i in pick], device="cuda"),
            "bias_tokens": tokens(n, b), "bias_lens": _u32([min(t, case["bias"]) for t in _spread(n, b, True)]),
            "bias_values": torch.empty(n, b, device="cuda").normal_(0, 3, generator=gen), "mask": mask}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    if case["kind"] in ("branch", "compact", "logits"):
        make = {"branch": _prepare_branch, "compact": _prepare_compact, "logits": _prepare_logits}[case["kind"]]
        return {"case": case, **make(case, gen)}
    nh, n_kv, hd = HEADS[case["heads"]]
    n = case["seqs"]
    st = {"case": case, **_cache(case, gen)}
    lens, new = _lens(case)
    rows = n * case["new"]
    st["new_lens"] = _u32(new)
    qt = TYPES[case["q"]][0]
    if case["kind"] == "store":
        st["qkv"] = torch.empty(rows, (nh + 2 * n_kv) * hd, device="cuda").normal_(0, 1.3, generator=gen)
        st["cos"], st["sin"] = _rope(case, rows, hd, lens, new)
        st["norms"] = [torch.empty(hd, device="cuda").normal_(1.0, 0.1, generator=gen) for _ in range(2)] \
            if case["norm"] else None
        st["q_out"] = torch.zeros(rows, nh * hd, dtype=qt, device="cuda")
        st["top"] = max(lens)
        st["k_read"], st["v_read"] = (torch.zeros(n, n_kv, st["top"], hd, dtype=torch.float16, device="cuda")
                                      for _ in range(2))
        return st
    st["q"] = torch.empty(rows, nh * hd, device="cuda").normal_(0, 1.5, generator=gen).to(qt)
    st["out"] = torch.zeros(rows, nh * hd, dtype=qt, device="cuda")
    return st


# ------------------------------------------------------------------------------------ plain forms
def _dense(st, name):
    """K or V of every sequence as [seqs][n_kv][positions][hd]: bytes, and their exponents [seqs][n_kv][blocks]."""
    c = st["case"]
    _, n_kv, hd = HEADS[c["heads"]]
    ps, n, stride = c["page"], c["seqs"], st["stride"]
    at = st["table"].long()
    x = st[name][at]
    if name == "k":  # [n][stride][n_kv][hd / 16][ps][16]
        x = x.view(n, stride, n_kv, hd // 16, ps, 16).permute(0, 2, 1, 4, 3, 5)
    else:  # [n][stride][n_kv][ps / 16][hd][16]
        x = x.view(n, stride, n_kv, ps // 16, hd, 16).permute(0, 2, 1, 3, 5, 4)
    e = st[name + "_exp"][at].permute(0, 2, 1, 3)
    return x.reshape(n, n_kv, stride * ps, hd), e.reshape(n, n_kv, stride * ps // BLOCK)


def _put_dense(st, name, x, e):
    c = st["case"]
    _, n_kv, hd = HEADS[c["heads"]]
    ps, n, stride = c["page"], c["seqs"], st["stride"]
    at = st["table"].long()
    if name == "k":
        x = x.view(n, n_kv, stride, ps, hd // 16, 16).permute(0, 2, 1, 4, 3, 5)
    else:
        x = x.view(n, n_kv, stride, ps // 16, 16, hd).permute(0, 2, 1, 3, 5, 4)
    st[name][at] = x.reshape(n, stride, n_kv, hd * ps)
    st[name + "_exp"][at] = e.view(n, n_kv, stride, ps // BLOCK).permute(0, 2, 1, 3)


def _values(c, x):
    return x.view(torch.int8 if c["kv"] == "i8" else torch.float8_e4m3fn).float()


def _pow2(e):
    return torch.ldexp(torch.ones((), device="cuda"), e)


def _dequantised(c, x, e):
    return _values(c, x) * _pow2(e.int() - 127).repeat_interleave(BLOCK, -1)[..., None]


def _exponents(c, top):
    """The smallest e with top <= LARGEST 2^e."""
    m, e = torch.frexp(top)  # m in [0.5, 1)
    bits, edge = (6, 127.0 / 128.0) if c["kv"] == "i8" else (8, 448.0 / 512.0)
    e = torch.where(top > 0, e - 1 - bits + (m > edge).int(), torch.full_like(e, -126))
    return e.clamp(-126, TOP_EXP[c["kv"]])


def _put_rows(st, name, rows, real):
    """rows [n][new][n_kv][hd] f32 into the cache, requantising what their blocks hold."""
    c = st["case"]
    n, new = c["seqs"], c["new"]
    raw, e = _dense(st, name)
    cap = raw.shape[2]
    first = st["lens"] - st["new_lens"]
    p = torch.arange(cap, device="cuda")
    fresh = (p >= first[:, None]) & (p < st["lens"][:, None])               # [n][cap]
    t = (p - first[:, None]).clamp(0, new - 1)
    x = rows.gather(1, t[..., None, None].expand(n, cap, *rows.shape[2:]).long()).permute(0, 2, 1, 3)
    x = torch.where(fresh[:, None, :, None], x, torch.zeros_like(x))
    need = _exponents(c, x.abs().amax(-1).unflatten(-1, (-1, BLOCK)).amax(-1))  # [n][n_kv][blocks]
    touched = fresh.unflatten(-1, (-1, BLOCK)).any(-1)
    old = (p[::BLOCK] < first[:, None])[:, None]                             # the block holds earlier positions
    was = e.int() - 127
    now = torch.where(touched[:, None], torch.where(old, torch.maximum(need, was), need), was)
    y = torch.where(fresh[:, None, :, None], x, _dequantised(c, raw, e))
    y = y * _pow2(-now).repeat_interleave(BLOCK, -1)[..., None]
    y = y.clamp(-LARGEST[c["kv"]], LARGEST[c["kv"]])
    y = (y.round().to(torch.int8) if c["kv"] == "i8" else y.to(torch.float8_e4m3fn)).view(torch.uint8)
    keep = (p < st["lens"][:, None]) & touched.repeat_interleave(BLOCK, -1)
    _put_dense(st, name, torch.where(keep[:, None, :, None], y, raw), (now + 127).to(torch.uint8))


def _plain_store(st):
    c = st["case"]
    nh, n_kv, hd = HEADS[c["heads"]]
    n, new = c["seqs"], c["new"]
    x = st["qkv"].view(n * new, nh + 2 * n_kv, hd)
    q, k, v = x[:, :nh], x[:, nh:nh + n_kv], x[:, nh + n_kv:]
    if st["norms"] is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * st["norms"][0]
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * st["norms"][1]
    cos, sin = st["cos"][:, None], st["sin"][:, None]

    def turn(t):
        a, b = (t[..., :hd // 2], t[..., hd // 2:]) if c["split_half"] else (t[..., 0::2], t[..., 1::2])
        a, b = a * cos - b * sin, a * sin + b * cos
        return torch.cat([a, b], -1) if c["split_half"] else torch.stack([a, b], -1).flatten(-2)

    real = torch.arange(new, device="cuda")[None] < st["new_lens"][:, None]
    st["q_out"].copy_(torch.where(real.view(-1, 1), turn(q).flatten(1).to(st["q_out"].dtype), st["q_out"]))
    _put_rows(st, "k", turn(k).view(n, new, n_kv, hd), real)
    _put_rows(st, "v", v.reshape(n, new, n_kv, hd), real)
    seen = (torch.arange(st["top"], device="cuda") < st["lens"][:, None])[:, None, :, None]
    for name in ("k", "v"):
        y = _dequantised(c, *_dense(st, name))[:, :, :st["top"]].half()
        st[name + "_read"].copy_(torch.where(seen, y, st[name + "_read"]))
    return {"q": st["q_out"], "k": st["k_read"], "v": st["v_read"]}


def _plain_attend(st):
    c = st["case"]
    nh, n_kv, hd = HEADS[c["heads"]]
    n, new, g = c["seqs"], c["new"], nh // n_kv
    cap = st["stride"] * c["page"]
    q = st["q"].float().view(n, new, n_kv, g, hd).permute(0, 2, 1, 3, 4).reshape(n, n_kv, new * g, hd)
    s = torch.matmul(q, _dequantised(c, *_dense(st, "k")).transpose(-1, -2).contiguous())
    s *= 1.0 / math.sqrt(hd)
    t = torch.arange(new, device="cuda")
    last = st["lens"][:, None] - st["new_lens"][:, None] + t[None]        # [n][new]: last visible position
    real = t[None] < st["new_lens"][:, None]
    hidden = ~((torch.arange(cap, device="cuda") <= last[..., None]) & real[..., None])
    s.view(n, n_kv, new, g, cap).masked_fill_(hidden[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(-3e38)
    w = s.sub_(top).exp_()
    w /= w.sum(-1, keepdim=True).clamp_min(1e-38)
    o = torch.matmul(w, _dequantised(c, *_dense(st, "v")))
    o = o.view(n, n_kv, new, g, hd).permute(0, 2, 1, 3, 4).reshape(n, new, nh * hd).to(st["out"].dtype)
    out = st["out"].view(n, new, nh * hd)
    out.copy_(torch.where(real[..., None], o, out))
    return {"out": st["out"]}


def _plain_reserve(st, first, lens):
    """Rows given pages for lens positions, what [first, lens) shares with other rows replaced."""
    ps, pages, most = st["case"]["page"], st["pages"], st["max_pairs"]
    table, refs, held = st["table"], st["refs"], st["held"]
    j = torch.arange(st["stride"], device="cuda")[None]
    need = (lens + ps - 1) // ps
    at = table.long().clamp(0, pages - 1)
    drop = (j >= need[:, None]) & (j < held[:, None])
    refs.index_add_(0, at.view(-1), -drop.view(-1).int())
    mine = torch.minimum(held, need)[:, None]
    shared = (j >= (first // ps)[:, None]) & (j < mine) & (first < lens)[:, None] & (refs[at] > 1)
    want = shared | ((j >= mine) & (j < need[:, None]))
    count, cow = want.sum(1), shared.sum(1)
    before, cows = count.cumsum(0), cow.cumsum(0)
    free = torch.sort((refs != 0).int(), stable=True)[1]
    room = (refs == 0).sum()
    ok = (count == 0) | ((before <= room) & ((cow == 0) | (cows <= most)))
    rank = (want.view(-1).cumsum(0) - 1).view_as(want).clamp(0, pages - 1)
    want, shared = want & ok[:, None], shared & ok[:, None]
    fresh = free[rank].int()
    # pairs, and what else is written nowhere: one place behind the end
    place = torch.where(shared, (cows - cow)[:, None] + shared.cumsum(1) - 1, most)
    wide = torch.cat([st["pairs"], st["pairs"][:1]])
    wide[place.view(-1)] = torch.stack([table, fresh], -1).view(-1, 2)
    st["pairs"].copy_(wide[:most])
    st["n_pairs"].copy_(shared.sum().view(1))
    refs.index_add_(0, at.view(-1), -shared.view(-1).int())
    refs.index_add_(0, fresh.view(-1).long(), want.view(-1).int())
    table.copy_(torch.where(want, fresh, table))
    held.copy_(torch.where(ok, need, mine[:, 0]))
    st["granted"].copy_(ok)


def _plain_copy(st):
    k = torch.arange(st["max_pairs"], device="cuda")
    pairs = torch.where((k < st["n_pairs"])[:, None], st["pairs"], st["pairs"][:1])
    pairs = torch.where(st["n_pairs"] > 0, pairs, torch.zeros_like(pairs)).long()
    for name in ("kv", "exps"):
        st[name][:, pairs[:, 1]] = st[name][:, pairs[:, 0]]


def _plain_branch(st):
    table, ps = st["table"], st["case"]["page"]
    parents, children = st["parents"].long(), st["children"].long()
    j = torch.arange(st["stride"], device="cuda")[None]
    taken = torch.minimum(st["held"][parents], (st["lens"][parents] + ps - 1) // ps)
    mine = j < taken[:, None]
    rows = table[parents]
    table[children] = torch.where(mine, rows, table[children])
    st["refs"].index_add_(0, rows.view(-1).long(), mine.view(-1).int())
    st["held"][children] = taken
    _plain_reserve(st, st["first"], st["grown"])
    pairs, n_pairs, granted = st["pairs"].clone(), st["n_pairs"].clone(), st["granted"].clone()
    _plain_copy(st)
    _plain_reserve(st, st["lens"], st["lens"])
    for name, kept in (("pairs", pairs), ("n_pairs", n_pairs), ("granted", granted)):
        st[name].copy_(kept)
    return _branch_outputs(st)


def _branch_outputs(st):
    return {k: st[k] for k in ("table", "held", "refs", "pairs", "n_pairs", "granted", "kv", "exps")}


def _plain_compact(st):
    refs, pages, most = st["refs"], st["pages"], st["max_pairs"]
    p = torch.arange(pages, device="cuda")
    live = refs > 0
    n_live = live.sum()
    hole, high = ~live & (p < n_live), live & (p >= n_live)
    to = torch.sort((~hole).int(), stable=True)[1]                       # holes first, ascending
    at = torch.sort(torch.where(high, p, -1), descending=True)[0]        # the highest first
    total = hole.sum()
    moves = total.clamp_max(most)
    moved = p < moves
    src, dst = torch.where(moved, at, pages), torch.where(moved, to, pages)
    remap = torch.arange(pages + 1, device="cuda")
    remap[src] = dst
    held = torch.arange(st["stride"], device="cuda")[None] < st["held"][:, None]
    st["table_out"].copy_(torch.where(held, remap[st["table"].long().clamp(0, pages - 1)].int(), st["table"]))
    wide = torch.cat([refs, refs[:1]])
    wide[dst] = torch.cat([refs, refs[:1]])[src]
    wide[src] = 0
    st["refs_out"].copy_(wide[:pages])
    k = torch.arange(most, device="cuda").clamp_max(pages - 1)
    pairs = torch.stack([at[k], to[k]], -1).int()
    st["pairs"].copy_(torch.where((torch.arange(most, device="cuda") < moves)[:, None], pairs, st["pairs"]))
    st["n_pairs"].copy_(moves.view(1))
    st["extent"].copy_(torch.where(moves < total, at[moves.clamp_max(pages - 1)] + 1, n_live).view(1))
    _plain_copy(st)
    return _compact_outputs(st)


def _compact_outputs(st):
    return {k: st[k] for k in ("table_out", "refs_out", "pairs", "n_pairs", "extent", "kv", "exps")}


def _plain_logits(st):
    c = st["case"]
    n, rows, v = c["seqs"], c["rows"], VOCAB[c["vocab"]]
    x = st["logits"].float()
    j = torch.arange(st["history"].shape[1], device="cuda")[None]
    known, said = j < st["history_lens"][:, None], j >= st["prompt_lens"][:, None]
    at = st["history"].long()
    zero = torch.zeros(n, v, device="cuda")
    seen = zero.scatter_add(1, at, known.float())[:, None]
    count = zero.scatter_add(1, at, (known & said).float())[:, None]
    # row t has the drafts before it, too
    t = torch.arange(rows, device="cuda")
    before = (torch.arange(st["draft"].shape[1], device="cuda")[None] < t[:, None]).float()
    drafts = torch.zeros(n, rows, v, device="cuda").scatter_add(
        2, st["draft"].long()[:, None].expand(-1, rows, -1), before.expand(n, -1, -1))
    seen, count = seen + drafts, count + drafts
    r, f, p = (st[k][:, None, None] for k in ("repetition", "frequency", "presence"))
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - f * count
    x = x - torch.where(count > 0, p, 0.0)
    # of equal tokens the last bias counts
    b = st["bias_tokens"].shape[1]
    k = torch.arange(b, device="cuda")[None]
    listed_here = (k < st["bias_lens"][:, None]).int() * (k + 1)
    last = torch.zeros(n, v, dtype=torch.int32, device="cuda").scatter_reduce(
        1, st["bias_tokens"].long(), listed_here.int(), "amax")
    add = st["bias_values"].gather(1, (last - 1).clamp_min(0).long())
    x = x + torch.where(last > 0, add, 0.0)[:, None]
    if st["mask"] is not None:
        i = torch.arange(v, device="cuda")
        x = torch.where((st["mask"][..., i // 32] >> (i % 32)) & 1 > 0, x, -math.inf)
    live = (t[None] <= st["draft_lens"][:, None])[..., None]
    st["out"].copy_(torch.where(live, x.to(st["out"].dtype), st["out"]))
    return {"out": st["out"]}


# ------------------------------------------------------------------------------ the framework's calls
def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _workspace(st, n_bytes, *sizes):
    """The scratch memory that a program keeps between its calls of the same sizes."""
    if "workspace" not in st:
        st["workspace"] = torch.empty(max(1, n_bytes(*sizes)), dtype=torch.uint8, device="cuda")
    return st["workspace"]


def _own_copy(lib, check, st):
    if "buffers" not in st:  # a program's buffers stay where they are
        every = [x for t in (st["kv"], st["exps"]) for x in t]
        st["buffers"] = ((ctypes.c_void_p * len(every))(*[x.data_ptr() for x in every]),
                         (ctypes.c_size_t * len(every))(*[x.shape[1] for x in every]), len(every))
    where, sizes, n = st["buffers"]
    check(lib.camelid_hip_pages_copy(where, sizes, n, st["pages"], _p(st["pairs"]), st["max_pairs"], _p(st["n_pairs"]),
                                     None, _stream()))


def _own_pages(st, lib, check):
    c = st["case"]
    if c["kind"] == "compact":
        ws = _workspace(st, lib.camelid_hip_pages_compact_workspace, st["pages"])
        check(lib.camelid_hip_pages_compact(
            _p(st["table"]), st["stride"], _p(st["held"]), st["n"], _p(st["refs"]), st["pages"], _p(st["table_out"]),
            _p(st["refs_out"]), _p(st["pairs"]), st["max_pairs"], _p(st["n_pairs"]), _p(st["extent"]), _p(ws),
            ws.numel(), None, _stream()))
        _own_copy(lib, check, st)
        return _compact_outputs(st)
    rows = st["table"].shape[0]
    ws = _workspace(st, lib.camelid_hip_pages_reserve_workspace, rows, st["pages"])
    check(lib.camelid_hip_pages_fork(
        _p(st["table"]), st["stride"], _p(st["held"]), rows, _p(st["parents"]), _p(st["children"]),
        st["children"].numel(), _p(st["lens"]), c["page"], _p(st["refs"]), st["pages"], None, _stream()))
    check(lib.camelid_hip_pages_reserve(
        _p(st["table"]), st["stride"], _p(st["held"]), rows, _p(st["first"]), _p(st["grown"]), c["page"],
        _p(st["refs"]), st["pages"], _p(st["pairs"]), st["max_pairs"], _p(st["n_pairs"]), _p(st["granted"]), _p(ws),
        ws.numel(), None, _stream()))
    _own_copy(lib, check, st)
    # nothing is written behind this one: no pairs
    check(lib.camelid_hip_pages_reserve(
        _p(st["table"]), st["stride"], _p(st["held"]), rows, None, _p(st["lens"]), c["page"], _p(st["refs"]),
        st["pages"], None, 0, None, None, _p(ws), ws.numel(), None, _stream()))
    return _branch_outputs(st)


def _own(st):
    from camelid_amd import _native
    lib, c, check = _native.lib(), st["case"], _native.check
    if c["kind"] in ("branch", "compact"):
        return _own_pages(st, lib, check)
    if c["kind"] == "logits":
        n, rows, v = c["seqs"], c["rows"], VOCAB[c["vocab"]]
        check(lib.camelid_hip_adjust_logits(
            _p(st["logits"]), v, _p(st["out"]), v, TYPES[c["type"]][1], n, rows, v, _p(st["history"]),
            st["history"].shape[1], _p(st["history_lens"]), _p(st["prompt_lens"]), _p(st["draft"]) if rows > 1 else None,
            _p(st["draft_lens"]), _p(st["repetition"]), _p(st["frequency"]), _p(st["presence"]),
            _p(st["bias_tokens"]) if c["bias"] else None, _p(st["bias_values"]) if c["bias"] else None,
            st["bias_tokens"].shape[1], _p(st["bias_lens"]), _p(st["mask"]), -(-v // 32), _stream()))
        return {"out": st["out"]}
    nh, n_kv, hd = HEADS[c["heads"]]
    n, ps, kv = c["seqs"], c["page"], KV8[c["kv"]]
    if c["kind"] == "store":
        norms = st["norms"] or (None, None)
        check(lib.camelid_hip_paged8_rope_kv(
            _p(st["qkv"]), n, c["new"], _p(st["new_lens"]), nh, n_kv, hd, hd, int(c["split_half"]), _p(st["cos"]),
            _p(st["sin"]), _p(norms[0]), _p(norms[1]), 1e-6, _p(st["q_out"]), TYPES[c["q"]][1], _p(st["k"]),
            _p(st["v"]), _p(st["k_exp"]), _p(st["v_exp"]), kv, st["pages"], ps, _p(st["table"]), st["stride"],
            _p(st["lens"]), None, _stream()))
        check(lib.camelid_hip_paged8_read(
            _p(st["k"]), _p(st["v"]), _p(st["k_exp"]), _p(st["v_exp"]), kv, st["pages"], ps, n_kv, hd, _p(st["table"]),
            st["stride"], _p(st["lens"]), n, _p(st["k_read"]), _p(st["v_read"]), TYPES["f16"][1], st["top"], None,
            _stream()))
        return {"q": st["q_out"], "k": st["k_read"], "v": st["v_read"]}
    ws = _workspace(st, lib.camelid_hip_paged8_attention_workspace, n, c["new"], nh, n_kv, hd, ps, st["stride"])
    check(lib.camelid_hip_paged8_attention(
        _p(st["q"]), TYPES[c["q"]][1], nh * hd, n, c["new"], _p(st["new_lens"]), nh, n_kv, hd, _p(st["k"]), _p(st["v"]),
        _p(st["k_exp"]), _p(st["v_exp"]), kv, st["pages"], ps, _p(st["table"]), st["stride"], _p(st["lens"]),
        1.0 / math.sqrt(hd), _p(st["out"]), nh * hd, _p(ws), ws.numel(), None, _stream()))
    return {"out": st["out"]}


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attend": _plain_attend, "branch": _plain_branch, "compact": _plain_compact,
            "logits": _plain_logits}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    """Each input that the operator cannot do without read once, each output written once."""
    if case["kind"] == "logits":
        n, rows, v = case["seqs"], case["rows"], VOCAB[case["vocab"]]
        size = TYPES[case["type"]][0].itemsize
        live = sum(min(t, rows) for t in _spread(n, rows, True))
        known = sum(_spread(n, case["history"], True))
        if case["in_place"] and not case["mask"]:  # what the lists name
            return {"bytes": 4 * known + 2 * size * rows * known + 8 * n * case["bias"], "flops": 4 * rows * known}
        return {"bytes": live * v * (2 * size + (0.125 if case["mask"] else 0)) + 4 * known, "flops": live * v}
    nh, n_kv, hd = HEADS[case["heads"]]
    if case["kind"] == "branch":
        c, ps = case["children"], case["page"]
        lens = _spread(case["seqs"], case["len"], True)
        copied = (1 + c) * sum(x % ps != 0 for x in lens)
        page = 2 * case["layers"] * n_kv * ps * (hd + 1 / BLOCK)
        return {"bytes": 2 * copied * page + 4 * (2 + 2 * c) * sum(-(-x // ps) for x in lens), "flops": 0}
    if case["kind"] == "compact":
        pages = case["pages"]
        used = max(1, min(pages, int(pages * case["used"])))
        page = 2 * case["layers"] * n_kv * case["page"] * (hd + 1 / BLOCK)
        # on the average (used / pages) (pages - used) of the pages in use lie behind the front
        return {"bytes": 2 * used * (pages - used) / pages * page + 8 * (pages + used), "flops": 0}
    lens, new = _lens(case)
    q = TYPES[case["q"]][0].itemsize
    if case["kind"] == "store":
        rows = sum(new)
        store = rows * (4 * (nh + 2 * n_kv) * hd + 4 * hd + nh * hd * q + 2 * n_kv * hd)
        return {"bytes": store + sum(lens) * n_kv * hd * 2 * (1 + 2),
                "flops": rows * (nh + n_kv) * hd * (3 + 4 * case["norm"])}
    pairs = sum(t * x - t * (t - 1) // 2 for x, t in zip(lens, new)) * nh
    return {"bytes": sum(lens) * n_kv * 2 * (hd + 1 / BLOCK) + 2 * sum(new) * nh * hd * q, "flops": 4 * pairs * hd}


# ------------------------------------------------------------------------------------------ exact
def _stored(case, st, name, s):
    """K or V bytes of sequence s as (values in 64 bits [n_kv][positions][hd], exponents [n_kv][positions / 16])."""
    _, n_kv, hd = HEADS[case["heads"]]
    ps = case["page"]
    rows, exps = [], []
    for page in st["table"][s].tolist():
        x = _values(case, st[name][page]).double()
        x = x.view(n_kv, hd // 16, ps, 16).transpose(1, 2) if name == "k" else x.view(n_kv, ps // 16, hd, 16).transpose(2, 3)
        rows.append(x.reshape(n_kv, ps, hd))
        exps.append(st[name + "_exp"][page].double() - 127)
    return torch.cat(rows, 1), torch.cat(exps, 1)


def _exact_store(case):
    st = case["state"]
    nh, n_kv, hd = HEADS[case["heads"]]
    lens, new = _lens(case)
    q = st["q_out"].double()
    read = {"k": st["k_read"].double(), "v": st["v_read"].double()}
    half, low = hd // 2, torch.tensor(-126.0, dtype=torch.float64, device="cuda")
    for s, (x, t) in enumerate(zip(lens, new)):
        r = slice(s * case["new"], s * case["new"] + t)
        row = st["qkv"][r].double().view(t, -1, hd)
        z = torch.complex(st["cos"][r].double(), st["sin"][r].double())[:, None]
        parts = []
        for part, norm in ((row[:, :nh], 0), (row[:, nh:nh + n_kv], 1)):
            if st["norms"] is not None:
                part = part / ((part.square().sum(-1, keepdim=True) / hd + 1e-6).sqrt()) * st["norms"][norm].double()
            pair = torch.complex(part[..., :half], part[..., half:]) if case["split_half"] else \
                torch.view_as_complex(part.reshape(t, -1, half, 2).contiguous())
            y = torch.view_as_real(pair * z)
            parts.append((y.transpose(-1, -2) if case["split_half"] else y).reshape(t, -1, hd))
        q[r] = parts[0].reshape(t, -1)
        for name, rows in (("k", parts[1]), ("v", row[:, nh + n_kv:])):
            held, exps = _stored(case, st, name, s)
            first, begin = x - t, (x - t) // BLOCK * BLOCK
            end = -(-x // BLOCK) * BLOCK
            held = held * torch.exp2(exps).repeat_interleave(BLOCK, 1)[..., None]
            found = held[:, :x].clone()
            block = torch.zeros(n_kv, end - begin, hd, dtype=torch.float64, device="cuda")
            block[:, first - begin:x - begin] = rows.transpose(0, 1)
            top = block.abs().view(n_kv, -1, BLOCK * hd).amax(-1)
            e = torch.maximum(torch.ceil(torch.log2(top / LARGEST[case["kv"]])), low)
            if first > begin:
                e[:, 0] = torch.maximum(e[:, 0], exps[:, begin // BLOCK])
                block[:, :first - begin] = held[:, begin:first]
            step = torch.exp2(e).repeat_interleave(BLOCK, 1)[..., None]
            block = block / step
            if case["kv"] == "i8":
                block = block.round()
            else:  # 3 bits behind the leading one, 2^-9 at the least
                unit = torch.exp2(torch.floor(torch.log2(block.abs().clamp_min(2.0 ** -6))) - 3)
                block = (block / unit).round() * unit
            found[:, begin:] = (block * step)[:, :x - begin]
            read[name][s, :, :x] = found
    return {"q": q, **read}


def _exact_logits(case):
    st = case["state"]
    out = st["out"].double()
    v = VOCAB[case["vocab"]]
    for s in range(case["seqs"]):
        n, cut = int(st["history_lens"][s]), int(st["prompt_lens"][s])
        r, f, p = (float(st[k][s]) for k in ("repetition", "frequency", "presence"))
        bias = {}
        for i in range(int(st["bias_lens"][s])):
            bias[int(st["bias_tokens"][s, i])] = float(st["bias_values"][s, i])
        for t in range(int(st["draft_lens"][s]) + 1):
            drafts = st["draft"][s, :t].long()
            count = torch.bincount(torch.cat([st["history"][s, cut:n].long(), drafts]), minlength=v).double()
            seen = torch.bincount(torch.cat([st["history"][s, :n].long(), drafts]), minlength=v) > 0
            x = st["logits"][s, t].double()
            x = torch.where(seen, torch.where(x > 0, x / r, x * r), x) - f * count - p * (count > 0)
            if bias:
                x[torch.tensor(list(bias), device="cuda")] += torch.tensor(list(bias.values()), device="cuda").double()
            if st["mask"] is not None:
                bits = st["mask"][s, t].cpu().numpy().view("uint8")
                allowed = torch.from_numpy(np.unpackbits(bits, bitorder="little")[:v].copy()).cuda()
                x[allowed == 0] = -math.inf
            out[s, t] = x
    return {"out": out}


def exact(case, seed):
    if case["kind"] in ("branch", "compact"):  # whole numbers
        return None
    st = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_store({**case, "state": st})
    if case["kind"] == "logits":
        return _exact_logits({**case, "state": st})
    nh, n_kv, hd = HEADS[case["heads"]]
    lens, new = _lens(case)
    out, g = st["out"].double(), nh // n_kv
    for s, (x, t) in enumerate(zip(lens, new)):
        k, v = (z * torch.exp2(e).repeat_interleave(BLOCK, 1)[..., None]
                for z, e in (_stored(case, st, "k", s), _stored(case, st, "v", s)))
        rows = st["q"][s * case["new"]:s * case["new"] + t].double().view(t, nh, hd)
        for h in range(nh):
            for i in range(0, t, 512):
                part = rows[i:i + 512, h]
                m = x - t + i + part.shape[0]
                score = part @ k[h // g, :m].t() / math.sqrt(hd)
                late = torch.arange(m, device="cuda")[None] > x - t + i + torch.arange(part.shape[0], device="cuda")[:, None]
                w = torch.softmax(score.masked_fill(late, -math.inf), -1)
                out[s * case["new"] + i:s * case["new"] + i + part.shape[0], h * hd:(h + 1) * hd] = w @ v[h // g, :m]
    return {"out": out}

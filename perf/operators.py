"""The operators of batched serving over a paged key/value cache, as cases that can be timed and compared.

Kinds (head layouts and vocabularies are those of the framework's own model configurations):

  store   RoPE (with optional QK RMSNorm) of new tokens' q and k rows, their K and V written into
          the pages of a cache (camelid_hip_paged_rope_kv)
  attend  attention of one or a few new tokens per sequence over the paged cache, optionally adding
          each cached position's softmax weight to its accumulator (camelid_hip_paged_attention)
  evict   the positions of lowest accumulated weight leave a cache that has grown past its budget;
          the rest moves up in place (camelid_hip_paged_evict)
  verify  drafted tokens accepted or replaced by speculative sampling from the target's
          distribution with given uniform numbers, and the log-probabilities of what comes out
          (camelid_hip_verify_drafts); no drafts: the next token sampled

A cache is n_pages pages of page_size positions.  K of one page: [n_kv][hd / 8][page_size][8], V:
[n_kv][page_size / 8][hd][8]; position p of sequence s lies in page table[s][p / page_size].
"""
from __future__ import annotations

import math

import torch

own = False

# (n_heads, n_kv, head_dim) of the framework's configurations, and their vocabularies
HEADS = {"tinyllama": (32, 4, 64), "llama3b": (24, 8, 128), "mistral": (32, 8, 128), "qwen": (32, 8, 128)}
VOCAB = {"tinyllama": 32000, "llama3b": 128256, "mistral": 32768, "qwen": 151936}
TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 2)}


def listed():
    return [
        # the smallest call: one token of one sequence, where only latency counts
        {"name": "store tinyllama 1x1", "kind": "store", "heads": "tinyllama", "seqs": 1, "new": 1, "ragged": False,
         "history": 127, "page": 16, "norm": False, "split_half": False, "q": "f32", "kv": "f16"},
        # drafts of up to 5 tokens of a batch, with QK-norm and split-half pairs
        {"name": "store qwen 24x5", "kind": "store", "heads": "qwen", "seqs": 24, "new": 5, "ragged": True,
         "history": 300, "page": 32, "norm": True, "split_half": True, "q": "bf16", "kv": "bf16"},
        # the prompts of a small batch, one token short of whole pages
        {"name": "store llama3b 4x2047", "kind": "store", "heads": "llama3b", "seqs": 4, "new": 2047, "ragged": True,
         "history": 0, "page": 64, "norm": False, "split_half": False, "q": "f32", "kv": "f16"},
        # chat with one user on the smallest model: latency
        {"name": "attend tinyllama 1x127", "kind": "attend", "heads": "tinyllama", "seqs": 1, "new": 1, "len": 127,
         "ragged": False, "page": 16, "q": "f32", "kv": "f16", "weights": False},
        # one user far into a long document: the split over the length has to fill the GPU
        {"name": "attend mistral 1x8199", "kind": "attend", "heads": "mistral", "seqs": 1, "new": 1, "len": 8199,
         "ragged": False, "page": 64, "q": "f32", "kv": "f16", "weights": False},
        # a serving batch of every age, 16-bit activations
        {"name": "attend llama3b 64x4001", "kind": "attend", "heads": "llama3b", "seqs": 64, "new": 1, "len": 4001,
         "ragged": True, "page": 32, "q": "bf16", "kv": "bf16", "weights": False},
        # drafts verified over caches kept to a budget: the weights that eviction goes by
        {"name": "attend qwen 16x1100 d5", "kind": "attend", "heads": "qwen", "seqs": 16, "new": 5, "len": 1100,
         "ragged": True, "page": 32, "q": "f32", "kv": "f16", "weights": True},
        # the largest call: a few sequences of very long contexts
        {"name": "attend mistral 4x65536", "kind": "attend", "heads": "mistral", "seqs": 4, "new": 1, "len": 65536,
         "ragged": False, "page": 16, "q": "f16", "kv": "f16", "weights": False},
        # upkeep while decoding: every 64 steps back to the budget
        {"name": "evict qwen 16x1088", "kind": "evict", "heads": "qwen", "seqs": 16, "len": 1088, "ragged": False,
         "page": 32, "kv": "f16", "keep": 1024, "recent": 256},
        # after long prompts: the cache shrinks to an eighth
        {"name": "evict mistral 4x16383", "kind": "evict", "heads": "mistral", "seqs": 4, "len": 16383,
         "ragged": True, "page": 64, "kv": "bf16", "keep": 2048, "recent": 512},
        # one user, drafts looked up in the prompt (no draft distribution)
        {"name": "verify tinyllama 1x4", "kind": "verify", "vocab": "tinyllama", "seqs": 1, "drafts": 4,
         "ragged": False, "draft_logits": False, "type": "f32"},
        # a serving batch with a draft model's logits, greedy sequences among them
        {"name": "verify qwen 32x5", "kind": "verify", "vocab": "qwen", "seqs": 32, "drafts": 5, "ragged": True,
         "draft_logits": True, "type": "f32"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "evict", "verify"])
    c = {"kind": kind}
    if kind == "verify":
        c.update(vocab=rng.choice(sorted(VOCAB)), seqs=_log_int(rng, 1, 48), drafts=rng.randint(0, 7),
                 ragged=rng.random() < 0.5, draft_logits=rng.random() < 0.5, type=rng.choice(["f32", "f16", "bf16"]))
        if c["drafts"] == 0:
            c["draft_logits"] = False
        return c
    c.update(heads=rng.choice(sorted(HEADS)), ragged=rng.random() < 0.6, page=rng.choice([8, 16, 32, 64, 128, 256]),
             kv=rng.choice(["f16", "bf16"]))
    if kind == "store":
        c.update(seqs=_log_int(rng, 1, 64), new=_log_int(rng, 1, 2048), history=_log_int(rng, 1, 1024),
                 norm=rng.random() < 0.5, split_half=rng.random() < 0.5, q=rng.choice(["f32", c["kv"]]))
        c["new"] = min(c["new"], 8192 // c["seqs"])
        return c
    c.update(seqs=_log_int(rng, 1, 128))
    most = 200000 // c["seqs"]
    if kind == "attend":
        c.update(new=rng.choice([1, 1, rng.randint(2, 8)]), len=min(_log_int(rng, 8, 65536), most),
                 q=rng.choice(["f32", c["kv"]]), weights=rng.random() < 0.4)
        return c
    c.update(len=min(_log_int(rng, 64, 32768), most // 2))
    c.update(keep=max(1, int(c["len"] * rng.uniform(0.1, 1.1))))
    c.update(recent=int(c["keep"] * rng.uniform(0.0, 1.0)))
    return c


# ---------------------------------------------------------------------------------------- inputs
def _spread(n, top, ragged):
    """Lengths 1 ... top of n sequences, spread evenly without order (the first one is `top`)."""
    return [top if not ragged or i == 0 else 1 + int(top * ((i * 0.6180339887498949) % 1.0)) for i in range(n)]


def _lens(case):
    """(positions in the cache with the new tokens, new tokens) of each sequence."""
    n = case["seqs"]
    if case["kind"] == "evict":
        return _spread(n, case["len"], case["ragged"]), None
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
    kv = TYPES[case["kv"]][0]
    shape = (pages, n_kv, hd * ps)
    k = torch.empty(shape, dtype=kv, device="cuda").normal_(generator=gen)
    v = torch.empty(shape, dtype=kv, device="cuda").normal_(generator=gen)
    table = torch.randperm(pages, generator=gen, device="cuda")[:used].to(torch.int32).view(case["seqs"], stride)
    return {"k": k, "v": v, "table": table.contiguous(), "lens": _u32(lens), "pages": pages, "stride": stride}


def _rope(case, gen, rows, hd, lens, new):
    """cos and sin rows [rows][hd / 2] of each row's position."""
    n = case["new"]
    pos = torch.tensor([[x - t + i for i in range(n)] for x, t in zip(lens, new)], device="cuda").double().view(rows, 1)
    f = 500000.0 ** (-2.0 * torch.arange(hd // 2, device="cuda").double() / hd)
    return (pos * f).cos().float(), (pos * f).sin().float()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    st = {"case": case}
    if case["kind"] == "verify":
        n, k, v = case["seqs"], case["drafts"], VOCAB[case["vocab"]]
        dt = TYPES[case["type"]][0]
        target = torch.empty(n, k + 1, v, device="cuda").normal_(0, 2.5, generator=gen)
        st["draft_logits"] = None
        if case["draft_logits"]:  # a draft model's logits: the target's with an error
            noise = torch.empty(n, k, v, device="cuda").normal_(0, 0.7, generator=gen)
            st["draft_logits"] = (target[:, :k] + noise).to(dt).contiguous()
            probs = torch.softmax(st["draft_logits"].float(), -1).view(n * k, v)
            st["tokens"] = torch.multinomial(probs, 1, generator=gen).to(torch.int32).view(n, k)
        else:  # tokens looked up: some right, some wrong
            right = torch.rand(n, k, generator=gen, device="cuda") < 0.7
            guess = torch.randint(v, (n, k), generator=gen, device="cuda")
            best = target[:, :k].argmax(-1)
            st["tokens"] = torch.where(right, best, guess).to(torch.int32).contiguous()
            if k:  # what a prompt repeats, the target is sure of
                target[:, :k].scatter_add_(2, best[..., None], torch.full((n, k, 1), 8.0, device="cuda"))
        st["target"] = target.to(dt)
        st["uniforms"] = torch.rand(n, k + 1, generator=gen, device="cuda")
        st["temperature"] = torch.tensor([0.0 if i % 8 == 7 else 0.6 + 0.1 * (i % 6) for i in range(n)],
                                         device="cuda")
        st["draft_lens"] = _u32([min(x, k) for x in _spread(n, max(k, 1), case["ragged"])])
        st["accepted"] = torch.full((n,), -1, dtype=torch.int32, device="cuda")
        st["out"] = torch.full((n, k + 1), -1, dtype=torch.int32, device="cuda")
        st["logprobs"] = torch.zeros(n, k + 1, device="cuda")
        return st
    nh, n_kv, hd = HEADS[case["heads"]]
    n = case["seqs"]
    st.update(_cache(case, gen))
    lens, new = _lens(case)
    if case["kind"] == "evict":
        cap = st["stride"] * case["page"]
        # softmax weights add up to heavy tails: a few positions hold most of it
        st["weights"] = torch.empty(n, n_kv, cap, device="cuda").log_normal_(-2.0, 2.0, generator=gen)
        st["lens_out"] = torch.zeros(n, dtype=torch.int32, device="cuda")
        st["kept"] = torch.full((n, n_kv, case["keep"]), -1, dtype=torch.int32, device="cuda")
        return st
    rows = n * case["new"]
    st["new_lens"] = _u32(new)
    qt = TYPES[case["q"]][0]
    if case["kind"] == "store":
        st["qkv"] = torch.empty(rows, (nh + 2 * n_kv) * hd, device="cuda").normal_(0, 1.3, generator=gen)
        st["cos"], st["sin"] = _rope(case, gen, rows, hd, lens, new)
        st["norms"] = [torch.empty(hd, device="cuda").normal_(1.0, 0.1, generator=gen) for _ in range(2)] \
            if case["norm"] else None
        st["q_out"] = torch.zeros(rows, nh * hd, dtype=qt, device="cuda")
        return st
    st["q"] = torch.empty(rows, nh * hd, device="cuda").normal_(0, 1.5, generator=gen).to(qt)
    st["out"] = torch.zeros(rows, nh * hd, dtype=qt, device="cuda")
    st["weights"] = torch.empty(n, n_kv, st["stride"] * case["page"], device="cuda").uniform_(0, 3, generator=gen) \
        if case["weights"] else None
    return st


# ------------------------------------------------------------------------------------ plain forms
def _dense(st, name):
    """K or V of every sequence as [seqs][n_kv][positions][hd], in the cache's type."""
    c = st["case"]
    _, n_kv, hd = HEADS[c["heads"]]
    ps, n, stride = c["page"], c["seqs"], st["stride"]
    x = st[name][st["table"].long()]
    if name == "k":  # [n][stride][n_kv][hd / 8][ps][8]
        x = x.view(n, stride, n_kv, hd // 8, ps, 8).permute(0, 2, 1, 4, 3, 5)
    else:  # [n][stride][n_kv][ps / 8][hd][8]
        x = x.view(n, stride, n_kv, ps // 8, hd, 8).permute(0, 2, 1, 3, 5, 4)
    return x.reshape(n, n_kv, stride * ps, hd)


def _put(st, name, seq, head, pos, rows):
    """rows [...][hd] to positions of sequences; seq, head, pos: index tensors of rows' leading shape."""
    c = st["case"]
    _, n_kv, hd = HEADS[c["heads"]]
    ps = c["page"]
    page = st["table"].long()[seq, pos // ps]
    off = pos % ps
    if name == "k":
        st["k"].view(-1, n_kv, hd // 8, ps, 8)[page, head, :, off, :] = rows.unflatten(-1, (hd // 8, 8))
    else:
        st["v"].view(-1, n_kv, ps // 8, hd, 8)[page, head, off // 8, :, off % 8] = rows


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

    t = torch.arange(new, device="cuda")[None]
    real = (t < st["new_lens"][:, None]).view(-1)
    seq = torch.arange(n, device="cuda")[:, None].expand(n, new).reshape(-1)[real]
    pos = (st["lens"][:, None] - st["new_lens"][:, None] + t).view(-1).long()[real]
    st["q_out"][real] = turn(q).flatten(1).to(st["q_out"].dtype)[real]
    seq, pos, head = seq[:, None], pos[:, None], torch.arange(n_kv, device="cuda")[None]
    _put(st, "k", seq, head, pos, turn(k)[real].to(st["k"].dtype))
    _put(st, "v", seq, head, pos, v[real].to(st["v"].dtype))
    return {"q": st["q_out"], "k": st["k"], "v": st["v"]}


def _plain_attend(st):
    c = st["case"]
    nh, n_kv, hd = HEADS[c["heads"]]
    n, new, g = c["seqs"], c["new"], nh // n_kv
    cap = st["stride"] * c["page"]
    scale = 1.0 / math.sqrt(hd)
    q = st["q"].float().view(n, new, n_kv, g, hd).permute(0, 2, 1, 3, 4).reshape(n, n_kv, new * g, hd)
    s = torch.matmul(q, _dense(st, "k").float().transpose(-1, -2).contiguous()) * scale
    t = torch.arange(new, device="cuda")
    last = st["lens"][:, None] - st["new_lens"][:, None] + t[None]        # [n][new]: last visible position
    real = t[None] < st["new_lens"][:, None]
    p = torch.arange(cap, device="cuda")
    seen = ((p[None, None] <= last[..., None]) & real[..., None]).repeat_interleave(g, 1)[:, None]
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True)
    e = torch.where(seen, torch.exp(s - top), torch.zeros_like(s))
    w = e / e.sum(-1, keepdim=True).clamp_min(1e-38)
    o = torch.matmul(w, _dense(st, "v").float().contiguous())
    o = o.view(n, n_kv, new, g, hd).permute(0, 2, 1, 3, 4).reshape(n, new, nh * hd)
    st["out"].view(n, new, nh * hd)[real] = o[real].to(st["out"].dtype)
    if st["weights"] is None:
        return {"out": st["out"]}
    # the new tokens' own positions start at nothing
    first = (st["lens"] - st["new_lens"])[:, None, None]
    old = torch.where(p < first, st["weights"], torch.zeros_like(st["weights"]))
    st["weights"].copy_(torch.where(p < st["lens"][:, None, None], old + w.sum(2), st["weights"]))
    return {"out": st["out"], "weights": st["weights"]}


def _plain_evict(st):
    c = st["case"]
    _, n_kv, _ = HEADS[c["heads"]]
    n, cap = c["seqs"], st["stride"] * c["page"]
    p = torch.arange(cap, device="cuda")
    lens = st["lens"][:, None, None]
    key = torch.where((p >= lens - c["recent"]) | (lens <= c["keep"]), torch.full_like(st["weights"], math.inf),
                      st["weights"])
    key = torch.where(p < lens, key, torch.full_like(key, -math.inf))
    keep = min(c["keep"], cap)
    at = torch.sort(key, dim=-1, descending=True, stable=True)[1][..., :keep].sort(-1)[0]
    seq, head = torch.arange(n, device="cuda")[:, None, None], torch.arange(n_kv, device="cuda")[None, :, None]
    dest = p[:keep].expand(n, n_kv, keep)
    held = _dense(st, "k"), _dense(st, "v")
    _put(st, "k", seq, head, dest, held[0][seq, head, at])
    _put(st, "v", seq, head, dest, held[1][seq, head, at])
    st["weights"][..., :keep] = st["weights"].gather(2, at)
    st["lens_out"].copy_(st["lens"].clamp_max(c["keep"]))
    st["kept"][..., :keep] = torch.where(dest < lens, at, -1).to(torch.int32)
    return {"k": st["k"], "v": st["v"], "weights": st["weights"], "lens": st["lens_out"], "kept": st["kept"]}


def _plain_verify(st):
    """In 64 bits: the token drawn depends on which side of a border of 100000 partial sums a number lies."""
    c = st["case"]
    n, k, v = c["seqs"], c["drafts"], VOCAB[c["vocab"]]
    temp = st["temperature"].double().view(n, 1, 1)
    greedy = temp == 0

    def logs(x):  # a greedy sequence's as at temperature 1
        x = x.double()
        x = (x - x.amax(-1, keepdim=True)) / torch.where(greedy, 1.0, temp)
        return x - x.exp().sum(-1, keepdim=True).log()

    def probs(x):
        y = logs(x).exp()
        one = torch.zeros_like(y).scatter_(2, x.argmax(-1, keepdim=True), 1.0)
        return torch.where(greedy, one, y)

    p, lp = probs(st["target"]), logs(st["target"])
    tokens = st["tokens"].long()
    if c["draft_logits"]:
        # a greedy sequence's draft counts as certain
        q = torch.where(greedy, torch.zeros(n, k, v, dtype=torch.float64, device="cuda")
                        .scatter_(2, tokens[..., None], 1.0), probs(st["draft_logits"]))
    else:
        q = torch.zeros(n, k, v, dtype=torch.float64, device="cuda").scatter_(2, tokens[..., None], 1.0)
    u = st["uniforms"].double()
    px, qx = (z.gather(2, tokens[..., None])[..., 0] for z in (p[:, :k], q))
    t = torch.arange(k + 1, device="cuda")[None]
    ok = (u[:, :k] * qx < px) & (t[:, :k] < st["draft_lens"][:, None])
    took = ok.long().cumprod(1).sum(1)
    seq = torch.arange(n, device="cuda")
    pj = p[seq, took]
    qj = torch.cat([q, torch.zeros(n, 1, v, dtype=torch.float64, device="cuda")], 1)[seq, took]
    r = (pj - torch.where((took < st["draft_lens"])[:, None], qj, 0.0)).clamp_min(0)
    r = torch.where(r.sum(-1, keepdim=True) > 0, r, pj)
    sums = r.cumsum(-1)
    last = (torch.arange(v, device="cuda") * (r > 0)).amax(-1)
    pick = (sums <= u[:, k:] * sums[:, -1:]).sum(-1).minimum(last)
    st["accepted"].copy_(took)
    padded = torch.cat([tokens, torch.full((n, 1), -1, device="cuda")], 1)
    st["out"].copy_(torch.where(t < took[:, None], padded, torch.where(t == took[:, None], pick[:, None], -1)))
    told = lp.gather(2, st["out"].long().clamp_min(0)[..., None])[..., 0]
    st["logprobs"].copy_(torch.where(t <= took[:, None], told, 0.0))
    return {"accepted": st["accepted"], "tokens": st["out"], "logprobs": st["logprobs"]}


# ------------------------------------------------------------------------------ the framework's calls
def _p(t):
    return None if t is None else t.data_ptr()


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _workspace(st, n_bytes, *sizes):
    """The scratch memory that a program keeps between its calls of the same sizes."""
    if "workspace" not in st:
        st["workspace"] = torch.empty(n_bytes(*sizes), dtype=torch.uint8, device="cuda")
    return st["workspace"]


def _own(st):
    from camelid_amd import _native
    lib, c = _native.lib(), st["case"]
    if c["kind"] == "verify":
        n, k, v = c["seqs"], c["drafts"], VOCAB[c["vocab"]]
        ws = _workspace(st, lib.camelid_hip_verify_drafts_workspace, n, k, v)
        _native.check(lib.camelid_hip_verify_drafts(
            _p(st["target"]), _p(st["draft_logits"]), TYPES[c["type"]][1], _p(st["tokens"]), _p(st["draft_lens"]), n, k,
            v, _p(st["temperature"]), _p(st["uniforms"]), _p(st["accepted"]), _p(st["out"]),
            _p(st["logprobs"]), _p(ws), ws.numel(), _stream()))
        return {"accepted": st["accepted"], "tokens": st["out"], "logprobs": st["logprobs"]}
    nh, n_kv, hd = HEADS[c["heads"]]
    n, ps, kv = c["seqs"], c["page"], TYPES[c["kv"]][1]
    if c["kind"] == "store":
        norms = st["norms"] or (None, None)
        _native.check(lib.camelid_hip_paged_rope_kv(
            _p(st["qkv"]), n, c["new"], _p(st["new_lens"]), nh, n_kv, hd, hd, int(c["split_half"]), _p(st["cos"]),
            _p(st["sin"]), _p(norms[0]), _p(norms[1]), 1e-6, _p(st["q_out"]), TYPES[c["q"]][1], _p(st["k"]),
            _p(st["v"]), kv, st["pages"], ps, _p(st["table"]), st["stride"], _p(st["lens"]), None, _stream()))
        return {"q": st["q_out"], "k": st["k"], "v": st["v"]}
    if c["kind"] == "attend":
        ws = _workspace(st, lib.camelid_hip_paged_attention_workspace, n, c["new"], nh, n_kv, hd, ps, st["stride"],
                        int(c["weights"]))
        _native.check(lib.camelid_hip_paged_attention(
            _p(st["q"]), TYPES[c["q"]][1], nh * hd, n, c["new"], _p(st["new_lens"]), nh, n_kv, hd, _p(st["k"]),
            _p(st["v"]), kv, st["pages"], ps, _p(st["table"]), st["stride"], _p(st["lens"]), 1.0 / math.sqrt(hd),
            _p(st["out"]), nh * hd, _p(st["weights"]), _p(ws), ws.numel(), None, _stream()))
        return {"out": st["out"], "weights": st["weights"]} if c["weights"] else {"out": st["out"]}
    ws = _workspace(st, lib.camelid_hip_paged_evict_workspace, n, n_kv, ps, st["stride"], c["keep"])
    _native.check(lib.camelid_hip_paged_evict(
        _p(st["k"]), _p(st["v"]), st["pages"], ps, n_kv, hd, _p(st["table"]), st["stride"], _p(st["lens"]), n,
        _p(st["weights"]), c["keep"], c["recent"], _p(st["lens_out"]), _p(st["kept"]), _p(ws), ws.numel(), None,
        _stream()))
    return {"k": st["k"], "v": st["v"], "weights": st["weights"], "lens": st["lens_out"], "kept": st["kept"]}


def run(state):
    if own:
        return _own(state)
    return {"store": _plain_store, "attend": _plain_attend, "evict": _plain_evict,
            "verify": _plain_verify}[state["case"]["kind"]](state)


# ------------------------------------------------------------------------------------------- work
def work(case):
    """Each input that the operator cannot do without read once, each output written once."""
    if case["kind"] == "verify":
        n, k, v = case["seqs"], case["drafts"], VOCAB[case["vocab"]]
        lens = [min(x, k) for x in _spread(n, max(k, 1), case["ragged"])]
        rows = sum(x + 1 + (x if case["draft_logits"] else 0) for x in lens)
        size = 4 if case["type"] == "f32" else 2
        return {"bytes": rows * v * size + n * (12 * k + 16), "flops": 4 * rows * v}
    nh, n_kv, hd = HEADS[case["heads"]]
    lens, new = _lens(case)
    if case["kind"] == "evict":
        kept = sum(min(x, case["keep"]) for x in lens if x > case["keep"])
        seen = sum(x for x in lens if x > case["keep"])
        # weights read; what stays: K and V read and written, weights and index written
        return {"bytes": n_kv * (4 * seen + kept * (8 * hd + 8)) + 8 * case["seqs"],
                "flops": n_kv * seen}
    q = TYPES[case["q"]][0].itemsize
    if case["kind"] == "store":
        rows = sum(new)
        return {"bytes": rows * (4 * (nh + 2 * n_kv) * hd + 4 * hd + nh * hd * q + 4 * n_kv * hd),
                "flops": rows * (nh + n_kv) * hd * (3 + 4 * case["norm"])}
    held = sum(lens)
    pairs = sum(t * x - t * (t - 1) // 2 for x, t in zip(lens, new)) * nh
    return {"bytes": held * n_kv * hd * 4 + 2 * sum(new) * nh * hd * q + (8 * held * n_kv if case["weights"] else 0),
            "flops": 4 * pairs * hd}


# ------------------------------------------------------------------------------------------ exact
def _cells(c, st):
    """(sequence, position) -> index of K's and V's elements [n_kv][hd] in the flat buffers, one row a pair."""
    _, n_kv, hd = HEADS[c["heads"]]
    ps = c["page"]
    table = st["table"].cpu().tolist()
    h = torch.arange(n_kv, device="cuda").view(-1, 1) * (hd * ps)
    d = torch.arange(hd, device="cuda").view(1, -1)

    def at(s, positions):
        pages = torch.tensor([table[s][p // ps] for p in positions], device="cuda").view(-1, 1, 1)
        o = torch.tensor([p % ps for p in positions], device="cuda").view(-1, 1, 1)
        base = pages * (n_kv * hd * ps) + h
        return base + (d // 8 * ps + o) * 8 + d % 8, base + (o // 8 * hd + d) * 8 + o % 8
    return at


def _exact_logprobs(case, st):
    """One sequence and one draft after the other, as the definition reads."""
    found = torch.zeros(case["seqs"], case["drafts"] + 1, dtype=torch.float64, device="cuda")
    temps, lens, tokens, u = (st[k].tolist() for k in ("temperature", "draft_lens", "tokens", "uniforms"))
    for s, temp in enumerate(temps):
        for t in range(lens[s] + 1):
            x = st["target"][s, t].double()
            told = torch.log_softmax(x / (temp or 1.0), 0)
            p = torch.softmax(x / temp, 0) if temp else torch.nn.functional.one_hot(x.argmax(), x.numel()).double()
            rest = p
            if t < lens[s]:
                d = tokens[s][t]
                if case["draft_logits"] and temp:
                    q = torch.softmax(st["draft_logits"][s, t].double() / temp, 0)
                else:
                    q = torch.zeros_like(p)
                    q[d] = 1.0
                if u[s][t] * q[d].item() < p[d].item():
                    found[s, t] = told[d]
                    continue
                rest = (p - q).clamp_min(0)
            sums = rest.cumsum(0)
            found[s, t] = told[torch.searchsorted(sums, sums[-1:] * u[s][-1], right=True)][0]
            break
    return found


def exact(case, seed):
    if case["kind"] == "verify":
        return {"accepted": None, "tokens": None, "logprobs": _exact_logprobs(case, prepare(case, seed))}
    st = prepare(case, seed)
    nh, n_kv, hd = HEADS[case["heads"]]
    lens, new = _lens(case)
    at = _cells(case, st)
    if case["kind"] == "evict":
        k0, v0, w0 = st["k"].double().view(-1), st["v"].double().view(-1), st["weights"].double()
        k, v, w = k0.clone(), v0.clone(), w0.clone()
        host, heads = st["weights"].cpu().tolist(), torch.arange(n_kv, device="cuda")
        for s, x in enumerate(lens):
            if x <= case["keep"]:
                continue
            cut = x - case["recent"]
            kept = []
            for h in range(n_kv):
                best = sorted(range(cut), key=lambda p: (-host[s][h][p], p))[:case["keep"] - case["recent"]]
                kept.append(sorted(best) + list(range(cut, x)))
            src_k, src_v = at(s, range(x))
            dst_k, dst_v = at(s, range(case["keep"]))
            rows = torch.tensor(kept, device="cuda").t()  # [keep][n_kv]
            k[dst_k] = k0[src_k[rows, heads]]
            v[dst_v] = v0[src_v[rows, heads]]
            w[s, :, :case["keep"]] = w0[s].gather(1, rows.t())
        return {"k": k.view_as(st["k"]), "v": v.view_as(st["v"]), "weights": w, "lens": None, "kept": None}
    if case["kind"] == "store":
        k, v, q = st["k"].double().view(-1), st["v"].double().view(-1), st["q_out"].double()
        half = hd // 2
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
            for p in range(0, t, 4096):
                ik, iv = at(s, range(x - t + p, min(x, x - t + p + 4096)))
                k[ik], v[iv] = parts[1][p:p + 4096], row[p:p + 4096, nh + n_kv:]
        return {"q": q, "k": k.view_as(st["k"]), "v": v.view_as(st["v"])}
    out, g = st["out"].double(), nh // n_kv
    weights = st["weights"].double() if case["weights"] else None
    fk, fv = st["k"].view(-1), st["v"].view(-1)
    for s, (x, t) in enumerate(zip(lens, new)):
        ik, iv = at(s, range(x))
        for h in range(n_kv):
            keys, vals = fk[ik[:, h]].double(), fv[iv[:, h]].double()
            if weights is not None:
                weights[s, h, x - t:x] = 0
            rows = st["q"][s * case["new"]:s * case["new"] + t].double().view(t, nh, hd)[:, h * g:(h + 1) * g]
            for i in range(t):
                m = x - t + i + 1
                w = torch.softmax(rows[i] @ keys[:m].t() / math.sqrt(hd), -1)
                out[s * case["new"] + i].view(nh, hd)[h * g:(h + 1) * g] = w @ vals[:m]
                if weights is not None:
                    weights[s, h, :m] += w.sum(0)
    return {"out": out, "weights": weights} if weights is not None else {"out": out}

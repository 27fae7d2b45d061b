"""Performance cases of the decoder's operators around an attention cache in 8 bits and the greedy pick.

Four operators, as a decode step or a prompt uses them one after the other:

- ``rope``: the norm of every query and key head, the rotation by its position, and the store of keys and values
  into the f32 cache (``qlin_launch_qk_norm_rope_store_kv``);
- ``store``: the same into the 8-bit cache (``qlin_launch_qk_norm_rope_store_kv8``), and the stored positions read
  back as the values they stand for (``qlin_launch_kv8_read``);
- ``attend``: attention over the 8-bit cache (``qlin_launch_attend_kv8``);
- ``logits``: penalties for repeated tokens, biases, a grammar mask and the greedy pick
  (``qlin_launch_logits_controls``).

The 8-bit cache: blocks of 32 positions.  A complete block of a key head is a record of 64 * head_dim + 16 bytes in a
page: int8 codes of the keys, of the values, then the two f32 scales (``key_codes`` and ``value_codes`` below have the
order of the codes).  The last 64 positions also stand in an f32 ring, from which the open block is read.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
BLOCK, RING = 32, 64
EPS, THETA = 1e-6, 1e6
NEG = -math.inf


def listed():
    return [
        # one decode step of the 0.5B decoder (14 query and 2 key heads of 64): the smallest launch
        {"name": "rope_token", "op": "rope", "heads": 14, "kv": 2, "d": 64, "rd": 64, "pairs": 0, "rows": 1, "start": 159},
        # a ragged prompt of a 7B decoder (28 query and 4 key heads of 128), continued in mid conversation
        {"name": "rope_prompt", "op": "rope", "heads": 28, "kv": 4, "d": 128, "rd": 128, "pairs": 0, "rows": 1877,
         "start": 411},
        # one decode step of a batch of 24 sequences at positions of their own
        {"name": "store_batch", "op": "store", "heads": 28, "kv": 4, "d": 128, "rd": 128, "pairs": 0, "seqs": 24, "rows": 1,
         "start": 3000, "norms": True},
        # a prompt into an empty cache
        {"name": "store_prompt", "op": "store", "heads": 28, "kv": 4, "d": 128, "rd": 128, "pairs": 0, "seqs": 1,
         "rows": 2011, "start": 0, "norms": True},
        # the 0.5B decoder's decode step early in a conversation: latency
        {"name": "attend_token", "op": "attend", "heads": 14, "kv": 2, "d": 64, "seqs": 1, "rows": 1, "start": 159},
        # one long conversation of a 7B decoder
        {"name": "attend_long", "op": "attend", "heads": 28, "kv": 4, "d": 128, "seqs": 1, "rows": 1, "start": 32001},
        # a batch of 24 sequences of up to 8000 positions, pages in no order
        {"name": "attend_batch", "op": "attend", "heads": 28, "kv": 4, "d": 128, "seqs": 24, "rows": 1, "start": 8000},
        # a whole prompt, and a chunk of one far into its context
        {"name": "attend_prompt", "op": "attend", "heads": 28, "kv": 4, "d": 128, "seqs": 1, "rows": 2011, "start": 0},
        {"name": "attend_chunk", "op": "attend", "heads": 32, "kv": 8, "d": 128, "seqs": 1, "rows": 250, "start": 6000},
        # one conversation's pick over a vocabulary of 151936 under a grammar
        {"name": "logits_token", "op": "logits", "rows": 1, "vocab": 151936, "history": 600, "biases": 0, "mask": True},
        # a batch of 48 requests, each with penalties, biases and a mask
        {"name": "logits_batch", "op": "logits", "rows": 48, "vocab": 151936, "history": 4000, "biases": 64, "mask": True},
        # penalties alone, over a vocabulary of 102400
        {"name": "logits_penalties", "op": "logits", "rows": 7, "vocab": 102400, "history": 1500, "biases": 0,
         "mask": False},
    ]


def log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "store", "store", "attend", "attend", "attend", "logits", "logits"])
    if op == "logits":
        rows = log_int(rng, 1, 48)
        return {"op": op, "rows": rows, "vocab": log_int(rng, 20000, 151936), "history": log_int(rng, 1, 4000),
                "biases": rng.choice([0, log_int(rng, 1, 64)]), "mask": rng.random() < 0.6}
    d = rng.choice([64, 96, 128, 128, 192, 256])
    kv = rng.choice([1, 2, 4, 5, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 7, 8])
    size = heads * d  # of a row's queries
    if op == "attend":
        kind = rng.choice(["token", "batch", "prompt", "chunk"])
        if kind in ("token", "batch"):
            seqs = 1 if kind == "token" else log_int(rng, 2, 32)
            rows = rng.choice([1, 1, 1, rng.randint(2, 5)])
            start = log_int(rng, 1, 32000)
            # at most the largest listed batch: 24 * 8000 positions of 4 * 128, and its products
            start = max(1, min(start, 24 * 8000 * 4 * 128 // (seqs * kv * d), 24 * 8000 * 28 * 128 // (seqs * rows * size)))
            return {"op": op, "heads": heads, "kv": kv, "d": d, "seqs": seqs, "rows": rows, "start": start}
        start = 0 if kind == "prompt" else log_int(rng, 1, 6000)
        rows = min(log_int(rng, 16, 2000), 32 + 2011 * 28 * 128 // size)
        while rows > 16 and size * rows * (start + rows / 2) > 28 * 128 * 2011 * 2011 / 2:
            rows //= 2
        return {"op": op, "heads": heads, "kv": kv, "d": d, "seqs": 1, "rows": rows, "start": start}
    rd = d if rng.random() < 0.7 else d // 2
    case = {"op": op, "heads": heads, "kv": kv, "d": d, "rd": rd, "pairs": rng.choice([0, 0, 1])}
    most = 1877 * 32 * 128 // ((heads + kv) * d)
    if op == "rope":
        return {**case, "rows": min(log_int(rng, 1, 1877), most), "start": log_int(rng, 1, 30000)}
    norms = rng.random() < 0.8
    if rng.random() < 0.5:  # a decode step, or a few drafted tokens
        return {**case, "seqs": log_int(rng, 1, 32), "rows": rng.choice([1, 1, rng.randint(2, 8)]),
                "start": log_int(rng, 1, 4000), "norms": norms}
    # a prompt's chunk, which begins with a block: one that begins inside a block replaces the ring's rows that it
    # reads, and the same pass could not be run again
    seqs = rng.choice([1, 1, 2, 3])
    return {**case, "seqs": seqs, "rows": max(1, min(log_int(rng, 33, 2011), most // seqs)),
            "start": BLOCK * rng.choice([0, rng.randint(1, 40)]), "norms": norms}


# ---- inputs ------------------------------------------------------------------------------------

def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def normal(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def starts_of(c):
    """The position of every sequence's first row: the longest first, the others down to an eighth of it."""
    n = c["seqs"]
    if n == 1:
        return [c["start"]]
    if c["op"] == "store" and c["rows"] > BLOCK:
        return [c["start"] // BLOCK * (n - i) // n * BLOCK for i in range(n)]
    return [max(1, c["start"] - (c["start"] * 7 * i) // (8 * (n - 1))) for i in range(n)]


def rotation_table(n, rd):
    """[n, rd] f32: the cosines, then the sines, of pos / theta^(2i / rd)."""
    i = torch.arange(rd // 2, dtype=torch.float64, device=DEV)
    angle = torch.arange(n, dtype=torch.float64, device=DEV)[:, None] * THETA ** (-2 * i / rd)
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def norm_weights(g, d):
    """bf16 weights as a trained norm's: around one, and above it."""
    return (1.2 + 0.3 * normal(g, d)).to(torch.bfloat16).view(torch.int16)


def key_codes(natural):
    """[pages, heads, 32, d] int8 to a record's key codes [pages, heads, 32 d]: for each 32 dims, groups of 8 dims,
    positions m and m + 16 beside each other."""
    p, h, _, d = natural.shape
    return natural.view(p, h, 2, 16, d // 32, 4, 8).permute(0, 1, 4, 5, 3, 2, 6).reshape(p, h, 32 * d)


def value_codes(natural):
    """The same for the value codes: for each 32 dims, groups of positions 4g .. 4g + 3 and 16 + 4g .. 16 + 4g + 3,
    dims m and m + 16 beside each other."""
    p, h, _, d = natural.shape
    return natural.view(p, h, 2, 4, 4, d // 32, 2, 16).permute(0, 1, 5, 3, 7, 6, 2, 4).reshape(p, h, 32 * d)


def key_values(codes, d):
    """key_codes' inverse."""
    p, h, _ = codes.shape
    return codes.view(p, h, d // 32, 4, 16, 2, 8).permute(0, 1, 5, 4, 2, 3, 6).reshape(p, h, 32, d)


def value_values(codes, d):
    """value_codes' inverse."""
    p, h, _ = codes.shape
    return codes.view(p, h, d // 32, 4, 16, 2, 2, 4).permute(0, 1, 5, 3, 6, 2, 4, 7).reshape(p, h, 32, d)


def prepare_logits(c, g):
    r, v, h, b = c["rows"], c["vocab"], c["history"], c["biases"]
    st = {"logits": 2.5 * normal(g, r, v), "out": torch.zeros(r, v, device=DEV),
          "pick": torch.zeros(r, dtype=torch.int32, device=DEV)}
    # text repeats itself: tokens from a part of the vocabulary that grows slowly with its length
    words = torch.randint(0, v, (r, 1 + h // 3), dtype=torch.int32, device=DEV, generator=g)
    st["history"] = words.gather(1, torch.randint(0, words.shape[1], (r, h), device=DEV, generator=g)).contiguous()
    st["lens"] = torch.clamp((h * (0.3 + 0.7 * torch.rand(r, device=DEV, generator=g))).int(), min=1)
    # the likely next tokens are often ones that were there
    st["logits"].scatter_add_(1, st["history"].long(), 0.5 * normal(g, r, h).abs())
    st["repetition"] = 1.0 + 0.3 * torch.rand(r, device=DEV, generator=g)
    st["frequency"] = 0.2 * torch.rand(r, device=DEV, generator=g)
    st["presence"] = 0.4 * torch.rand(r, device=DEV, generator=g)
    if b:
        st["bias_ids"] = torch.randint(0, v, (r, b), dtype=torch.int32, device=DEV, generator=g)
        st["bias_values"] = 3.0 * normal(g, r, b)
        st["bias_ids"][:, b - b // 4:] = -1  # requests with fewer biases than the longest list
    if c["mask"]:
        # a grammar allows about one token in four
        w = (v + 31) // 32
        bits = [torch.randint(-2 ** 31, 2 ** 31, (r, w), dtype=torch.int64, device=DEV, generator=g) for _ in range(2)]
        st["mask"] = (bits[0] & bits[1]).to(torch.int32)
    return st


def prepare(case, seed):
    c, g = case, generator(seed)
    st = {"case": c}
    if c["op"] == "logits":
        st.update(prepare_logits(c, g))
        return st
    h, kv, d, rows, n = c["heads"], c["kv"], c["d"], c["rows"], c.get("seqs", 1)
    if c["op"] != "attend":
        # queries, keys and values as one linear's output, whose norms differ from head to head
        width = (h + 2 * kv) * d
        scale = (0.5 + 1.5 * torch.rand(h + 2 * kv, device=DEV, generator=g)).repeat_interleave(d)
        st.update(qkv=normal(g, n, rows, width) * scale, q=torch.zeros(n, rows, h, d, device=DEV))
        if c.get("norms", True):
            st.update(q_norm=norm_weights(g, d), k_norm=norm_weights(g, d))
    if c["op"] == "rope":
        m = c["start"] + rows
        st.update(table=rotation_table(m, c["rd"]), start=ints([c["start"]]),
                  kc=torch.zeros(m, kv * d, device=DEV), vc=torch.zeros(m, kv * d, device=DEV))
        return st
    starts = starts_of(c)
    per = (max(starts) + rows + BLOCK - 1) // BLOCK  # blocks of a sequence
    # pages in no order, a few more than the tables name
    pages = n * per + 3
    table = torch.randperm(pages, device=DEV, generator=g)[:n * per].view(n, per).int().contiguous()
    st.update(start=ints(starts), table=table, per=per, n_pages=pages,
              ring=normal(g, n, kv, 2, RING, d) * torch.tensor([1.3, 0.8], device=DEV).view(2, 1, 1),
              pages=torch.zeros(pages, kv, 64 * d + 16, dtype=torch.uint8, device=DEV))
    if c["op"] == "store":
        m = max(starts) + rows
        span = rows + BLOCK - 1  # from the start of the block that a chunk begins in
        st.update(rotation=rotation_table(m, c["rd"]), first=st["start"] // BLOCK * BLOCK, lens=st["start"] + rows,
                  k=torch.zeros(n, span, kv, d, device=DEV), v=torch.zeros(n, span, kv, d, device=DEV))
        return st
    # keys and values of normed heads, some dims of the keys larger than the others, as blocks of codes
    for i in range(0, pages, 512):
        p = min(512, pages - i)
        outliers = 1 + 4 * (torch.rand(kv, 1, d, device=DEV, generator=g) < 0.03)
        for j, (x, order) in enumerate(((1.3 * outliers * normal(g, p, kv, BLOCK, d), key_codes),
                                        (0.8 * normal(g, p, kv, BLOCK, d), value_codes))):
            s = x.abs().amax((2, 3)) / 127
            codes = torch.round(x / s[:, :, None, None]).clamp(-127, 127).to(torch.int8)
            st["pages"][i:i + p, :, 32 * d * j:32 * d * (j + 1)] = order(codes).view(torch.uint8)
            st["pages"][i:i + p, :, 64 * d + 4 * j:64 * d + 4 * j + 4] = s.view(torch.uint8).view(p, kv, 4)
    st.update(q=1.3 * normal(g, n, rows, h, d), attn=torch.zeros(n, rows, h, d, device=DEV))
    return st


# ---- one pass ----------------------------------------------------------------------------------

def workspace(st, size):
    if "ws" not in st:  # as a program's, from its first call on
        st["ws"] = torch.empty(max(16, size()), dtype=torch.uint8, device=DEV)
    return st["ws"]


def how(st, table, rd, pairs):
    from blog_amd import qlin
    if "how" not in st:
        st["how"] = qlin.QkRope(st.get("q_norm"), st.get("k_norm"), 0, EPS, 0, table, rd, pairs)
    return st["how"]


def cache_of(st):
    from blog_amd import qlin
    if "cache" not in st:
        st["cache"] = qlin.Kv8Cache(st["pages"], st["ring"], st["table"])
    return st["cache"]


def run_own(st):
    from blog_amd import qlin
    c = st["case"]
    qlin.set_stream(torch.cuda.current_stream())
    if c["op"] == "logits":
        ws = workspace(st, lambda: qlin.logits_controls_scratch_bytes(c["rows"], c["vocab"]))
        qlin.logits_controls(st["logits"], st["out"], c["rows"], c["vocab"], history=st["history"],
                             history_lens=st["lens"], repetition=st["repetition"], frequency=st["frequency"],
                             presence=st["presence"], bias_ids=st.get("bias_ids"), bias_values=st.get("bias_values"),
                             mask=st.get("mask"), picks=st["pick"], scratch=ws)
        return {"logits": st["out"], "pick": st["pick"]}
    h, kv, d, rows = c["heads"], c["kv"], c["d"], c["rows"]
    if c["op"] == "attend":
        ws = workspace(st, lambda: qlin.attend_kv8_workspace_bytes(c["seqs"], rows, h, kv, d, st["per"]))
        qlin.attend_kv8(cache_of(st), st["q"], st["attn"], rows, h, st["start"], None, d ** -0.5, ws)
        return st["attn"]
    width = (h + 2 * kv) * d
    q = st["qkv"].data_ptr()
    k, v = q + 4 * h * d, q + 4 * (h + kv) * d
    if c["op"] == "rope":
        qlin.qk_norm_rope_store_kv(how(st, st["table"], c["rd"], c["pairs"]), q, width, k, width, v, width, st["q"], st["kc"],
                                   st["vc"], rows, h, kv, d, c["start"] + rows, st["start"])
        return {"q": st["q"], "k": st["kc"], "v": st["vc"]}
    qlin.qk_norm_rope_store_kv8(how(st, st["rotation"], c["rd"], c["pairs"]), cache_of(st), q, width, k, width, v, width,
                                st["q"], rows, h, st["start"], None)
    qlin.kv8_read(cache_of(st), st["first"], st["lens"], rows + BLOCK - 1, st["k"], st["v"])
    return {"q": st["q"], "k": st["k"], "v": st["v"]}


def weights(w, like):
    return (w.view(torch.int16).int() << 16).view(torch.float32).to(like)


def normed_and_rotated(x, w, cs, rd, pairs):
    """x [.., rows, heads, d]; cs [.., rows, rd], the cosines and then the sines."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weights(w, x)
    cos, sin = cs[..., None, :rd // 2], cs[..., None, rd // 2:]
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if pairs else (x[..., :rd // 2], x[..., rd // 2:rd])
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if pairs else torch.cat([u, v], -1)
    return torch.cat([turned, x[..., rd:]], -1)


def plain_rope(st):
    c = st["case"]
    h, kv, d, rows = c["heads"], c["kv"], c["d"], c["rows"]
    q, k, v = st["qkv"][0].split([h * d, kv * d, kv * d], 1)
    at = slice(c["start"], c["start"] + rows)
    cs = st["table"][at]
    st["q"][0] = normed_and_rotated(q.reshape(rows, h, d), st["q_norm"], cs, c["rd"], c["pairs"])
    st["kc"][at] = normed_and_rotated(k.reshape(rows, kv, d), st["k_norm"], cs, c["rd"], c["pairs"]).flatten(1)
    st["vc"][at] = v
    return {"q": st["q"], "k": st["kc"], "v": st["vc"]}


def quantized(x):
    """x [.., 32, heads, d] in codes of 8 bits, as the values that these stand for."""
    s = x.abs().amax((-3, -1), keepdim=True) / 127
    codes = torch.where(s > 0, torch.round(x / s).clamp(-127, 127), 0)
    return torch.where(s.isfinite(), codes * s, math.nan)


def plain_store(st):
    c = st["case"]
    h, kv, d, rows, n = c["heads"], c["kv"], c["d"], c["rows"], c["seqs"]
    q, k, v = st["qkv"].split([h * d, kv * d, kv * d], 2)
    pos = st["start"].long()[:, None] + torch.arange(rows, device=DEV)
    cs = st["rotation"][pos]
    st["q"].copy_(normed_and_rotated(q.reshape(n, rows, h, d), st.get("q_norm"), cs, c["rd"], c["pairs"]))
    # (64 bits: a key next to a border between two codes has to come out as the same f32 value everywhere)
    k = normed_and_rotated(k.reshape(n, rows, kv, d).double(), st.get("k_norm"), cs.double(), c["rd"], c["pairs"]).float()
    blocks = (rows + 2 * BLOCK - 2) // BLOCK
    span = blocks * BLOCK
    at = st["first"].long()[:, None] + torch.arange(span, device=DEV)  # the positions from the first block on
    held = at < st["start"][:, None]
    seq = torch.arange(n, device=DEV)[:, None]
    new = (at - st["start"][:, None]).clamp(0, rows - 1)
    done = at // BLOCK * BLOCK + BLOCK <= st["lens"][:, None]
    for out, x, j in ((st["k"], k, 0), (st["v"], v.reshape(n, rows, kv, d), 1)):
        old = st["ring"][:, :, j].transpose(1, 2)[seq, at % RING]
        x = torch.where(held[..., None, None], old, x[seq, new])
        x = torch.where(done[..., None, None], quantized(x.view(n, blocks, BLOCK, kv, d)).view(n, span, kv, d), x)
        x = torch.where((at < st["lens"][:, None])[..., None, None], x, 0.0)
        out.copy_(x[:, :rows + BLOCK - 1])
    return {"q": st["q"], "k": st["k"], "v": st["v"]}


def plain_attend(st):
    c = st["case"]
    h, kv, d, rows, n, per = c["heads"], c["kv"], c["d"], c["rows"], c["seqs"], st["per"]
    records = st["pages"][st["table"].long().flatten()]
    scales = records[:, :, 64 * d:64 * d + 8].contiguous().view(torch.float32)
    pos = torch.arange(per * BLOCK, device=DEV)
    length = (st["start"] + rows).long()[:, None]
    recent = (pos >= length // BLOCK * BLOCK)[:, None, :, None]

    def of_cache(j, natural):
        codes = records[:, :, 32 * d * j:32 * d * (j + 1)].contiguous().view(torch.int8)
        x = natural(codes, d).float() * scales[:, :, j, None, None]
        x = x.view(n, per, kv, BLOCK, d).transpose(1, 2).reshape(n, kv, per * BLOCK, d)
        return torch.where(recent, st["ring"][:, :, j, pos % RING], x)

    q = st["q"].view(n, rows, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(n, kv, h // kv * rows, d)
    s = (q * d ** -0.5) @ of_cache(0, key_values).transpose(2, 3).contiguous()
    own_pos = st["start"].long()[:, None] + torch.arange(rows, device=DEV)
    unseen = (pos[None, None] > own_pos[:, :, None])[:, None, None]
    s = s.view(n, kv, h // kv, rows, per * BLOCK).masked_fill_(unseen, NEG).view(n, kv, h // kv * rows, per * BLOCK)
    e = s.sub_(s.amax(-1, keepdim=True)).exp_()
    o = (e @ of_cache(1, value_values)) / e.sum(-1, keepdim=True)
    return o.view(n, kv, h // kv, rows, d).permute(0, 3, 1, 2, 4).reshape(n, rows, h, d)


def plain_logits(st):
    c = st["case"]
    r, v, h = c["rows"], c["vocab"], c["history"]
    there = torch.arange(h, device=DEV) < st["lens"][:, None]
    count = torch.zeros(r, v, device=DEV).scatter_add_(1, st["history"].long(), there.float())
    x, rep = st["logits"], st["repetition"][:, None]
    seen = count > 0
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - st["frequency"][:, None] * count - st["presence"][:, None] * seen
    if c["biases"]:
        ids = st["bias_ids"].long()
        x = x.scatter_add(1, ids.clamp(min=0), torch.where(ids >= 0, st["bias_values"], 0.0))
    if c["mask"]:
        bits = torch.arange(32, dtype=torch.int32, device=DEV)
        x = torch.where(((st["mask"][:, :, None] >> bits) & 1).view(r, -1)[:, :v].bool(), x, NEG)
    at = torch.arange(v, dtype=torch.int32, device=DEV)
    return {"logits": x, "pick": torch.where(x == x.amax(1, keepdim=True), at, v).amin(1).int()}


def run(st):
    if own:
        return run_own(st)
    return {"rope": plain_rope, "store": plain_store, "attend": plain_attend, "logits": plain_logits}[st["case"]["op"]](st)


def work(case):
    c = case
    if c["op"] == "logits":
        each = 8 + (1 / 8 if c["mask"] else 0)
        return {"bytes": c["rows"] * (c["vocab"] * each + 4 * c["history"] + 8 * c["biases"] + 20), "flops": c["rows"] * c["vocab"]}
    h, kv, d, rows = c["heads"], c["kv"], c["d"], c["rows"]
    if c["op"] == "rope":
        return {"bytes": 4 * rows * (2 * (h + 2 * kv) * d + c["rd"]), "flops": 10 * rows * (h + kv) * d}
    starts = starts_of(c)
    if c["op"] == "store":
        n = c["seqs"]
        # q, k and v in, q out, the table's rows; then what is stored (the blocks in codes and the ring) and read back
        size = 4 * n * rows * ((h + 2 * kv) * d + h * d + c["rd"])
        for s in starts:
            done = ((s + rows) // BLOCK - s // BLOCK) * BLOCK
            read = s + rows - s // BLOCK * BLOCK
            held = s % BLOCK if done else 0
            size += kv * d * (2 * (2 * done + 4 * min(rows, RING) + 4 * held) + 2 * 4 * read + 2 * (done + 4 * (read - done)))
        return {"bytes": size, "flops": 10 * n * rows * (h + 3 * kv) * d}
    size = flops = 0
    for s in starts:
        done = (s + rows) // BLOCK
        size += kv * (done * (64 * d + 8) + 8 * d * ((s + rows) % BLOCK))
        flops += 4 * d * h * (rows * s + rows * (rows + 1) // 2)
    return {"bytes": size + 8 * c["seqs"] * rows * h * d, "flops": flops}


# ---- in 64 bits --------------------------------------------------------------------------------

def turn_exactly(x, w, pos, rd, pairs):
    """x [rows, heads, d] f64 of one sequence at positions pos; the table's entries are inputs, in 32 bits."""
    if w is not None:
        gain = w.view(torch.bfloat16).double()
        x = gain * x / torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
    x = x.clone()
    for i in range(rd // 2):
        angle = pos.double() * math.pow(THETA, -2.0 * i / rd)
        cos, sin = angle.cos().float().double()[:, None], angle.sin().float().double()[:, None]
        a, b = (2 * i, 2 * i + 1) if pairs else (i, i + rd // 2)
        xa, xb = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = xa * cos - xb * sin, xa * sin + xb * cos
    return x


def exact_store(c, st):
    h, kv, d, rows, n = c["heads"], c["kv"], c["d"], c["rows"], c["seqs"]
    q_out = torch.zeros(n, rows, h, d, dtype=torch.float64, device=DEV)
    kept = [torch.zeros(n, rows + BLOCK - 1, kv, d, dtype=torch.float64, device=DEV) for _ in range(2)]
    for s, begin in enumerate(starts_of(c)):
        pos = torch.arange(begin, begin + rows, device=DEV)
        x = st["qkv"][s].double().view(rows, h + 2 * kv, d)
        q_out[s] = turn_exactly(x[:, :h], st.get("q_norm"), pos, c["rd"], c["pairs"])
        fresh = (turn_exactly(x[:, h:h + kv], st.get("k_norm"), pos, c["rd"], c["pairs"]), x[:, h + kv:])
        base = begin - begin % BLOCK
        for j, (out, y) in enumerate(zip(kept, fresh)):
            y = y.float()  # (the cache's own type)
            if begin > base:
                slots = [p % RING for p in range(base, begin)]
                y = torch.cat([st["ring"][s, :, j, slots].transpose(0, 1), y])
            whole = y.shape[0] // BLOCK * BLOCK
            values = y.double()
            for b in range(0, whole, BLOCK):
                top = y[b:b + BLOCK].abs().amax((0, 2))
                step = (top / 127)[None, :, None]  # (and the scale's)
                values[b:b + BLOCK] = torch.round(y[b:b + BLOCK] / step).double() * step.double()
            out[s, :y.shape[0]] = values
    return {"q": q_out, "k": kept[0], "v": kept[1]}


def exact_attend(c, st):
    h, kv, d, rows, n = c["heads"], c["kv"], c["d"], c["rows"], c["seqs"]
    out = torch.zeros(n, rows, h, d, dtype=torch.float64, device=DEV)
    for s, begin in enumerate(starts_of(c)):
        length = begin + rows
        done = length // BLOCK
        rec = st["pages"][st["table"][s, :done].long()]
        slots = [p % RING for p in range(done * BLOCK, length)]
        for k in range(kv):
            step = rec[:, k, 64 * d:64 * d + 8].contiguous().view(torch.float32).double()
            held = []
            for j, natural in ((0, key_values), (1, value_values)):
                codes = natural(rec[:, k:k + 1, 32 * d * j:32 * d * (j + 1)].contiguous().view(torch.int8), d)[:, 0]
                held.append(torch.cat([(codes.double() * step[:, j, None, None]).reshape(-1, d), st["ring"][s, k, j, slots].double()]))
            for m in range(k * (h // kv), (k + 1) * (h // kv)):
                score = st["q"][s, :, m].double() @ held[0].T / math.sqrt(d)
                later = torch.arange(length, device=DEV)[None] > begin + torch.arange(rows, device=DEV)[:, None]
                out[s, :, m] = torch.softmax(score.masked_fill(later, NEG), -1) @ held[1]
    return out


def exact_logits(c, st):
    r, v = c["rows"], c["vocab"]
    out = st["logits"].double()
    for i in range(r):
        count = torch.bincount(st["history"][i, :int(st["lens"][i])].long(), minlength=v).double()
        rep, freq, pres = (float(st[k][i]) for k in ("repetition", "frequency", "presence"))
        was = out[i].clone()
        out[i] = torch.where(count > 0, torch.where(was > 0, was / rep, was * rep) - pres, was) - freq * count
        if c["biases"]:
            for t, b in zip(st["bias_ids"][i].tolist(), st["bias_values"][i].tolist()):
                if t >= 0:
                    out[i, t] += b
        if c["mask"]:
            words = st["mask"][i].long() & 0xffffffff
            token = torch.arange(v, device=DEV)
            out[i, ((words[token // 32] >> (token % 32)) & 1) == 0] = NEG
    return {"logits": out, "pick": None}


def exact(case, seed):
    c, st = case, prepare(case, seed)
    if c["op"] == "rope":
        kv, d, h, rows = c["kv"], c["d"], c["heads"], c["rows"]
        pos = torch.arange(c["start"], c["start"] + rows, device=DEV)
        x = st["qkv"][0].double().view(rows, h + 2 * kv, d)
        kc, vc = st["kc"].double(), st["vc"].double()
        kc[pos] = turn_exactly(x[:, h:h + kv], st["k_norm"], pos, c["rd"], c["pairs"]).flatten(1)
        vc[pos] = x[:, h + kv:].flatten(1)
        return {"q": turn_exactly(x[:, :h], st["q_norm"], pos, c["rd"], c["pairs"])[None], "k": kc, "v": vc}
    return {"store": exact_store, "attend": exact_attend, "logits": exact_logits}[c["op"]](c, st)

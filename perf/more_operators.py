"""Operators that serve several sequences from one paged KV cache: the cases their
speed and results are held to.

A serving program keeps the k and v of many sequences in pages of a shared pool.  In
each step it runs a few new rows of every sequence (one token, a chain of drafted
ones, or a chunk of a prompt): row r of sequence s with m rows sits in slot
length[s] - m + (r - start[s]), slot p being entry p mod page_size of page
table[s, p / page_size].  Four operators carry that:

  append   of the rows' projections q, k, v the norm of each head of q and k and their
           rotation by the position, q rounded to f16, k and v written into the pages:
             y = x / sqrt(mean x^2 + eps) w;  pairs (y[i], y[i + D/2]) turned by the
             angle position theta^(-2i/D)
           8-bit pages hold round(y / scale) with scale = f32(max |y| / 127) for
           each token and kv head.
  attn     attention of the rows over their sequence's slots up to their own, with
           each row's log-sum-exp:
             s[r,h,j] = scale q[r,h] . k[j,h']      h' = h / (q_heads / kv_heads)
             lse[r,h] = log sum_j exp s,  out[r,h] = sum_j exp(s - lse) v[j,h']
  read     whole sequences out of their pages into a flat f16 cache, all layers.
  verify   drafted tokens against the model: row i of a sequence gives the target's
           probabilities p of the token behind it, softmax(logits / temperature)
           (temperature 0: all on the lowest index of the maximum).  With q the
           drafter's probabilities (without them: all on the drafted token x), x is
           accepted if u q(x) < p(x).  Behind the accepted ones one more token is
           taken from max(p - q, 0) of the row that refused, or from p behind the
           last row: the lowest index whose running sum exceeds u times the sum.

  listed()       the named cases
  draw(rng)      one more case of the same ranges
  prepare        what the program holds before the call
  run            the call, and what it wrote
  work           bytes and operations the call cannot do without
  exact          the same results in 64 bits
"""
from __future__ import annotations

import importlib.util
import math
import random
import sys
from pathlib import Path

import torch

own = False

MODEL = {"q_heads": 16, "kv_heads": 8, "head_dim": 128}
VOCAB = 151936
EPS, THETA = 1e-6, 1e6
# what a case may hold, by its largest listed ones
MOST_SLOTS = 4 * 131072 * 8 * 128    # 8-bit values of k in the padded cache of all layers
MOST_SCORES = 100_000_000            # scores of all layers, padded
MOST_ROWS = 4096 * 16 * 128 * 2      # values of q that are appended
MOST_READ = 28 * 4096 * 8 * 128      # values of k that are read back
MOST_LOGITS = 320 * VOCAB


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # One token of one short chat, one layer: the smallest call.
        {"name": "attn_1x300_f16", "op": "attn", "layers": 1, **MODEL, "seqs": 1, "len": 300,
         "new": 1, "mix": 1, "ragged": False, "page": 16, "bits": 16},
        # One token of each of 48 conversations of all lengths, four layers.
        {"name": "attn_48x4096_q8_4l", "op": "attn", "layers": 4, **MODEL, "seqs": 48, "len": 4096,
         "new": 1, "mix": 2, "ragged": True, "page": 64, "bits": 8},
        # Chains of drafted tokens behind long documents.
        {"name": "attn_16x8000_new5_f16", "op": "attn", "layers": 1, **MODEL, "seqs": 16,
         "len": 8000, "new": 5, "mix": 3, "ragged": True, "page": 32, "bits": 16},
        # A few very long contexts: the largest.
        {"name": "attn_4x131072_q8", "op": "attn", "layers": 1, **MODEL, "seqs": 4, "len": 131072,
         "new": 1, "mix": 4, "ragged": False, "page": 128, "bits": 8},
        # One decoded token into f16 pages.
        {"name": "append_1x300_f16", "op": "append", "layers": 1, **MODEL, "seqs": 1, "len": 300,
         "new": 1, "mix": 5, "ragged": False, "page": 16, "bits": 16, "given": False},
        # A batch's drafted chains into 8-bit pages in every layer, and read back.
        {"name": "append_64x1000_new4_q8_28l", "op": "append", "layers": 28, **MODEL, "seqs": 64,
         "len": 1000, "new": 4, "mix": 6, "ragged": True, "page": 64, "bits": 8, "given": False},
        # Prompts of a few thousand tokens into 8-bit pages, positions of their own.
        {"name": "append_3x2999_q8", "op": "append", "layers": 1, **MODEL, "seqs": 3, "len": 2999,
         "new": 2999, "mix": 7, "ragged": False, "page": 64, "bits": 8, "given": True},
        # A short sequence out of f16 pages, a layer.
        {"name": "read_1x333_f16", "op": "read", "layers": 1, "kv_heads": 8, "head_dim": 128,
         "seqs": 1, "len": 333, "mix": 8, "ragged": False, "page": 16, "bits": 16},
        # A conversation out of 8-bit pages, every layer.
        {"name": "read_1x4096_q8_28l", "op": "read", "layers": 28, "kv_heads": 8, "head_dim": 128,
         "seqs": 1, "len": 4096, "mix": 9, "ragged": False, "page": 64, "bits": 8},
        # A token sampled for one sequence, no draft.
        {"name": "verify_1x1", "op": "verify", "seqs": 1, "new": 1, "vocab": VOCAB, "mix": 10,
         "draft": False},
        # A chain looked up in the text so far: no probabilities of a drafter.
        {"name": "verify_7x6", "op": "verify", "seqs": 7, "new": 6, "vocab": VOCAB, "mix": 11,
         "draft": False},
        # A batch's chains against their drafter's probabilities.
        {"name": "verify_64x5_draft", "op": "verify", "seqs": 64, "new": 5, "vocab": VOCAB,
         "mix": 12, "draft": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    if rng.random() < 0.4:
        return dict(MODEL)
    q, kv, d = rng.choice([(14, 2, 64), (8, 8, 128), (32, 8, 128), (32, 4, 128), (9, 3, 64),
                           (16, 16, 64), (28, 4, 128), (16, 1, 128), (64, 2, 64)])
    return {"q_heads": q, "kv_heads": kv, "head_dim": d}


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "append", "read", "verify"])
    if op == "verify":
        new = rng.randint(1, 9)
        c = {"op": op, "seqs": _log(rng, 1, 256), "new": new, "vocab": _log(rng, 1000, VOCAB),
             "mix": rng.randrange(1 << 20), "draft": rng.random() < 0.5}
        while c["seqs"] * new * c["vocab"] > MOST_LOGITS:
            c["seqs"] = (c["seqs"] + 1) // 2
        return c
    h = _heads(rng)
    c = {"op": op, "layers": rng.choice([1, 2, 4] if op == "attn" else [1, 4, 28]), **h,
         "seqs": _log(rng, 1, 256), "len": _log(rng, 1, 131072 if op == "attn" else 8192),
         "mix": rng.randrange(1 << 20), "ragged": rng.random() < 0.7,
         "page": rng.choice([16, 32, 48, 64, 128, 256]), "bits": rng.choice([8, 16])}
    if op == "read":
        del c["q_heads"]
        while c["layers"] * c["seqs"] * c["len"] * h["kv_heads"] * h["head_dim"] > MOST_READ:
            shrink = rng.choice(["layers", "seqs", "len"])
            c[shrink] = (c[shrink] + 1) // 2
        return c
    x = rng.random()
    c["new"] = 1 if x < 0.5 else rng.randint(2, 8) if x < 0.85 else _log(rng, 9, 256)
    if op == "append":
        c["given"] = rng.random() < 0.3
        if rng.random() < 0.3:
            c["new"] = c["len"]
    c["new"] = min(c["new"], c["len"])
    width = h["q_heads"] * h["head_dim"]
    while (c["layers"] * c["seqs"] * (c["len"] + c["page"]) * h["kv_heads"] * h["head_dim"]
           > MOST_SLOTS * 8 // c["bits"]
           or (op == "attn" and c["layers"] * c["seqs"] * c["new"] * h["q_heads"] * c["len"] > MOST_SCORES)
           or (op == "append" and c["layers"] * c["seqs"] * c["new"] * width > MOST_ROWS)):
        shrink = rng.choice(["layers", "seqs", "len"])
        c[shrink] = (c[shrink] + 1) // 2
        c["new"] = min(c["new"], c["len"])
    return c


def _shape(case):
    """Lengths and new rows of a case's sequences: the same for every seed."""
    rng = random.Random(case["mix"])
    n, seqs = case.get("new", 0), case["seqs"]
    if case["op"] == "verify":
        # a sequence in twenty has nothing to run in this step
        counts = [n if n == 1 else 0 if rng.random() < 0.05 else rng.randint(1, n)
                  for _ in range(seqs)]
        return None, counts if any(counts) else [1] * seqs
    top = case["len"]
    lengths = [_log(rng, max(1, top // 16), top) if case["ragged"] else top for _ in range(seqs)]
    lengths[rng.randrange(seqs)] = top
    if case["op"] == "read" or n == top:
        return lengths, list(lengths)
    counts = [1 if n == 1 else 0 if case["ragged"] and rng.random() < 0.05
              else min(l, rng.randint(1, n)) for l in lengths]
    return lengths, counts if any(counts) else [1] * seqs


# ----------------------------------------------------------------- inputs ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 31)
    return g


def _normal(g, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g)


def _pool(s, g, name, pages):
    """Pages of normal values, f16 or 8-bit codes with the scale of each row."""
    c = s["case"]
    shape = (c["layers"], pages, c["kv_heads"], c["page"], c["head_dim"])
    if c["bits"] == 16:
        s[name] = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(0.0, 1.0, generator=g)
        return
    s[name] = torch.empty(shape, dtype=torch.int8, device="cuda")
    s[name + "_scale"] = torch.empty(shape[:-1], device="cuda")
    for l in range(c["layers"]):
        x = _normal(g, shape[1:])
        scale = x.abs().amax(-1) / 127.0
        s[name + "_scale"][l] = scale
        s[name][l] = torch.round(x / scale[..., None]).to(torch.int8)


def _start(counts):
    at = [0]
    for m in counts:
        at.append(at[-1] + m)
    return torch.tensor(at, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    op = case["op"]
    g = _gen(seed)
    s = {"case": case, "keep": {}}
    lengths, counts = _shape(case)
    rows, seqs = sum(counts), case["seqs"]
    s["rows"], s["most"] = rows, max(1, max(counts))
    # one row a sequence: no list of first rows
    s["start"] = None if all(m == 1 for m in counts) else _start(counts)
    seq = [i for i, m in enumerate(counts) for _ in range(m)]
    s["seq"] = torch.tensor(seq, dtype=torch.int64, device="cuda")
    s["nth"] = torch.tensor([i for m in counts for i in range(m)], dtype=torch.int64, device="cuda")
    s["counts"] = torch.tensor(counts, dtype=torch.int64, device="cuda")
    if op == "verify":
        return _prepare_verify(s, g, rows)
    layers, kvh, d, page = case["layers"], case["kv_heads"], case["head_dim"], case["page"]
    s["length"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    wide = max((l + page - 1) // page for l in lengths)
    spare = 3
    used = [(l + page - 1) // page for l in lengths]
    pages = sum(used) + spare
    # the pages of a pool in use lie anywhere; entries behind a sequence's last are not set
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((seqs, wide), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    s["table"] = table
    _pool(s, g, "k", pages)
    _pool(s, g, "v", pages)
    if op == "read":
        s["max_seq"] = rows + 5
        s["k_to"] = torch.zeros((layers, s["max_seq"], kvh, d), dtype=torch.float16, device="cuda")
        s["v_to"] = torch.zeros_like(s["k_to"])
        return s
    qh = case["q_heads"]
    s["q_out"] = torch.empty((layers, rows, qh * d), dtype=torch.float16, device="cuda")
    if op == "attn":
        s["q"] = _normal(g, (layers, rows, qh * d), 1.2).half()
        s["scale"] = 1.0 / math.sqrt(d)
        s["lse"] = torch.empty((layers, rows, qh), device="cuda")
        return s
    # the rows of a fused q/k/v product, with the few large channels that k has
    x = _normal(g, (layers, rows, (qh + 2 * kvh) * d))
    loud = torch.where(torch.rand((1, 1, (qh + 2 * kvh) * d), generator=g, device="cuda") < 0.03, 6.0, 1.0)
    s["qkv"] = (x * loud).half()
    s["q_norm"] = (1.0 + 0.2 * _normal(g, (layers, d))).half()
    s["k_norm"] = (1.0 + 0.2 * _normal(g, (layers, d))).half()
    s["positions"] = None
    if case["given"]:
        # a cache whose early slots have been dropped: positions ahead of slots
        s["positions"] = (s["length"].long()[s["seq"]] - s["counts"][s["seq"]] + s["nth"]
                          + 1000 * (s["seq"] + 1)).int()
    s["k_rows"] = torch.empty((layers, rows, kvh * d), dtype=torch.float16, device="cuda")
    s["v_rows"] = torch.empty_like(s["k_rows"])
    return s


def _prepare_verify(s, g, rows):
    c = s["case"]
    vocab, seqs = c["vocab"], c["seqs"]
    # a few tokens a row have a chance, the rest are a long tail
    x = _normal(g, (rows, vocab), 2.0)
    likely = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")
    x.scatter_add_(1, likely, 8.0 + 4.0 * torch.rand((rows, 8), generator=g, device="cuda"))
    s["logits"] = x.half()
    s["tokens"] = likely[:, 0].roll(1).int().contiguous()
    heat = 0.5 + torch.rand((seqs,), generator=g, device="cuda")
    s["temperature"] = torch.where(torch.rand((seqs,), generator=g, device="cuda") < 0.1,
                                   torch.zeros_like(heat), heat)
    s["uniform"] = torch.rand((rows,), generator=g, device="cuda")
    # the rows with a drafted token behind them
    s["from"] = torch.nonzero(s["nth"] < s["counts"][s["seq"]] - 1)[:, 0]
    s["draft"] = None
    if c["draft"]:
        s["draft"] = torch.softmax(x + _normal(g, (rows, vocab), 0.7), 1)
        if s["from"].numel():
            picked = torch.multinomial(s["draft"][s["from"]], 1, generator=g)[:, 0]
            s["tokens"][s["from"] + 1] = picked.int()
    elif s["from"].numel():
        # what followed in the text: mostly the likeliest token
        best = s["logits"][s["from"]].argmax(1).int()
        hit = torch.rand((best.numel(),), generator=g, device="cuda") < 0.7
        s["tokens"][s["from"] + 1] = torch.where(hit, best, s["tokens"][s["from"] + 1])
    wide = s["most"]
    s["out"] = torch.empty((seqs, wide), dtype=torch.int32, device="cuda")
    s["accepted"] = torch.empty((seqs,), dtype=torch.int32, device="cuda")
    s["logprob"] = torch.empty((seqs, wide), device="cuda")
    return s


# ------------------------------------------------------------ plain forms ----

def _padded(s, name):
    """[layers * seqs * kv_heads, slots, head_dim] f32: the pages of every sequence."""
    c = s["case"]
    at = s["table"].long().clamp(min=0)
    x = s[name][:, at].float()
    if c["bits"] == 8:
        x = x * s[name + "_scale"][:, at][..., None]
    l, n, wide, h, p, d = x.shape
    return x.transpose(2, 3).reshape(l * n * h, wide * p, d)


def _plain_attn(s):
    c = s["case"]
    layers, seqs, kvh, d, qh = c["layers"], c["seqs"], c["kv_heads"], c["head_dim"], c["q_heads"]
    g, m = qh // kvh, s["most"]
    q = torch.zeros((layers, seqs, m, kvh, g, d), device="cuda")
    q[:, s["seq"], s["nth"]] = s["q"].view(layers, s["rows"], kvh, g, d).float()
    q = q.permute(0, 1, 3, 2, 4, 5).reshape(layers * seqs * kvh, m * g, d)
    scores = torch.bmm(q, _padded(s, "k").transpose(1, 2).contiguous()) * s["scale"]
    slots = scores.shape[2]
    sees = (s["length"].long() - s["counts"])[:, None] + 1 + torch.arange(m, device="cuda")
    ok = torch.arange(slots, device="cuda") < sees[:, :, None]
    scores = scores.view(layers, seqs, kvh, m, g, slots)
    scores.masked_fill_(~ok[None, :, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = scores.sub_(top).exp_()
    total = e.sum(-1, keepdim=True)
    p = e.div_(total).view(layers * seqs * kvh, m * g, slots)
    v = _padded(s, "v")
    # slots behind a sequence's last hold anything
    inside = torch.arange(slots, device="cuda") < s["length"][:, None]
    v.view(layers, seqs, kvh, slots, d).masked_fill_(~inside[None, :, None, :, None], 0.0)
    out = torch.bmm(p, v).view(layers, seqs, kvh, m, g, d)
    out = out.permute(0, 1, 3, 2, 4, 5)[:, s["seq"], s["nth"]].reshape(layers, s["rows"], qh * d)
    lse = (top + torch.log(total))[..., 0].permute(0, 1, 3, 2, 4)[:, s["seq"], s["nth"]]
    return {"out": out.half(), "lse": lse.reshape(layers, s["rows"], qh)}


def _slots(s):
    """The slot of every row, and its page and entry."""
    slot = s["length"].long()[s["seq"]] - s["counts"][s["seq"]] + s["nth"]
    page = s["case"]["page"]
    return slot, s["table"].long()[s["seq"], slot // page], slot % page


def _turned(x, norm, position, d):
    """x f16 [layers, rows, heads, d]: each head's norm and rotation, in f64 (the
    result is rounded to codes: sums in another order must not move it over a border)."""
    x = x.double()
    x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * norm.double()[:, None, None]
    i = torch.arange(d // 2, device="cuda", dtype=torch.float64)
    angle = position.double()[:, None] * torch.pow(torch.tensor(THETA, device="cuda", dtype=torch.float64), -2.0 * i / d)
    cos, sin = torch.cos(angle)[None, :, None], torch.sin(angle)[None, :, None]
    a, b = x[..., :d // 2], x[..., d // 2:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    c = s["case"]
    layers, kvh, d, qh, rows = c["layers"], c["kv_heads"], c["head_dim"], c["q_heads"], s["rows"]
    slot, page, entry = _slots(s)
    position = s["positions"] if c["given"] else slot
    x = s["qkv"].view(layers, rows, qh + 2 * kvh, d)
    q = _turned(x[:, :, :qh], s["q_norm"], position, d)
    k = _turned(x[:, :, qh:qh + kvh], s["k_norm"], position, d)
    v = x[:, :, qh + kvh:].double()
    out = {"q": q.float().half().reshape(layers, rows, qh * d)}
    if c["bits"] == 16:
        s["k"][:, page, :, entry] = k.float().half().transpose(0, 1)
        s["v"][:, page, :, entry] = v.half().transpose(0, 1)
        return {**out, "k": s["k"], "v": s["v"]}
    _write_codes(s, "k", k, page, entry)
    _write_codes(s, "v", v, page, entry)
    return {**out, "k": _read_rows(s, "k", page, entry), "v": _read_rows(s, "v", page, entry)}


def _write_codes(s, name, y, page, entry):
    scale = (y.abs().amax(-1) / 127.0).float()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale)).double()
    code = torch.round(y / safe[..., None]).clamp(-127, 127).to(torch.int8)
    s[name][:, page, :, entry] = code.transpose(0, 1)
    s[name + "_scale"][:, page, :, entry] = scale.transpose(0, 1)


def _read_rows(s, name, page, entry):
    x = s[name][:, page, :, entry].transpose(0, 1)
    if s["case"]["bits"] == 8:
        x = (x.float() * s[name + "_scale"][:, page, :, entry].transpose(0, 1)[..., None]).half()
    return x.reshape(x.shape[0], x.shape[1], -1)


def _plain_read(s):
    _, page, entry = _slots(s)
    rows, shape = s["rows"], s["k_to"].shape
    s["k_to"][:, :rows] = _read_rows(s, "k", page, entry).view(shape[0], rows, *shape[2:])
    s["v_to"][:, :rows] = _read_rows(s, "v", page, entry).view(shape[0], rows, *shape[2:])
    return {"k": s["k_to"], "v": s["v_to"]}


def _plain_verify(s):
    c = s["case"]
    seqs, vocab, rows = c["seqs"], c["vocab"], s["rows"]
    at = torch.arange(vocab, device="cuda")
    x = s["logits"].double()
    top = x.amax(1, keepdim=True)
    heat = s["temperature"][s["seq"]].double()[:, None]
    first = torch.where(x == top, at, vocab).amin(1, keepdim=True)
    warm = torch.exp((x - top) / torch.where(heat > 0, heat, torch.ones_like(heat)))
    e = torch.where(heat > 0, warm, (at == first).double())
    p = e / e.sum(1, keepdim=True)
    # the drafted tokens, row by row of the ones they were taken from
    row = s["from"]
    told = s["tokens"].long()[row + 1]
    q_told = torch.ones((row.numel(),), dtype=torch.float64, device="cuda")
    if s["draft"] is not None:
        q_told = s["draft"][row, told].double()
    yes = torch.zeros((seqs, s["most"]), dtype=torch.int64, device="cuda")
    p_told = torch.gather(p[row], 1, told[:, None])[:, 0]
    fine = s["uniform"][row].double() * q_told < p_told
    yes[s["seq"][row], s["nth"][row]] = fine.long()
    accepted = torch.cumprod(yes, 1).sum(1)
    # the row that the last token of each sequence comes from
    has = torch.nonzero(s["counts"] > 0)[:, 0]
    begin = torch.cumsum(s["counts"], 0) - s["counts"]
    n = accepted[has]
    last = begin[has] + n
    left = p[last]
    refused = n < s["counts"][has] - 1
    if row.numel():
        if s["draft"] is not None:
            taken = s["draft"][last].double()
        else:
            taken = (at == s["tokens"].long()[(last + 1).clamp(max=rows - 1)][:, None]).double()
        rest = torch.clamp(left - taken, min=0.0)
        refused = refused & (rest.sum(1) > 0)
        left = torch.where(refused[:, None], rest, left)
    run_sum = torch.cumsum(left, 1)
    u = s["uniform"][begin[has] + s["counts"][has] - 1].double()
    token = (run_sum <= u[:, None] * run_sum[:, -1:]).sum(1)
    token = torch.minimum(token, torch.where(left > 0, at, -1).amax(1))
    # what goes out: the accepted ones, the last one, -1 behind
    places = torch.arange(s["most"], device="cuda")
    out = torch.full((seqs, s["most"] + 1), -1, dtype=torch.int64, device="cuda")
    out[s["seq"][row], s["nth"][row]] = told
    out = torch.where(places <= accepted[:, None], out[:, :-1], -1)
    out[has, n] = token
    out[s["counts"] == 0] = -1
    real = out >= 0
    from_row = (begin[:, None] + places).clamp(max=max(0, rows - 1))
    chosen = torch.gather(p[from_row.reshape(-1)], 1, out.clamp(min=0).reshape(-1, 1)).view(out.shape)
    logprob = torch.where(real, torch.log(chosen), torch.zeros_like(chosen))
    return {"tokens": out.int(), "accepted": accepted.int(), "logprob": logprob.float()}


# -------------------------------------------------- the framework's calls ----

def _ops():
    name = "qwen3_iree_amd"
    if name not in sys.modules:
        pkg = Path(__file__).resolve().parent.parent / "qwen3-iree_amd"
        spec = importlib.util.spec_from_file_location(
            name, pkg / "__init__.py", submodule_search_locations=[str(pkg)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    import qwen3_iree_amd.pages as pages
    import qwen3_iree_amd.q8gemv as q8gemv
    q8gemv.init()
    return pages


def _kept(s, key, make):
    """What a program makes once and keeps beside its buffers."""
    if key not in s["keep"]:
        s["keep"][key] = make()
    return s["keep"][key]


def _address(t):
    return None if t is None else t.data_ptr()


def _held(s):
    """The module, the pool and the batch."""
    def make():
        P = _ops()
        c = s["case"]
        pool = P.Pages(s["k"].data_ptr(), s["v"].data_ptr(), s["k"].shape[1], c["page"], c["layers"],
                       c["kv_heads"], c["head_dim"], k_scale=_address(s.get("k_scale")),
                       v_scale=_address(s.get("v_scale")))
        batch = P.Batch(s["table"].data_ptr(), s["length"].data_ptr(), c["seqs"],
                        s["table"].shape[1], s["rows"], s["most"], start=_address(s["start"]))
        return P, pool, batch
    return _kept(s, "held", make)


def _workspace(nbytes):
    return torch.zeros((max(1, nbytes),), dtype=torch.uint8, device="cuda")


def _own_attn(s):
    P, pool, batch = _held(s)
    c = s["case"]
    qh, d, rows = c["q_heads"], c["head_dim"], s["rows"]
    ws = _kept(s, "ws", lambda: _workspace(P.attn_workspace_bytes(pool, batch, qh)))
    stream = torch.cuda.current_stream().cuda_stream
    q, out, lse = s["q"].data_ptr(), s["q_out"].data_ptr(), s["lse"].data_ptr()
    for l in range(c["layers"]):
        P.attn(pool, l, batch, q + 2 * l * rows * qh * d, qh * d, qh, s["scale"],
               out + 2 * l * rows * qh * d, qh * d, lse + 4 * l * rows * qh, ws.data_ptr(),
               ws.numel(), stream)
    return {"out": s["q_out"], "lse": s["lse"]}


def _own_append(s):
    P, pool, batch = _held(s)
    c = s["case"]
    qh, kvh, d, rows = c["q_heads"], c["kv_heads"], c["head_dim"], s["rows"]
    cols = (qh + 2 * kvh) * d
    stream = torch.cuda.current_stream().cuda_stream
    qkv, q_out = s["qkv"].data_ptr(), s["q_out"].data_ptr()
    for l in range(c["layers"]):
        q = qkv + 2 * l * rows * cols
        P.append(pool, l, batch, q + 2 * qh * d, cols, q + 2 * (qh + kvh) * d, cols,
                 k_norm=s["k_norm"].data_ptr() + 2 * l * d, q=q, q_stride=cols, q_heads=qh,
                 q_norm=s["q_norm"].data_ptr() + 2 * l * d, q_out=q_out + 2 * l * rows * qh * d,
                 q_out_stride=qh * d, eps=EPS, theta=THETA, positions=_address(s["positions"]),
                 stream=stream)
    if c["bits"] == 16:
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    P.read(pool, 0, c["layers"], batch, s["k_rows"].data_ptr(), s["v_rows"].data_ptr(), kvh * d,
           rows * kvh * d, stream)
    return {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}


def _own_read(s):
    P, pool, batch = _held(s)
    c = s["case"]
    row = c["kv_heads"] * c["head_dim"]
    P.read(pool, 0, c["layers"], batch, s["k_to"].data_ptr(), s["v_to"].data_ptr(), row,
           s["max_seq"] * row, torch.cuda.current_stream().cuda_stream)
    return {"k": s["k_to"], "v": s["v_to"]}


def _own_verify(s):
    P = _kept(s, "ops", _ops)
    c = s["case"]
    seqs, vocab = c["seqs"], c["vocab"]
    ws = _kept(s, "ws", lambda: _workspace(P.verify_workspace_bytes(s["rows"], seqs, vocab)))
    P.verify(s["logits"].data_ptr(), vocab, vocab, s["rows"], s["tokens"].data_ptr(), seqs,
             s["most"], s["uniform"].data_ptr(), s["out"].data_ptr(), s["most"],
             s["accepted"].data_ptr(), start=_address(s["start"]),
             temperature=s["temperature"].data_ptr(), draft=_address(s["draft"]),
             draft_stride=vocab, logprob=s["logprob"].data_ptr(), workspace=ws.data_ptr(),
             workspace_bytes=ws.numel(), stream=torch.cuda.current_stream().cuda_stream)
    return {"tokens": s["out"], "accepted": s["accepted"], "logprob": s["logprob"]}


PLAIN = {"attn": _plain_attn, "append": _plain_append, "read": _plain_read, "verify": _plain_verify}
OWN = {"attn": _own_attn, "append": _own_append, "read": _own_read, "verify": _own_verify}


def run(state):
    if own:
        return OWN[state["case"]["op"]](state)
    return PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------- work and exact ----

def work(case):
    lengths, counts = _shape(case)
    rows = sum(counts)
    if case["op"] == "verify":
        # every row's logits; of the drafter's probabilities only those that a
        # refused token's row has, which the inputs decide
        return {"bytes": rows * (2 * case["vocab"] + 8) + case["seqs"] * (8 + 8 * max(counts)),
                "flops": rows * case["vocab"]}
    layers, kvh, d = case["layers"], case["kv_heads"], case["head_dim"]
    slot = 2 * kvh * (d + 4 if case["bits"] == 8 else 2 * d)  # k and v of a slot in a layer
    if case["op"] == "read":
        return {"bytes": layers * rows * (slot + 4 * kvh * d), "flops": layers * rows * 2 * kvh * d}
    qh = case["q_heads"]
    if case["op"] == "append":
        back = slot + 4 * kvh * d if case["bits"] == 8 else 0
        return {"bytes": layers * rows * (2 * (qh + 2 * kvh) * d + 2 * qh * d + slot + back),
                "flops": layers * rows * 10 * (qh + kvh) * d}
    pairs = sum(m * (l - m) + m * (m + 1) // 2 for l, m in zip(lengths, counts))
    seen = sum(l for l, m in zip(lengths, counts) if m)
    return {"bytes": layers * (seen * slot + rows * qh * (4 * d + 4)),
            "flops": layers * 4 * qh * d * pairs}


def _exact_pages(s, name, l, i):
    """[slots, kv_heads, head_dim] of sequence i in layer l."""
    n, page = int(s["length"][i]), s["case"]["page"]
    at = s["table"][i, :(n + page - 1) // page].long()
    x = s[name][l].index_select(0, at).double()
    if s["case"]["bits"] == 8:
        x = x * s[name + "_scale"][l].index_select(0, at).double().unsqueeze(-1)
    return x.permute(0, 2, 1, 3).flatten(0, 1)[:n]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    lengths, counts = _shape(case)
    if op == "verify":
        return _exact_verify(s, counts)
    layers, kvh, d = case["layers"], case["kv_heads"], case["head_dim"]
    if op == "read":
        out = {}
        for name in ("k", "v"):
            to = torch.zeros(s["k_to"].shape, dtype=torch.float64, device="cuda")
            for l in range(layers):
                to[l, :s["rows"]] = torch.cat([_exact_pages(s, name, l, i) for i in range(case["seqs"])])
            out[name] = to
        return out
    qh = case["q_heads"]
    g = qh // kvh
    if op == "attn":
        out = torch.zeros((layers, s["rows"], qh, d), dtype=torch.float64, device="cuda")
        lse = torch.full((layers, s["rows"], qh), -math.inf, dtype=torch.float64, device="cuda")
        for l in range(layers):
            r = 0
            for i, (n, m) in enumerate(zip(lengths, counts)):
                if not m:
                    continue
                k = _exact_pages(s, "k", l, i).transpose(0, 1).contiguous()
                v = _exact_pages(s, "v", l, i).transpose(0, 1).contiguous()
                q = s["q"][l, r:r + m].double().view(m, kvh, g, d).permute(1, 2, 0, 3)
                for h in range(kvh):
                    e = (q[h].reshape(g * m, d) @ k[h].t().contiguous()).view(g, m, n) * s["scale"]
                    late = torch.ones((m, n), dtype=torch.bool, device="cuda").triu(n - m + 1)
                    e = e.masked_fill(late, -math.inf)
                    t = torch.logsumexp(e, -1)
                    lse[l, r:r + m, h * g:(h + 1) * g] = t.t()
                    o = torch.exp(e - t[..., None]).view(g * m, n) @ v[h]
                    out[l, r:r + m, h * g:(h + 1) * g] = o.view(g, m, d).transpose(0, 1)
                r += m
        return {"out": out.view(layers, s["rows"], qh * d), "lse": lse}
    return _exact_append(s, lengths, counts)


def _exact_append(s, lengths, counts):
    c = s["case"]
    layers, kvh, d, qh, rows = c["layers"], c["kv_heads"], c["head_dim"], c["q_heads"], s["rows"]
    slot = [n - m + i for n, m in zip(lengths, counts) for i in range(m)]
    seq = [i for i, m in enumerate(counts) for _ in range(m)]
    where = slot if s["positions"] is None else s["positions"].tolist()
    half = d // 2
    turn = torch.tensor(where, dtype=torch.float64, device="cuda")[:, None] * torch.tensor(
        [THETA ** (-2.0 * i / d) for i in range(half)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones_like(turn), turn)[:, None]  # e^(i angle)
    heads = s["qkv"].view(layers, rows, qh + 2 * kvh, d)
    out = {"q": torch.empty((layers, rows, qh * d), dtype=torch.float64, device="cuda")}
    new = {}
    for name, lo, hi in (("q", 0, qh), ("k", qh, qh + kvh)):
        y = torch.empty((layers, rows, hi - lo, d), dtype=torch.float64, device="cuda")
        for l in range(layers):
            x = heads[l, :, lo:hi].double()
            x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / d + EPS) * s[name + "_norm"][l].double()
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
            y[l] = torch.cat([z.real, z.imag], -1)
        new[name] = y
    out["q"] = new["q"].reshape(layers, rows, qh * d)
    new["v"] = heads[:, :, qh + kvh:].double()
    page = [int(p) for p in s["table"].long()[torch.tensor(seq, device="cuda", dtype=torch.long),
                                              torch.tensor([x // c["page"] for x in slot], device="cuda", dtype=torch.long)].tolist()]
    for name in ("k", "v"):
        y = new[name]
        if c["bits"] == 16:
            pool = s[name].double()
            flat = pool.permute(1, 3, 0, 2, 4).contiguous().view(-1, layers, kvh, d)
            flat[torch.tensor([p * c["page"] + x % c["page"] for p, x in zip(page, slot)], device="cuda",
                              dtype=torch.long)] = y.transpose(0, 1)
            out[name] = flat.view(pool.shape[1], c["page"], layers, kvh, d).permute(2, 0, 3, 1, 4).contiguous()
        else:
            # what the codes stand for, by their definition
            scale = (torch.linalg.vector_norm(y, ord=math.inf, dim=-1, keepdim=True) / 127).float().double()
            out[name] = (torch.round(y / scale.clamp(min=1e-300)) * scale).reshape(layers, rows, -1)
    return out


def _exact_verify(s, counts):
    c = s["case"]
    wide, heat = s["most"], s["temperature"].tolist()
    told, u = s["tokens"].tolist(), s["uniform"].tolist()
    tokens = torch.full((c["seqs"], wide), -1, dtype=torch.int32)
    accepted = torch.zeros((c["seqs"],), dtype=torch.int32)
    logprob = torch.zeros((c["seqs"], wide), dtype=torch.float64)
    r = 0
    for i, m in enumerate(counts):
        n, done = 0, m == 0
        while not done:
            x = s["logits"][r + n].double()
            if heat[i] > 0:
                logp = torch.log_softmax(x / s["temperature"][i].double(), 0)
            else:
                logp = torch.full_like(x, -math.inf)
                logp[torch.nonzero(x == x.max())[0, 0]] = 0.0
            p = logp.exp()
            left = p
            if n < m - 1:
                t = told[r + n + 1]
                q = torch.zeros_like(p)
                q[t] = 1.0
                if s["draft"] is not None:
                    q = s["draft"][r + n].double()
                if u[r + n] * float(q[t]) < float(p[t]):
                    tokens[i, n], logprob[i, n] = t, float(logp[t])
                    n += 1
                    continue
                rest = (p - q).clamp(min=0.0)
                left = rest if float(rest.sum()) > 0 else p
            some = torch.nonzero(left)[:, 0]
            sums = torch.cumsum(left[some], 0)
            j = int(torch.searchsorted(sums, sums[-1] * u[r + m - 1], right=True))
            t = int(some[min(j, some.numel() - 1)])
            tokens[i, n], logprob[i, n] = t, float(logp[t])
            done = True
        accepted[i] = n
        r += m
    return {"tokens": tokens, "accepted": accepted, "logprob": logprob}

"""Operators over a KV cache and over the vocabulary for drafted tokens: the cases
their speed and results are held to.

A serving program drafts a tree of tokens, runs all of them through the model at
once, keeps the path the model agrees with, and drops the cache positions that get
the least attention when the cache is full.  Four operators carry that:

  tree     attention of the n nodes of a tree over `len` cached positions and over
           each node's own ancestors (their k and v already in the n slots behind
           the cache), with each row's log-sum-exp:
             s[i,h,j] = scale q[i,h] . k[j,h']      h' = h / (q_heads / kv_heads)
             lse[i,h] = log sum_j exp s,  out[i,h] = sum_j exp(s - lse) v[j,h']
           over j < len and the slots len + a of i's ancestors a (i among them);
           a node that is padding (a parent outside -1 .. i - 1, or such an
           ancestor) has out 0 and lse -inf and is nobody's ancestor.
  weights  what attention the positions got: for the accepted tokens i = 0 .. n - 1
           at slots len + i, weights[l,h',j] += sum over the rows i with j <= len + i
           and the heads h of h' of exp(s[l,i,h,j] - lse[l,i,h]); in the n new slots
           the sum replaces what was there.
  evict    per layer and kv head the first `sinks`, the last `recent` and the most
           attended positions between (equal weights: the lower position first),
           `budget` in all, in order, moved into a smaller cache with their weights.
  vocab    logits[i] = f16(W x[i]) for n token rows over the vocabulary and their
           argmax (lowest index of the largest f16 logit).

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

HIDDEN, VOCAB = 1024, 151936
MODEL = {"q_heads": 16, "kv_heads": 8, "head_dim": 128}


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # One token over a short chat, one layer: the smallest call.
        {"name": "tree_n1_len300", "op": "tree", "layers": 1, **MODEL, "n": 1, "len": 300,
         "slack": 211, "pad": 0, "fused": False},
        # A small tree in every layer of a model, q rows inside a q/k/v product.
        {"name": "tree_n13_len1024_28l", "op": "tree", "layers": 28, **MODEL, "n": 13,
         "len": 1024, "slack": 500, "pad": 1, "fused": True},
        # A wide tree over a long document, ragged.
        {"name": "tree_n61_len8191_4l", "op": "tree", "layers": 4, **MODEL, "n": 61, "len": 8191,
         "slack": 900, "pad": 3, "fused": False},
        # The largest tree over the longest context.
        {"name": "tree_n256_len16384", "op": "tree", "layers": 1, **MODEL, "n": 256,
         "len": 16384, "slack": 0, "pad": 0, "fused": False},
        # What one decoded token adds to the weights of every layer.
        {"name": "weights_n1_len1000_28l", "op": "weights", "layers": 28, **MODEL, "n": 1,
         "nodes": 1, "len": 1000, "slack": 24},
        # The accepted path of a tree over a long context, every layer.
        {"name": "weights_n5_len16384_28l", "op": "weights", "layers": 28, **MODEL, "n": 5,
         "nodes": 24, "len": 16384, "slack": 77},
        # A chunk of a prompt on top of an earlier one, one layer.
        {"name": "weights_n256_len2047", "op": "weights", "layers": 1, **MODEL, "n": 256,
         "nodes": 256, "len": 2047, "slack": 33},
        # One layer's cache, just over its budget.
        {"name": "evict_len601_to_512", "op": "evict", "layers": 1, "kv_heads": 8,
         "head_dim": 128, "len": 601, "budget": 512, "sinks": 4, "recent": 64, "slack": 23,
         "room": 128},
        # A conversation at half its length again, every layer.
        {"name": "evict_len2048_28l", "op": "evict", "layers": 28, "kv_heads": 8, "head_dim": 128,
         "len": 2048, "budget": 1024, "sinks": 4, "recent": 256, "slack": 0, "room": 512},
        # A long document cut to a quarter.
        {"name": "evict_len16384_28l", "op": "evict", "layers": 28, "kv_heads": 8,
         "head_dim": 128, "len": 16384, "budget": 4096, "sinks": 4, "recent": 1024, "slack": 0,
         "room": 1},
        # Next tokens of a small tree, and of the largest.
        {"name": "vocab_n13", "op": "vocab", "rows": VOCAB, "n": 13},
        {"name": "vocab_n256", "op": "vocab", "rows": VOCAB, "n": 256},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    if rng.random() < 0.5:
        return dict(MODEL)
    q, kv, d = rng.choice([(14, 2, 64), (8, 8, 128), (32, 8, 128), (32, 4, 128), (9, 3, 64),
                           (16, 16, 64), (28, 4, 128), (16, 1, 128)])
    return {"q_heads": q, "kv_heads": kv, "head_dim": d}


def draw(rng):
    op = rng.choice(["tree", "tree", "weights", "evict", "vocab"])
    if op == "tree":
        h, n = _heads(rng), _log(rng, 1, 256)
        length = 0 if rng.random() < 0.1 else _log(rng, 1, 16384)
        layers = rng.choice([1, 2, 4, 28])
        while layers > 1 and layers * n * h["q_heads"] * (length + n) > 16 * 256 * 8192:
            layers //= 2
        while n * h["q_heads"] * (length + n) > 16 * 256 * 16640:
            length //= 2
        return {"op": op, "layers": layers, **h, "n": n, "len": length,
                "slack": rng.randint(0, 600), "pad": rng.choice([0, rng.randint(0, n // 3)]),
                "fused": rng.random() < 0.5}
    if op == "weights":
        h, n = _heads(rng), _log(rng, 1, 256)
        length = 0 if rng.random() < 0.1 else _log(rng, 1, 16384)
        layers = rng.choice([1, 4, 28])
        while layers > 1 and layers * n * h["q_heads"] * (length + n) > 16 * 256 * 8192:
            layers //= 2
        while n * h["q_heads"] * (length + n) > 16 * 256 * 16640:
            length //= 2
        return {"op": op, "layers": layers, **h, "n": n, "nodes": n + rng.randint(0, 40),
                "len": length, "slack": rng.randint(0, 600)}
    if op == "evict":
        h = _heads(rng)
        length = _log(rng, 2, 16384)
        budget = max(1, int(length * rng.uniform(0.1, 1.0)))
        sinks = rng.randint(0, min(16, budget))
        recent = int((budget - sinks) * rng.uniform(0.0, 0.9))
        return {"op": op, "layers": rng.choice([1, 4, 28]), "kv_heads": min(8, h["kv_heads"]),
                "head_dim": h["head_dim"], "len": length, "budget": budget, "sinks": sinks,
                "recent": recent, "slack": rng.randint(0, 300), "room": rng.randint(0, 300)}
    return {"op": op, "rows": _log(rng, 1000, VOCAB), "n": _log(rng, 1, 256)}


# ----------------------------------------------------------------- inputs ----

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 7919 + 29)
    return g


def _normal(g, shape, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g).half()


def _cache(g, layers, max_seq, kv_heads, head_dim):
    return torch.empty((layers, max_seq, kv_heads, head_dim), dtype=torch.float16,
                       device="cuda").normal_(0.0, 1.0, generator=g)


def _tree(seed, n, pad):
    """Parents of a tree as a drafter makes them: about half of the nodes
    continue the one before, the rest branch off an earlier one; `pad` entries
    at the end are padding."""
    rng = random.Random(seed * 31 + 7)
    p = [-1] + [i - 1 if rng.random() < 0.5 else rng.randint(-1 if rng.random() < 0.05 else 0, i - 1)
                for i in range(1, n)]
    if pad:
        p[n - pad:] = [-2] * pad
    return p


def prepare(case, seed):
    op = case["op"]
    g = _gen(seed)
    s = {"case": case, "keep": {}}
    if op == "vocab":
        rows, n = case["rows"], case["n"]
        s["w"] = _normal(g, (rows, HIDDEN), 0.02)
        # hidden rows as a trained model's final norm leaves them: one row of
        # the matrix stands out, so that the next token is clear
        target = torch.randint(0, rows, (n,), generator=g, device="cuda")
        lift = torch.empty((n, 1), device="cuda").uniform_(0.4, 1.0, generator=g)
        s["x"] = (_normal(g, (n, HIDDEN)).float() + lift * s["w"][target].float() / 0.02).half()
        s["logits"] = torch.empty((n, rows), dtype=torch.float16, device="cuda")
        s["tokens"] = torch.empty((n,), dtype=torch.int32, device="cuda")
        return s
    layers, kvh, d, length = case["layers"], case["kv_heads"], case["head_dim"], case["len"]
    if op == "evict":
        max_seq, small = length + case["slack"], case["budget"] + case["room"]
        s["k"] = _cache(g, layers, max_seq, kvh, d)
        s["v"] = _cache(g, layers, max_seq, kvh, d)
        # accumulated weights: a few positions take most, some have none at all
        w = torch.empty((layers, kvh, max_seq), device="cuda")
        w = torch.exp(2.0 * w.normal_(0.0, 1.0, generator=g) - 4.0)
        none = torch.empty_like(w).uniform_(0.0, 1.0, generator=g) < 0.05
        s["weights"] = torch.where(none, torch.zeros_like(w), w)
        s["k_to"] = torch.zeros((layers, small, kvh, d), dtype=torch.float16, device="cuda")
        s["v_to"] = torch.zeros_like(s["k_to"])
        s["weights_to"] = torch.zeros((layers, kvh, small), device="cuda")
        s["kept"] = torch.empty((layers, kvh, case["budget"]), dtype=torch.int32, device="cuda")
        return s
    n, qh = case["n"], case["q_heads"]
    max_seq = length + n + case["slack"]
    s["scale"] = 1.0 / math.sqrt(d)
    s["k"] = _cache(g, layers, max_seq, kvh, d)
    s["v"] = _cache(g, layers, max_seq, kvh, d)
    if op == "tree":
        cols = (qh + 2 * kvh) * d if case["fused"] else qh * d
        s["q"] = _normal(g, (layers, n, cols), 1.5)
        s["parents"] = torch.tensor(_tree(seed, n, case["pad"]), dtype=torch.int32, device="cuda")
        s["mask"] = torch.empty((n, (n + 31) // 32), dtype=torch.int32, device="cuda")
        s["depth"] = torch.empty((n,), dtype=torch.int32, device="cuda")
        s["out"] = torch.empty((layers, n, qh * d), dtype=torch.float16, device="cuda")
        s["lse"] = torch.empty((layers, n, qh), device="cuda")
        return s
    nodes = case["nodes"]
    s["q"] = _normal(g, (layers, nodes, qh * d), 1.5)
    rng = random.Random(seed * 31 + 11)
    s["path"] = torch.tensor(sorted(rng.sample(range(nodes), n)), dtype=torch.int32, device="cuda")
    s["lse"] = torch.zeros((layers, nodes, qh), device="cuda")
    at = s["path"].long()
    scores = _path_scores(s, torch.float32)
    s["lse"][:, at] = torch.logsumexp(scores, -1).view(layers, kvh, n, qh // kvh).permute(
        0, 2, 1, 3).reshape(layers, n, qh)
    # about what 50 earlier tokens left
    s["weights"] = torch.empty((layers, kvh, max_seq), device="cuda").uniform_(
        0.0, 100.0 * qh / kvh / (length + 1), generator=g)
    return s


def _path_scores(s, dtype):
    """[layers, kv_heads, n * group, len + n]: the accepted rows' scores, -inf
    behind each row's own slot."""
    c = s["case"]
    layers, kvh, d, n, length = c["layers"], c["kv_heads"], c["head_dim"], c["n"], c["len"]
    g = c["q_heads"] // kvh
    q = s["q"][:, s["path"].long()].view(layers, n, kvh, g, d).permute(0, 2, 1, 3, 4)
    q = q.reshape(layers * kvh, n * g, d).to(dtype)
    k = s["k"][:, :length + n].permute(0, 2, 3, 1).reshape(layers * kvh, d, length + n).to(dtype)
    scores = (torch.bmm(q, k.contiguous()) * s["scale"]).view(layers, kvh, n, g, length + n)
    at = torch.arange(length + n, device="cuda")
    ok = at[None, :] <= length + torch.arange(n, device="cuda")[:, None]
    scores = scores.masked_fill(~ok[None, None, :, None], -math.inf)
    return scores.view(layers, kvh, n * g, length + n)


# ------------------------------------------------------------ plain forms ----

def _ancestors(parents, dtype):
    """[n, n] truth values: j is i or an ancestor of i, and i is no padding."""
    n = parents.numel()
    p = parents.long()
    at = torch.arange(n, device=p.device)
    ok = (p >= -1) & (p < at)
    reach = torch.eye(n, dtype=dtype, device=p.device)
    reach = reach + ((at[None, :] == p[:, None]) & ok[:, None]).to(dtype)
    # a chain of n nodes is closed after 8 squarings (n <= 256)
    for _ in range(8):
        reach = ((reach @ reach) > 0.5).to(dtype)
    lost = (reach @ (~ok).to(dtype)[:, None])[:, 0] > 0.5
    return (reach > 0.5) & ~lost[:, None]


def _mask_words(see):
    n = see.shape[0]
    words = (n + 31) // 32
    bits = torch.zeros((n, words * 32), dtype=torch.int64, device=see.device)
    bits[:, :n] = see.long()
    w = (bits.view(n, words, 32) << torch.arange(32, device=see.device)).sum(-1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).int()


def _tree_attention(s, dtype):
    c = s["case"]
    layers, kvh, d, n, length = c["layers"], c["kv_heads"], c["head_dim"], c["n"], c["len"]
    qh = c["q_heads"]
    g = qh // kvh
    see = _ancestors(s["parents"], torch.float32)
    q = s["q"][:, :, :qh * d].reshape(layers, n, kvh, g, d).permute(0, 2, 1, 3, 4)
    q = q.reshape(layers * kvh, n * g, d).to(dtype)
    k = s["k"][:, :length + n].permute(0, 2, 3, 1).reshape(layers * kvh, d, length + n).to(dtype)
    v = s["v"][:, :length + n].permute(0, 2, 1, 3).reshape(layers * kvh, length + n, d).to(dtype)
    scores = (torch.bmm(q, k.contiguous()) * s["scale"]).view(layers, kvh, n, g, length + n)
    live = see.any(1)
    ok = torch.cat([live[:, None].expand(n, length), see], 1)
    scores = scores.masked_fill(~ok[None, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    e = torch.exp(scores - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.bmm(p.view(layers * kvh, n * g, length + n), v.contiguous())
    out = out.view(layers, kvh, n, g, d).permute(0, 2, 1, 3, 4).reshape(layers, n, qh * d)
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(layers, n, qh)
    return out, lse, see


def _plain_tree(s):
    out, lse, see = _tree_attention(s, torch.float32)
    return {"out": out.half(), "lse": lse, "mask": _mask_words(see),
            "depth": see.sum(1).int() - 1}


def _plain_weights(s):
    c = s["case"]
    layers, kvh, n, length = c["layers"], c["kv_heads"], c["n"], c["len"]
    g = c["q_heads"] // kvh
    lse = s["lse"][:, s["path"].long()].view(layers, n, kvh, g).permute(0, 2, 1, 3)
    p = torch.exp(_path_scores(s, torch.float32) - lse.reshape(layers, kvh, n * g, 1))
    got = p.sum(2)
    s["weights"][:, :, :length] += got[:, :, :length]
    s["weights"][:, :, length:length + n] = got[:, :, length:]
    return {"weights": s["weights"]}


def _plain_evict(s):
    c = s["case"]
    layers, kvh, length, budget = c["layers"], c["kv_heads"], c["len"], c["budget"]
    sinks, recent = c["sinks"], c["recent"]
    w = s["weights"][:, :, sinks:length - recent]
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    middle = torch.sort(order[:, :, :budget - sinks - recent], dim=-1).values + sinks
    at = torch.arange(length, device="cuda").expand(layers, kvh, length)
    kept = torch.cat([at[:, :, :sinks], middle, at[:, :, length - recent:]], -1)
    s["kept"].copy_(kept)
    l = torch.arange(layers, device="cuda")[:, None, None]
    h = torch.arange(kvh, device="cuda")[None, :, None]
    s["k_to"][:, :budget] = s["k"][l, kept, h].transpose(1, 2)
    s["v_to"][:, :budget] = s["v"][l, kept, h].transpose(1, 2)
    s["weights_to"][:, :, :budget] = torch.gather(s["weights"], 2, kept)
    return {"kept": s["kept"], "k": s["k_to"], "v": s["v_to"], "weights": s["weights_to"]}


def _plain_vocab(s):
    logits = (s["x"].float() @ s["w"].float().t()).half()
    rows = logits.shape[1]
    at = torch.arange(rows, device="cuda", dtype=torch.int32)
    top = logits.amax(1, keepdim=True)
    tokens = torch.where(logits == top, at, torch.full_like(at, rows)).amin(1)
    return {"logits": logits, "tokens": tokens}


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
    import qwen3_iree_amd.cache as cache
    import qwen3_iree_amd.q8gemv as q8gemv
    q8gemv.init()
    return cache, q8gemv


def _kept(s, key, make):
    """What a program makes once and keeps beside its buffers."""
    if key not in s["keep"]:
        s["keep"][key] = make()
    return s["keep"][key]


def _cache_of(C, s, k="k", v="v", weights=None):
    c = s["case"]
    return C.Cache(s[k].data_ptr(), s[v].data_ptr(), s[k].shape[1], c["layers"], c["kv_heads"],
                   c["head_dim"], weights=s[weights].data_ptr() if weights else None)


def _own_tree(s):
    C, Q = _kept(s, "ops", _ops)
    c = s["case"]
    n, qh, d, stream = c["n"], c["q_heads"], c["head_dim"], torch.cuda.current_stream().cuda_stream
    cache = _kept(s, "cache", lambda: _cache_of(C, s))
    ws = _kept(s, "ws", lambda: torch.empty(
        max(1, C.attn_tree_workspace_bytes(cache, c["len"], n, qh)), dtype=torch.uint8,
        device="cuda"))
    C.tree_mask(s["parents"].data_ptr(), n, s["mask"].data_ptr(), s["depth"].data_ptr(), stream)
    cols = s["q"].shape[2]
    q, out, lse = s["q"].data_ptr(), s["out"].data_ptr(), s["lse"].data_ptr()
    for l in range(c["layers"]):
        C.attn_tree(cache, l, c["len"], q + 2 * l * n * cols, cols, qh, s["mask"].data_ptr(), n,
                    s["scale"], out + 2 * l * n * qh * d, qh * d, lse + 4 * l * n * qh,
                    ws.data_ptr(), ws.numel(), stream)
    return {"out": s["out"], "lse": s["lse"], "mask": s["mask"], "depth": s["depth"]}


def _own_weights(s):
    C, Q = _kept(s, "ops", _ops)
    c = s["case"]
    nodes, qh, d = c["nodes"], c["q_heads"], c["head_dim"]
    cache = _kept(s, "cache", lambda: _cache_of(C, s, weights="weights"))
    C.attn_weights_add(cache, c["len"], s["q"].data_ptr(), nodes * qh * d, qh * d, qh,
                       s["lse"].data_ptr(), nodes * qh, nodes, s["path"].data_ptr(), c["n"],
                       s["scale"], torch.cuda.current_stream().cuda_stream)
    return {"weights": s["weights"]}


def _own_evict(s):
    C, Q = _kept(s, "ops", _ops)
    c = s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    src = _kept(s, "src", lambda: _cache_of(C, s, weights="weights"))
    dst = _kept(s, "dst", lambda: _cache_of(C, s, "k_to", "v_to", "weights_to"))
    C.cache_select(src, c["len"], c["budget"], c["sinks"], c["recent"], s["kept"].data_ptr(),
                   stream)
    C.cache_compact(src, dst, s["kept"].data_ptr(), True, 0, c["budget"], stream)
    return {"kept": s["kept"], "k": s["k_to"], "v": s["v_to"], "weights": s["weights_to"]}


def _own_vocab(s):
    C, Q = _kept(s, "ops", _ops)
    c = s["case"]
    ws = _kept(s, "ws", lambda: torch.zeros(Q.gemm_argmax_workspace_bytes(c["n"]),
                                            dtype=torch.uint8, device="cuda"))
    Q.f16_gemm_argmax(s["w"].data_ptr(), c["rows"], s["x"].data_ptr(), c["n"],
                      s["logits"].data_ptr(), s["tokens"].data_ptr(), ws.data_ptr(),
                      torch.cuda.current_stream().cuda_stream)
    return {"logits": s["logits"], "tokens": s["tokens"]}


PLAIN = {"tree": _plain_tree, "weights": _plain_weights, "evict": _plain_evict,
         "vocab": _plain_vocab}
OWN = {"tree": _own_tree, "weights": _own_weights, "evict": _own_evict, "vocab": _own_vocab}


def run(state):
    if own:
        return OWN[state["case"]["op"]](state)
    return PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------- work and exact ----

def work(case):
    op = case["op"]
    if op == "vocab":
        rows, n = case["rows"], case["n"]
        return {"bytes": 2 * (rows * HIDDEN + n * HIDDEN + n * rows) + 4 * n,
                "flops": 2 * n * rows * HIDDEN}
    layers, kvh, d, length = case["layers"], case["kv_heads"], case["head_dim"], case["len"]
    if op == "evict":
        b = case["budget"]
        # the weights to choose from, the kept rows read and written, their
        # positions and weights written
        return {"bytes": layers * kvh * (4 * length + 2 * 2 * 2 * b * d + 4 * b + 4 * b),
                "flops": layers * kvh * length}
    n, qh = case["n"], case["q_heads"]
    if op == "tree":
        rows = n * (length + 1)  # at least: the cache and itself
        return {"bytes": layers * (2 * 2 * (length + n) * kvh * d + 2 * 2 * n * qh * d + 4 * n * qh)
                + 4 * n * (2 + (n + 31) // 32),
                "flops": layers * 4 * qh * d * rows}
    rows = n * length + n * (n + 1) // 2
    return {"bytes": layers * (2 * (length + n) * kvh * d + 4 * kvh * (2 * length + n)
                               + 2 * n * qh * d + 4 * n * qh) + 4 * n,
            "flops": layers * 2 * qh * d * rows}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "vocab":
        w, x = s["w"], s["x"].double()
        parts = [x @ w[i:i + 16384].double().t() for i in range(0, case["rows"], 16384)]
        logits = torch.cat(parts, 1)
        return {"logits": logits, "tokens": None}
    layers, kvh, d, length = case["layers"], case["kv_heads"], case["head_dim"], case["len"]
    if op == "evict":
        w, b = s["weights"].double(), case["budget"]
        first, last = case["sinks"], length - case["recent"]
        at = torch.arange(length, device="cuda")
        # always kept before anything else, then by weight, then by position
        rank = torch.where((at < first) | (at >= last), torch.full_like(w[:, :, :length], math.inf),
                           w[:, :, :length])
        by = torch.sort(-rank, dim=-1, stable=True).indices[:, :, :b]
        kept = torch.sort(by, dim=-1).values
        out = {"kept": kept.int()}
        for name in ("k", "v"):
            to = torch.zeros(s[name + "_to"].shape, dtype=torch.float64, device="cuda")
            for l in range(layers):
                for h in range(kvh):
                    to[l, :b, h] = s[name][l, kept[l, h], h].double()
            out[name] = to
        to = torch.zeros(s["weights_to"].shape, dtype=torch.float64, device="cuda")
        to[:, :, :b] = torch.gather(w, 2, kept)
        out["weights"] = to
        return out
    n, qh = case["n"], case["q_heads"]
    g = qh // kvh
    if op == "tree":
        parents = s["parents"].tolist()
        sees = []  # each node's ancestors and itself, or nothing for padding
        for i, p in enumerate(parents):
            mine = ([i] if p == -1 else (sees[p] + [i] if 0 <= p < i and sees[p] else []))
            sees.append(mine)
        see = torch.zeros((n, n), dtype=torch.bool)
        for i, mine in enumerate(sees):
            see[i, mine] = True
        see = see.cuda()
        ok = torch.cat([see.any(1)[:, None].expand(n, length), see], 1)
        out = torch.zeros((layers, n, qh, d), dtype=torch.float64, device="cuda")
        lse = torch.full((layers, n, qh), -math.inf, dtype=torch.float64, device="cuda")
        live = see.any(1)
        for l in range(layers):
            for h in range(qh):
                k = s["k"][l, :length + n, h // g].double()
                v = s["v"][l, :length + n, h // g].double()
                q = s["q"][l, :, h * d:(h + 1) * d].double()
                e = (q @ k.t()) * s["scale"]
                e = e.masked_fill(~ok, -math.inf)[live]
                if e.shape[0]:
                    t = torch.logsumexp(e, -1)
                    lse[l, live, h] = t
                    out[l, live, h] = torch.exp(e - t[:, None]) @ v
        return {"out": out.view(layers, n, qh * d), "lse": lse, "mask": _mask_words(see),
                "depth": torch.tensor([len(m) - 1 for m in sees], dtype=torch.int32)}
    w = s["weights"].double()
    w[:, :, length:length + n] = 0.0
    row = s["path"].long()
    ok = torch.arange(length + n, device="cuda")[None] <= length + torch.arange(n, device="cuda")[:, None]
    for l in range(layers):
        for h in range(qh):
            k = s["k"][l, :length + n, h // g].double()
            q = s["q"][l, row, h * d:(h + 1) * d].double()
            e = (q @ k.t()) * s["scale"] - s["lse"][l, row, h].double()[:, None]
            w[l, h // g, :length + n] += torch.exp(e.masked_fill(~ok, -math.inf)).sum(0)
    return {"weights": w}

"""Workloads of the tree-decoding operators: rows written to a quantised KV cache and read back, accepted rows moved
together, attention of a tree of drafted tokens over a cache, and penalties, biases and grammar masks on logits.

listed() and draw() name the cases, prepare() makes a case's inputs on the GPU, run() makes one pass: in plain torch
operations in 32 bits, or, with `own` set, by the library's calls. exact() gives the same outputs in 64 bits.

The caches are the library's (include/synapse_b200.h, syn_kv_cache): F16 rows [position][head][dim]; Q8_0 and Q4_0 as
planes, quants [head][position][dim] and then, 256-byte aligned, binary16 scales [head][position][dim / 32].
"""
import math

import numpy as np
import torch

own = False

F16, Q4_0, Q8_0 = "f16", "q4_0", "q8_0"
QUANT_BYTES = {Q8_0: 32, Q4_0: 16}  # quants of 32 values; their scale has 2 bytes more


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of 16 sequences: each appends its token's row (RoPE, quantise, store), read back as stored
        {"name": "write-decode-16", "op": "write", "type": Q8_0, "n_seq": 16, "n": 1, "ctx": 4096, "n_head": 32, "n_kv": 8, "dim": 128, "neox": False},
        # a prompt chunk of one sequence, in the smallest cache type
        {"name": "write-prompt-2048", "op": "write", "type": Q4_0, "n_seq": 1, "n": 2048, "ctx": 8192, "n_head": 32, "n_kv": 8, "dim": 128, "neox": False},
        # a short prefix brought back in floats (a sequence handed to another engine), odd length
        {"name": "read-513", "op": "read", "type": Q4_0, "n_seq": 1, "n": 513, "ctx": 1024, "n_kv": 8, "dim": 64, "half": False},
        # a whole long context brought back in binary16
        {"name": "read-32768", "op": "read", "type": Q8_0, "n_seq": 1, "n": 32768, "ctx": 32768, "n_kv": 8, "dim": 128, "half": True},
        # one sequence's accepted path of a small tree, every layer of a small model
        {"name": "move-1x4", "op": "move", "type": Q4_0, "n_seq": 1, "n": 4, "tree": 16, "layers": 16, "ctx": 96, "n_kv": 8, "dim": 64},
        # a batch's accepted paths, every layer of an 8B-shaped model
        {"name": "move-16x8", "op": "move", "type": Q8_0, "n_seq": 16, "n": 8, "tree": 64, "layers": 32, "ctx": 128, "n_kv": 8, "dim": 128},
        # single-token decode of one sequence over a plain cache: latency counts
        {"name": "attend-1-4096-f16", "op": "attend", "type": F16, "n_seq": 1, "tree": 1, "ctx": 4096, "n_head": 32, "n_kv": 8, "dim": 128},
        # single-token decode of 16 sequences of different lengths over an 8-bit cache
        {"name": "attend-16x1-8191-q8", "op": "attend", "type": Q8_0, "n_seq": 16, "tree": 1, "ctx": 8191, "n_head": 32, "n_kv": 8, "dim": 128},
        # an ordinary tree of 16 drafted tokens in 4 sequences over an 8-bit cache
        {"name": "attend-4x16-4096-q8", "op": "attend", "type": Q8_0, "n_seq": 4, "tree": 16, "ctx": 4096, "n_head": 32, "n_kv": 8, "dim": 128},
        # the widest tree over a long context, 70B-shaped heads
        {"name": "attend-64-32768-f16", "op": "attend", "type": F16, "n_seq": 1, "tree": 64, "ctx": 32768, "n_head": 64, "n_kv": 8, "dim": 128},
        # one row of logits: a single sequence's next token
        {"name": "logits-1", "op": "logits", "n_seq": 1, "tree": 1, "vocab": 128256, "history": 1000, "biases": 16, "grammar": True},
        # the logits of 16 sequences' trees of 16 nodes, each node with its own path and grammar mask
        {"name": "logits-16x16", "op": "logits", "n_seq": 16, "tree": 16, "vocab": 128256, "history": 4096, "biases": 300, "grammar": True},
    ]


HEADS = [(32, 8, 128), (64, 8, 128), (4, 2, 32), (12, 12, 64), (24, 8, 96), (20, 4, 64), (16, 2, 256), (7, 1, 128)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "move", "attend", "attend", "logits"])
    n_head, n_kv, dim = rng.choice(HEADS)
    ty = rng.choice([F16, Q8_0, Q4_0])
    if op == "write":
        n_seq = _log(rng, 1, 32)
        n = _log(rng, 1, max(1, 2048 * 8 * 128 // (n_seq * n_kv * dim)))
        return {"op": op, "type": ty, "n_seq": n_seq, "n": n, "ctx": n + _log(rng, 1, 2048), "n_head": n_head, "n_kv": n_kv, "dim": dim, "neox": rng.random() < 0.5}
    if op == "read":
        n = _log(rng, 3, 16 * 1024 * 1024 // (n_kv * dim))
        return {"op": op, "type": ty, "n_seq": 1, "n": n, "ctx": n + _log(rng, 1, 1000), "n_kv": n_kv, "dim": dim, "half": rng.random() < 0.5}
    if op == "move":
        tree = _log(rng, 2, 64)
        return {"op": op, "type": ty, "n_seq": _log(rng, 1, 16), "n": rng.randint(1, min(tree, 12)), "tree": tree, "layers": _log(rng, 1, 32), "ctx": tree + _log(rng, 1, 64), "n_kv": n_kv, "dim": dim}
    if op == "attend":
        tree = rng.choice([1, 1, _log(rng, 2, 64)])
        n_seq = _log(rng, 1, 16) if tree == 1 else _log(rng, 1, 6)
        most = min(32768, 64 * 64 * 32768 * 128 // (n_seq * tree * n_head * dim), (1 << 27) // (n_seq * n_kv * dim))
        return {"op": op, "type": ty, "n_seq": n_seq, "tree": tree, "ctx": _log(rng, 1, most), "n_head": n_head, "n_kv": n_kv, "dim": dim}
    n_seq = _log(rng, 1, 16)
    return {"op": op, "n_seq": n_seq, "tree": _log(rng, 1, 16), "vocab": rng.choice([128256, 32000, 50257, _log(rng, 500, 120000)]), "history": _log(rng, 1, 4096), "biases": rng.choice([0, _log(rng, 1, 300)]), "grammar": rng.random() < 0.6}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _lens(case):
    """The sequences' lengths before the tree: full for the first, shorter in steps for the others."""
    n = case["n_seq"]
    return [case["ctx"] - (i * case["ctx"]) // (2 * n) for i in range(n)]


def _plane(n):
    return (n + 255) // 256 * 256


def _cache_bytes(ty, n_kv, dim, ctx):
    if ty == F16:
        return ctx * n_kv * dim * 2
    blocks = n_kv * ctx * (dim // 32)
    return _plane(blocks * QUANT_BYTES[ty]) + _plane(blocks * 2)


def _views(cache, ty, n_kv, dim, ctx):
    """The planes of caches [n][bytes]: F16 rows [n][ctx][n_kv][dim], or (quants as bytes, scales) [n][n_kv][ctx][...]."""
    n = cache.shape[0]
    if ty == F16:
        return cache.view(torch.float16).view(n, ctx, n_kv, dim)
    size = n_kv * ctx * (dim // 32)
    at = _plane(size * QUANT_BYTES[ty])
    return cache[:, :size * QUANT_BYTES[ty]].view(n, n_kv, ctx, -1), cache[:, at:at + size * 2].view(torch.float16).view(n, n_kv, ctx, dim // 32)


def _fill(gen, ty, n, n_kv, dim, ctx, sigma):
    """n caches as a decode leaves them: keys and values of spread sigma with a few loud channels, in the cache's type."""
    cache = torch.zeros(n, _cache_bytes(ty, n_kv, dim, ctx), dtype=torch.uint8, device="cuda")
    loud = torch.ones(dim, device="cuda")
    loud[::max(1, dim // 6)] = 3.0
    if ty == F16:
        _views(cache, ty, n_kv, dim, ctx).copy_(torch.randn(n, ctx, n_kv, dim, generator=gen, device="cuda") * sigma * loud)
        return cache
    quants, scales = _views(cache, ty, n_kv, dim, ctx)
    for i in range(n):
        q, d = _quantise(ty, torch.randn(n_kv, ctx, dim, generator=gen, device="cuda") * sigma * loud)
        quants[i], scales[i] = q, d
    return cache


def _trees(rng, n_seq, tree):
    """Each sequence's tree as mask words: bit j of a node's words is set when it sees node j (its ancestors and itself)."""
    words = (tree + 31) // 32
    mask = np.zeros((n_seq, tree, words), dtype=np.uint32)
    for s in range(n_seq):
        for i in range(tree):
            if i:
                mask[s, i] = mask[s, rng.integers(max(0, i - 8), i)]
            mask[s, i, i // 32] |= np.uint32(1 << (i % 32))
    return torch.from_numpy(mask.view(np.int32)).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    s = dict(case)
    op, n_seq = case["op"], case["n_seq"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    if op == "logits":
        tree, vocab = case["tree"], case["vocab"]
        s["logits"] = randn(n_seq * tree, vocab) * 3
        # a text repeats its words: few tokens often, many once
        s["past"] = (torch.rand(n_seq, case["history"], generator=gen, device="cuda").pow(3) * (vocab - 1)).int()
        s["past_len"] = torch.tensor([case["history"] - i * case["history"] // (2 * n_seq) for i in range(n_seq)], dtype=torch.int32).cuda()
        s["draft"] = ints(0, vocab, n_seq, tree)
        s["mask"] = _trees(rng, n_seq, tree)
        s["penalties"] = torch.tensor([[1.1 + 0.01 * i, 0.3, 0.2 - 0.01 * i] for i in range(n_seq)]).cuda()
        n = min(case["biases"], vocab)
        per = [n - i * n // (2 * n_seq) for i in range(n_seq)]
        s["bias_begin"] = torch.tensor([sum(per[:i]) for i in range(n_seq + 1)], dtype=torch.int32).cuda()
        s["bias_seq"] = torch.repeat_interleave(torch.arange(n_seq), torch.tensor(per)).cuda()
        picked = [rng.choice(vocab, k, replace=False) for k in per]
        s["bias_token"] = torch.from_numpy(np.concatenate(picked).astype(np.int32)).cuda()
        s["bias_value"] = randn(sum(per)) * 4
        # a grammar leaves a quarter of the words of the vocabulary, or a handful at a forced place
        words = (vocab + 31) // 32
        allowed = ints(-2**31, 2**31 - 1, n_seq * tree, words) & ints(-2**31, 2**31 - 1, n_seq * tree, words)
        s["allowed"] = allowed if case["grammar"] else None
        return s
    n_kv, dim, ctx = case["n_kv"], case["dim"], case["ctx"]
    if op == "write":
        n, n_head = case["n"], case["n_head"]
        s["q"], s["k"], s["v"] = randn(n_seq * n, n_head * dim), randn(n_seq * n, n_kv * dim), randn(n_seq * n, n_kv * dim)
        s["cache_k"], s["cache_v"] = (torch.zeros(n_seq, _cache_bytes(case["type"], n_kv, dim, ctx), dtype=torch.uint8, device="cuda") for _ in "kv")
        begin = ints(0, ctx - n + 1, n_seq, 1)
        s["slot"] = (begin + torch.arange(n, device="cuda", dtype=torch.int32)).contiguous()
        angle = torch.arange(ctx, dtype=torch.float64, device="cuda")[:, None] * 500000.0 ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64, device="cuda") / dim)
        s["table"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        return s
    if op == "read":
        s["cache_k"], s["cache_v"] = (_fill(gen, case["type"], n_seq, n_kv, dim, ctx, sigma) for sigma in (1.0, 0.5))
        return s
    if op == "move":
        layers, tree, n = case["layers"], case["tree"], case["n"]
        size = _cache_bytes(case["type"], n_kv, dim, ctx)
        s["caches"] = ints(0, 256, layers, 2, n_seq, size).to(torch.uint8)
        begin = rng.integers(0, ctx - tree + 1, n_seq)
        s["begin"] = torch.from_numpy(begin.astype(np.int32)).cuda()
        path = [begin[i] + np.sort(rng.choice(tree, n, replace=False)) for i in range(n_seq)]
        s["path"] = torch.from_numpy(np.stack(path).astype(np.int32)).cuda()
        s["count"] = torch.full((n_seq,), n, dtype=torch.int32, device="cuda")
        return s
    tree, n_head = case["tree"], case["n_head"]
    s["room"] = ctx + tree
    s["cache_k"], s["cache_v"] = (_fill(gen, case["type"], n_seq, n_kv, dim, ctx + tree, sigma) for sigma in (1.0, 0.5))
    s["q"] = randn(n_seq * tree, n_head * dim) * 1.5
    s["len"] = torch.tensor(_lens(case), dtype=torch.int32).cuda()
    s["mask"] = _trees(rng, n_seq, tree)
    s["scale"] = 1.0 / math.sqrt(dim)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _quantise(ty, x):
    """Blocks of 32 along the last axis -> (quants as bytes, binary16 scales): the library's Q8_0 and Q4_0."""
    b = x.unflatten(-1, (-1, 32))
    if ty == Q8_0:
        d = b.abs().amax(-1) / 127.0
        y = b * torch.where(d != 0, 1.0 / d, 0.0)[..., None]
        a = y.abs()
        whole = a.floor()
        q = torch.copysign(whole + (a - whole >= 0.5), y).to(torch.int8).flatten(-2)
        return q.view(torch.uint8), d.half()
    at = b.abs().argmax(-1, keepdim=True)
    d = b.gather(-1, at) / -8.0
    q = (b * torch.where(d != 0, 1.0 / d, 0.0) + 8.5).to(torch.int32).clamp(0, 15).to(torch.uint8)
    return (q[..., :16] | (q[..., 16:] << 4)).flatten(-2), d[..., 0].half()


def _dequantise(ty, quants, scales):
    """(quants as bytes, scales) [..., blocks] -> floats [..., dims]."""
    if ty == Q8_0:
        q = quants.view(torch.int8).float().unflatten(-1, (-1, 32))
    else:
        b = quants.unflatten(-1, (-1, 16))
        q = torch.cat([b & 15, b >> 4], -1).float() - 8.0
    return (q * scales.float()[..., None]).flatten(-2)


def _floats(cache, ty, n_kv, dim, ctx):
    """Caches as floats [n][n_kv][ctx][dim]."""
    if ty == F16:
        return _views(cache, ty, n_kv, dim, ctx).float().transpose(1, 2)
    return _dequantise(ty, *_views(cache, ty, n_kv, dim, ctx))


def _rotate(x, table, pos, neox):
    """x [n][heads][dim] at positions pos [n]."""
    c, sn = table[pos.long(), None, :, 0], table[pos.long(), None, :, 1]
    half = x.shape[-1] // 2
    a, b = (x[..., :half], x[..., half:]) if neox else (x[..., 0::2], x[..., 1::2])
    out = torch.empty_like(x)
    (out[..., :half] if neox else out[..., 0::2]).copy_(a * c - b * sn)
    (out[..., half:] if neox else out[..., 1::2]).copy_(a * sn + b * c)
    return out


def _bits(words, n):
    """Mask words [...][w] -> truth values [...][n]."""
    shift = torch.arange(32, device=words.device, dtype=torch.int32)
    return ((words[..., None] >> shift) & 1).bool().flatten(-2)[..., :n]


def _plain_write(s):
    ty, n_seq, n, n_kv, dim, ctx = s["type"], s["n_seq"], s["n"], s["n_kv"], s["dim"], s["ctx"]
    pos = s["slot"].flatten()
    q = _rotate(s["q"].view(n_seq * n, -1, dim), s["table"], pos, s["neox"]).flatten(1)
    rows = [_rotate(s["k"].view(-1, n_kv, dim), s["table"], pos, s["neox"]), s["v"].view(-1, n_kv, dim)]
    seq = torch.arange(n_seq, device="cuda").repeat_interleave(n)
    back = []
    for x, cache in zip(rows, (s["cache_k"], s["cache_v"])):
        at = pos.long()
        if ty == F16:
            rows16 = _views(cache, ty, n_kv, dim, ctx)
            rows16[seq, at] = x.half()
            back.append(rows16[seq, at])
        else:
            quants, scales = _views(cache, ty, n_kv, dim, ctx)
            quants[seq, :, at], scales[seq, :, at] = _quantise(ty, x)
            back.append(_dequantise(ty, quants[seq, :, at], scales[seq, :, at]).half())
    return q, back[0].view(n_seq, n, n_kv, dim), back[1].view(n_seq, n, n_kv, dim)


def _plain_read(s):
    ty, n_kv, dim, ctx = s["type"], s["n_kv"], s["dim"], s["ctx"]
    out = torch.float16 if s["half"] else torch.float32
    return tuple(_floats(c, ty, n_kv, dim, ctx)[:, :, :s["n"]].transpose(1, 2).to(out).contiguous() for c in (s["cache_k"], s["cache_v"]))


def _plain_move(s):
    ty, n_kv, dim, ctx, n_seq = s["type"], s["n_kv"], s["dim"], s["ctx"], s["n_seq"]
    seq = torch.arange(n_seq, device="cuda")[:, None]
    src, dst = s["path"].long(), s["begin"].long()[:, None] + torch.arange(s["n"], device="cuda")
    flat = s["caches"].view(-1, s["caches"].shape[-1])
    planes = _views(flat, ty, n_kv, dim, ctx)
    for p in ((planes,) if ty == F16 else planes):
        p = p.unflatten(0, (-1, n_seq))
        if ty == F16:
            p[:, seq, dst] = p[:, seq, src].clone()
        else:
            p[:, seq, :, dst] = p[:, seq, :, src].clone()
    return s["caches"]


def _plain_attend(s):
    n_seq, tree, n_head, n_kv, dim, room = s["n_seq"], s["tree"], s["n_head"], s["n_kv"], s["dim"], s["room"]
    group = n_head // n_kv
    k, v = (_floats(c, s["type"], n_kv, dim, room) for c in (s["cache_k"], s["cache_v"]))
    q = s["q"].view(n_seq, tree, n_kv, group, dim).permute(0, 2, 1, 3, 4).reshape(n_seq, n_kv, tree * group, dim)
    score = q @ k.transpose(2, 3) * s["scale"]
    at = torch.arange(room, device="cuda") - s["len"].long()[:, None]  # a position's node in the tree: [n_seq][room]
    node = at.clamp(0, tree - 1)[:, None].expand(-1, tree, -1)
    sees = (at < 0)[:, None] | ((at < tree)[:, None] & _bits(s["mask"], tree).gather(2, node))
    score = score.view(n_seq, n_kv, tree, group, room).masked_fill(~sees[:, None, :, None], -math.inf)
    e = (score - score.amax(-1, keepdim=True)).exp()
    p = (e / e.sum(-1, keepdim=True)).view(n_seq, n_kv, tree * group, room)
    out = (p @ v).view(n_seq, n_kv, tree, group, dim).permute(0, 2, 1, 3, 4)
    return out.reshape(n_seq * tree, n_head * dim)


def _plain_logits(s):
    n_seq, tree, vocab = s["n_seq"], s["tree"], s["vocab"]
    x = s["logits"].view(n_seq, tree, vocab)
    bias = torch.zeros(n_seq, vocab, device="cuda")
    bias[s["bias_seq"], s["bias_token"].long()] = s["bias_value"]
    inside = torch.arange(s["past"].shape[1], device="cuda") < s["past_len"][:, None]
    count = torch.zeros(n_seq, vocab, device="cuda").scatter_add_(1, s["past"].long(), inside.float())
    count = count[:, None].repeat(1, tree, 1)
    count.scatter_add_(2, s["draft"].long()[:, None].expand(-1, tree, -1), _bits(s["mask"], tree).float())
    repeat, presence, frequency = s["penalties"][:, None, None].unbind(-1)
    x = x + bias[:, None]
    seen = count > 0
    x = torch.where(seen, torch.where(x > 0, x / repeat, x * repeat) - (count * frequency + presence), x)
    x = x.view(n_seq * tree, vocab)
    if s["allowed"] is not None:
        x = x.masked_fill(~_bits(s["allowed"], vocab), -math.inf)
    return x, x.argmax(-1).int()


# ---- the library's calls ----------------------------------------------------------------------------------------------
def _handle(s):
    """The program's caches as the library takes them, and its scratch: made at a state's first pass and kept."""
    if "handle" not in s:
        import synapse_b200 as syn
        ty = {F16: syn.F16, Q8_0: syn.Q8_0, Q4_0: syn.Q4_0}
        if s["op"] == "logits":
            s["handle"] = syn, syn.logits_scratch(s["n_seq"] * s["tree"])
        elif s["op"] == "move":
            k, v = s["caches"][:, 0], s["caches"][:, 1]
            s["handle"] = syn, syn.KVCache.over(ty[s["type"]], k, v, s["n_kv"], s["dim"], s["ctx"])
        else:
            cache = syn.KVCache.over(ty[s["type"]], s["cache_k"], s["cache_v"], s["n_kv"], s["dim"], s.get("room", s["ctx"]))
            s["handle"] = syn, cache, syn.tree_attention_scratch(cache, s["tree"], s["n_head"], s["room"]) if s["op"] == "attend" else None
    return s["handle"]


def _own(s):
    syn, cache, *scratch = _handle(s)
    op = s["op"]
    if op == "write":
        q = syn.kv_append(cache, s["k"], s["v"], s["slot"], rope_table=s["table"], rope_mode=int(s["neox"]), q=s["q"])
        return (q, *syn.kv_read(cache, s["n"], rows=s["slot"], dtype=torch.float16))
    if op == "read":
        return syn.kv_read(cache, s["n"], dtype=torch.float16 if s["half"] else torch.float32)
    if op == "move":
        syn.kv_move(cache, s["path"], s["count"], s["begin"])
        return s["caches"]
    if op == "attend":
        return syn.tree_attention(cache, s["q"], s["len"], s["n_head"], s["scale"], tree=s["tree"], mask=s["mask"], max_len=s["room"], scratch=scratch[0])
    return syn.logits_process(s["logits"], s["n_seq"], penalties=s["penalties"], history=s["past"], history_len=s["past_len"], draft=s["draft"],
                              mask=s["mask"], bias=(s["bias_begin"], s["bias_token"], s["bias_value"]), allowed=s["allowed"], scratch=cache)


PLAIN = {"write": _plain_write, "read": _plain_read, "move": _plain_move, "attend": _plain_attend, "logits": _plain_logits}


def run(state):
    return _own(state) if own else PLAIN[state["op"]](state)


# ---- the work of one pass ---------------------------------------------------------------------------------------------
def _row_bytes(case):
    """Bytes of one position's keys (or values) in the cache."""
    values = case["n_kv"] * case["dim"]
    return values * 2 if case["type"] == F16 else values // 32 * (QUANT_BYTES[case["type"]] + 2)


def work(case):
    op, n_seq = case["op"], case["n_seq"]
    if op == "logits":
        rows = n_seq * case["tree"]
        return {"bytes": rows * (8 * case["vocab"] + (case["vocab"] // 8 if case["grammar"] else 0) + 4) + n_seq * (4 * case["history"] + 8 * case["biases"]), "flops": 0}
    values = case["n_kv"] * case["dim"]
    if op == "write":
        n = n_seq * case["n"]
        # q in and out, k and v in, the rows stored, and the rows read back in binary16
        return {"bytes": n * (8 * case["n_head"] * case["dim"] + 8 * values + 2 * _row_bytes(case) + 4 * values), "flops": 0}
    if op == "read":
        return {"bytes": 2 * n_seq * case["n"] * (_row_bytes(case) + values * (2 if case["half"] else 4)), "flops": 0}
    if op == "move":
        return {"bytes": 4 * n_seq * case["layers"] * case["n"] * _row_bytes(case), "flops": 0}
    seen = sum(n + case["tree"] for n in _lens(case))
    rows = n_seq * case["tree"] * case["n_head"] * case["dim"]
    return {"bytes": 2 * seen * _row_bytes(case) + 8 * rows, "flops": 4 * seen * case["tree"] * case["n_head"] * case["dim"]}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------
def _exact_values(s, cache, ctx):
    """A cache's stored values in 64 bits, [n][ctx][n_kv][dim], from its bytes."""
    n, n_kv, dim, ty = cache.shape[0], s["n_kv"], s["dim"], s["type"]
    if ty == F16:
        return cache.view(torch.float16).double().reshape(n, ctx, n_kv, dim)
    blocks = n_kv * ctx * dim // 32
    raw = cache[:, :blocks * QUANT_BYTES[ty]]
    first = -(-blocks * QUANT_BYTES[ty] // 256) * 256
    d = cache[:, first:first + 2 * blocks].view(torch.float16).double().reshape(n, blocks, 1)
    if ty == Q8_0:
        q = raw.to(torch.int16)
        q = torch.where(q > 127, q - 256, q).double().reshape(n, blocks, 32)
    else:
        raw = raw.reshape(n, blocks, 16).to(torch.int16)
        q = torch.cat([raw % 16, raw // 16], 2).double() - 8
    return (q * d).reshape(n, n_kv, ctx, dim).transpose(1, 2)


def _exact_block(ty, x):
    """x [..., dim] as a cache of type ty holds it, in 64 bits but for the scale, which is stored in binary16."""
    if ty == F16:
        return x.half().double()
    b = x.reshape(*x.shape[:-1], -1, 32)
    if ty == Q8_0:
        d = b.abs().max(-1, keepdim=True).values / 127
        q = torch.sign(b) * (b.abs() / d.clamp_min(1e-300) + 0.5).floor()
    else:
        low, high = b.min(-1, keepdim=True).values, b.max(-1, keepdim=True).values
        d = torch.where(high > -low, high, low) / -8
        q = (b / torch.where(d == 0, 1.0, d) + 8.5).floor().clamp(max=15) - 8
    return (q * d.half().double()).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    op, n_seq = case["op"], case["n_seq"]
    if op == "move":
        return None
    if op == "read":
        return tuple(_exact_values(s, s[c], case["ctx"])[:, :case["n"]] for c in ("cache_k", "cache_v"))
    if op == "write":
        n, dim = case["n"], case["dim"]
        turn = torch.view_as_complex(s["table"].double())[s["slot"].long()][:, :, None]

        def rotated(x):
            x = x.double().reshape(n_seq, n, -1, dim)
            pair = x.unflatten(-1, (2, -1)).transpose(-1, -2) if case["neox"] else x.unflatten(-1, (-1, 2))
            y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
            return (y.transpose(-1, -2) if case["neox"] else y).reshape(x.shape)
        v = s["v"].double().reshape(n_seq, n, -1, dim)
        return rotated(s["q"]).reshape(n_seq * n, -1), _exact_block(case["type"], rotated(s["k"])), _exact_block(case["type"], v)
    words = s["mask"].cpu().numpy().view(np.uint32)
    tree = case["tree"]
    sees = [[[j for j in range(tree) if int(words[i, t, j // 32]) >> (j % 32) & 1] for t in range(tree)] for i in range(n_seq)]
    if op == "logits":
        out = s["logits"].double().clone()
        past, lens, draft, pen = (s[c].cpu().tolist() for c in ("past", "past_len", "draft", "penalties"))
        begin = s["bias_begin"].tolist()
        for i in range(n_seq):
            at = slice(begin[i], begin[i + 1])
            rep, pres, freq = (float(x) for x in pen[i])
            for t in range(tree):
                row = out[i * tree + t]
                row[s["bias_token"][at].long()] += s["bias_value"][at].double()
                tokens, counts = np.unique(past[i][:lens[i]] + [draft[i][j] for j in sees[i][t]], return_counts=True)
                tokens, counts = torch.from_numpy(tokens).cuda(), torch.from_numpy(counts).cuda().double()
                x = row[tokens]
                row[tokens] = torch.where(x > 0, x / rep, x * rep) - counts * freq - pres
        if s["allowed"] is not None:
            place = torch.arange(case["vocab"], device="cuda")
            for r in range(n_seq * tree):
                out[r][(s["allowed"][r].long()[place // 32] >> (place % 32)) & 1 == 0] = -math.inf
        return out, None
    room, n_head, dim = s["room"], case["n_head"], case["dim"]
    group = n_head // case["n_kv"]
    out = torch.zeros(n_seq, tree, n_head, dim, dtype=torch.float64, device="cuda")
    for i, n in enumerate(_lens(case)):
        k, v = (_exact_values(s, s[c][i:i + 1], room)[0] for c in ("cache_k", "cache_v"))
        hidden = torch.ones(tree, n + tree, dtype=torch.bool, device="cuda")
        hidden[:, :n] = False
        for t in range(tree):
            hidden[t, [n + j for j in sees[i][t]]] = False
        for h in range(n_head):
            q = s["q"].view(n_seq, tree, n_head, dim)[i, :, h].double()
            score = torch.einsum("td,pd->tp", q, k[:n + tree, h // group]) / math.sqrt(dim)
            p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
            out[i, :, h] = torch.einsum("tp,pd->td", p, v[:n + tree, h // group])
    return out.reshape(n_seq * tree, n_head * dim)

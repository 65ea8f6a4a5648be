"""Greedy decoding with trees of drafted tokens over a quantised KV cache.

  python -m synapse_b200.tree_decode [--cache f16|q8_0|q4_0] [--tree N] [--steps N] [--seqs N] [--layers N]

Runs the tree operators together, as a serving program does, on a Llama-shaped
model of random weights: every step drafts a tree of continuations from the
pairs of neighbouring tokens in the sequence and in a corpus (here an earlier
decode of the same prompts, a fifth of its tokens changed), appends the drafted tokens' K and V rows to the cache
(syn_kv_append), attends with the tree's mask (syn_tree_attention), picks a
token at every node under penalties, biases and a grammar mask
(syn_logits_process), keeps the longest path that the picks confirm and moves
its rows together (syn_kv_move). The tokens are those of decoding one at a time,
up to near ties that the orders of summing decide; the command decodes both ways
and compares.
"""
import argparse
import json
import math

import numpy as np

from . import F16, F32, LAYOUT_PLANAR, Q4_0, Q8_0, KVCache, embed, kv_append, kv_move, kv_read, logits_process, \
    logits_scratch, mul_mat, rms_norm, rope_table, silu_mul, tree_attention, tree_attention_scratch, upload_weight
from .model import random_llama_weights

CACHES = {"f16": F16, "q8_0": Q8_0, "q4_0": Q4_0}
MOST_NODES = 1024  # of a tree (syn_tree_attention)


def tree_mask(parents):
    """Mask words (int32 [nodes][words]) and depths of a tree given by each node's parent (-1 for the root; a parent
    comes before its children): a node sees its ancestors and itself."""
    n = len(parents)
    words = np.zeros((n, (n + 31) // 32), np.uint32)
    depth = np.zeros(n, np.int32)
    for i, p in enumerate(parents):
        if p >= 0:
            words[i], depth[i] = words[p], depth[p] + 1
        words[i, i // 32] |= np.uint32(1 << (i % 32))
    return words.view(np.int32), depth


def draft_pairs(history, size, corpus=(), branch=2):
    """A tree of `size` nodes from the last token on: what followed each token earlier, in the history or the corpus,
    most recent first. (tokens, parents); node 0 is the last token itself. The tree is filled up with copies of it under
    the root."""
    follow = {}
    for a, b in [*zip(corpus, corpus[1:]), *zip(history, history[1:])]:
        f = follow.setdefault(int(a), [])
        if b in f:
            f.remove(b)
        f.insert(0, int(b))
    tokens, parents, at = [int(history[-1])], [-1], 0
    while len(tokens) < size:
        while at < len(tokens) and tokens[at] not in follow:
            at += 1
        if at == len(tokens):
            parents += [0] * (size - len(tokens))
            tokens += [tokens[0]] * (size - len(tokens))
            break
        for b in follow[tokens[at]][:branch]:
            if len(tokens) < size:
                tokens.append(b)
                parents.append(at)
        at += 1
    return tokens, parents


class TreeDecoder:
    """A Llama-shaped model and the caches of n_seq sequences, decoded a tree per sequence and step."""

    def __init__(self, cfg, weights, cache_type, n_seq, max_ctx, tree, device="cuda"):
        import torch
        self.torch, self.cfg, self.n_seq, self.max_ctx = torch, cfg, n_seq, max_ctx
        self.w = {}
        for name, (ty, a) in weights.items():
            if name.endswith("norm"):
                self.w[name] = torch.from_numpy(np.ascontiguousarray(a, np.float32)).to(device)
            else:
                cols = {"attn_output": cfg["n_head"] * cfg["head_dim"], "ffn_down": cfg["n_ff"]}.get(name.split(".")[-1], cfg["n_embd"])
                rows = a.shape[0]
                self.w[name] = (ty, upload_weight(ty, a, rows, cols, LAYOUT_PLANAR, device), rows, cols)
        self.cache = KVCache(cache_type, cfg["n_layer"], n_seq, cfg["n_head_kv"], cfg["head_dim"], max_ctx, device)
        self.table = rope_table(max_ctx, cfg["head_dim"], cfg["rope_base"] ** (-2.0 / cfg["head_dim"]), device=device)
        self.scratch = {n: tree_attention_scratch(self.cache, n, cfg["n_head"]) for n in {1, tree}}
        self.pick_scratch = logits_scratch(n_seq * tree, device)
        self.corpus = [()] * n_seq                   # texts to draft from
        self.histories = [[] for _ in range(n_seq)]  # committed tokens and the one to feed next
        self.lens = np.zeros(n_seq, np.int32)        # rows committed

    def dev(self, a):
        return self.torch.from_numpy(np.ascontiguousarray(a)).to(self.cache.device)

    def forward(self, tokens, parents):
        """Logits [n_seq * nodes][n_vocab] of one tree per sequence appended after its committed rows, and the mask.
        Raises ValueError when a tree does not fit its sequence's cache."""
        c, w, n = self.cfg, self.w, tokens.shape[1]
        if self.lens.max() + n > self.max_ctx:
            raise ValueError(f"{n} rows after {self.lens.max()} do not fit a cache of {self.max_ctx}")
        masks, depths = zip(*(tree_mask(p) for p in parents))
        mask = self.dev(np.stack(masks))
        slot = self.dev((self.lens[:, None] + np.arange(n, dtype=np.int32)).reshape(-1))
        pos = self.dev((self.lens[:, None] + np.stack(depths)).reshape(-1).astype(np.int32))
        lens = self.dev(self.lens)
        mm = lambda name, x: mul_mat(w[name][0], w[name][1], LAYOUT_PLANAR, w[name][2], w[name][3], x)  # noqa: E731
        ty, table, rows, cols = w["token_embd"]
        x = embed(ty, table, LAYOUT_PLANAR, rows, cols, self.dev(tokens.reshape(-1)))
        for i in range(c["n_layer"]):
            b = f"blk.{i}."
            h, _ = rms_norm(x, w[b + "attn_norm"], c["rms_eps"])
            q = kv_append(self.cache, mm(b + "attn_k", h), mm(b + "attn_v", h), slot, pos=pos, rope_table=self.table,
                          q=mm(b + "attn_q", h), layer=i)
            a = tree_attention(self.cache, q, lens, c["n_head"], 1 / math.sqrt(c["head_dim"]), tree=n, mask=mask,
                               scratch=self.scratch.get(n), layer=i)
            x = x + mm(b + "attn_output", a)
            h, _ = rms_norm(x, w[b + "ffn_norm"], c["rms_eps"])
            g, _ = silu_mul(mm(b + "ffn_gate", h), mm(b + "ffn_up", h))
            x = x + mm(b + "ffn_down", g)
        h, _ = rms_norm(x, w["output_norm"], c["rms_eps"])
        return mm("output" if "output" in w else "token_embd", h), mask

    def step(self, size, rules):
        """One step of a tree of `size` nodes per sequence: the tokens that it commits, for every sequence. Raises ValueError,
        with nothing committed, where the rules leave a sequence no token."""
        drafts = [draft_pairs(h, size, c) for h, c in zip(self.histories, self.corpus)]
        tokens = np.array([d[0] for d in drafts], np.int32)
        logits, mask = self.forward(tokens, [d[1] for d in drafts])
        most = max(len(h) for h in self.histories)
        past = np.full((self.n_seq, most), -1, np.int32)  # without the last token: it is node 0 of the tree
        for s, h in enumerate(self.histories):
            past[s, :len(h) - 1] = h[:-1]
        _, picks = logits_process(logits, self.n_seq, penalties=rules.get("penalties"), history=self.dev(past),
                                  history_len=self.dev(np.array([len(h) - 1 for h in self.histories], np.int32)),
                                  draft=self.dev(tokens), mask=mask, bias=rules.get("bias"),
                                  allowed=None if "allowed" not in rules else rules["allowed"].repeat(logits.shape[0], 1),
                                  out=logits, scratch=self.pick_scratch)
        picks = picks.cpu().numpy().reshape(self.n_seq, size)
        path = np.zeros((self.n_seq, size), np.int32)
        count = np.zeros(self.n_seq, np.int32)
        out = []
        for s, (toks, parents) in enumerate(drafts):
            node, kept, new = 0, [0], [int(picks[s, 0])]
            while True:  # the child whose token is the pick, if the tree has it
                node = next((i for i in range(node + 1, size) if parents[i] == node and toks[i] == new[-1]), None)
                if node is None:
                    break
                kept.append(node)
                new.append(int(picks[s, node]))
            if min(new) < 0:
                raise ValueError(f"no logit of sequence {s} is above -inf: no token to go on with")
            path[s, :len(kept)] = self.lens[s] + np.array(kept)
            count[s] = len(kept)
            out.append(new)
        kv_move(self.cache, self.dev(path), self.dev(count), self.dev(self.lens))
        for s, new in enumerate(out):
            self.lens[s] += count[s]
            self.histories[s] += new
        return out

    def keep(self, n):
        """Takes the tokens past the first n of every sequence back; their rows are written again."""
        for s, h in enumerate(self.histories):
            if len(h) > n:
                del h[n:]
                self.lens[s] = n - 1

    def start(self, prompts):
        """Prompts of one length: all but the last token are run as chains through the cache."""
        self.histories = [list(map(int, p)) for p in prompts]
        self.lens[:] = 0
        tokens = np.array([p[:-1] for p in prompts], np.int32)
        for i in range(0, tokens.shape[1], MOST_NODES):
            part = tokens[:, i:i + MOST_NODES]
            self.forward(part, [list(range(-1, part.shape[1] - 1))] * self.n_seq)
            self.lens += part.shape[1]


def decode(model, prompts, steps, size, rules):
    """`steps` tokens per sequence by trees of `size` nodes: (tokens [n_seq][steps], forward passes). The caches need room
    for the prompt, the steps and a tree; a sequence that is done waits for the others."""
    model.start(prompts)
    first, passes = len(prompts[0]), 0
    while min(len(h) for h in model.histories) < first + steps:
        model.step(size, rules)
        model.keep(first + steps)
        passes += 1
    return [h[first:first + steps] for h in model.histories], passes


def changed(texts, vocab, seed=0):
    """Texts with a fifth of their tokens replaced by others."""
    rng = np.random.default_rng(seed)
    return [[int(rng.integers(vocab)) if rng.random() < 0.2 else t for t in x] for x in texts]


def default_rules(torch, cfg, n_seq, seed=0):
    """Penalties, a few biases and a grammar that forbids a tenth of the vocabulary."""
    rng = np.random.default_rng(seed)
    vocab = cfg["n_vocab"]
    allowed = np.zeros((1, (vocab + 31) // 32 * 32), np.uint8)
    allowed[0, :vocab] = rng.random(vocab) > 0.1
    words = np.packbits(allowed, axis=1, bitorder="little").view(np.int32)
    tokens = np.concatenate([rng.choice(vocab, 4, replace=False) for _ in range(n_seq)]).astype(np.int32)
    return {"penalties": torch.tensor([[1.05, 0.0, 0.02]] * n_seq, device="cuda"),
            "bias": (torch.arange(0, 4 * n_seq + 1, 4, dtype=torch.int32, device="cuda"), torch.from_numpy(tokens).cuda(),
                     torch.full((4 * n_seq,), 0.1, device="cuda")),
            "allowed": torch.from_numpy(words).cuda()}


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--cache", choices=sorted(CACHES), default="q8_0")
    p.add_argument("--tree", type=int, default=16)
    p.add_argument("--steps", type=int, default=64)
    p.add_argument("--seqs", type=int, default=2)
    p.add_argument("--layers", type=int, default=2)
    a = p.parse_args()
    import torch
    cfg = dict(n_layer=a.layers, n_embd=512, n_ff=1024, n_head=8, n_head_kv=2, head_dim=64, n_vocab=2048, rms_eps=1e-5,
               rope_base=10000.0)
    weights = random_llama_weights(cfg, seed=1, type_layers=F32, type_embd=F32, tied=True, sigma=0.05)
    prompts = np.random.default_rng(2).integers(0, cfg["n_vocab"], (a.seqs, 24)).tolist()
    rules = default_rules(torch, cfg, a.seqs)
    model = TreeDecoder(cfg, weights, CACHES[a.cache], a.seqs, 24 + a.steps + 2 * a.tree, a.tree)
    one, n_one = decode(model, prompts, a.steps, 1, rules)
    model.corpus = changed([p + o for p, o in zip(prompts, one)], cfg["n_vocab"])
    many, n_many = decode(model, prompts, a.steps, a.tree, rules)
    k, _ = kv_read(model.cache, int(model.lens[0]), layer=a.layers - 1)
    print(json.dumps({"cache": a.cache, "tree": a.tree, "tokens": a.steps, "sequences": a.seqs, "passes_one": n_one,
                      "passes_tree": n_many, "same_tokens": one == many, "cache_bytes": int(2 * model.cache.k.numel()),
                      "last_layer_k_rms": float(k.square().mean().sqrt())}))


if __name__ == "__main__":
    main()

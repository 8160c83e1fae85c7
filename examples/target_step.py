"""The target model's side of one speculative step, on one full-attention layer and one gated-delta layer
with random projections: prompts into the paged cache and the recurrent states, a draft tree verified
against both, the accepted path committed, a plain decode.

    PYTHONPATH=. python examples/target_step.py [--cache e4m3|fp16] [--prompts 700,33,1]
"""
from __future__ import annotations

import argparse

import torch

from chain_flow_b200.attention import PagedAttention
from chain_flow_b200.gdn import ChunkedGdn, ancestor_chains, gdn_step, gdn_verify, make_tree
from chain_flow_b200.kv_cache import PagedKVCache
from chain_flow_b200.tree import ancestor_mask, tree_attn_merge

HEADS, KV_HEADS, HEAD_DIM = 16, 4, 256           # the attention layer
KEY_HEADS, VALUE_HEADS, KEY_DIM, VALUE_DIM = 16, 32, 128, 128    # the gated-delta layer
PAGE = 16


class TargetLayers:
    """The two layers' state for ``requests`` requests of up to ``max_len`` tokens, and trees of up to
    ``nodes`` nodes. State slots: one per request, then one per tree row."""

    def __init__(self, requests: int, max_len: int, nodes: int, dtype=torch.float16, cache_dtype=torch.float8_e4m3fn, seed: int = 0):
        per = -(-max_len // PAGE)
        self.requests, self.nodes, self.dtype = requests, nodes, dtype
        self.cache = PagedKVCache(requests * per, PAGE, KV_HEADS, HEAD_DIM, cache_dtype)
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.table = torch.randperm(requests * per, generator=g, device="cuda").view(requests, per).int()
        self.kv_len = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.attention = PagedAttention(HEADS, KV_HEADS, HEAD_DIM)
        self.chunks = ChunkedGdn(requests * max_len, requests, VALUE_HEADS)
        self.state = torch.zeros(requests * (1 + nodes), VALUE_HEADS, VALUE_DIM, KEY_DIM, device="cuda")
        self.slot = torch.arange(requests, dtype=torch.int32, device="cuda")          # where a request's state is
        self.A_log = torch.rand(VALUE_HEADS, device="cuda", generator=g)
        self.dt_bias = torch.randn(VALUE_HEADS, device="cuda", generator=g)
        self.scale = KEY_DIM ** -0.5

    def slots_of(self, request, position):
        """The cache's flat slots of positions of requests."""
        return self.table[request.long(), (position // PAGE).long()].long() * PAGE + position.long() % PAGE

    def _gdn(self, x, o):
        return self.A_log, self.dt_bias, x["a"], x["b"], x["gq"], x["gk"], x["gv"], o, self.state

    def prompt(self, x, news):
        """Whole prompts of news[b] tokens, request after request. Returns both layers' outputs."""
        cu = torch.tensor([0] + list(news), device="cuda").cumsum(0).int()
        request = torch.repeat_interleave(torch.arange(len(news), device="cuda"), torch.tensor(news, device="cuda"))
        position = torch.arange(len(request), device="cuda") - cu[request]
        self.cache.write(x["k"], x["v"], self.slots_of(request, position))
        self.kv_len = cu.diff().int()
        attn, _ = self.attention(x["q"], self.cache, self.table, self.kv_len, cu)
        o = torch.empty_like(x["gv"])
        self.chunks(*self._gdn(x, o), cu, torch.full_like(self.slot, -1), self.slot, scale=self.scale)
        return attn, o

    def verify(self, x, parents):
        """A tree of N nodes a request (parents [S, N], -1: the committed token): every node sees its request's
        context and its own ancestors. Nothing is committed: the nodes' states go to the tree's slots."""
        S, N = parents.shape
        rows = torch.arange(S * N, device="cuda")
        cu = torch.arange(0, S * N + 1, N, device="cuda").int()
        prefix, lse = self.attention(x["q"], self.cache, self.table, self.kv_len, cu, causal=False)
        attn = tree_attn_merge(x["q"], x["k"], x["v"], torch.empty_like(prefix), prefix, lse, rows.view(S, N),
                               ancestor_mask(parents), HEAD_DIM ** -0.5)
        flat = torch.where(parents >= 0, parents + torch.arange(S, device="cuda")[:, None] * N, parents)
        chain, depth = ancestor_chains(flat.view(-1), N)
        o = torch.empty_like(x["gv"])
        gdn_verify(*self._gdn(x, o), chain, depth, self.requests + rows.int(), self.slot.repeat_interleave(N), scale=self.scale)
        return attn, o

    def commit(self, x, paths):
        """The accepted nodes of each request (paths[b]: node numbers from the root down) join its context; its
        state is the last one's."""
        request = torch.tensor([b for b, p in enumerate(paths) for _ in p], device="cuda", dtype=torch.long)
        depth = torch.tensor([i for p in paths for i in range(len(p))], device="cuda", dtype=torch.int32)
        rows = torch.tensor([b * self.nodes + n for b, p in enumerate(paths) for n in p], device="cuda", dtype=torch.long)
        self.cache.write(x["k"][rows], x["v"][rows], self.slots_of(request, self.kv_len[request] + depth))
        self.kv_len = self.kv_len + torch.tensor([len(p) for p in paths], device="cuda", dtype=torch.int32)
        last = torch.tensor([self.requests + b * self.nodes + p[-1] if p else b for b, p in enumerate(paths)], device="cuda")
        self.state[:self.requests] = self.state[last]

    def decode(self, x):
        """One token of every request."""
        self.cache.write(x["k"], x["v"], self.slots_of(self.slot, self.kv_len))
        self.kv_len = self.kv_len + 1
        cu = torch.arange(self.requests + 1, device="cuda", dtype=torch.int32)
        attn, _ = self.attention(x["q"], self.cache, self.table, self.kv_len, cu)
        o = torch.empty_like(x["gv"])
        gdn_step(*self._gdn(x, o), self.slot, self.slot, scale=self.scale)
        return attn, o


def projections(tokens: int, dtype=torch.float16, seed: int = 0):
    """What the two layers' projections would give for ``tokens`` tokens."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda *shape, t=dtype: torch.randn(*shape, device="cuda", generator=g).to(t)
    return dict(q=draw(tokens, HEADS, HEAD_DIM), k=draw(tokens, KV_HEADS, HEAD_DIM), v=draw(tokens, KV_HEADS, HEAD_DIM),
                gq=draw(tokens, KEY_HEADS, KEY_DIM), gk=draw(tokens, KEY_HEADS, KEY_DIM), gv=draw(tokens, VALUE_HEADS, VALUE_DIM),
                a=draw(tokens, VALUE_HEADS, t=torch.float32), b=draw(tokens, VALUE_HEADS, t=torch.float32))


def main():
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--cache", choices=("e4m3", "fp16"), default="e4m3")
    p.add_argument("--prompts", default="700,33,1")
    p.add_argument("--nodes", type=int, default=12)
    a = p.parse_args()
    news = [int(n) for n in a.prompts.split(",")]
    layers = TargetLayers(len(news), max(news) + a.nodes + 1, a.nodes,
                          cache_dtype=torch.float8_e4m3fn if a.cache == "e4m3" else torch.float16)
    out = layers.prompt(projections(sum(news), seed=1), news)
    print("prompts ", news, *(tuple(t.shape) for t in out))
    parents = torch.stack([make_tree(a.nodes, 4, 3, seed=b)[0] for b in range(len(news))]).cuda()
    tree = projections(len(news) * a.nodes, seed=2)
    out = layers.verify(tree, parents)
    print("verified", list(parents.shape), *(tuple(t.shape) for t in out))
    paths = []
    for row in parents.tolist():                     # a target would accept by its logits: here, the last node's path
        path = [len(row) - 1]
        while row[path[0]] >= 0:
            path.insert(0, row[path[0]])
        paths.append(path)
    layers.commit(tree, paths)
    out = layers.decode(projections(len(news), seed=3))
    layers.attention.check()
    layers.chunks.check()
    print("accepted", paths, "decoded", *(tuple(t.shape) for t in out), "contexts", layers.kv_len.tolist())


if __name__ == "__main__":
    main()

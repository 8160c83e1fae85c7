"""Performance cases of what closes a sampled speculative step: drafted tokens verified against the
target's probabilities from given random numbers (a tree or chain without draft probabilities, a chain
with them), accepted rows moved together in the paged caches of all layers, and the caches' pages taken,
given back, forked and copied.

``run`` computes a case in its plain form (elementary torch operations; the probabilities in 64 bits,
since a draw next to a border of two tokens decides a whole number) or, with ``own`` set, through
chain_flow_b200's public entry points. ``exact`` is the same from the definition in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}
VOCAB, SHORTLIST = 248320, 62642


def listed():
    return [
        # one request, a chain of five drafts: the latency of a step's verification
        dict(name="sample_chain_one", op="sample", requests=1, width=1, depth=5, vocab=VOCAB, dtype="bf16", accept=0.8,
             temp="one", keep=0),
        # one request, a tree of 40 nodes under the committed token
        dict(name="sample_tree_one", op="sample", requests=1, width=10, depth=4, vocab=VOCAB, dtype="bf16", accept=0.8,
             temp="one", keep=0),
        # a serving batch of such trees
        dict(name="sample_tree_batch", op="sample", requests=64, width=10, depth=4, vocab=VOCAB, dtype="bf16", accept=0.8,
             temp="mixed", keep=0),
        # fp32 logits of an odd vocabulary behind a top-k filter (-inf outside), greedy and sampling requests mixed
        dict(name="sample_filtered", op="sample", requests=17, width=3, depth=3, vocab=32003, dtype="fp32", accept=0.7,
             temp="mixed", keep=50),
        # one request's chain with the draft model's probabilities over a shortlist
        dict(name="reject_one", op="reject", requests=1, drafts=5, vocab=VOCAB, shortlist=SHORTLIST, dtype="bf16", temp="one"),
        # a batch of chains with probabilities over the whole vocabulary
        dict(name="reject_batch", op="reject", requests=48, drafts=5, vocab=VOCAB, shortlist=0, dtype="fp16", temp="mixed"),
        # one request's accepted nodes moved together in the caches of eight layers (4B target's heads)
        dict(name="keep_one", op="keep", requests=1, nodes=40, depth=5, context=500, layers=8, kv_heads=4, dim=256, page=16,
             cache="bf16"),
        # a batch's, quantised caches
        dict(name="keep_batch", op="keep", requests=64, nodes=40, depth=5, context=500, layers=8, kv_heads=4, dim=256, page=16,
             cache="fp8"),
        # a scheduler's step: finished requests give their pages back, new prompts and growing requests take theirs
        dict(name="pages_step", op="pages", requests=256, pages=65536, length=4000, page=16),
        # eight samples of one long prompt: full pages shared, the last one copied in eight layers
        dict(name="fork_samples", op="fork", parents=1, children=8, length=9001, layers=8, kv_heads=4, dim=256, page=16,
             cache="bf16"),
        # samples of a batch of prompts, quantised caches
        dict(name="fork_batch", op="fork", parents=16, children=4, length=1500, layers=8, kv_heads=8, dim=128, page=48,
             cache="fp8"),
        # pages moved for good: the contexts of a batch copied to other pages of the pool
        dict(name="copy_pages", op="copy", count=2048, page=16, layers=4, kv_heads=4, dim=256, cache="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["sample", "sample", "reject", "keep", "pages", "fork", "copy"])
    heads, dim = rng.choice([(4, 256), (2, 256), (8, 128), (1, 64), (3, 64)])
    pool = dict(kv_heads=heads, dim=dim, page=rng.choice([16, 17, 32, 48, 64]), layers=rng.randint(1, 8),
                cache=rng.choice(["fp8", "fp16", "bf16"]))
    if op in ("sample", "reject"):
        vocab, dtype = rng.choice([VOCAB, 32000, 32003, _log_int(rng, 1000, VOCAB)]), rng.choice(["fp16", "bf16", "fp32"])
        temp = rng.choice(["one", "mixed"])
        if op == "reject":
            return dict(op=op, requests=_log_int(rng, 1, 48), drafts=rng.randint(1, 8), vocab=vocab, dtype=dtype, temp=temp,
                        shortlist=rng.choice([0, max(vocab // 4, 1)]))
        return dict(op=op, requests=_log_int(rng, 1, 32), width=rng.choice([1, 1, 2, 4, 10]), depth=rng.randint(1, 6),
                    vocab=vocab, dtype=dtype, accept=rng.choice([0.5, 0.8, 0.95]), temp=temp, keep=rng.choice([0, 0, 20, 200]))
    if op == "keep":
        depth = rng.randint(1, 8)
        return dict(op=op, requests=_log_int(rng, 1, 64), nodes=rng.randint(depth, 64), depth=depth, context=_log_int(rng, 1, 500), **pool)
    if op == "pages":
        requests = _log_int(rng, 1, 256)
        return dict(op=op, requests=requests, length=_log_int(rng, 1, 4000), pages=_log_int(rng, 64, 65536), page=rng.choice([16, 17, 48]))
    if op == "fork":
        length = _log_int(rng, 1, 9001)
        return dict(op=op, parents=max(1, min(_log_int(rng, 1, 16), 20000 // length)), children=_log_int(rng, 1, 8), length=length, **pool)
    return dict(op=op, count=_log_int(rng, 1, 2048 * 64 // pool["page"] // 8), **pool)


def _cumulative(lengths):
    cu = []
    for n in lengths:
        cu.append(n + (cu[-1] if cu else 0))
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


# ---- inputs -----------------------------------------------------------------------------------------
def _parents(case):
    """A request's tree: `depth` levels of `width` nodes; a node hangs below one of the first nodes of the level above."""
    w = case["width"]
    return [-1 if i < w else (i // w - 1) * w + (i % w) * (i % w) // (2 * w) for i in range(w * case["depth"])]


def _temperatures(case, h):
    """One number a request: 1, or mixed ones with greedy requests (0) among them."""
    if case["temp"] == "one":
        return None
    t = 0.4 + 1.1 * torch.rand(case["requests"], generator=h)
    t[::7] = 0
    return t


def _rows(n, vocab, dtype, g):
    """Logits of n rows: most tokens far below a few, as a language model's are."""
    x = torch.randn(n, vocab, device=DEV, generator=g, dtype=torch.float32 if dtype == torch.float32 else torch.bfloat16)
    return x.mul_(2.5).to(dtype)


def _prepare_sample(case, g, h):
    B, V, dt = case["requests"], case["vocab"], TYPES[case["dtype"]]
    par = _parents(case)
    n = len(par)
    logits = _rows(B * (n + 1), V, dt, g)
    token = torch.randint(V, (B, n), device=DEV, generator=g)
    temp = _temperatures(case, h)
    tau = torch.ones(B) if temp is None else torch.where(temp > 0, temp, torch.ones_like(temp))
    for node in range(-1, n):
        kids = [i for i in range(n) if par[i] == node]
        if kids:                                     # siblings carry different tokens
            token[:, kids] = (token[:, kids[:1]] + torch.arange(len(kids), device=DEV) * (V // len(kids))) % V
        row = logits[node + 1::n + 1]
        if case["keep"]:
            bound = row.float().topk(min(case["keep"], V), dim=1).values[:, -1:]
            row[row.float() < bound] = -math.inf
        if kids:                                     # together the children get `accept` of the row's mass
            t = tau.to(DEV)[:, None]
            rest = torch.logsumexp(row.float() / t, 1, keepdim=True)
            share = torch.tensor([2.0 ** -(k + 1) for k in range(len(kids))], device=DEV)
            want = rest + math.log(case["accept"] / (1 - case["accept"])) + torch.log(share / share.sum())
            row.scatter_(1, token[:, kids], (want * t).to(dt))
    return dict(logits=logits, cu_draft=_cumulative([n] * B), cu_sampled=_cumulative([n + 1] * B),
                tokens=token.flatten().int(), parents=torch.tensor(par * B, dtype=torch.int32, device=DEV),
                uniform=torch.rand(B * (n + 1), device=DEV, generator=g), temp=None if temp is None else temp.to(DEV),
                nodes=n, depth=case["depth"])


def _prepare_reject(case, g, h):
    B, K, V, R, dt = case["requests"], case["drafts"], case["vocab"], case["shortlist"], TYPES[case["dtype"]]
    logits = _rows(B * (K + 1), V, dt, g)
    temp = _temperatures(case, h)
    ids = torch.randperm(V, device=DEV, generator=g)[:R].sort().values if R else None
    if R:                                            # a shortlist holds the tokens that matter
        out = torch.ones(V, dtype=torch.bool, device=DEV)
        out[ids] = False
        logits[:, out] -= 3
    tau = torch.ones(B) if temp is None else torch.where(temp > 0, temp, torch.ones_like(temp))
    probs, token = [], []
    for b in range(B):                               # the draft model: the target's logits, off by a little
        x = logits[b * (K + 1):b * (K + 1) + K].float()
        x = x if ids is None else x[:, ids]
        x = (x + 0.7 * torch.randn(x.shape, device=DEV, generator=g)) / float(tau[b])
        p = torch.softmax(x, 1)
        t = torch.multinomial(p, 1, generator=g)[:, 0]
        probs.append(p)
        token.append(t if ids is None else ids[t])
    return dict(logits=logits, cu_draft=_cumulative([K] * B), cu_sampled=_cumulative([K + 1] * B), tokens=torch.cat(token).int(),
                probs=torch.cat(probs), ids=ids, uniform=torch.rand(B * K, device=DEV, generator=g),
                resample=torch.rand(B, device=DEV, generator=g), temp=None if temp is None else temp.to(DEV), drafts=K)


def _pools(case, pages, g):
    """The layers' key and value pools [pages, kv_heads, page, dim], and their scales where they are quantised."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    out = []
    for _ in range(case["layers"]):
        layer = {}
        for name in ("k", "v"):
            x = torch.randn(shape, device=DEV, generator=g, dtype=torch.bfloat16)
            layer[name] = (x * 100 if case["cache"] == "fp8" else x).to(TYPES[case["cache"]])
            layer[name + "_scale"] = torch.rand(shape[:3], device=DEV, generator=g) if case["cache"] == "fp8" else None
        out.append(layer)
    return out


def _path(n, depth, h):
    """An accepted path: increasing nodes of a tree of n, up to `depth` of them."""
    a = int(torch.randint(0, min(depth, n) + 1, (1,), generator=h))
    return sorted(torch.randperm(n, generator=h)[:a].tolist())


def _prepare_keep(case, g, h):
    B, n, depth = case["requests"], case["nodes"], case["depth"]
    base = [case["context"] - (7 * b) % max(1, case["context"] // 2) for b in range(B)]
    width = max(-(-(x + n) // case["page"]) for x in base)
    order = torch.randperm(B * width + 3, generator=h)
    paths = [_path(n, depth, h) for _ in range(B)]
    path = torch.full((B, depth), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    return dict(layers=_pools(case, B * width + 3, g), table=order[:B * width].view(B, width).int().to(DEV),
                base=torch.tensor(base, dtype=torch.int32, device=DEV), path=path.to(DEV),
                count=torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV), depth=depth)


def _pages_lengths(case):
    """(positions kept, positions that pages are held for) of every request: the case's own, whatever the seed. A quarter of
    the requests has ended and makes room for new prompts; the others give back what was taken for refused drafts, and take
    as much for the next ones."""
    B, rng = case["requests"], random.Random(case["requests"] * 1000003 + case["length"])
    mean = max(1, min(case["length"], case["pages"] * case["page"] // (2 * B)))
    left = [0 if b % 4 == 0 else rng.randint(0, 2 * mean - 1) for b in range(B)]
    held = [rng.randint(1, 2 * mean - 1) if b % 4 == 0 else left[b] + rng.choice([1, 5, case["page"], 40]) for b in range(B)]
    return left, held


def _prepare_pages(case, g, h):
    left, held = _pages_lengths(case)
    page, B = case["page"], case["requests"]
    width = max(-(-n // page) for n in held)
    order = torch.randperm(case["pages"], generator=h, dtype=torch.int32)
    refs = torch.zeros(case["pages"], dtype=torch.int32)
    table = torch.full((B, width), -1, dtype=torch.int32)
    at = 0
    for b, x in enumerate(held):
        n = min(-(-x // page), case["pages"] - at)
        table[b, :n] = order[at:at + n]
        refs[order[at:at + n].long()] = 1
        at += n
    return dict(refs=refs.to(DEV), table=table.to(DEV), held=torch.tensor(held, dtype=torch.int32, device=DEV),
                left=torch.tensor(left, dtype=torch.int32, device=DEV))


def _prepare_fork(case, g, h):
    P, C, L, page = case["parents"], case["children"], case["length"], case["page"]
    lens = [max(1, L - (L // 5) * (p % 4) - p % 3) for p in range(P)]
    width = -(-max(lens) // page)
    used = sum(-(-n // page) for n in lens)
    pages = used + P * C + 5
    order = torch.randperm(pages, generator=h, dtype=torch.int32)
    rows = P + P * C
    table = torch.full((rows, width), -1, dtype=torch.int32)
    refs = torch.zeros(pages, dtype=torch.int32)
    at = 0
    for p, n in enumerate(lens):
        m = -(-n // page)
        table[p, :m] = order[at:at + m]
        refs[order[at:at + m].long()] = 1
        at += m
    length = torch.tensor(lens + [0] * (P * C), dtype=torch.int32)
    return dict(layers=_pools(case, pages, g), refs=refs.to(DEV), table=table.to(DEV), length=length.to(DEV),
                parent=torch.arange(P, dtype=torch.int32, device=DEV).repeat_interleave(C),
                child=torch.arange(P, rows, dtype=torch.int32, device=DEV), zero=torch.zeros(rows, dtype=torch.int32, device=DEV),
                was=torch.tensor([0] * P + [n for n in lens for _ in range(C)], dtype=torch.int32, device=DEV))


def _prepare_copy(case, g, h):
    n = case["count"]
    order = torch.randperm(2 * n + 1, generator=h, dtype=torch.int32).to(DEV)
    return dict(layers=_pools(case, 2 * n + 1, g), src=order[:n], dst=order[n:2 * n])


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    make = dict(sample=_prepare_sample, reject=_prepare_reject, keep=_prepare_keep, pages=_prepare_pages, fork=_prepare_fork,
                copy=_prepare_copy)[case["op"]]
    s = dict(make(case, g, h), case=case)
    if own:                                          # what a program keeps: the verifier, the caches' and the pool's handles
        from chain_flow_b200.kv_cache import PagedKVCache, PagePool
        from chain_flow_b200.tree import RejectionVerifier, SampledVerifier
        if case["op"] == "sample":
            s["verifier"] = SampledVerifier(len(s["logits"]), case["requests"], s["nodes"])
        elif case["op"] == "reject":
            s["verifier"] = RejectionVerifier(len(s["logits"]), case["requests"], case["drafts"], case["vocab"], draft_ids=s["ids"])
        if "layers" in s:
            s["caches"] = [PagedKVCache.from_tensors(x["k"], x["v"], x["k_scale"], x["v_scale"]) for x in s["layers"]]
        if "refs" in s:
            s["pool"] = PagePool.from_refs(s["refs"], case["page"])
    return s


# ---- the plain forms --------------------------------------------------------------------------------
def _weights(row, tau):
    """(weights of the rows' tokens, the rows' largest, rows that take their argmax) in 64 bits."""
    x = row.double()
    top = x.amax(1, keepdim=True)
    greedy = (tau < 2.0 ** -126) | torch.isnan(top[:, 0])
    t = torch.where(tau < 2.0 ** -126, torch.ones_like(tau), tau).double()[:, None]
    w = torch.exp((x - top) / t)
    w = torch.where(x == top, torch.ones_like(w), torch.where(torch.isfinite(top), w, torch.zeros_like(w)))
    return torch.where(x == -math.inf, torch.zeros_like(w), w), top, t, greedy


def _pick(w, u):
    """The first index at which the running sum of w passes u times the whole."""
    c = torch.cumsum(w, 1)
    return (c <= u.double()[:, None] * c[:, -1:]).sum(1).clamp_max(w.shape[1] - 1)


def _log_prob(row, w, top, t, token):
    x = row.gather(1, token.clamp_min(0)[:, None]).double()
    lp = torch.where(x == top, torch.zeros_like(x), (x - top) / t) - torch.log(w.sum(1, keepdim=True))
    return lp[:, 0].float()


def _tau(s, B):
    return torch.ones(B, device=DEV) if s["temp"] is None else s["temp"]


def _plain_sample(s):
    B, n = s["case"]["requests"], s["nodes"]
    cu = s["cu_sampled"].long()
    first = cu - (n + 1)
    tau = _tau(s, B)
    tokens, parents = s["tokens"].view(B, n), s["parents"].view(B, n)
    out = torch.full((B, n + 1), -1, dtype=torch.int32, device=DEV)
    path = torch.full((B, n), -1, dtype=torch.int32, device=DEV)
    logp = torch.zeros(B, n + 1, device=DEV)
    count = torch.zeros(B, dtype=torch.int32, device=DEV)
    node = torch.full((B,), -1, dtype=torch.int64, device=DEV)
    live = torch.ones(B, dtype=torch.bool, device=DEV)
    at = torch.arange(n, device=DEV)
    for level in range(s["depth"] + 1):
        row = s["logits"][first + node + 1]
        w, top, t, greedy = _weights(row, tau)
        token = torch.where(greedy, row.argmax(1), _pick(w, s["uniform"][first + node + 1]))
        token = torch.where(top[:, 0] == -math.inf, torch.full_like(token, -1), token)
        lp = _log_prob(row, w, top, t, token)
        out[:, level] = torch.where(live, token, torch.full_like(token, -1)).int()
        logp[:, level] = torch.where(live & (token >= 0), lp, torch.zeros_like(lp))
        hit = (parents == node[:, None]) & (tokens == token[:, None]) & live[:, None]
        kid = torch.where(hit, at, n).amin(1)
        live = kid < n
        if level < n:
            path[:, level] = torch.where(live, kid, torch.full_like(kid, -1)).int()
        count += live
        node = torch.where(live, kid, node)
    return out, path, count, logp


def _draft_row(s, rows):
    """The draft probabilities of the drafts `rows`, over the whole vocabulary, in 64 bits."""
    p = s["probs"][rows].double()
    p = torch.where(p > 0, p, torch.zeros_like(p))
    if s["ids"] is None:
        return p
    full = torch.zeros(len(p), s["case"]["vocab"], dtype=torch.float64, device=DEV)
    full[:, s["ids"]] = p
    return full


def _plain_reject(s):
    B, K = s["case"]["requests"], s["drafts"]
    first, d0 = s["cu_sampled"].long() - (K + 1), s["cu_draft"].long() - K
    tau = _tau(s, B)
    out = torch.full((B, K + 1), -1, dtype=torch.int32, device=DEV)
    logp = torch.zeros(B, K + 1, device=DEV)
    count = torch.zeros(B, dtype=torch.int32, device=DEV)
    live = torch.ones(B, dtype=torch.bool, device=DEV)
    for i in range(K + 1):
        row = s["logits"][first + i]
        w, top, t, greedy = _weights(row, tau)
        best = row.argmax(1)
        if i < K:
            draft = s["tokens"][d0 + i].long()
            q = _draft_row(s, d0 + i)
            p = w / w.sum(1, keepdim=True)
            pd, qd = (x.gather(1, draft[:, None])[:, 0] for x in (p, q))
            accept = torch.where(greedy, best == draft, s["uniform"][d0 + i].double() * qd < pd)
            rest = (p - q).clamp_min(0)
            rest = torch.where(rest.sum(1, keepdim=True) > 0, rest, p)
            other = torch.where(greedy, best, _pick(rest, s["resample"]))
            token = torch.where(accept, draft, other)
        else:
            accept = torch.zeros_like(live)
            token = torch.where(greedy, best, _pick(w, s["resample"]))
        token = torch.where(top[:, 0] == -math.inf, torch.full_like(token, -1), token)
        lp = _log_prob(row, w, top, t, token)
        out[:, i] = torch.where(live, token, torch.full_like(token, -1)).int()
        logp[:, i] = torch.where(live & (token >= 0), lp, torch.zeros_like(lp))
        live = live & accept
        count += live
    return out, count, logp


def _pool_outputs(s):
    return [[x[n] for n in ("k", "v", "k_scale", "v_scale") if x[n] is not None] for x in s["layers"]]


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _plain_keep(s):
    page, depth = s["case"]["page"], s["depth"]
    j = torch.arange(depth, device=DEV)
    src, dst = s["base"][:, None] + s["path"], (s["base"][:, None] + j).expand(-1, depth)
    live = j < s["count"][:, None]
    dst = torch.where(live, dst, s["base"][:, None])
    src = torch.where(live & (s["path"] >= 0), src, dst)          # a row that stays is written with itself
    at = lambda x: (s["table"].gather(1, (x // page).long()).long().flatten(), (x % page).long().flatten())  # noqa: E731
    (sp, so), (dp, do) = at(src), at(dst)
    moves = live.flatten().nonzero()[:, 0]
    sp, so, dp, do = sp[moves], so[moves], dp[moves], do[moves]
    for x in s["layers"]:
        for t in x.values():
            if t is not None:
                _bytes(t)[dp, :, do] = _bytes(t)[sp, :, so]
    return _pool_outputs(s)


def _ceil(x, page):
    return (x.clamp_min(0).long() + page - 1) // page


def _plain_reserve(refs, table, h, w):
    """Pages [h, w) of every request from the lowest free ones, in order; (granted) per request."""
    need = (w - h).clamp_min(0)
    total = torch.cumsum(need, 0)
    free = refs == 0
    granted = (need == 0) | (total <= free.sum())
    low = torch.argsort((~free).int(), stable=True)               # free pages first, each kind in order
    j = torch.arange(table.shape[1], device=DEV)
    mine = (j >= h[:, None]) & (j < w[:, None]) & granted[:, None]
    rank = (total - need)[:, None] + j - h[:, None]
    page = low[rank.clamp(0, len(refs) - 1)]
    table.copy_(torch.where(mine, page.int(), table))
    taken = torch.zeros(len(refs) + 1, dtype=torch.int32, device=DEV)
    taken[torch.where(mine, page, len(refs)).flatten()] = 1
    refs += taken[:-1]
    return granted


def _plain_release(refs, table, k, h):
    j = torch.arange(table.shape[1], device=DEV)
    mine = (j >= k[:, None]) & (j < h[:, None]) & (table >= 0)
    drop = torch.zeros(len(refs) + 1, dtype=torch.int32, device=DEV)
    drop.scatter_add_(0, torch.where(mine, table, len(refs)).flatten().long(), torch.ones_like(table).flatten())
    refs -= drop[:-1]
    table.copy_(torch.where((j >= k[:, None]) & (j < h[:, None]), torch.full_like(table, -1), table))


def _plain_pages(s):
    left, held = _ceil(s["left"], s["case"]["page"]), _ceil(s["held"], s["case"]["page"])
    _plain_release(s["refs"], s["table"], left, held)
    granted = _plain_reserve(s["refs"], s["table"], left, held)
    return s["table"], s["refs"], granted.int()


def _plain_copy(s, src, dst, slots):
    """Leading slots of pages src to pages dst, in every layer."""
    live = torch.arange(s["case"]["page"], device=DEV) < slots[:, None]
    for x in s["layers"]:
        for t in x.values():
            if t is not None:
                b = _bytes(t)
                m = live[:, None, :] if t.dim() == 3 else live[:, None, :, None]
                b[dst] = torch.where(m, b[src], b[dst])


def _plain_fork(s):
    page = s["case"]["page"]
    # the children of the last pass end
    _plain_release(s["refs"], s["table"], _ceil(s["zero"], page), _ceil(s["was"], page))
    L = s["length"][s["parent"].long()]
    full, part = (L // page).long(), L % page
    rows = s["table"][s["parent"].long()]
    need = torch.where(part > 0, full + 1, full)
    mine = s["table"][s["child"].long()]
    granted = _plain_reserve(s["refs"], mine, full, need)
    j = torch.arange(rows.shape[1], device=DEV)
    shared = (j < full[:, None]) & granted[:, None] & (rows >= 0)
    more = torch.zeros(len(s["refs"]) + 1, dtype=torch.int32, device=DEV)
    more.scatter_add_(0, torch.where(shared, rows, len(s["refs"])).flatten().long(), torch.ones_like(rows).flatten())
    s["refs"] += more[:-1]
    mine = torch.where(shared, rows, mine)
    s["table"][s["child"].long()] = mine
    s["length"][s["child"].long()] = torch.where(granted, L, s["length"][s["child"].long()])
    cut = ((part > 0) & granted).nonzero()[:, 0]
    at = full[cut][:, None]
    _plain_copy(s, rows[cut].gather(1, at)[:, 0].long(), mine[cut].gather(1, at)[:, 0].long(), part[cut])
    return s["table"], s["length"], s["refs"], granted.int(), _pool_outputs(s)


def _plain_copy_pages(s):
    for x in s["layers"]:
        for t in x.values():
            if t is not None:
                _bytes(t)[s["dst"].long()] = _bytes(t)[s["src"].long()]
    return _pool_outputs(s)


# ---- the framework's own ----------------------------------------------------------------------------
def _own(s):
    op = s["case"]["op"]
    if op == "sample":
        out, path, count, logp = s["verifier"](s["logits"], s["cu_draft"], s["cu_sampled"], s["tokens"], s["parents"], s["uniform"],
                                               temperature=s["temp"])
        return out, path, count, logp
    if op == "reject":
        return s["verifier"](s["logits"], s["cu_draft"], s["cu_sampled"], s["tokens"], s["probs"], s["uniform"], s["resample"],
                             temperature=s["temp"])
    from chain_flow_b200.kv_cache import copy_pages, keep_path
    if op == "keep":
        keep_path(s["caches"], s["table"], s["base"], s["path"], s["count"])
        return _pool_outputs(s)
    if op == "copy":
        copy_pages(s["caches"], s["src"], s["dst"])
        return _pool_outputs(s)
    if op == "pages":
        s["pool"].release(s["table"], s["held"], s["left"])
        granted = s["pool"].reserve(s["table"], s["left"], s["held"])
        return s["table"], s["refs"], granted
    s["pool"].release(s["table"], s["was"])                       # the children of the last pass end
    granted = s["pool"].fork(s["table"], s["length"], s["parent"], s["child"], s["caches"])
    return s["table"], s["length"], s["refs"], granted, _pool_outputs(s)


def run(state):
    if own:
        return _own(state)
    plain = dict(sample=_plain_sample, reject=_plain_reject, keep=_plain_keep, pages=_plain_pages, fork=_plain_fork,
                 copy=_plain_copy_pages)
    return plain[state["case"]["op"]](state)


# ---- the definitions in 64 bits ---------------------------------------------------------------------
def _exact_row(row, tau):
    """(probabilities, log-probabilities) of one row of finite or masked logits, and whether it takes its argmax."""
    x = row.to(torch.float64)
    greedy = tau < 2.0 ** -126
    lp = torch.log_softmax(x if greedy else x / tau, 0)
    return lp.exp(), lp, greedy


def _exact_pick(p, u):
    c = p.cumsum(0)
    return int(torch.searchsorted(c, c[-1:] * u, right=True)[0])


def exact(case, seed):
    if case["op"] in ("keep", "fork", "copy", "pages"):
        return None                                               # copies and indices: no computed numbers
    s = prepare(case, seed)
    B = case["requests"]
    tau = [1.0] * B if s["temp"] is None else s["temp"].tolist()
    if case["op"] == "sample":
        n, par = s["nodes"], _parents(case)
        tokens, u = s["tokens"].view(B, n).tolist(), s["uniform"].tolist()
        out, path = torch.full((B, n + 1), -1), torch.full((B, n), -1)
        logp, count = torch.zeros(B, n + 1, dtype=torch.float64), torch.zeros(B, dtype=torch.int64)
        for b in range(B):
            node, pos = -1, 0
            while True:
                r = b * (n + 1) + node + 1
                p, lp, greedy = _exact_row(s["logits"][r], tau[b])
                t = int(s["logits"][r].argmax()) if greedy else _exact_pick(p, u[r])
                out[b, pos], logp[b, pos] = t, float(lp[t])
                kids = [i for i in range(n) if par[i] == node and tokens[b][i] == t]
                if not kids:
                    break
                node = kids[0]
                path[b, pos] = node
                pos += 1
            count[b] = pos
        return out, path, count, logp
    K = case["drafts"]
    tokens, u, v = s["tokens"].tolist(), s["uniform"].tolist(), s["resample"].tolist()
    out, count = torch.full((B, K + 1), -1), torch.zeros(B, dtype=torch.int64)
    logp = torch.zeros(B, K + 1, dtype=torch.float64)
    for b in range(B):
        for i in range(K + 1):
            row = s["logits"][b * (K + 1) + i]
            p, lp, greedy = _exact_row(row, tau[b])
            if i == K:
                t = int(row.argmax()) if greedy else _exact_pick(p, v[b])
            else:
                d = tokens[b * K + i]
                q = torch.zeros_like(p)
                q[slice(None) if s["ids"] is None else s["ids"]] = s["probs"][b * K + i].to(torch.float64)
                if int(row.argmax()) == d if greedy else u[b * K + i] * float(q[d]) < float(p[d]):
                    t = d
                elif greedy:
                    t = int(row.argmax())
                else:
                    t = _exact_pick(torch.relu(p - q), v[b])
            out[b, i], logp[b, i] = t, float(lp[t])
            if i == K or t != tokens[b * K + i]:
                break
            count[b] += 1
    return out, count, logp


# ---- what a pass cannot do without ------------------------------------------------------------------
def work(case):
    op = case["op"]
    size = 4 if case.get("dtype") == "fp32" else 2
    if op == "sample":
        # the rows that the walk is expected to reach: a node's children are taken by `accept`, each by half of the one before
        par = _parents(case)
        reach = [1.0] + [0.0] * len(par)
        for node in range(-1, len(par)):
            kids = [i for i in range(len(par)) if par[i] == node]
            for k, i in enumerate(kids):
                reach[i + 1] = reach[node + 1] * case["accept"] * 2.0 ** -(k + 1) / (1 - 2.0 ** -len(kids))
        rows = case["requests"] * sum(reach)
        return dict(bytes=rows * case["vocab"] * size, flops=4 * rows * case["vocab"])
    if op == "reject":
        # drafts accepted seven times in ten, then the refusing row's draft probabilities
        rows = case["requests"] * sum(0.7 ** i for i in range(case["drafts"] + 1))
        refused = case["requests"] * (1 - 0.7 ** case["drafts"])
        return dict(bytes=rows * case["vocab"] * size + refused * 4 * (case["shortlist"] or case["vocab"]),
                    flops=4 * (rows + refused) * case["vocab"])
    if op == "pages":
        # every count read; of the pages given back and taken, the table's entries and the counts
        moved = sum(-(-h // case["page"]) - -(-k // case["page"]) for k, h in zip(*_pages_lengths(case)))
        return dict(bytes=4 * (case["pages"] + 6 * moved), flops=0)
    row = 2 * case["kv_heads"] * (case["dim"] + 4 if case["cache"] == "fp8" else 2 * case["dim"]) * case["layers"]
    if op == "keep":
        return dict(bytes=2 * row * case["requests"] * min(case["depth"], case["nodes"]) / 2, flops=0)
    if op == "copy":
        return dict(bytes=2 * row * case["count"] * case["page"], flops=0)
    forks = case["parents"] * case["children"]
    return dict(bytes=2 * row * forks * (case["page"] / 2) + forks * 3 * 4 * (case["length"] // case["page"]), flops=0)

"""Performance cases of the target-side operators: the paged key/value cache (written, quantised,
read back), attention of new tokens over it, and the gated delta rule over prompts (chunked) and
single tokens (recurrent).

``run`` computes a case in its plain form (elementary torch operations, fp32, rounded once at the
end) or, with ``own`` set, through chain_flow_b200's public entry points. ``exact`` is the same from
the definition in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp8": torch.float8_e4m3fn}


def listed():
    return [
        # the K/V rows of one decode step of 64 requests, quantised into the cache (4B target's heads)
        dict(name="write_decode", op="write", tokens=64, kv_heads=4, dim=256, page=16, dtype="bf16", cache="fp8"),
        # a scheduler step's worth of prompt tokens, quantised
        dict(name="write_prompt", op="write", tokens=8192, kv_heads=4, dim=256, page=16, dtype="fp16", cache="fp8"),
        # a request's context read back to 16 bits (moved to another engine, re-quantised, inspected)
        dict(name="read_context", op="read", tokens=20001, kv_heads=8, dim=128, page=48, dtype="bf16", cache="fp8"),
        # one request, one new token: the latency of a plain decode step (4B target's heads)
        dict(name="attn_decode_one", op="attn", requests=1, new=1, context=9001, heads=16, kv_heads=4, dim=256, page=16,
             dtype="bf16", cache="bf16", causal=True, ragged=False),
        # a batch of decoding requests of mixed lengths over a quantised cache
        dict(name="attn_decode_batch", op="attn", requests=48, new=1, context=8192, heads=16, kv_heads=4, dim=256, page=16,
             dtype="bf16", cache="fp8", causal=True, ragged=True),
        # the tree verify's prefix attention: 41 rows of a draft tree per request, no mask (27B target's heads)
        dict(name="attn_tree_prefix", op="attn", requests=4, new=41, context=4000, heads=24, kv_heads=4, dim=256, page=16,
             dtype="fp16", cache="fp16", causal=False, ragged=False),
        # a long prompt's last chunk
        dict(name="attn_prompt_chunk", op="attn", requests=1, new=2048, context=16384, heads=16, kv_heads=4, dim=256, page=16,
             dtype="bf16", cache="bf16", causal=True, ragged=False),
        # several whole prompts of mixed lengths in one step, quantised cache, 128-wide heads
        dict(name="attn_prompts", op="attn", requests=5, new=1500, context=1500, heads=32, kv_heads=8, dim=128, page=48,
             dtype="fp16", cache="fp8", causal=True, ragged=True),
        # a long prompt through a gated-delta layer (4B target's heads)
        dict(name="gdn_prompt", op="gdn_chunk", requests=1, tokens=8191, heads=16, value_heads=32, vdim=128, dtype="bf16"),
        # a scheduler step of prompts of mixed lengths
        dict(name="gdn_prompts", op="gdn_chunk", requests=9, tokens=1500, heads=16, value_heads=32, vdim=128, dtype="fp16"),
        # one decoding request: latency
        dict(name="gdn_decode_one", op="gdn_step", requests=1, heads=16, value_heads=32, vdim=128, dtype="bf16"),
        # a batch of decoding requests: the states' bytes
        dict(name="gdn_decode_batch", op="gdn_step", requests=96, heads=16, value_heads=32, vdim=128, dtype="fp16"),
    ]


def _log_int(rng, lo, hi):
    n = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return n + 1 if n == 3072 and n < hi else n


def draw(rng):
    op = rng.choice(["write", "read", "attn", "attn", "gdn_chunk", "gdn_step"])
    dtype = rng.choice(["fp16", "bf16"])
    if op in ("write", "read"):
        kv_heads, dim = rng.choice([(4, 256), (2, 256), (8, 128), (1, 64), (8, 64), (3, 128)])
        tokens = _log_int(rng, 1, 20000 if op == "read" else 8192)
        return dict(op=op, tokens=tokens, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 17, 32, 48, 64]), dtype=dtype,
                    cache=rng.choice(["fp8", dtype]))
    if op == "attn":
        heads, kv_heads, dim = rng.choice([(16, 4, 256), (24, 4, 256), (32, 8, 128), (8, 8, 64), (28, 4, 128), (7, 1, 64), (16, 2, 256)])
        kind = rng.choice(["decode", "tree", "prompt", "chunk"])
        if kind == "decode":
            new, context, causal = 1, _log_int(rng, 1, 9001), True
            requests = min(_log_int(rng, 1, 48), max(1, 96000 // context))
        elif kind == "tree":
            requests, new, context, causal = _log_int(rng, 1, 8), rng.randint(2, 64), _log_int(rng, 16, 4000), False
        elif kind == "prompt":
            requests, new, causal = _log_int(rng, 1, 5), _log_int(rng, 2, 1500), True
            context = new
        else:
            requests, new, causal = 1, _log_int(rng, 16, 1500), True
            context = new + _log_int(rng, 16, 12000)
        return dict(op=op, requests=requests, new=new, context=context, heads=heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 17, 32, 48, 64]), dtype=dtype, cache=rng.choice(["fp8", dtype]), causal=causal,
                    ragged=rng.random() < 0.5)
    heads, value_heads = rng.choice([(16, 32), (16, 16), (4, 8), (8, 32), (3, 6)])
    vdim = rng.choice([128, 128, 64, 32])
    if op == "gdn_chunk":
        requests = _log_int(rng, 1, 9)
        return dict(op=op, requests=requests, tokens=_log_int(rng, 2, 1500 if requests > 1 else 6000), heads=heads,
                    value_heads=value_heads, vdim=vdim, dtype=dtype)
    return dict(op=op, requests=_log_int(rng, 1, 96), heads=heads, value_heads=value_heads, vdim=vdim, dtype=dtype)


def _lengths(case):
    """(new tokens, context length with them) of every request: the case's own, whatever the seed."""
    B, ragged = case["requests"], case.get("ragged", True)
    new, ctx = (case["new"], case["context"]) if case["op"] == "attn" else (case["tokens"], case["tokens"])
    if not ragged:
        return [new] * B, [ctx] * B
    rng = random.Random(B * 1000003 + new * 1009 + ctx)
    news = [new] + [rng.randint(1, new) for _ in range(B - 1)]
    return news, [ctx] + [n if new == ctx else rng.randint(min(n, ctx), ctx) for n in news[1:]]


def _cumulative(lengths):
    cu = [0]
    for n in lengths:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32, device=DEV)


def _quantised(x):
    """e4m3 codes and one fp32 scale per row of the last dim: what the cache's write makes of x."""
    x = x.float()
    amax = x.abs().amax(-1, keepdim=True)
    floor = amax.clamp_min(2.0 ** -24)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    scale = torch.where(bad, torch.full_like(amax, math.nan), floor / 448.0)
    code = torch.where(bad, torch.zeros_like(x), (x * torch.div(torch.full_like(floor, 448.0), floor)).clamp(-448.0, 448.0))
    return code.to(torch.float8_e4m3fn), scale.squeeze(-1)


def _pool(case, pages, g):
    """A cache pool [pages, kv_heads, page, dim] (and its scales) holding random rows."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.randn(shape, device=DEV, generator=g, dtype=torch.float32)
    if case["cache"] == "fp8":
        return _quantised(x.to(TYPES[case["dtype"]]))
    return x.to(TYPES[case["cache"]]), None


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    s = dict(case=case)
    if case["op"] in ("write", "read"):
        pages = -(-case["tokens"] // case["page"]) + 8
        slots = torch.randperm(pages * case["page"], device=DEV, generator=g)[:case["tokens"]]
        if case["tokens"] > 8:                       # padded rows of a step: skipped
            slots[case["tokens"] // 2] = -1
        s.update(slots=slots, pages=pages)
        s["k"], s["k_scale"] = _pool(case, pages, g)
        s["v"], s["v_scale"] = _pool(case, pages, g)
        if case["op"] == "write":
            # rows of a fused projection: strided views
            d, kv = case["dim"], case["kv_heads"]
            x = torch.randn(case["tokens"], 2 * kv, d, device=DEV, generator=g).to(TYPES[case["dtype"]])
            s["key"], s["value"] = x[:, :kv], x[:, kv:]
        return s
    if case["op"] == "attn":
        news, lens = _lengths(case)
        per = [-(-n // case["page"]) for n in lens]
        pages = sum(per) + 4
        order = torch.randperm(pages, generator=h, dtype=torch.int32)
        table = torch.zeros(len(lens), max(per), dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        s["k"], s["k_scale"] = _pool(case, pages, g)
        s["v"], s["v_scale"] = _pool(case, pages, g)
        s.update(table=table.to(DEV), kv_len=torch.tensor(lens, dtype=torch.int32, device=DEV), cu_q=_cumulative(news),
                 max_new=max(news), max_len=max(lens))
        q = torch.randn(sum(news), case["heads"], case["dim"], device=DEV, generator=g)
        s["q"] = (q * 1.5).to(TYPES[case["dtype"]])
        return s
    H, HV, V, K = case["heads"], case["value_heads"], case["vdim"], 128
    if case["op"] == "gdn_chunk":
        lens, _ = _lengths(case)
        s["cu"], s["max_tokens"] = _cumulative(lens), max(lens)
    else:
        lens = [1] * case["requests"]
    T, B = sum(lens), len(lens)
    dt = TYPES[case["dtype"]]
    s["q"] = torch.randn(T, H, K, device=DEV, generator=g).to(dt)
    s["k"] = torch.randn(T, H, K, device=DEV, generator=g).to(dt)
    s["v"] = torch.randn(T, HV, V, device=DEV, generator=g).to(dt)
    s["a"] = torch.randn(T, HV, device=DEV, generator=g).to(dt)
    s["b"] = torch.randn(T, HV, device=DEV, generator=g).to(dt)
    # decays of a trained layer: exp(A_log) in [1, 16], the step size's bias log-uniform in [0.001, 0.1]
    s["A_log"] = torch.log(1 + 15 * torch.rand(HV, device=DEV, generator=g))
    step = torch.exp(math.log(1e-3) + (math.log(1e-1) - math.log(1e-3)) * torch.rand(HV, device=DEV, generator=g))
    s["dt_bias"] = step + torch.log(-torch.expm1(-step))
    slots = B + 3
    s["state"] = torch.randn(slots, HV, V, K, device=DEV, generator=g) * 0.1
    order = torch.randperm(slots, generator=h, dtype=torch.int32)[:B]
    init = order.clone()
    if B > 1:
        init[B // 2] = -1                            # a request that starts here: zero state
    s.update(init=init.to(DEV), kept=order.to(DEV), scale=K ** -0.5)
    s["o"] = torch.empty(T, HV, V, device=DEV, dtype=dt)
    s["out_state"] = torch.zeros_like(s["state"])
    return s


# ---- the plain forms ------------------------------------------------------------------------------
def _plain_write(s):
    case = s["case"]
    keep = (s["slots"] >= 0).nonzero().squeeze(1)
    slot = s["slots"][keep]
    page, at = slot // case["page"], slot % case["page"]
    out = {}
    for name in ("key", "value"):
        x, pool, scale = s[name][keep], s[name[0]], s[name[0] + "_scale"]
        if scale is None:
            pool[page, :, at] = x.to(pool.dtype)
        else:
            code, sc = _quantised(x)
            pool.view(torch.uint8)[page, :, at] = code.view(torch.uint8)
            scale[page, :, at] = sc
            out[name[0] + "_scale"] = scale
        out[name[0]] = pool
    return out


def _rows(s, name, slots):
    """The rows at `slots`, dequantised in fp32: [..., kv_heads, dim]."""
    page = s["case"]["page"]
    x = s[name].view(torch.uint8)[slots // page, :, slots % page].view(s[name].dtype) if s[name + "_scale"] is not None \
        else s[name][slots // page, :, slots % page]
    x = x.float()
    return x if s[name + "_scale"] is None else x * s[name + "_scale"][slots // page, :, slots % page][..., None]


def _plain_read(s):
    live = (s["slots"] >= 0)[:, None, None]
    at = s["slots"].clamp_min(0)
    dt = TYPES[s["case"]["dtype"]]
    return tuple(torch.where(live, _rows(s, n, at), torch.zeros((), device=DEV)).to(dt) for n in ("k", "v"))


def _padded(s, lmax):
    """(key slots of every request [B, lmax], token rows [B, max_new], live rows, allowed keys [B, max_new, lmax])."""
    page = s["case"]["page"]
    j = torch.arange(lmax, device=DEV)
    slots = s["table"].long()[:, j // page] * page + j % page
    n = (s["cu_q"][1:] - s["cu_q"][:-1]).long()[:, None]
    i = torch.arange(s["max_new"], device=DEV)[None]
    live = i < n
    rows = (s["cu_q"][:-1].long()[:, None] + i)
    length = s["kv_len"].long()[:, None, None]
    limit = length - n[..., None] + i[..., None] + 1 if s["case"]["causal"] else length.expand(-1, s["max_new"], 1)
    return slots, rows, live, j[None, None] < limit


def _plain_attn(s):
    case = s["case"]
    slots, rows, live, allowed = _padded(s, s["max_len"])
    rep = case["heads"] // case["kv_heads"]
    B, n = rows.shape
    T = s["q"].shape[0]
    q = s["q"].float()[rows.clamp_max(T - 1)].view(B, n, case["kv_heads"], rep, case["dim"]).permute(0, 2, 3, 1, 4)
    q = q.reshape(B, case["kv_heads"], rep * n, case["dim"])
    k = _rows(s, "k", slots).permute(0, 2, 3, 1)                     # [B, kv, dim, L]
    score = ((q @ k) * case["dim"] ** -0.5).view(B, case["kv_heads"], rep, n, -1)
    score = torch.where(allowed[:, None, None], score, torch.full((), -math.inf, device=DEV))
    top = score.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, torch.zeros_like(top))
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    lse = (top + torch.log(total)).squeeze(-1)
    v = _rows(s, "v", slots).permute(0, 2, 1, 3)
    p = torch.where(total > 0, p / total, torch.zeros_like(p))
    o = (p.view(B, case["kv_heads"], rep * n, -1) @ v).view(B, case["heads"], n, case["dim"])
    o = o.permute(0, 2, 1, 3)[live]
    return o.to(s["q"].dtype), lse.view(B, case["heads"], n).permute(0, 2, 1)[live].t().contiguous()


def _gates(s, f):
    """(decay, beta, normalised k, normalised scaled q, v) of every token, heads repeated for the value heads."""
    rep = s["case"]["value_heads"] // s["case"]["heads"]
    x = s["a"].to(f) + s["dt_bias"].to(f)
    decay = torch.exp(-torch.exp(s["A_log"].to(f)) * torch.where(x > 20, x, torch.log1p(torch.exp(x.clamp_max(20)))))
    beta = 1 / (1 + torch.exp(-s["b"].to(f)))
    q, k = s["q"].to(f), s["k"].to(f)
    k = (k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)).repeat_interleave(rep, 1)
    q = (q * (s["scale"] / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6))).repeat_interleave(rep, 1)
    return decay, beta, k, q, s["v"].to(f)


def _recurrent(s, f):
    """The recurrence token by token over all requests at once, in the type f: (o [T, HV, V], new states [B, HV, V, K])."""
    decay, beta, k, q, v = _gates(s, f)
    init = s["init"].long()
    S = torch.where((init >= 0)[:, None, None, None], s["state"].to(f)[init.clamp_min(0)], torch.zeros((), dtype=f, device=DEV))
    if s["case"]["op"] == "gdn_step":
        first, steps, count = torch.arange(len(init), device=DEV), 1, None
    else:
        first, steps, count = s["cu"][:-1].long(), s["max_tokens"], (s["cu"][1:] - s["cu"][:-1]).long()
    T = v.shape[0]
    out = torch.zeros(T + 1, *v.shape[1:], dtype=f, device=DEV)
    # a request that has ended takes steps of no decay and no update, and its outputs go to a spare row
    decay = torch.cat([decay, torch.ones_like(decay[:1])])
    beta = torch.cat([beta, torch.zeros_like(beta[:1])])
    k, q, v = (torch.cat([x, torch.zeros_like(x[:1])]) for x in (k, q, v))
    for i in range(steps):
        at = first + i if count is None else torch.where(count > i, first + i, T)
        kn = k[at][..., None]                                          # [B, HV, K, 1]
        S = S * decay[at][..., None, None]
        S = torch.addcmul(S, (beta[at][..., None] * (v[at] - (S @ kn).squeeze(-1)))[..., None], kn.transpose(-1, -2))
        out[at] = (S @ q[at][..., None]).squeeze(-1)
    return out[:T], S


def _plain_gdn(s):
    o, S = _recurrent(s, torch.float32)
    s["o"].copy_(o)
    s["out_state"][s["kept"].long()] = S
    return s["o"], s["out_state"]


# ---- the framework's own -----------------------------------------------------------------------------
def _own(s):
    from chain_flow_b200.attention import PagedAttention
    from chain_flow_b200.gdn import ChunkedGdn, gdn_step
    from chain_flow_b200.kv_cache import PagedKVCache
    case = s["case"]
    if case["op"] in ("write", "read", "attn") and "cache" not in s:      # kept by a program as long as its pool
        s["cache"] = PagedKVCache.from_tensors(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if case["op"] == "write":
        s["cache"].write(s["key"], s["value"], s["slots"])
        return {n: s[n] for n in ("k", "v", "k_scale", "v_scale") if s[n] is not None}
    if case["op"] == "read":
        return s["cache"].read(s["slots"], dtype=TYPES[case["dtype"]])
    if case["op"] == "attn":
        if "attention" not in s:
            s["attention"] = PagedAttention(case["heads"], case["kv_heads"], case["dim"])
        return s["attention"](s["q"], s["cache"], s["table"], s["kv_len"], s["cu_q"], causal=case["causal"])
    args = (s["A_log"], s["dt_bias"], s["a"], s["b"], s["q"], s["k"], s["v"], s["o"], s["state"])
    if case["op"] == "gdn_step":
        gdn_step(*args, s["init"], s["kept"], scale=s["scale"], out_state=s["out_state"])
    else:
        if "gdn" not in s:
            s["gdn"] = ChunkedGdn(s["q"].shape[0], case["requests"], case["value_heads"])
        s["gdn"](*args, s["cu"], s["init"], s["kept"], scale=s["scale"], out_state=s["out_state"])
    return s["o"], s["out_state"]


def run(state):
    if own:
        return _own(state)
    plain = {"write": _plain_write, "read": _plain_read, "attn": _plain_attn, "gdn_chunk": _plain_gdn, "gdn_step": _plain_gdn}
    return plain[state["case"]["op"]](state)


# ---- the definitions in 64 bits --------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "write":
        if case["cache"] != "fp8":
            return None                                  # a copy: no computed numbers
        out = {}
        keep = s["slots"] >= 0
        slot = s["slots"][keep]
        for name in ("key", "value"):
            x = s[name].to(f)[keep]
            sc = s[name[0] + "_scale"].to(f)
            sc[slot // case["page"], :, slot % case["page"]] = x.abs().max(-1).values.clamp_min(2.0 ** -24) / 448
            out[name[0]], out[name[0] + "_scale"] = None, sc
        return out

    def values(name):
        x = s[name].to(torch.float32).to(f)
        return x if s[name + "_scale"] is None else x * s[name + "_scale"].to(f).unsqueeze(-1)

    def flat(name):                                      # [slot, kv head, dim]
        return values(name).transpose(1, 2).flatten(0, 1)

    if case["op"] == "read":
        out = []
        for name in ("k", "v"):
            x = flat(name)[s["slots"].clamp_min(0)]
            x[s["slots"] < 0] = 0
            out.append(x)
        return tuple(out)
    if case["op"] == "attn":
        k, v = flat("k"), flat("v")
        rep, page = case["heads"] // case["kv_heads"], case["page"]
        out = torch.zeros(s["q"].shape, dtype=f, device=DEV)
        lse = torch.full((case["heads"], s["q"].shape[0]), -math.inf, dtype=f, device=DEV)
        cu, lens = s["cu_q"].tolist(), s["kv_len"].tolist()
        for b, length in enumerate(lens):
            j = torch.arange(length, device=DEV)
            slot = s["table"][b].long()[j // page] * page + j % page
            n = cu[b + 1] - cu[b]
            last = length - n + torch.arange(n, device=DEV) if case["causal"] else torch.full((n,), length - 1, device=DEV)
            for h in range(case["heads"]):
                kh, vh = k[slot, h // rep], v[slot, h // rep]
                w = (s["q"][cu[b]:cu[b + 1], h].to(f) @ kh.T) / math.sqrt(case["dim"])
                w.masked_fill_(j[None] > last[:, None], -math.inf)
                lse[h, cu[b]:cu[b + 1]] = torch.logsumexp(w, -1)
                out[cu[b]:cu[b + 1], h] = torch.nan_to_num(torch.softmax(w, -1)) @ vh
        return out, lse
    return _exact_gdn(s, case)


def _exact_gdn(s, case):
    f = torch.float64
    rep = case["value_heads"] // case["heads"]
    g = -torch.exp(s["A_log"].to(f)) * torch.nn.functional.softplus(s["a"].to(f) + s["dt_bias"].to(f))
    alpha, beta = torch.exp(g), torch.sigmoid(s["b"].to(f))
    norm = lambda x: x * torch.rsqrt(x.square().sum(-1, keepdim=True) + 1e-6)  # noqa: E731
    k = norm(s["k"].to(f)).repeat_interleave(rep, 1)
    q = norm(s["q"].to(f)).repeat_interleave(rep, 1) * s["scale"]
    v = s["v"].to(f)
    out = torch.zeros(v.shape, dtype=f, device=DEV)
    states = torch.zeros(s["state"].shape, dtype=f, device=DEV)
    B = case["requests"]
    cu = s["cu"].tolist() if case["op"] == "gdn_chunk" else list(range(B + 1))
    init, kept = s["init"].tolist(), s["kept"].tolist()
    # the requests' states side by side, longest first, so that step i touches a leading block of them
    order = sorted(range(B), key=lambda b: cu[b] - cu[b + 1])
    S = torch.stack([s["state"][init[b]].to(f) if init[b] >= 0 else torch.zeros_like(states[0]) for b in order])
    first = torch.tensor([cu[b] for b in order], device=DEV)
    lens = [cu[b + 1] - cu[b] for b in order]
    for i in range(lens[0]):
        m = sum(n > i for n in lens)
        t = first[:m] + i
        A = S[:m].mul_(alpha[t][..., None, None])
        miss = (v[t] - torch.einsum("bhvk,bhk->bhv", A, k[t])) * beta[t][..., None]
        A.add_(torch.einsum("bhv,bhk->bhvk", miss, k[t]))
        out[t] = torch.einsum("bhvk,bhk->bhv", A, q[t])
    for x, b in enumerate(order):
        states[kept[b]] = S[x]
    return out, states


# ---- what a pass cannot do without ----------------------------------------------------------------
def work(case):
    if case["op"] in ("write", "read"):
        rows = 2 * case["tokens"] * case["kv_heads"]
        row = case["dim"] * 2 + (case["dim"] + 4 if case["cache"] == "fp8" else case["dim"] * 2)
        return dict(bytes=rows * row + 8 * case["tokens"], flops=rows * case["dim"])
    if case["op"] == "attn":
        sets = list(zip(*_lengths(case)))
        pairs = sum(n * (c - (n - 1) / 2) if case["causal"] else n * c for n, c in sets)
        row = 2 * case["kv_heads"] * (case["dim"] + 4 if case["cache"] == "fp8" else case["dim"] * 2)
        tokens = sum(n for n, _ in sets)
        return dict(bytes=row * sum(c for _, c in sets) + tokens * case["heads"] * (case["dim"] * 4 + 4),
                    flops=4 * case["dim"] * case["heads"] * pairs)
    H, HV, V, K, B = case["heads"], case["value_heads"], case["vdim"], 128, case["requests"]
    T = B if case["op"] == "gdn_step" else sum(_lengths(case)[0])
    states = B * 2 - (B > 1)
    return dict(bytes=T * (2 * H * K * 2 + 2 * HV * V * 2 + 4 * HV) + states * HV * V * K * 4, flops=7 * K * V * HV * T)

"""Oracle: drafted tokens verified against the target's probabilities from given random numbers (64 bits, CPU, test
infrastructure)."""
from __future__ import annotations

import math

import torch


def row_weights(row, tau: float):
    """(weights of a logits row's tokens relative to its largest, log of their sum, the row takes its argmax) at
    temperature tau: (w, log_z, greedy); w is None where nothing has mass."""
    x = row.double()
    greedy = not tau >= 2.0 ** -126
    if bool(torch.isnan(x).any()):
        return None, math.nan, True
    top = x.max()
    if top == -math.inf:
        return None, math.nan, greedy
    t = 1.0 if greedy else min(tau, 2.0 ** 100)
    w = (x == top).double() if top == math.inf else torch.exp((x - top) / t)
    return w, math.log(float(w.sum())), greedy


def number(u) -> float:
    u = float(u)
    return 0.0 if math.isnan(u) else min(max(u, 0.0), 1 - 2.0 ** -32)


def draw(w, u) -> int:
    """The first token at which the running sum of w passes u of the whole."""
    c = torch.cumsum(w, 0)
    over = (c > number(u) * c[-1]).nonzero()
    return int(over[0]) if len(over) else int((w > 0).nonzero()[-1])


def log_prob(row, tau: float, token: int) -> float:
    w, log_z, greedy = row_weights(row, tau)
    if w is None:
        return math.nan
    x, top = float(row[token]), float(row.double().max())
    t = 1.0 if greedy else min(tau, 2.0 ** 100)
    return (0.0 if x == top else (x - top) / t) - log_z


def row_token(row, tau: float, u):
    """The token that a row draws with the number u, -1 where nothing has mass (a NaN: the first)."""
    w, _, greedy = row_weights(row, tau)
    if bool(torch.isnan(row).any()):
        return int(torch.isnan(row).nonzero()[0])
    if w is None:
        return -1
    return int(row.double().argmax()) if greedy else draw(w, u)


def _requests(cu_num_draft, cu_num_sampled):
    d = 0
    for r, (d1, s1) in enumerate(zip(cu_num_draft.tolist(), cu_num_sampled.tolist())):
        n = d1 - d
        yield r, d, n, s1 - (n + 1)
        d = d1


def tree_verify_sampled(logits, cu_num_draft, cu_num_sampled, draft_tokens, parents, uniforms, temperature, max_spec_len: int):
    """-> (output_tokens [B, max_spec_len + 1], accepted_path [B, max_spec_len], accepted_len [B], logprobs)."""
    B = len(cu_num_draft)
    out, path = torch.full((B, max_spec_len + 1), -1), torch.full((B, max_spec_len), -1)
    logp, count = torch.zeros(B, max_spec_len + 1, dtype=torch.float64), torch.zeros(B, dtype=torch.int64)
    tok, par = draft_tokens.tolist(), parents.tolist()
    for r, d0, n, s0 in _requests(cu_num_draft, cu_num_sampled):
        tau = 1.0 if temperature is None else float(temperature[r])
        cur, pos = -1, 0
        while True:
            row = logits[s0 + cur + 1]
            t = row_token(row, tau, uniforms[s0 + cur + 1])
            out[r, pos] = t
            logp[r, pos] = log_prob(row, tau, t) if t >= 0 else 0.0
            nxt = next((i for i in range(n) if t >= 0 and par[d0 + i] == cur and tok[d0 + i] == t), -1)
            if nxt < 0 or pos >= max_spec_len:
                break
            path[r, pos] = nxt
            cur, pos = nxt, pos + 1
        count[r] = pos
    return out, path, count, logp


def chain_verify_rejection(logits, cu_num_draft, cu_num_sampled, draft_tokens, draft_probs, uniforms, resample, temperature,
                           max_spec_len: int, ids=None):
    """-> (output_tokens [B, max_spec_len + 1], accepted_len [B], logprobs); draft_probs over the tokens ids, or all."""
    B, V = len(cu_num_draft), logits.shape[1]
    out, count = torch.full((B, max_spec_len + 1), -1), torch.zeros(B, dtype=torch.int64)
    logp = torch.zeros(B, max_spec_len + 1, dtype=torch.float64)
    tok = draft_tokens.tolist()
    for r, d0, n, s0 in _requests(cu_num_draft, cu_num_sampled):
        tau = 1.0 if temperature is None else float(temperature[r])
        for i in range(n + 1):
            row = logits[s0 + i]
            w, _, greedy = row_weights(row, tau)
            d = tok[d0 + i] if i < n else -1
            stays = False
            if w is None or greedy:
                t = row_token(row, tau, 0.0)
                stays = i < n and t >= 0 and t == d
            elif i == n:
                t = draw(w, resample[r])
            else:
                p, q = w / w.sum(), torch.zeros(V, dtype=torch.float64)
                given = draft_probs[d0 + i].double()
                q[slice(None) if ids is None else ids.long()] = torch.where(given > 0, given, torch.zeros_like(given))
                stays = 0 <= d < V and number(uniforms[d0 + i]) * float(q[d]) < float(p[d])
                rest = (p - q).clamp_min(0)
                t = d if stays else draw(rest if float(rest.sum()) > 0 else p, resample[r])
            out[r, i] = t
            logp[r, i] = log_prob(row, tau, t) if t >= 0 else 0.0
            if not stays:
                break
            count[r] += 1
    return out, count, logp

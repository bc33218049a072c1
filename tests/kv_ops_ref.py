"""Plain 64-bit implementations of the cache operators, for their tests: one sequence and one
query head at a time, straight from the definitions in include/jinf/kv_ops.h."""
import math

import torch

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # half the distance of two neighbours near 1


def sees(mask_words, nodes, past, device):
    """[nodes, past + nodes] truth values; mask_words int32 [nodes, words] or None (causal)."""
    see = torch.ones(nodes, past + nodes, dtype=torch.bool)
    for t in range(nodes):
        for u in range(nodes):
            if mask_words is None:
                see[t, past + u] = u <= t
            else:
                see[t, past + u] = bool((int(mask_words[t, u // 32]) >> (u % 32)) & 1)
    return see.to(device)


def attention(q, k, v, n_past, masks, scale):
    """q [S, T, H, hd], k / v [S, Hkv, ctx, hd] (any type), masks: per sequence words or None. Returns out,
    lse and, for the error bound of out, sum p |v| and sum |v| / sum e^(s - max) over the seen rows."""
    S, T, H, hd = q.shape
    group = H // k.shape[1]
    out = torch.zeros(S, T, H, hd, dtype=torch.float64, device=q.device)
    lse = torch.full((S, T, H), -math.inf, dtype=torch.float64, device=q.device)
    mag, flat = torch.zeros_like(out), torch.zeros_like(out)
    for s in range(S):
        past = int(n_past[s])
        see = sees(None if masks[s] is None else masks[s].cpu(), T, past, q.device)
        for h in range(H):
            kk, vv = k[s, h // group, :past + T].double(), v[s, h // group, :past + T].double()
            for t in range(T):
                at = see[t].nonzero()[:, 0]
                if len(at) == 0:
                    continue
                x = scale * (kk[at] @ q[s, t, h].double())
                m = x.max()
                e = torch.exp(x - m)
                out[s, t, h] = (e / e.sum()) @ vv[at]
                mag[s, t, h] = (e / e.sum()) @ vv[at].abs()
                flat[s, t, h] = vv[at].abs().sum(0) / e.sum()
                lse[s, t, h] = m + torch.log(e.sum())
    return out, lse, mag, flat


def mass(before, q, k, n_past, masks, lse, weight, scale):
    """The new mass [S, Hkv, ctx] and, for its error bound, what was added."""
    S, T, H, hd = q.shape
    group = H // k.shape[1]
    new, add = before.double().clone(), torch.zeros_like(before, dtype=torch.float64)
    for s in range(S):
        past = int(n_past[s])
        see = sees(None if masks[s] is None else masks[s].cpu(), T, past, q.device)
        new[s, :, past:past + T] = 0.0
        for h in range(H):
            kk = k[s, h // group, :past + T].double()
            for t in range(T):
                w = 1.0 if weight is None else float(weight[s, t])
                if w == 0.0 or float(lse[s, t, h]) == -math.inf:
                    continue
                at = see[t].nonzero()[:, 0]
                x = scale * (kk[at] @ q[s, t, h].double())
                add[s, h // group, at] += w * torch.exp(x - lse[s, t, h].double())
    return new + add, add


def evict_ids(mass_row, n, keep, sink, recent):
    """Kept rows (a list) of one sequence and head; mass_row a list of floats."""
    if n <= keep:
        return list(range(n))
    middle = list(range(sink, n - recent))
    rank = lambda x: -math.inf if math.isnan(x) else x  # noqa: E731
    chosen = sorted(middle, key=lambda i: (math.isnan(mass_row[i]), -rank(mass_row[i]), i))[:keep - sink - recent]
    return sorted(list(range(sink)) + chosen + list(range(n - recent, n)))

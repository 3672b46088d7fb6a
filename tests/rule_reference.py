"""Routing by a rule, restated row by row in float64 (include/osm_hip.h, osm_route_experts)."""

import numpy as np


def route(logits, rule, bias=None):
    """ids, weights and mass of logits [T, E]; rule: any object with osm_route_rule's fields."""
    T, E = logits.shape
    k, per = rule.top_k, E // rule.groups
    ids, weights, mass = np.zeros((T, k), np.uint32), np.zeros((T, k)), np.zeros(T)
    for t in range(T):
        l = np.asarray(logits[t], np.float64)
        avail = l > -np.inf
        s = np.zeros(E)
        if rule.score == 0 and avail.any():
            m = l[avail].max()
            d = np.where(l[avail] == m, 0.0, l[avail])  # also where the largest is infinite
            s[avail] = np.where(l[avail] == m, 1.0, np.exp(np.minimum(d - m, 0.0) if np.isfinite(m) else -np.inf))
            s /= s.sum()
        elif rule.score == 1:
            with np.errstate(over="ignore"):
                s[avail] = 1.0 / (1.0 + np.exp(-l[avail]))
        rank = (s + bias.astype(np.float64)) if bias is not None else l
        c = (s + bias.astype(np.float64)) if bias is not None else s
        ok = avail & (rank > -np.inf)
        if rule.groups > 1:
            g = np.where(ok, c, -np.inf).reshape(rule.groups, per)
            gs = np.sort(g, 1)[:, ::-1][:, :rule.group_score].sum(1)
            kept = np.argsort(-gs, kind="stable")[:rule.top_groups]
            keep = np.zeros(rule.groups, bool)
            keep[kept] = True
            ok &= np.repeat(keep, per)
        left = np.where(ok, rank, -np.inf)
        order = np.lexsort((np.arange(E), -left, ~ok))  # the unavailable ones last, by id
        pick = order[:k]
        ps = np.where(ok[pick], s[pick], 0.0)
        ids[t], mass[t] = pick, ps.sum()
        w = ps / ps.sum() if rule.renormalize and ps.sum() > 0 else (ps if not rule.renormalize else 0 * ps)
        weights[t] = rule.scale * w
    return ids, weights, mass

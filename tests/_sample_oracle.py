"""The choice of a token from a uniform, row by row in 64 bits."""

import math

import torch


def choose(x, u, T, k, tp, mp):
    """(token, log-prob, log-prob of what is drawn from) of one row; -1 and NaN without a distribution."""
    x = x.double().cpu()
    V = x.numel()
    if torch.isnan(x).any() or not torch.isfinite(x.max()) or math.isnan(T) or T == math.inf:
        return -1, math.nan, math.nan
    greedy = T <= 0
    T = 1.0 if greedy else T
    # from the maximum, so that temperatures next to 0 overflow nothing
    z = (x - x.max()) / T
    lp = z - z.exp().sum().log()
    if greedy:
        t = int((x == x.max()).nonzero()[0, 0])
        return t, float(lp[t]), 0.0
    order = torch.sort(x, descending=True, stable=True).indices
    w = z[order].exp()
    n = k if 0 < k < V else V
    if 0 < tp < 1:
        share = w[:n].cumsum(0) / w[:n].sum()
        n = max(1, int((share <= tp).sum()))
    if mp > 0:
        n = min(n, int((x[order] - x.max() >= T * math.log(min(mp, 1.0))).sum()))
    left = torch.sort(order[:n]).values
    run = z[left].exp().cumsum(0)
    over = (run > float(u) * run[-1]).nonzero()
    t = int(left[over[0, 0]]) if over.numel() else int(left[(z[left] > -700).nonzero()[-1, 0]])
    return t, float(lp[t]), float(z[t] - run[-1].log())

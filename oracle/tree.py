"""The cached step over sequences of different lengths, with a tree of drafted tokens, in
float64 from its definition: one sequence at a time, over exactly the keys that count."""

from __future__ import annotations

import torch

from . import diff


def lines(parents) -> list:
    """Each node's line of descent (itself last), or None outside the tree."""
    out: list = []
    for t, p in enumerate(int(x) for x in parents):
        if p == -1:
            out.append([t])
        elif 0 <= p < t and out[p] is not None:
            out.append(out[p] + [t])
        else:
            out.append(None)
    return out


def keep_of(T: int, n: int, parents=None, causal: bool = True):
    """(which of the T nodes are in the tree, what those see of n cached rows and the block)."""
    if parents is None:
        return list(range(T)), diff.causal_keep(T, n + T, causal)
    ls = lines(parents)
    live = [t for t in range(T) if ls[t] is not None]
    keep = torch.zeros(len(live), n + T, dtype=torch.bool)
    keep[:, :n] = True
    for i, t in enumerate(live):
        keep[i, [n + a for a in ls[t]]] = True
    return live, keep


def cases(q, k, v, ck, cv, lens, parents, scale, lam=None, causal=True):
    """For each sequence: its nodes in the tree and a diff.Case of their rows (None if none)."""
    B, T = q.shape[:2]
    for b in range(B):
        n = int(lens[b])
        own = None if parents is None else parents if parents.dim() == 1 else parents[b]
        live, keep = keep_of(T, n, own, causal)
        if not live:
            yield live, None
            continue
        keys, vals = (torch.cat([c[b, :, :n].transpose(0, 1), x[b]])[None]
                      for c, x in ((ck, k), (cv, v)))
        # Keys that nobody sees leave the problem (what they hold must not matter).
        seen = keep.any(0)
        yield live, diff.Case(q[b:b + 1, live], keys[:, seen], vals[:, seen], lam, scale, keep[:, seen])

"""Differential attention in float64, from its definition, and its gradients in closed form.

    P_m = softmax(scale * q_m k_m^T + mask),  out = (P_1 - lam_h P_2) v

on q [B,T,H,E], k/v [B,L,Hkv,E] (the halves m of the E dims of q and k), lam [H]; with lam None,
ordinary attention: one map of all E dims. Query t may see key j where ``keep`` [T, L] says so,
and sees one at least. Also bounds on what roundings do to each result, for
the tolerances of the tests.
"""

from __future__ import annotations

import dataclasses

import torch


def causal_keep(T: int, L: int, causal: bool) -> torch.Tensor:
    """Row t of the last T of L keys sees keys up to its own (all of them if not causal)."""
    keep = torch.ones(T, L, dtype=torch.bool)
    return keep.tril(L - T) if causal else keep


def _heads(x: torch.Tensor, H: int) -> torch.Tensor:
    """[B,T,h,E] -> float64 [B,H,T,E], kv heads repeated for their group."""
    x = x.detach().cpu().double().transpose(1, 2)
    return x.repeat_interleave(H // x.shape[1], 1)


def _fold(x: torch.Tensor, Hkv: int) -> torch.Tensor:
    """[B,H,T,E] -> [B,T,Hkv,E], summed over each kv head's group."""
    B, H, T, E = x.shape
    return x.reshape(B, Hkv, H // Hkv, T, E).sum(2).transpose(1, 2)


@dataclasses.dataclass
class Case:
    """One problem, its maps and everything the bounds are made of."""

    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor
    lam: torch.Tensor | None
    scale: float
    keep: torch.Tensor

    def __post_init__(self):
        H, E = self.q.shape[2], self.q.shape[3]
        self.H, self.Hkv, self.E = H, self.k.shape[2], E
        self.qh, self.kh, self.vh = (_heads(t, H) for t in (self.q, self.k, self.v))
        self.w = (torch.ones(1, 1, 1, 1, dtype=torch.float64),)
        self.half = (slice(0, E),)
        if self.lam is not None:
            self.w += (-self.lam.detach().cpu().double().reshape(1, H, 1, 1),)
            self.half = (slice(0, E // 2), slice(E // 2, E))
        self.P, self.lse = [], []
        for m in self.half:
            s = self.scale * self.qh[..., m] @ self.kh[..., m].transpose(-1, -2)
            s = s.masked_fill(~self.keep, float("-inf"))
            self.lse.append(torch.logsumexp(s, -1))
            self.P.append(torch.exp(s - self.lse[-1][..., None]))

    def out(self) -> torch.Tensor:
        """[B,T,H,E]"""
        o = sum(w * (P @ self.vh) for w, P in zip(self.w, self.P))
        return o.transpose(1, 2)

    def grads(self, do: torch.Tensor):
        """(dq, dk, dv, dlam) for the gradient ``do`` of out."""
        do = do.detach().cpu().double().transpose(1, 2)
        G = do @ self.vh.transpose(-1, -2)
        delta = [(P * G).sum(-1, keepdim=True) for P in self.P]
        dS = [self.scale * w * P * (G - d) for w, P, d in zip(self.w, self.P, delta)]
        dq = torch.cat([S @ self.kh[..., m] for S, m in zip(dS, self.half)], -1).transpose(1, 2)
        dk = torch.cat([S.transpose(-1, -2) @ self.qh[..., m] for S, m in zip(dS, self.half)], -1)
        W = sum(w * P for w, P in zip(self.w, self.P))
        dv = W.transpose(-1, -2) @ do
        return dq, _fold(dk, self.Hkv), _fold(dv, self.Hkv), -delta[1].sum((0, 2, 3))

    # What the roundings of a computation can do, element by element. `u` is half a unit in
    # the last place, relative (eps / 2), of the type that P, W and dS enter their products
    # in and that the results are stored in, and `tiny` half of its smallest step: what a
    # rounding is off by at most under the type's normal range (float16: 2^-25 below 2^-14;
    # the other types reach 2^-126). Sums are taken in float32.
    def _slack(self) -> float:
        """Relative error of a P, and of a sum of products, in float32: the scores' own
        (at most E products, then a few units of the largest score's exponent) and the length
        of the sums."""
        f = 2.0 ** -24
        big = max(float((abs(self.scale) * self.qh[..., m].abs() @ self.kh[..., m].abs().transpose(-1, -2))
                        .max()) for m in self.half) if self.qh.numel() and self.kh.numel() else 0.0
        return f * (self.E * big + 4 * big + 64 + self.E + self.keep.shape[0] + self.keep.shape[1])

    def _value_bounds(self, u, tiny):
        """|error| of P_m v before it is rounded, from P's rounding and float32. (The forward
        rounds exp(s - m) with m <= the row's largest score: e^(m - lse) <= 1 times P.)"""
        r = u + self._slack()
        seen = self.keep.double()
        return [r * (P @ self.vh.abs()) + tiny * (seen @ self.vh.abs()) for P in self.P]

    def out_bound(self, u: float, tiny: float = 0.0) -> torch.Tensor:
        e = sum(w.abs() * b for w, b in zip(self.w, self._value_bounds(u, tiny)))
        return (e + u * (self.out().transpose(1, 2).abs() + e) + tiny).transpose(1, 2)

    def lse_bound(self) -> torch.Tensor:
        """|error| of a map's LSE: its scores' absolute error and its sum's relative one, and
        its own rounding."""
        return self._slack() + 2.0 ** -23 * self.lse[0].abs()

    def grad_bounds(self, do: torch.Tensor, u: float, tiny: float = 0.0):
        a = do.detach().cpu().double().transpose(1, 2)
        G = a @ self.vh.transpose(-1, -2)
        A = a.abs() @ self.vh.abs().transpose(-1, -2)
        sl = self._slack()
        r = u + sl
        lam = self.w[1].abs()
        vb = self._value_bounds(u, tiny)
        seen = self.keep.double()
        o = self.out().transpose(1, 2)
        O2 = self.P[1] @ self.vh
        ob = vb[0] + lam * vb[1]
        e_o = ob + u * (o.abs() + ob) + tiny                   # as stored
        e_o2 = vb[1] + u * (O2.abs() + vb[1]) + tiny
        # delta_1 = do . (out + lam O2), delta_2 = do . O2, in float32 from the stored ones.
        e_d = [(a.abs() * (e_o + lam * e_o2 + sl * (o.abs() + lam * O2.abs()))).sum(-1, keepdim=True),
               (a.abs() * (e_o2 + sl * O2.abs())).sum(-1, keepdim=True)]
        delta = [(P * G).sum(-1, keepdim=True) for P in self.P]
        e_S, S = [], []
        for w, P, d, ed in zip(self.w, self.P, delta, e_d):
            S.append(abs(self.scale) * w.abs() * P * (G - d).abs())
            e = abs(self.scale) * w.abs() * P * (ed + sl * (A + d.abs()) + sl * (G - d).abs())
            # dS enters as P (G - delta), with or without lam; the scale comes after.
            e_S.append(e + r * (S[-1] + e) + tiny * abs(self.scale) * w.abs().clamp(min=1) * seen)
        W = sum(w * P for w, P in zip(self.w, self.P)).abs()
        e_W = u * W + sl * sum(w.abs() * P for w, P in zip(self.w, self.P)) + tiny * seen
        e_q = torch.cat([(e + sl * s) @ self.kh[..., m].abs() for e, s, m in zip(e_S, S, self.half)], -1)
        e_k = torch.cat([(e + sl * s).transpose(-1, -2) @ self.qh[..., m].abs()
                         for e, s, m in zip(e_S, S, self.half)], -1)
        e_v = (e_W + sl * W).transpose(-1, -2) @ a.abs()
        rows = a.shape[0] * a.shape[2]
        e_l = ((e_d[1] + rows * 2.0 ** -24 * delta[1].abs()).sum((0, 2, 3)))
        dq, dk, dv, dl = self.grads(do)
        out = []
        for g, e in ((dq, e_q.transpose(1, 2)), (dk, _fold(e_k, self.Hkv)), (dv, _fold(e_v, self.Hkv)),
                     (dl, e_l)):
            out.append(e + u * (g.abs() + e) + tiny)
        return out

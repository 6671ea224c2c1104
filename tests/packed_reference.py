"""Plain 64-bit attention over packed sequences with a bound on what a kernel of a given type may be off by.

The bounds follow from the arithmetic and were written down before the first run.  With u half a step of the type
(bf16 2^-8, fp16 2^-11, fp32 2^-24 relative), e = 2^-24 and n keys (queries for dk, dv):
  * a score is a sum of D products in fp32: off by at most (D + 8) e scale sum|q||k| =: es absolutely, so P by the factor
    exp(+-2 es) (numerator and denominator), and the exponential and the sums add 2^-20 + 2 n e: together r;
  * P (and dS) are rounded to the type once as operands of the next product, results once more:
      |o error|  <= (u + r) sum P|v| + u |o|
      |dv error| <= (u + r) sum P|do| + u |dv|
    dS = P (dP - delta) with delta = sum do * o from the rounded o (u sum|do||o|), dP a sum of D products:
      |dS error| <= P (u_o sum|do||o| + (D + 8) e (sum|do||v| + sum|do||o|)) + (u + r) P (|dP| + |delta|)
      |dq error| <= scale sum |dS error||k| + n e scale sum|dS||k| + u |dq|, dk alike with q and the group's heads.
  fp16 has a smallest step: 2^-25 is added for each rounding of a value (P is off by at most 2^-25 absolutely, and so on).
"""
import math

import torch

HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def packed_reference(q, k, v, lens_q, lens_k, causal, scale, d_out=None):
    """``{name: (value, bound)}`` for o, lse and, with ``d_out``, dq, dk, dv; rows of no sequence are zeros."""
    u, tiny, e = HALF[q.dtype], TINY[q.dtype], 2.0 ** -24
    T, H, D = q.shape
    S, Hk = k.shape[:2]
    dev = q.device
    z = lambda *shape: torch.zeros(shape, dtype=torch.float64, device=dev)
    q, k, v = q.double(), k.double(), v.double()
    o, ob, lse, lb = z(T, H, D), z(T, H, D), torch.full((H, T), -math.inf, dtype=torch.float64, device=dev), z(H, T)
    dq, dqb, dk, dkb, dv, dvb = z(T, H, D), z(T, H, D), z(S, Hk, D), z(S, Hk, D), z(S, Hk, D), z(S, Hk, D)
    a = c = 0
    for lq, lk in zip(lens_q, lens_k):
        for h in range(H if lq and lk else 0):
            g = h // (H // Hk)
            Q, K, V = q[a:a + lq, h], k[c:c + lk, g], v[c:c + lk, g]
            s = Q @ K.T * scale
            es = (D + 8) * e * scale * (Q.abs() @ K.abs().T).amax(1, keepdim=True)
            seen = torch.ones(lq, lk, dtype=torch.bool, device=dev)
            if causal:
                seen = torch.arange(lk, device=dev)[None] <= torch.arange(lq, device=dev)[:, None] + (lk - lq)
            s = s.masked_fill(~seen, -math.inf)
            alive = seen.any(1)
            P = torch.where(alive[:, None], torch.softmax(s.masked_fill(~alive[:, None], 0.0), 1), torch.zeros_like(s))
            r = torch.expm1(2 * es) + 2.0 ** -20 + 2 * lk * e
            rows = slice(a, a + lq)
            O = P @ V
            o[rows, h] = O
            ob[rows, h] = (u + r) * (P @ V.abs()) + u * O.abs() + tiny * (1 + seen.double() @ V.abs())
            lse[h, rows] = torch.where(alive, torch.logsumexp(s.masked_fill(~alive[:, None], 0.0), 1), lse[h, rows])
            lb[h, rows] = (es + 2.0 ** -20 + lk * e)[:, 0] + 4 * e * lse[h, rows].abs().nan_to_num(0, 0, 0)
            if d_out is None:
                continue
            G = d_out[rows, h].double()
            dP = G @ V.T
            delta = (G * O).sum(1, keepdim=True)
            dS = P * (dP - delta)
            go = (G.abs() * O.abs()).sum(1, keepdim=True)
            # the saved o carries the forward's own error
            go_err = (G.abs() * (ob[rows, h])).sum(1, keepdim=True)
            dSb = P * (go_err + (D + 8) * e * (G.abs() @ V.abs().T + go)) + (u + r) * P * (dP.abs() + delta.abs()) + tiny * seen
            rq = 2.0 ** -20 + 2 * lq * e
            dq[rows, h] = dS @ K * scale
            dqb[rows, h] = scale * (dSb @ K.abs() + lk * e * (dS.abs() @ K.abs())) + u * dq[rows, h].abs() + tiny
            dk[c:c + lk, g] += dS.T @ Q * scale
            dkb[c:c + lk, g] += scale * (dSb.T @ Q.abs() + rq * (dS.abs().T @ Q.abs()))
            dv[c:c + lk, g] += P.T @ G
            dvb[c:c + lk, g] += ((u + r + rq) * P + tiny * seen).T @ G.abs()
        a, c = a + lq, c + lk
    out = {"o": (o, ob), "lse": (lse, lb)}
    if d_out is not None:
        out.update(dq=(dq, dqb), dk=(dk, dkb + u * dk.abs() + tiny), dv=(dv, dvb + u * dv.abs() + tiny))
    return out


def assert_within(name, got, ref):
    value, bound = ref
    got = got.double()
    finite = torch.isfinite(value)
    assert torch.equal(torch.where(finite, torch.zeros_like(got), got), torch.where(finite, torch.zeros_like(value), value)), \
        f"{name}: infinities differ"
    assert torch.isfinite(got[finite]).all(), f"{name}: not finite"
    excess = ((got - value).abs() - bound)[finite]
    if excess.numel():
        worst = int(excess.argmax())
        assert excess.max() <= 0, f"{name}: error {(got - value)[finite][worst].abs():.3e} above its bound {bound[finite][worst]:.3e}"


def borders(lens, device):
    t = torch.zeros(len(lens) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lens, dtype=torch.int64).cumsum(0).to(torch.int32) if lens else t[1:]
    return t.to(device)

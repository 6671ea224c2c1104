"""Gradients of the packed attention over the range of sizes that incoming gradients have: unscaled losses (small), loss scaling
(large), rows and keys of very different sizes.

Limits, written down before the first run.  With u half a step of the type, a kernel rounds each P and each dS = P (dP - D) to the type
once, independently of one another and by at most u of the value, whatever the value's size; so a row of dq is off by a vector whose
square is at most u^2 / 3 sum_j dS_j^2 |k_j|^2 scale^2 on average, over sums of four terms and more: 2.5 u of that root is four to
five standard deviations.  dk and dv alike, over the queries of all heads of the group.  D comes from an output whose P were
rounded: its error is u / sqrt(3) sqrt(sum_j P_j^2 dP_j^2) alike and moves the row by that times P k.  P itself is off by a common factor
of at most 2^-16 (the exponent, of size 64 at most, in fp32).  The result is rounded once more.
"""
import math

import pytest
import torch

from tests.packed_reference import HALF, borders

pytestmark = pytest.mark.gpu


def _limits(q, k, v, g, lens_q, lens_k, causal):
    """``{name: (value, limit of each row's error)}`` in 64 bits, without the last rounding."""
    u = HALF[q.dtype]
    q, k, v, g = [x.double() for x in (q, k, v, g)]
    H, D = q.shape[1:]
    group, scale = H // k.shape[1], D ** -0.5
    val = {"dq": torch.zeros_like(q), "dk": torch.zeros_like(k), "dv": torch.zeros_like(v)}
    var = {n: torch.zeros(x.shape[:2], dtype=torch.float64, device=x.device) for n, x in val.items()}
    a = c = 0
    for lq, lk in zip(lens_q, lens_k):
        for h in range(H if lq and lk else 0):
            e = h // group
            Q, K, V, G = q[a:a + lq, h], k[c:c + lk, e], v[c:c + lk, e], g[a:a + lq, h]
            s = Q @ K.T * scale
            if causal:
                s = s.masked_fill(torch.arange(lk, device=s.device)[None] > torch.arange(lq, device=s.device)[:, None] + (lk - lq), -math.inf)
            P = torch.softmax(s, 1)
            dP = G @ V.T
            dS = P * (dP - (P * dP).sum(1, keepdim=True))
            d_var = (P * dP).square().sum(1, keepdim=True)  # of D, in units of u^2 / 3
            val["dq"][a:a + lq, h] = dS @ K * scale
            val["dk"][c:c + lk, e] += dS.T @ Q * scale
            val["dv"][c:c + lk, e] += P.T @ G
            qq, kk, gg = [x.square().sum(1) for x in (Q, K, G)]
            var["dq"][a:a + lq, h] = (dS.square() @ kk + d_var[:, 0] * (P @ K).square().sum(1)) * scale ** 2
            var["dk"][c:c + lk, e] += (dS.square() + P.square() * d_var).T @ qq * scale ** 2
            var["dv"][c:c + lk, e] += P.square().T @ gg
        a, c = a + lq, c + lk
    return {n: (val[n], 2.5 * u * var[n].sqrt() + 2.0 ** -16 * val[n].norm(dim=-1)) for n in val}


def _check(q, k, v, g, lens_q, lens_k, causal):
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func

    want = _limits(q, k, v, g, lens_q, lens_k, causal)
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    o = packed_flash_attn_func(*leaves, borders(lens_q, q.device), borders(lens_k, q.device), causal)
    got = torch.autograd.grad(o, leaves, g)
    check_status()
    for (name, (value, limit)), x in zip(want.items(), got):
        assert torch.isfinite(x).all(), name
        rounding = (value.to(x.dtype).double() - value).norm(dim=-1)
        excess = (x.double() - value).norm(dim=-1) - limit - rounding
        at = excess.argmax().item()
        assert excess.max() <= 0, (f"{name} row {at // x.shape[1]} head {at % x.shape[1]}: off by {(x.double() - value).norm(dim=-1).flatten()[at]:.3e} of "
                                   f"{value.norm(dim=-1).flatten()[at]:.3e}, rounding {rounding.flatten()[at]:.3e}, limit {limit.flatten()[at]:.3e}")


def _draw(lens_q, lens_k, H, Hk, D, dtype, seed, sizes):
    g = torch.Generator().manual_seed(seed)
    mk = lambda n, h, size: (torch.randn(n, h, D, generator=g) * size).to(dtype).cuda()
    return mk(sum(lens_q), H, sizes[0]), mk(sum(lens_k), Hk, sizes[1]), mk(sum(lens_k), Hk, sizes[2]), mk(sum(lens_q), H, sizes[3])


DTYPES = [torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3])
@pytest.mark.parametrize("lens_q,lens_k,H,Hk,D,causal", [
    ([300], [4099], 2, 1, 64, False), ([130], [8328], 2, 2, 64, True), ([260], [8328], 1, 1, 128, False), ([1500, 77], [1500, 900], 4, 2, 64, True),
    ([1500, 77], [1500, 900], 4, 1, 128, True), ([700], [700], 8, 1, 96, False),
])
def test_small_incoming_gradients(lens_q, lens_k, H, Hk, D, causal, size, dtype):
    _check(*_draw(lens_q, lens_k, H, Hk, D, dtype, D + H, (1.0, 1.0, 1.0, size)), lens_q, lens_k, causal)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_scaled_losses(D, dtype):
    """dS beyond the largest fp16 number, with gradients that are within it."""
    lens = [4] * 30 + [300, 150]
    q, k, v, g = _draw(lens, lens, 2, 2, D, dtype, 5, (1 / 16, 1 / 16, 4.0, 8192.0))
    _check(q, k, v, g.clamp(-32768, 32768), lens, lens, False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128, 40])
@pytest.mark.parametrize("falling", [False, True])
def test_sizes_that_change_along_the_sequence(D, falling, dtype):
    """Incoming gradients from 2^-9 to 2^9 along the queries, values from 2^-3 to 2^5 along the keys: sums in which later tiles
    outweigh, or are lost beside, the earlier ones."""
    n = 1100
    for lens_q, H, Hk in (([n], 2, 2), ([n], 4, 1)):
        q, k, v, g = _draw(lens_q, [n], H, Hk, D, dtype, D, (0.5, 0.5, 1.0, 1.0))
        ramp = torch.linspace(-1, 1, n, device=q.device)[:, None, None] * (-1 if falling else 1)
        g, v = (g * torch.exp2((9 * ramp).round())).to(dtype), (v * torch.exp2((1 + 4 * ramp).round())).to(dtype)
        _check(q, k, v, g, lens_q, [n], False)
        _check(q, k, v, g, lens_q, [n], True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_gradient_at_all_and_one_row_of_it(dtype):
    lens = [200, 333]
    q, k, v, g = _draw(lens, lens, 2, 1, 64, dtype, 9, (1.0, 1.0, 1.0, 1.0))
    _check(q, k, v, torch.zeros_like(g), lens, lens, True)
    g[:-1] = 0
    _check(q, k, v, g, lens, lens, True)

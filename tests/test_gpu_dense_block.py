"""The documented replacement of a dense block's attention, as the integration guide prints it, against that attention in 64 bits."""
import os
import re

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _example():
    text = open(os.path.join(ROOT, "INTEGRATION.md")).read()
    return re.search(r"### Dense blocks.*?```python\n(.*?)```", text, re.S).group(1)


class _Attention(torch.nn.Module):
    """The parts of a dense block's attention that the example names; ``norm``: q and k of each head normalised, as in VGGT and Pi3."""

    def __init__(self, dim, heads, norm):
        super().__init__()
        self.qkv, self.proj = torch.nn.Linear(dim, 3 * dim), torch.nn.Linear(dim, dim)
        self.q_norm, self.k_norm = [torch.nn.LayerNorm(dim // heads) if norm else torch.nn.Identity() for _ in range(2)]
        with torch.no_grad():
            for p in self.parameters():  # norms with weights and offsets of their own too
                p.add_(torch.randn(p.shape) * 0.02 if p.dim() == 2 else torch.randn(p.shape) * 0.3)


def _definition(attn, x, pos, views, heads):
    """The block's attention from its definition: projection, norm, rotation of the pairs (j, j + 16) of each half, softmax, projection."""
    n = x.shape[0] * x.shape[1]
    q, k, v = attn.qkv(x).view(n, 3, heads, 64).unbind(1)
    rate = 100.0 ** (-torch.arange(16, device=x.device, dtype=torch.float64) / 16)

    def turn(y):
        out = []
        for axis in range(2):
            z = torch.complex(y[..., 32 * axis:32 * axis + 16], y[..., 32 * axis + 16:32 * axis + 32])
            angle = pos.reshape(n, 2)[:, axis].double()[:, None] * rate
            z = z * torch.polar(torch.ones_like(angle), angle)[:, None]
            out += [z.real, z.imag]
        return torch.cat(out, -1)

    q, k, v = [y.reshape(views, n // views, heads, 64).transpose(1, 2) for y in (turn(attn.q_norm(q)), turn(attn.k_norm(k)), v)]
    out = torch.softmax(q @ k.transpose(-1, -2) / 8, -1) @ v
    return attn.proj(out.transpose(1, 2).reshape(x.shape))


@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_documented_dense_block_is_the_block_it_replaces(dtype, norm):
    from geoweave_b200 import check_status
    from tests.gpu_util import dev

    torch.manual_seed(3)
    views, rows, cols, heads = 3, 9, 7, 4
    tokens_per_view, dim = 5 + rows * cols, heads * 64
    attn = _Attention(dim, heads, norm).to(dev(), dtype)
    x = torch.randn(views, tokens_per_view, dim).to(dev(), dtype).requires_grad_()
    up = torch.randn(views, tokens_per_view, dim).to(dev(), dtype)
    grid = torch.cartesian_prod(torch.arange(rows), torch.arange(cols)) + 1
    pos = torch.cat((torch.zeros(5, 2, dtype=torch.int64), grid)).to(dev()).expand(views, -1, -1).contiguous()
    names = {"torch": torch, "attn": attn, "x": x, "pos": pos, "views": views, "rows": rows, "cols": cols, "heads": heads,
             "tokens_per_view": tokens_per_view}
    exec(_example(), names)
    (grad,) = torch.autograd.grad(names["x"], x, up)
    check_status()

    twice = x.detach().double().requires_grad_()
    want = _definition(attn.double(), twice, pos, views, heads)
    (want_grad,) = torch.autograd.grad(want, twice, up.double())
    # On the way values are rounded to the type six times (projection, norm, rotary, P, output, projection), each by u at most and about
    # u / 2 on average, and a score's error counts as one of P: below 16 u of the norm.  Sums of 256 products in fp32 add 2^-18.  A block without
    # its norms is off by a large part of the norm.  The backward pass doubles the number of roundings.
    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
    assert (names["x"].double() - want).norm() <= (16 * u + 2.0 ** -18) * want.norm()
    assert (grad.double() - want_grad).norm() <= (32 * u + 2.0 ** -17) * want_grad.norm()

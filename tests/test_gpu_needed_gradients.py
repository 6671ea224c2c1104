"""Gradients of some of the inputs only: the same numbers as with all of them, and no work for the others."""
import itertools

import pytest
import torch

from tests.packed_reference import borders

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _some(call, inputs, needed, up):
    leaves = [x.detach().clone().requires_grad_(n) for x, n in zip(inputs, needed)]
    out = call(*leaves)
    asked = [x for x, n in zip(leaves, needed) if n]
    outs = [x for x in (out if isinstance(out, tuple) else (out,)) if x.requires_grad]
    got = iter(torch.autograd.grad(outs, asked, up[:len(outs)]))
    return [next(got) if n else None for n in needed]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_attention(D, dtype, monkeypatch):
    from geoweave_b200 import check_status
    from geoweave_b200.custom_flash_attn import packed_flash_attn, packed_flash_attn_func

    made = []
    whole = packed_flash_attn.packed_attention_backward
    monkeypatch.setattr(packed_flash_attn, "packed_attention_backward", lambda *a, **k: made.append(whole(*a, **k)) or made[-1])
    g = torch.Generator().manual_seed(D)
    lens = [130, 0, 77]
    mk = lambda h: torch.randn(sum(lens) + 20, h, D, generator=g).to(dtype).cuda()
    inputs, up = [mk(4), mk(2), mk(2)], [mk(4)]
    call = lambda q, k, v: packed_flash_attn_func(q, k, v, borders(lens, q.device), None, True)
    every = _some(call, inputs, (True, True, True), up)
    for needed in itertools.product((True, False), repeat=3):
        if any(needed):
            made.clear()
            for a, b, n in zip(every, _some(call, inputs, needed, up), needed):
                assert b is None if not n else torch.equal(a, b)
            assert [x is not None for x in made[0]] == [True, any(needed[1:]), any(needed[1:])]
    empty = [x[:0] for x in inputs[1:]]
    (dq, _, _) = _some(lambda q, k, v: packed_flash_attn_func(q, k, v, borders(lens, q.device), borders([0, 0, 0], q.device)),
                       [inputs[0], *empty], (True, False, False), up)
    assert (dq == 0).all()
    check_status()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary(dtype, monkeypatch):
    from geoweave_b200 import rotary

    g = torch.Generator().manual_seed(1)
    mk = lambda h: torch.randn(50, h, 64, generator=g).to(dtype).cuda()
    inputs, up = [mk(4), mk(2)], [mk(4), mk(2)]
    pos = torch.randint(0, 30, (50, 3), generator=g).cuda()
    axes = rotary.rotary_axes((16, 24, 24), 30, "cuda")
    call = lambda q, k: rotary.apply_rotary_axes(q, k, pos, axes)
    every = _some(call, inputs, (True, True), up)
    turned = []
    whole = rotary._rotate
    monkeypatch.setattr(rotary, "_rotate", lambda q, k, *a: turned.append((q.shape[-2], k is not None)) or whole(q, k, *a))
    for needed, backward in (((True, False), (4, False)), ((False, True), (2, False)), ((True, True), (4, True))):
        turned.clear()
        for a, b, n in zip(every, _some(call, inputs, needed, up), needed):
            assert b is None if not n else torch.equal(a, b)
        assert turned[1] == backward


def test_what_the_output_lost_must_be_on_the_same_device():
    from geoweave_b200.custom_flash_attn.packed_flash_attn import packed_attention_backward, packed_attention_forward

    x = torch.randn(20, 2, 64, dtype=torch.bfloat16, device="cuda")
    cu, low = borders([20], x.device), torch.empty_like(x)
    o, lse = packed_attention_forward(x, x, x, cu, return_lse=True, o_low=low)
    packed_attention_backward(x, x, x, cu, None, o, lse, x, o_low=low)
    for bad in (low.cpu(), low.float(), low[:10], low.transpose(0, 1)):
        with pytest.raises(ValueError):
            packed_attention_backward(x, x, x, cu, None, o, lse, x, o_low=bad)
        with pytest.raises(ValueError):
            packed_attention_forward(x, x, x, cu, o_low=bad)

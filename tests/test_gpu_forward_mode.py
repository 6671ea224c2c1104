"""Forward-mode derivatives: no operator has them, so a dual tensor is refused; it never comes back without its tangent."""
import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


def _calls():
    """(differentiable inputs, call of them) for each operator with a gradient."""
    from geoweave_b200.custom_flash_attn import packed_flash_attn_func, sparse_index_flash_attn_bhtd_func, sparse_index_flash_attn_func
    from geoweave_b200.custom_indexer import sparse_topk_indexer_func
    from geoweave_b200.rotary import apply_rotary_axes, rotary_axes
    from tests.gpu_util import dev

    mk = lambda *s: torch.randn(*s, device=dev(), dtype=torch.bfloat16)
    cu = torch.tensor([0, 40, 64], dtype=torch.int32, device=dev())
    pos = torch.zeros(64, 2, dtype=torch.int64, device=dev())
    axes = rotary_axes((32, 32), 4, dev())
    lists = torch.arange(16, dtype=torch.int32, device=dev()).expand(1, 64, 16).contiguous()
    return {
        "packed attention": ([mk(64, 2, 64) for _ in range(3)], lambda q, k, v: packed_flash_attn_func(q, k, v, cu)),
        "rotary": ([mk(64, 2, 64) for _ in range(2)], lambda q, k: apply_rotary_axes(q, k, pos, axes)),
        "rotary of q": ([mk(64, 2, 64)], lambda q: apply_rotary_axes(q, None, pos, axes)),
        "sparse attention": ([mk(1, 64, 16, 64) for _ in range(3)], lambda q, k, v: sparse_index_flash_attn_func(q, k, v, lists)),
        "sparse attention, head-major": ([mk(1, 16, 64, 64) for _ in range(3)], lambda q, k, v: sparse_index_flash_attn_bhtd_func(q, k, v, lists)),
        "indexer": ([mk(1, 64, 4, 64), mk(1, 64, 4, 64), mk(1, 64, 4)],
                    lambda q, k, w: sparse_topk_indexer_func(q, k, w, None, 16, 0.125, 0)),
    }


def test_dual_tensors_are_refused_and_plain_ones_are_not():
    from geoweave_b200 import check_status

    for name, (inputs, call) in _calls().items():
        plain = call(*inputs)
        with forward_ad.dual_level():
            for grad in (True, False):
                with torch.set_grad_enabled(grad):
                    for i in range(len(inputs)):
                        args = list(inputs)
                        args[i] = forward_ad.make_dual(inputs[i], torch.ones_like(inputs[i]))
                        with pytest.raises((NotImplementedError, RuntimeError)):
                            call(*args)
                    again = call(*inputs)  # beside a level that none of them belongs to
        for a, b in zip(*(x if isinstance(x, tuple) else (x,) for x in (plain, again))):
            assert (a is None and b is None) or torch.equal(a, b), name
    check_status()

"""Corners of the training operators: sizes at the ends of their ranges, layouts and transforms outside the usual ones, what the
host does during a call, and results that must not depend on how a launch is divided."""
import pytest
import torch

from icsa_hip import rotary_func, rotary_table

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


# ------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("H", [1 << 20, (1 << 20) - 3])
def test_rotary_of_one_token_with_as_many_heads_as_there_may_be(gpu, H):
    """Every head is written: heads are alike, so each result is the first one's."""
    x = torch.randn(1, 1, 1, 512, device=gpu).to(BF)
    cos, sin = rotary_table(9, 512)
    pos = torch.full((1, 1), 7, dtype=torch.int32, device=gpu)
    want = rotary_func(x, None, cos, sin, pos)
    fill = torch.full((H, 512), float("nan"), dtype=BF, device=gpu)        # what the result's memory may hold
    del fill
    y = rotary_func(x.expand(1, 1, H, 512), None, cos, sin, pos)
    assert bool((y == want).all())


def test_rotary_tables_with_a_tangent_are_refused(gpu):
    """Forward mode, as with q and k."""
    q = torch.randn(1, 5, 2, 64, device=gpu)
    cos, sin = rotary_table(5, 64)
    pos = torch.arange(5, dtype=torch.int32, device=gpu)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual
        for c, s in ((dual(cos, -sin), sin), (cos, dual(sin, cos))):
            for grad in (False, True):
                with pytest.raises(NotImplementedError), torch.set_grad_enabled(grad):
                    rotary_func(q, None, c, s, pos)

"""Top logits and distillation: rows at the edges of what numbers hold, and calls repeated."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, K", [(20, 6), (9000, 40), (20, 300), (20, 3000)])
def test_a_barred_student_whose_teacher_holds_everything_outside_the_list(rows, K):
    """No class is open to the student and the listed classes' shares are too small for a number: the loss is infinite (the rest
    has weight and the student none), not NaN, and the gradient zero."""
    from devis_amd import criterions
    z = torch.zeros((rows, K), device="cuda")
    z[::2] = -math.inf
    z.requires_grad_(True)
    v, i = torch.zeros((rows, 2), device="cuda"), torch.tensor([1, 3], dtype=torch.int32, device="cuda").expand(rows, 2).contiguous()
    rest = torch.full((rows,), 2000.0, device="cuda")
    loss = criterions.distill_top_loss(z, v, i, rest, reduction="none")
    assert (loss[::2] == math.inf).all() and torch.isfinite(loss[1::2]).all()
    (dz,) = torch.autograd.grad(loss, z, torch.ones_like(loss))
    assert (dz[::2] == 0).all() and torch.isfinite(dz).all()
    assert criterions.distill_top_loss(z, v, i, rest).item() == math.inf

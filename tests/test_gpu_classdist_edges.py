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


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, K, k, spread", [(1500, 131072, 64, 2.0), (800, 151936, 128, 2.0), (3000, 40000, 128, 0.01), (100, 262147, 128, 0.5),
                                                (3000, 1031, 100, 1.0), (1000, 20000, 100, 0.0), (2000, 1000, 100, 2.0)])
def test_top_logits_are_the_same_every_time(rows, K, k, spread, dtype):
    """Bit for bit: nothing depends on the order in which waves run, whatever is read again, listed and left over."""
    from devis_amd import ops
    g = torch.Generator(device="cuda").manual_seed(7)
    z = (torch.randn((rows, K), generator=g, device="cuda") * spread).to(dtype)
    z[::3, 100:200] += 30.0                        # more large classes than are kept, side by side
    strided = z[:64].t().contiguous().t()          # and classes that are not adjacent
    first = None
    for _ in range(12):
        out = [ops.top_logits(x, k, temperature=0.7) for x in (z, strided)]
        got = [o[n] for o in out for n in ("values", "indices", "rest")]
        if first is None:
            first = got
        else:
            assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, K, k, T", [(300, 1000, 20, 1.0), (300, 1031, 3, 2.0), (200, 9001, 128, 1.0), (64, 50257, 64, 1.25), (300, 131072, 64, 1.0),
                                           (12, 131073, 8, 4.0), (300, 151936, 64, 1.0), (12, 256000, 32, 2.0), (2, 1100003, 64, 1.0)])
def test_rest_is_as_good_as_its_sums(rows, K, k, T, dtype):
    """Long vocabularies, with vectors and groups that end inside a tile.  A class d T below the largest has an exponential good
    to 3 d E + 2 E, twice (against its group, and its group against all); what counts of it is its weight.  A thread adds
    vectors in turn, 4 classes or more each, as trees.  The logarithm is rounded once."""
    from devis_amd import ops
    E = 2.0 ** -24
    g = torch.Generator(device="cuda").manual_seed(K)
    z = (torch.randn((rows, K), generator=g, device="cuda") * 2).to(dtype)
    z.scatter_add_(1, torch.randint(0, K, (rows, 16), generator=g, device="cuda"), (torch.rand((rows, 16), generator=g, device="cuda") * 12).to(dtype))
    out = ops.top_logits(z, k, temperature=T)
    order = torch.sort(z, dim=1, descending=True, stable=True)
    assert torch.equal(out["indices"].long(), order[1][:, :k]) and torch.equal(out["values"], order[0][:, :k])
    left = order[0][:, k:].double() / T
    want = torch.logsumexp(left, 1)
    weight = (left - want[:, None]).exp()
    far = (weight * (left[:, :1] - left)).sum(1) + (order[0][:, k - 1].double() / T - left[:, 0])
    adds = 16 + K / ((64 if K <= 1024 else 256) * 4)
    tol = (6 * far + adds + 16) * E + want.abs() * E
    assert ((out["rest"].double() - want).abs() <= tol).all(), ((out["rest"].double() - want).abs() / tol).max()

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


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows, K, k", [(8192, 17, 4), (8192, 40, 4), (24576, 256, 4), (24574, 256, 4), (38400, 100, 16), (38398, 100, 16), (98304, 256, 16),
                                        (4096, 1500, 20), (4094, 1500, 20), (4100, 2048, 100), (4096, 4096, 5), (4096, 4098, 5)])
def test_both_sides_of_the_rules_for_short_rows(rows, K, k, dtype, first):
    """A lane a row from here on, a wave a row below; a wave a row and a block a row: the same lists, losses and gradients, as the formulas in 64 bits give them."""
    from devis_amd import criterions, ops
    from tests.test_gpu_classdist_near import exact
    E, T = 2.0 ** -24, 2.0
    g = torch.Generator(device="cuda").manual_seed(K + k)
    t = (torch.randn((rows, K), generator=g, device="cuda") * 2).to(dtype)
    z = (t.float() + torch.randn((rows, K), generator=g, device="cuda")).to(dtype)
    t[5:9] = 0.5                                   # ties: the lowest classes
    z[7:11, K // 2:] = torch.finfo(dtype).min
    put = (lambda x: x.view(2, rows // 2, -1).movedim(-1, 1).contiguous()) if first else lambda x: x
    back = (lambda x: x.movedim(1, -1).reshape(rows, -1)) if first else lambda x: x
    top = ops.top_logits(put(t), k, channels_last=not first, temperature=T)
    order = torch.sort(t, dim=1, descending=True, stable=True)
    v, i, rest = back(top["values"]), back(top["indices"]).long(), top["rest"].reshape(rows)
    assert torch.equal(i, order[1][:, :k]) and torch.equal(v, order[0][:, :k])
    want = torch.logsumexp(order[0][:, k:].double() / T, 1)
    assert ((rest.double() - want).abs() <= (3 * 10 + K / 64 + 16) * E + want.abs() * E).all()
    student = put(z).requires_grad_(True)
    loss = criterions.distill_top_loss(student, top["values"], top["indices"], top["rest"], channels_last=not first, temperature=T, reduction="none")
    (dz,) = torch.autograd.grad(loss, student, torch.ones_like(loss))
    want, tol = (x.to("cuda") for x in exact(z, v, i, rest, T))
    assert ((loss.reshape(rows).double() - want).abs() <= tol).all()
    zd = z.double().requires_grad_(True)
    log_p = torch.log_softmax(torch.cat([v.double() / T, rest.double()[:, None]], 1), 1)
    log_q = torch.log_softmax(zd / T, 1)
    out = torch.logsumexp(log_q.scatter(1, i, -math.inf), 1, keepdim=True)
    kl = (log_p.exp() * (log_p - torch.cat([log_q.gather(1, i), out], 1))).sum() * T * T
    (grad,) = torch.autograd.grad(kl, zd)
    # shares q, p and p_rest of a class are good to their exponents' roundings and their sums', and the type rounds once
    q = log_q.detach().exp()
    scale = q.scatter_add(1, i, log_p[:, :k].exp()) + (q / out.detach().exp()).scatter(1, i, 0.0) * log_p[:, k:].exp()
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    bound = T * scale * (2 * (3 * 20 + K / 64 + 12) + 16) * E + half * grad.abs() + 1e-37
    assert ((back(dz).double() - grad).abs() <= bound).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K, times", [(40, 376), (40, 374), (256, 2400)])
def test_verification_of_many_sequences_of_dozens_of_classes(K, times, dtype):
    """A lane a sequence from here on, a block each below: every copy as the first ones, and those as the oracle says."""
    from devis_amd import ops
    from tests.test_gpu_classdist import check_verify, drafts, many
    tok, p, q, u, r = drafts(41, 3, K, dtype, K, True, torch.int32)
    p[5] = 0.0
    p[8], q[8] = q[8, :1].expand(p.shape[1:]), p[8, :3]
    u[9:20] *= 0.01
    lengths = torch.arange(41) % 4
    for x, n in ((q, None), (q, lengths), (None, lengths)):
        one = check_verify(tok, p, x, u, r, n)
        out = ops.verify_drafts(many(tok, times).cuda(), many(p.cuda(), times), None if x is None else many(x.cuda(), times),
                                many(u, times).cuda(), many(r, times).cuda(), None if n is None else many(n, times).cuda())
        assert torch.equal(out["tokens"], many(one["tokens"], times)) and torch.equal(out["accepted"], many(one["accepted"], times))


@pytest.mark.parametrize("B, K", [(255, 16385), (256, 16385), (2, 16384), (2, 16385), (256, 65537)])
def test_verification_on_both_sides_of_the_rule_for_long_rows(B, K):
    from tests.test_gpu_classdist import check_verify, drafts
    for dtype in (torch.float32, torch.bfloat16):
        tok, p, q, u, r = drafts(B, 2, K, dtype, K)
        check_verify(tok, p, q, u, r)
        check_verify(tok, p, None, u, r, torch.arange(B) % 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N, K, V, k", [(5, 4, 2, 2), (5000, 4, 2, 2), (4097, 7, 3, 3), (300, 16, 31, 16), (300, 16, 32, 16), (9000, 2, 1, 1), (33, 3, 5, 1)])
def test_many_small_images_channels_first(N, K, V, k, dtype):
    """Classes first, few rows side by side: as the same rows one behind the other give it, near enough."""
    from devis_amd import criterions, ops
    from tests.test_gpu_classdist_near import exact
    g = torch.Generator(device="cuda").manual_seed(N)
    t = (torch.randn((N, K, V), generator=g, device="cuda") * 3).to(dtype)
    z = (t.float() + torch.randn((N, K, V), generator=g, device="cuda")).to(dtype).requires_grad_(True)
    mask = torch.rand((N, V), generator=g, device="cuda") < 0.8
    top = ops.top_logits(t, k, channels_last=False, temperature=2.0)
    last = ops.top_logits(t.movedim(1, -1).contiguous(), k, temperature=2.0)
    assert torch.equal(top["values"].movedim(1, -1), last["values"]) and torch.equal(top["indices"].movedim(1, -1), last["indices"])
    assert torch.allclose(top["rest"], last["rest"], rtol=2.0 ** -22, atol=2.0 ** -20)
    rows = lambda x: x.movedim(1, -1).reshape(N * V, -1)
    want, tol = (x.cuda() for x in exact(rows(z.detach()), rows(top["values"]), rows(top["indices"]), top["rest"].reshape(-1), 2.0))
    want, tol = torch.where(mask.view(-1), want, 0.0), torch.where(mask.view(-1), tol, 0.0)
    call = lambda x, **kw: criterions.distill_top_loss(x, top["values"], top["indices"], top["rest"], channels_last=False, temperature=2.0, row_mask=mask, **kw)
    assert ((call(z, reduction="none").reshape(-1).double() - want).abs() <= tol).all()
    loss = call(z, reduction="sum")
    assert abs(loss.item() - want.sum().item()) <= tol.sum().item() + 2.0 ** -23 * want.sum().item()
    (dz,) = torch.autograd.grad(loss, z)
    flat = rows(z.detach()).requires_grad_(True)
    one = criterions.distill_top_loss(flat, rows(top["values"]), rows(top["indices"]), top["rest"].reshape(-1), temperature=2.0, row_mask=mask.reshape(-1), reduction="sum")
    (want,) = torch.autograd.grad(one, flat)
    # each side is within 2 x 12 roundings of its shares (at most 2 in all, times T), and the type's own
    half = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    assert ((rows(dz).double() - want.double()).abs() <= 2 * (2 * 2 * 2 * (3 * 12 + 24) * 2.0 ** -24 + half * want.double().abs())).all()


@pytest.mark.parametrize("N, V", [(6, 2), (6, 40)])
def test_saved_tensors_that_come_back_in_another_layout(N, V):
    """Rows of few classes keep nothing for the backward, whichever layout their tensors come back in."""
    from devis_amd import criterions, ops
    g = torch.Generator(device="cuda").manual_seed(V)
    t = torch.randn((N, V, 4), generator=g, device="cuda")
    z = torch.randn((N, V, 4), generator=g, device="cuda")
    top = ops.top_logits(t, 2)
    got = []
    for unpack in (lambda x: x, lambda x: x.clone(memory_format=torch.contiguous_format) if x.dim() == 3 else x.clone()):
        x = z.clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda s: s, unpack):
            loss = criterions.distill_top_loss(x.movedim(-1, 1), top["values"].movedim(-1, 1), top["indices"].movedim(-1, 1), top["rest"], channels_last=False)
        loss.backward()
        got.append(x.grad)
    assert torch.equal(*got)


@pytest.mark.parametrize("rows, K", [(20, 4), (9000, 12), (9000, 40), (20, 300), (20, 3000)])
def test_a_closed_class_that_the_teacher_hardly_gives(rows, K):
    """A class that is closed to the student makes the loss infinite however little the teacher gives it (e^-120 here, too little for
    fp32), listed or not: in the mean, the sum and row by row."""
    from devis_amd import criterions
    v, i = torch.tensor([0.0, -120.0], device="cuda").expand(rows, 2).contiguous(), torch.tensor([1, 2], dtype=torch.uint8, device="cuda").expand(rows, 2).contiguous()
    z = torch.zeros((rows, K), device="cuda")
    z[:, 2] = -math.inf
    rest = torch.full((rows,), -64.0, device="cuda")
    for reduction in ("mean", "sum", "none"):
        for r in (rest, None):
            assert (criterions.distill_top_loss(z, v, i, r, reduction=reduction) == math.inf).all()
    z[:] = -math.inf
    z[:, 1:3] = 0.0
    for reduction in ("mean", "sum", "none"):
        assert (criterions.distill_top_loss(z, v, i, rest - 60.0, reduction=reduction) == math.inf).all()
        assert torch.isfinite(criterions.distill_top_loss(z, v, i, rest * math.inf, reduction=reduction)).all()


@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("rows, K", [(20, 4), (9000, 12), (9000, 40), (20, 300), (20, 3000)])
def test_a_rest_that_the_student_holds_at_the_lowest_value(rows, K, T):
    """One part in 1e28 of the teacher lies outside the list, where the student's mask left the type's lowest value: that adds T times
    the distance times the share, a number, in the mean and the sum as row by row."""
    from devis_amd import criterions
    low = torch.finfo(torch.float32).min
    v, i = torch.tensor([0.0, -120.0], device="cuda").expand(rows, 2).contiguous(), torch.tensor([1, 2], dtype=torch.uint8, device="cuda").expand(rows, 2).contiguous()
    z = torch.full((rows, K), low, device="cuda")
    z[:, 1], z[:, 2] = 0.0, -120.0
    want = T * math.exp(-64.0) * -float(low)       # and terms of order one, far below its last digit
    for reduction, n in (("mean", 1), ("sum", rows), ("none", 1)):
        loss = criterions.distill_top_loss(z, v, i, torch.full((rows,), -64.0, device="cuda"), temperature=T, reduction=reduction).double()
        # the share is an fp32 exponential of 64 nats (192 E + 3 E); a sum of rows in fp64
        assert ((loss / n - want).abs() <= 200 * 2.0 ** -24 * want).all()

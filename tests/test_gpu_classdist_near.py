"""Distillation of a student near its teacher, and the mean of many rows: what is left when logarithms cancel.

Tolerances.  A row's loss is T^2 times the sum over its classes (the listed ones, and what is left as one) of p (r - 1 - log r),
r = q / p.  With E = 2^-24, an error e_j of log r_j changes that by (q_j - p_j) e_j + p_j e_j^2 / 2.  What is in every e_j of a
row alike (the logarithms of both models' sums) drops out in first order, because the q and the p both sum to one; its square
stays.  Left over are
  of a listed class: the roundings of its two distances from the row's largest, E (|t_j - t_max| + |z_j - z_max|) / T, and 4 E;
  of the rest: its own sum, good to (3 D + adds + 12) E as in test_gpu_classdist.py, with D = the largest distance of a class
    that counts, and adds = the additions one thread makes in turn; and E |rest - t_max / T| and 4 E.
The roundings of shares and terms scale with the loss: 3 E of p and of q, and where the term is q - p - p log r, |log r| >= 1/2, the
magnitudes of what is taken off are at most (q + p + p |log r|) / (p (r - 1 - log r)) <= 20 times it: 24 E with the sums'.  A row's own loss ("none") of few classes is a
difference of logarithms in 64 bits, of an exponential's series that ends at 0.3466^10 / 10! = 7e-12: two sums of them and the
two Newton steps of their logarithms, 3e-11 T^2.
"""
import math

import numpy as np
import pytest
import torch

from oracle import classdist_oracle as O

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def additions(K):
    """Additions that one thread makes in turn: vectors of 4 classes dealt to 64, 256 or 1024 threads (at least), summed as trees."""
    return 8 + K / ((64 if K <= 4096 else 256) * 4)


def exact(z, v, i, rest, T):
    """(rows,) losses in 64 bits and how far off they may be, from the definitions; distinct listed classes."""
    z, t, i = z.double() / T, v.double() / T, i.long()
    k = t.shape[1]
    r = torch.full_like(t[:, 0], -math.inf) if rest is None else rest.double()
    log_p = torch.log_softmax(torch.cat([t, r[:, None]], 1), 1)
    log_q = torch.log_softmax(z, 1)
    out = torch.logsumexp(log_q.scatter(1, i, -math.inf), 1)
    log_q = torch.cat([log_q.gather(1, i), out[:, None]], 1)
    p, q = log_p.exp(), log_q.exp()
    loss = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
    high, top = t.max(1)[0][:, None], z.max(1)[0][:, None]
    near = torch.where(z > top - 110, top - z, torch.zeros_like(z)).max(1)[0]
    sums = (3 * near + additions(z.shape[1]) + 12) * E
    each = torch.cat([(high - t) + (top - z.gather(1, i)) + 4, torch.where(r > -math.inf, (r - high[:, 0]).abs(), torch.zeros_like(r))[:, None] + 4], 1) * E
    each[:, k] += sums
    first = ((q - p).abs() * each).sum(1) + (p * each * each).sum(1) + (2 * sums + 8 * E) ** 2
    if rest is None:                               # the listed q do not sum to one: what they leave out scales what is common
        first = first + q[:, k] * (2 * sums + 8 * E)
    return T * T * loss, T * T * (first + 3e-11) + 24 * E * T * T * loss


def near_pair(rows, K, k, T, noise, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    t = (torch.randn((rows, K), generator=g) * 3).to(dtype)
    z = (t.float() + noise * torch.randn((rows, K), generator=g)).to(dtype)
    order = torch.sort(t.float(), dim=1, descending=True, stable=True)[1]
    v, i = torch.gather(t, 1, order[:, :k]), order[:, :k].to(torch.int32)
    rest = torch.logsumexp(torch.gather(t, 1, order[:, k:]).double() / T, 1).float() if k < K else torch.full((rows,), -math.inf)
    return z, v, i, rest


# rows of few classes; a lane a row; a wave a row; long rows
SHAPES = [(1, 4, 2), (1, 9, 3), (1, 16, 16), (300, 2, 1), (64, 9, 3), (20000, 4, 2), (20000, 7, 3), (20000, 9, 3), (20000, 12, 12),
          (9000, 21, 4), (9000, 40, 40), (9000, 100, 12), (1, 100, 5), (300, 300, 20), (300, 1000, 100), (50, 5003, 20), (8, 33001, 16),
          (300, 9001, 64), (2, 151936, 64), (9700, 100, 4), (25000, 256, 4), (38500, 100, 16), (98400, 256, 9)]


@pytest.mark.parametrize("noise", [0.1, 0.01, 0.001, 0.0])
@pytest.mark.parametrize("T", [1.0, 4.0, 1.3])
@pytest.mark.parametrize("rows, K, k", SHAPES)
def test_a_student_near_its_teacher(rows, K, k, T, noise):
    from devis_amd import criterions
    T = float(np.float32(T))                       # what the kernels are given
    z, v, i, rest = near_pair(rows, K, k, T, noise, torch.float32, K + k)
    args = z.cuda(), v.cuda(), i.cuda()
    for r in (rest, None):
        loss, tol = exact(z, v, i, r, T)
        kw = dict(rest=None if r is None else r.cuda(), temperature=T)
        have = criterions.distill_top_loss(*args, reduction="none", **kw).cpu().double()
        assert (((have - loss).abs() - tol) <= 1e-37).all(), ((have - loss).abs() / tol.clamp_min(1e-37)).max()
        mean = criterions.distill_top_loss(*args, **kw).item()
        assert abs(mean - loss.mean().item()) <= tol.mean().item() + E * loss.mean().item(), (mean, loss.mean().item(), tol.mean().item())
        assert r is None or mean >= 0
        total = criterions.distill_top_loss(*args, reduction="sum", **kw).item()
        assert abs(total - loss.sum().item()) <= tol.sum().item() + E * loss.sum().item()


@pytest.mark.parametrize("rows, K, k", [(20000, 4, 2), (20000, 9, 5), (9000, 40, 6), (300, 1000, 20), (50, 9001, 30)])
def test_the_mean_is_the_mean_of_the_rows(rows, K, k):
    """bf16, classes first: both reductions are within their own bounds of the same 64-bit losses, so of each other."""
    from devis_amd import criterions
    for noise in (1.0, 0.1):
        z, v, i, rest = near_pair(rows, K, k, 4.0, noise, torch.bfloat16, K)
        loss, tol = exact(z, v, i, rest, 4.0)
        put = lambda x: x.view(2, rows // 2, -1).movedim(-1, 1).contiguous().cuda()
        args = put(z), put(v), put(i)
        kw = dict(rest=rest.view(2, -1).cuda(), temperature=4.0, channels_last=False)
        each = criterions.distill_top_loss(*args, reduction="none", **kw).cpu().double().reshape(-1)
        assert ((each - loss).abs() <= tol).all()
        mean = criterions.distill_top_loss(*args, **kw).item()
        assert abs(mean - loss.mean().item()) <= tol.mean().item() + E * loss.mean().item()
        assert abs(mean - each.mean().item()) <= 2 * (tol.mean().item() + E * loss.mean().item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [4, 6, 16, 40, 3000])
def test_odd_rows_one_by_one(K, dtype):
    """Empty and repeated slots, masks of the lowest value, barred classes, nothing left outside the list: each row's sum is
    its own loss, whatever form it takes; a NaN on either side makes it NaN."""
    from devis_amd import criterions
    from tests.test_gpu_classdist import odd_rows, oracle_rows
    z, v, i, r, _, _ = odd_rows(K, dtype)
    for n in range(14):
        one = slice(n, n + 1)
        for rest in (None, r[one]):
            for T in (1.0, 0.25, 3.0):
                want, _, _, _, err = oracle_rows(z[one], v[one], i[one], rest, None, T)
                for reduction in ("sum", "mean"):
                    have = criterions.distill_top_loss(z[one].cuda(), v[one].cuda(), i[one].cuda(), None if rest is None else rest.cuda(),
                                                       temperature=T, reduction=reduction).item()
                    with np.errstate(over="ignore"):
                        assert have == np.float32(want[0]) or abs(have - want[0]) <= err[0] + 24 * E * want[0], (n, T, have, want, err)
    z[6, 0], v[7, 1] = math.nan, math.nan          # among barred classes
    for n in (6, 7):
        one = slice(n, n + 1)
        for rest in (None, r[one].cuda()):
            assert math.isnan(criterions.distill_top_loss(z[one].cuda(), v[one].cuda(), i[one].cuda(), rest).item())


@pytest.mark.parametrize("T", [1.0, 0.25])
@pytest.mark.parametrize("rows, K, k", [(4000, 3, 3), (4000, 5, 2), (4000, 9, 6), (9000, 40, 5), (300, 300, 20), (50, 5003, 20)])
def test_a_class_in_two_slots_of_a_student_near_its_teacher(rows, K, k, T):
    """Two slots p1 > p2 of one class whose share is q: their terms are p1 (r - 1 - log r), r = q / p1, and -p2 - p2 log(q / p2).  Where p2
    is small nothing of it is lost beside q: the error is a few E of each term and second order in what is common."""
    from devis_amd import criterions
    z, v, i, rest = near_pair(rows, K, k, T, 0.0, torch.float32, K)
    i[:, k - 1] = i[:, 0]                          # the last slot, the least share, names the first's class
    v[:, k - 1] = v[:, 0] - T * torch.linspace(0.0, 18.0, rows)
    zt, t = z.double() / T, v.double() / T
    log_p = torch.log_softmax(torch.cat([t, rest.double()[:, None]], 1), 1)
    log_q = torch.log_softmax(zt, 1)
    out = torch.logsumexp(log_q.scatter(1, i.long(), -math.inf), 1, keepdim=True)
    log_q = torch.cat([log_q.gather(1, i.long()), out], 1)
    p, q = log_p.exp(), log_q.exp()
    term = torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)) + q - p
    term[:, k - 1] -= q[:, 0]
    want = T * T * term.sum(1)
    top = zt.max(1)[0][:, None]
    near = torch.where(zt > top - 110, top - zt, torch.zeros_like(zt)).max(1)[0]
    sums = (3 * near + additions(K) + 12) * E      # as in exact()
    each = torch.cat([(t[:, :1] - t) + (top - zt.gather(1, i.long())) + 4, torch.full_like(out, 4.0) + sums[:, None] / E + (rest.double()[:, None] - t[:, :1]).abs().nan_to_num(0, 0, 0)], 1) * E
    change = q - p
    change[:, k - 1] = -p[:, k - 1]
    tol = T * T * ((change.abs() * each).sum(1) + (2 * sums + 8 * E) ** 2 + 3e-11 + 24 * E * term.abs().sum(1)) + E * want.abs()
    args = z.cuda(), v.cuda(), i.cuda(), rest.cuda()
    for reduction in ("none", "rows"):
        if reduction == "none":
            have = criterions.distill_top_loss(*args, temperature=T, reduction="none").cpu().double()
        else:                                      # the form of the mean, row by row
            some = range(0, rows, max(1, rows // 200))
            have = want.clone()
            for n in some:
                have[n] = criterions.distill_top_loss(*(x[n:n + 1] for x in args), temperature=T, reduction="sum").item()
        assert ((have - want).abs() <= tol).all(), (reduction, ((have - want).abs() / tol).max())


@pytest.mark.parametrize("T", [1.5, 3.0, 0.75, 1.3, 48.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K, times", [(6, 1), (16, 700), (40, 2100), (300, 1), (3001, 1)])
def test_a_teacher_of_lowest_values_at_other_temperatures(K, times, dtype, T):
    """A masked teacher's row: its rest is the row's value over T, and so is every slot, to the last digit or far from it; a quotient by
    way of a rounded 1 / T would be 1e22 off and give all to one side."""
    from tests.test_gpu_classdist import check_distill, logits, teacher_of
    T = float(np.float32(T))
    z = logits(4, K, dtype, K, 2.0)
    t = torch.full((4, K), torch.finfo(dtype).min).to(dtype)
    t[1] = torch.finfo(dtype).min / 2
    t[2, :1] = 1.0
    t[3] = -1e30
    if T < 1:
        t[0] /= 16
    for k in {1, 2, 6}:
        v, i, rest = teacher_of(t, k, T)
        for reduction in ("mean", "none"):
            check_distill(z, v, i, rest, None, T, reduction, times=times)

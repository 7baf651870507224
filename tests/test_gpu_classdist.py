"""Top logits, distillation from them and verification of drafted classes on the GPU, against the 64-bit oracle.

Tolerances.  Let e = 2^-24 (fp32) and D = the largest |z - max z| / T that is finite.  An exponential of the kernels is
exp2((z - m) * c): the difference, c and the product are rounded (3e of an exponent of D nats), the exponential itself is
good to 2e: 3 D e + 2e relative.  A thread adds its classes in turn, at most K/64 of them, in groups: (K/64 + 8) e.  So
every sum of exponentials is within S = (3 D + K/64 + 12) e relative, which is also the absolute error of its logarithm.
Teacher's shares are good to 4e relative where they count for something (fp64 and rounded once in most paths, fp32 exponentials
in the gradients of few and of dozens of classes).  Bounds relative to the loss: test_gpu_classdist_near.py.
"""
import math

import numpy as np
import pytest
import torch

from oracle import classdist_oracle as O

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}      # one rounding to the type, relative


def sum_error(z, T, listed=()):
    """Of the sum over a row and, where classes are `listed`, of the sum over the others; classes more than 110 T below
    the largest add nothing (exp(-104) is below the smallest fp32)."""
    z = np.asarray(z, np.float64)
    D = 0.0
    for f in (z, np.delete(z, listed)):
        f = f[np.isfinite(f)]
        if f.size:
            near = f[f >= f.max() - 110 * T]
            D = max(D, (f.max() - near.min()) / T)
    return (3 * D + z.size / 64 + 12) * E


def logits(rows, K, dtype, seed, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, K), generator=g) * spread).to(dtype)


# ------------------------------------------------------------------ top logits
def check_top(z, k, T=1.0, channels_last=True, device_z=None, times=1):
    """z (rows, K) on the CPU as the oracle sees it; device_z the tensor given to the call (default z, `times` over)."""
    from devis_amd import ops
    out = ops.top_logits(torch.cat([z] * times).cuda() if device_z is None else device_z, k, channels_last=channels_last, temperature=T)
    if times > 1:
        for n in out:
            assert torch.equal(out[n].reshape(times, -1).nan_to_num(7.25), out[n].reshape(times, -1)[:1].expand(times, -1).nan_to_num(7.25))
            out[n] = out[n][:z.shape[0]]
    vals, idx, rest = out["values"], out["indices"], out["rest"]
    K = z.shape[1]
    assert vals.dtype == z.dtype and idx.dtype == (torch.uint8 if K <= 256 else torch.int32) and rest.dtype == torch.float32
    if not channels_last:
        vals, idx = vals.movedim(1, -1), idx.movedim(1, -1)
    vals, idx, rest = vals.reshape(-1, k).cpu(), idx.reshape(-1, k).cpu().long(), rest.reshape(-1).cpu().double().numpy()
    zd = z.double().numpy()
    for r in range(z.shape[0]):
        order, want = O.top_row(zd[r], k, T)
        assert np.array_equal(idx[r].numpy(), order), (r, idx[r], order)
        assert torch.equal(vals[r].float().nan_to_num(7.25), z[r][torch.as_tensor(order.copy())].float().nan_to_num(7.25))
        with np.errstate(over="ignore"):
            want32 = np.float32(want)            # -3.4e38 / T is below every fp32 number for T < 1: it rounds to -inf
        if np.isinf(want32):
            assert rest[r] == want32, (r, rest[r], want)
        else:
            left = np.delete(zd[r], order)
            assert abs(rest[r] - want) <= sum_error(left, T) + abs(want) * E, (r, rest[r], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K, k", [(1, 1), (2, 1), (2, 2), (3, 2), (4, 2), (7, 7), (8, 3), (9, 4), (16, 5), (17, 1), (31, 31), (33, 8),
                                  (64, 64), (65, 65), (100, 17), (128, 128), (255, 20), (256, 128), (257, 3), (1000, 128),
                                  (1023, 64), (1024, 1), (1025, 127), (2047, 128), (4099, 8), (33001, 64), (131072, 100)])
def test_top_sizes(K, k, dtype):
    check_top(logits(5, K, dtype, K + k), k, T=1.5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K, times", [(5, 1), (100, 1), (3001, 1), (30, 700)])
def test_top_ties_masks_and_infinities(K, times, dtype):
    inf, low = math.inf, torch.finfo(dtype).min
    rows = [torch.zeros(K),                                         # every class alike: the lowest classes
            torch.arange(K).float() // 7,                           # rising plateaus
            -(torch.arange(K).float() // 3),                        # falling plateaus
            torch.full((K,), -inf),                                 # a mask that leaves nothing
            torch.where(torch.arange(K) % 4 == 1, 0.5, -inf),       # a quarter is left
            torch.where(torch.arange(K) == K - 1, 3.0, -inf),       # one class is left
            torch.full((K,), low),
            torch.where(torch.arange(K) < 2, 1.0, low),
            torch.where(torch.arange(K) == 3, math.nan, 0.25),      # NaN orders as +inf
            torch.where(torch.arange(K) >= K - 2, inf, -1.0),
            torch.where(torch.arange(K) % 2 == 0, 0.0, -0.0),       # the zeros are equal
            torch.where(torch.arange(K) < 3, 300.0, -torch.arange(K) / K)]      # the rest far below the listed
    z = torch.stack([r.expand(K).float() for r in rows]).to(dtype)
    for k in (1, 3, 5):
        check_top(z, k, times=times)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("below", [-200.0, -3.0e4, torch.finfo(torch.float32).min, -math.inf])
@pytest.mark.parametrize("K, k", [(300, 2), (1000, 5), (3001, 2), (9001, 7), (40000, 2), (40000, 20)])
def test_top_large_classes_side_by_side(K, k, below, dtype):
    """Many more large classes than are kept, next to each other, all others far below: what is left of them is the rest,
    though it lies far above what the other threads hold."""
    g = torch.Generator().manual_seed(K + k)
    low = max(below, torch.finfo(dtype).min) if below > -math.inf else below
    z = torch.full((4, K), low) + (torch.randn((4, K), generator=g) * 4 if abs(low) < 1e5 else 0.0)
    for r, (at, n) in enumerate([(96, 8), (100, 24), (0, 64), (K - 25, 25)]):
        z[r, at:at + n] = torch.randn(n, generator=g) * 3
    z = z.to(dtype)
    check_top(z, k)
    check_top(z, k, T=0.25)
    check_top(z, k, channels_last=False, device_z=z.t().contiguous().cuda()[None].expand(1, K, 4).contiguous())


def test_top_all_infinite_rows():
    check_top(torch.full((2, 600), math.inf), 3)
    check_top(torch.full((2, 600), math.nan, dtype=torch.bfloat16), 3)


@pytest.mark.parametrize("descending", [True, False])
@pytest.mark.parametrize("dtype, K", [(torch.float32, 60001), (torch.bfloat16, 5000)])
def test_top_sorted_rows(dtype, K, descending):
    z = torch.arange(K).float() / K * 8
    z = (z.flip(0) if descending else z).to(dtype)[None]
    for k in (1, 64, 128):
        check_top(z, k)


def test_top_more_large_classes_than_the_list_holds():
    """All large classes fall to the same threads, so the threshold of the first pass keeps far more than k of them."""
    K = 600001
    z = torch.where(torch.arange(K) % 1024 < 4, torch.arange(K) / K + 5.0, -torch.arange(K) / K)[None]
    for k in (2, 3, 100):
        check_top(z, k)
    z = torch.where(torch.arange(K) % 1024 < 4, 5.0, 0.0)[None]             # and all of them alike
    check_top(z, 40)


def test_top_layouts_and_strides():
    g = torch.Generator().manual_seed(5)
    for shape in ((2, 3, 5, 4, 6), (3, 7, 9), (2, 300, 4, 3)):
        x = torch.randn(shape, generator=g)
        for dtype in (torch.float32, torch.bfloat16):
            xd = x.to(dtype).cuda()
            rows = x.to(dtype).movedim(1, -1).reshape(-1, shape[1])
            k = min(3, shape[1])
            check_top(rows, k, channels_last=False, device_z=xd)
            check_top(rows, k, device_z=xd.movedim(1, -1))
            check_top(rows, k, channels_last=False, device_z=xd.movedim(1, -1).contiguous().movedim(-1, 1))
    wide = torch.randn((6, 5003), generator=g).to(torch.bfloat16)
    check_top(wide[:, 1:4002], 9, device_z=wide.cuda()[:, 1:4002])            # rows at odd addresses
    check_top(wide[::2, ::3], 9, device_z=wide.cuda()[::2, ::3])
    check_top(wide[:1].expand(4, 5003), 5, device_z=wide.cuda()[:1].expand(4, 5003))
    check_top(wide[0][None], 5, device_z=wide.cuda()[0])
    v = torch.randn((2, 4, 6, 5, 4), generator=g).cuda()
    check_top(v[:, :, ::2, 1:].cpu().movedim(1, -1).reshape(-1, 4), 2, channels_last=False, device_z=v[:, :, ::2, 1:])


def test_top_without_rest_and_without_rows():
    from devis_amd import ops
    z = logits(3, 50, torch.float32, 1).cuda()
    a, b = ops.top_logits(z, 4), ops.top_logits(z, 4, want_rest=False)
    assert b["rest"] is None and torch.equal(a["indices"], b["indices"]) and torch.equal(a["values"], b["values"])
    e = ops.top_logits(z[:0], 4)
    assert e["values"].shape == (0, 4) and e["rest"].shape == (0,)


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K, k", [(5, 3), (17, 1), (37, 4), (64, 5), (100, 16), (256, 7), (300, 6), (37, 20)])
def test_top_many_rows(K, k, dtype, first):
    """More rows than blocks run at once, all of them against sorting; bf16 rows hold many ties."""
    from devis_amd import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    z = torch.randn((9, 8001, K), generator=g, device="cuda").to(dtype)
    z[0, :, K // 2:] = -math.inf
    z[1, :, 3:] = 1.0
    z[2] = z[2].float().round().to(dtype)
    z[3, :, ::3] = torch.finfo(dtype).min
    order = torch.sort(z, dim=-1, descending=True, stable=True)
    want = torch.logsumexp(order[0][..., k:].double(), -1)
    out = ops.top_logits(z.movedim(-1, 1).contiguous() if first else z, k, channels_last=not first)
    vals, idx = (x.movedim(1, -1) if first else x for x in (out["values"], out["indices"]))
    assert torch.equal(idx.long(), order[1][..., :k]) and torch.equal(vals, order[0][..., :k])
    off = (out["rest"].double() - want).abs()
    off = torch.where(out["rest"].double() == want, torch.zeros_like(off), off)
    assert (off / (1 + want.abs())).max().item() < (3 * 12 + K / 64 + 13) * E


# ------------------------------------------------------------------ distillation
def oracle_rows(z, v, i, rest, mask, T):
    z, v, i = z.double().numpy(), v.double().numpy(), i.numpy()
    rows = len(z)
    loss, grad, counted = np.zeros(rows), np.zeros(z.shape), np.zeros(rows, bool)
    scale, err = np.zeros(z.shape), np.zeros(rows)
    for r in range(rows):
        if mask is not None and not mask[r]:
            continue
        rr = None if rest is None else float(rest[r])
        loss[r], grad[r], counted[r] = O.distill_row(z[r], v[r], i[r], rr, T)
        if not counted[r] or np.isnan(loss[r]):
            continue
        scale[r] = O.distill_scale(z[r], v[r], i[r], rr, T)
        if not np.isfinite(loss[r]):
            continue
        # two logarithms of sums, shares wrong by 4e of what they multiply, one rounding at the end
        log_p = O._log_softmax(np.append(v[r] / T, -np.inf if rr is None else rr))
        log_q = O._log_softmax(z[r] / T)[i[r][v[r] > -np.inf]]
        p = np.exp(log_p)
        far = np.abs(log_p[p > 0]).max() + np.abs(log_q[np.isfinite(log_q)]).max()
        err[r] = T * T * (2 * sum_error(z[r], T, i[r][v[r] > -np.inf]) + 8 * E * far) + E * abs(loss[r])
    return loss, grad, counted, scale, err


def check_distill(z, v, i, rest=None, mask=None, T=1.0, reduction="mean", layout=None, g=0.7, times=1):
    """z (rows, K), v, i (rows, k) on the CPU.  `layout`: (rows, c) CPU tensor -> what the call takes, channels_last.
    `times`: the rows are given that often, one lot behind the other."""
    from devis_amd import criterions
    last, put = (True, lambda x: x) if layout is None else layout
    out = oracle_rows(z, v, i, rest, mask, T)
    loss, grad, counted, scale, err = (np.concatenate([x] * times) for x in out)
    z, v, i, rest, mask = (None if x is None else torch.cat([x] * times) for x in (z, v, i, rest, mask))
    zd = put(z).cuda().detach().requires_grad_(True)
    one = lambda x: None if x is None else put(x[:, None]).select(-1 if last else 1, 0).cuda()
    got = criterions.distill_top_loss(zd, put(v).cuda(), put(i).cuda(), one(rest), last, T, one(mask), reduction)
    assert got.dtype == torch.float32
    n = max(int(counted.sum()), 1)
    if reduction == "none":
        up = torch.linspace(0.2, 1.2, z.shape[0], dtype=torch.float32)
        dz = torch.autograd.grad(got, zd, one(up).reshape(got.shape))[0]
        have = got.detach().cpu().double().reshape(-1).numpy()
        ok = np.isfinite(loss)
        assert np.all(np.abs(have[ok] - loss[ok]) <= err[ok]), np.abs(have[ok] - loss[ok]).max()
        assert np.array_equal(have[~ok], loss[~ok], equal_nan=True)
        f = up.double().numpy()[:, None]
    else:
        dz = torch.autograd.grad(got, zd, torch.tensor(g, device="cuda"))[0]
        want = loss.sum() / (n if reduction == "mean" else 1)
        tol = err.sum() / (n if reduction == "mean" else 1) + E * abs(want)
        with np.errstate(over="ignore"):
            rounded = float(np.float32(want))          # the loss is fp32: a sum past 3.4e38 is infinite
        assert np.isnan(want) and math.isnan(got.item()) or abs(got.item() - want) <= tol or got.item() == rounded, (got.item(), want, tol)
        f = np.full((z.shape[0], 1), float(np.float32(g)) / (n if reduction == "mean" else 1))
    assert dz.dtype == z.dtype and dz.shape == zd.shape
    d = (dz if last else dz.movedim(1, -1)).reshape(z.shape).cpu().double().numpy()
    want = grad * f
    listed = [np.unique(a[(b > -np.inf).numpy() & (a >= 0).numpy() & (a < z.shape[1]).numpy()].numpy()) for a, b in zip(i.long(), v)]
    sums = {}
    for r in range(z.shape[0]):
        # q, the shares and the factor of the row: a sum, an exponential and four roundings each; then the type's
        n = r % (z.shape[0] // times)
        if n not in sums:
            sums[n] = 2 * sum_error(z[r].double().numpy(), T, listed[r]) + 8 * E
        tol = np.abs(f[r]) * scale[r] * sums[n] + HALF[z.dtype] * np.abs(want[r]) + 1e-37
        if np.isnan(loss[r]):
            assert np.isnan(d[r]).all()
        else:
            assert np.all(np.abs(d[r] - want[r]) <= tol), (r, np.abs(d[r] - want[r]).max(), tol[np.abs(d[r] - want[r]).argmax()])
    return got, dz


def teacher_of(t, k, T, itype=torch.int32):
    rows = [O.top_row(r, k, T) for r in t.double().numpy()]
    i = torch.as_tensor(np.stack([r[0] for r in rows]))
    return torch.gather(t, 1, i), i.to(itype), torch.tensor([r[1] for r in rows], dtype=torch.float32)


def pair(rows, K, k, T, dtype, seed, itype=torch.int32, vtype=None):
    t = logits(rows, K, vtype or dtype, seed)
    z = (t.float() + logits(rows, K, torch.float32, seed + 1, 1.0)).to(dtype)
    return (z,) + teacher_of(t, k, T, itype)


SIZES = [(1, 1), (2, 1), (2, 2), (3, 2), (4, 2), (7, 3), (8, 8), (9, 1), (10, 4), (16, 16), (17, 5), (33, 33), (64, 20), (100, 65),
         (255, 7), (257, 128), (1000, 30), (1024, 128), (1025, 3), (2051, 100), (8191, 64), (33001, 16), (131073, 64)]


@pytest.mark.parametrize("rest", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K, k", SIZES)
def test_distill_sizes(K, k, dtype, rest):
    z, v, i, r = pair(5, K, k, 2.0, dtype, 3 * K + k)
    check_distill(z, v, i, r if rest else None, T=2.0, reduction="none")
    check_distill(z, v, i, r if rest else None, T=2.0)


@pytest.mark.parametrize("itype", [torch.uint8, torch.int32, torch.int64])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_distill_types_masks_reductions(itype, reduction):
    for K, k, T in ((4, 2, 1.0), (10, 3, 4.0), (200, 40, 0.5)):
        z, v, i, r = pair(12, K, k, T, torch.bfloat16, K, itype, torch.float32)
        mask = torch.arange(12) % 3 != 1
        for m in (mask, mask.to(torch.uint8) * 5, torch.zeros(12, dtype=torch.bool)):
            check_distill(z, v, i, r, m, T, reduction)
            check_distill(z, v, i, None, m, T, reduction)


@pytest.mark.parametrize("K", [6, 40, 3000])
def test_distill_empty_slots_masked_classes_and_bad_rows(K):
    z, v, i, r, r8, ok = odd_rows(K, torch.float32)
    for rest in (None, r8):
        check_distill(z, v, i, rest, None, 1.0, "none")
    check_distill(z, v, i, r8, ok, 1.0, "mean")
    # masked rows may hold anything
    z[6], v[7], i[8] = math.nan, math.nan, 2 ** 30
    check_distill(z, v, i, r8, ok, 1.0, "mean")


def odd_rows(K, dtype):
    """Fourteen rows of what can go wrong, and which of them have finite losses."""
    inf = math.inf
    z, v, i, r = pair(14, K, 4, 1.0, dtype, K)
    low = torch.finfo(dtype).min
    v[1, 2:] = -inf                                # a short list
    v[2] = -inf                                    # no list: not counted
    i[2] = 2 ** 30
    i[1, 3] = -5                                   # an empty slot's class is not looked at
    v[3, 0] = -inf                                 # an empty slot in front
    z[4, :] = low                                  # the student's mask: the lowest value everywhere
    z[5, 1:] = low
    z[6, i[6].long()] = -inf                       # listed classes the student may not use: infinite loss, finite gradient
    z[7, :] = -inf
    keep = torch.zeros(K, dtype=torch.bool)
    keep[i[8].long()] = True
    z[8, ~keep] = -inf                             # nothing is left outside the list
    v[8], i[8] = v[8], i[8]
    i[9, 1] = i[9, 0]                              # a class in two slots
    i[10] = i[10, 0]
    z[11, i[11].long()] += 200.0                   # the rest far below
    z[12, i[12].long()] -= 200.0                   # the list far below
    r[13] = -inf                                   # no rest in this row
    ok = torch.ones(14, dtype=torch.bool)
    ok[6] = ok[7] = ok[8] = False
    return z, v, i, r, r.clone(), ok


LANES = 586                                        # 14 rows 586 times: enough rows for one thread each


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [17, 31, 64, 100, 256])
def test_distill_many_rows_of_some_classes(K, dtype, first):
    layout = (False, lambda x: x.view(14, -1, x.shape[1]).movedim(-1, 1).contiguous()) if first else None
    z, v, i, r, r8, ok = odd_rows(K, dtype)
    for rest in (None, r8):
        check_distill(z, v, i, rest, None, 1.0, "none", layout, times=LANES)
    check_distill(z, v, i, r8, ok, 1.0, "mean", layout, times=LANES)
    z[6], v[7], i[8] = math.nan, math.nan, 2 ** 30
    check_distill(z, v, i, r8, ok, 1.0, "sum", layout, times=LANES)
    i[9, 1], i[10, 3] = K, -1                      # filled slots that name no class
    check_distill(z, v, i, r8, ok, 1.0, "none", layout, times=LANES)
    for k, T in ((1, 3.0), (16, 2.0)):
        z, v, i, r = pair(14, K, k, T, dtype, K, torch.int64)
        check_distill(z, v, i, r, None, T, "none", layout, times=LANES)


@pytest.mark.parametrize("K", [5, 3000])
def test_distill_makes_bad_rows_nan(K):
    z, v, i, r = pair(6, K, 3, 1.0, torch.float32, K)
    i[1, 1] = K
    i[2, 0] = -1
    got, dz = check_distill(z, v, i, r, None, 1.0, "none")
    assert torch.isnan(got[1]) and torch.isnan(got[2]) and torch.isfinite(got[0])
    i64 = i.long()
    i64[3, 2] = 2 ** 40
    got, _ = check_distill(z, v, i64, None, None, 1.0, "none")
    assert torch.isnan(got[3])
    for bad in (math.nan, math.inf):
        z2 = z.clone()
        z2[4, K - 1] = bad
        from devis_amd import criterions
        out = criterions.distill_top_loss(z2.cuda(), v.cuda(), i.cuda(), reduction="none")
        assert torch.isnan(out[4]) and torch.isfinite(out[5])


@pytest.mark.parametrize("T", [0.25, 1.0, 8.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K, times", [(2, 1), (6, 1), (16, 700), (40, 1), (40, 2100), (1001, 1), (3001, 1), (20000, 1)])
def test_distill_teacher_of_lowest_values(K, times, dtype, T):
    """A teacher's row that its mask left at the type's lowest value: the listed classes and the rest share alike, as what
    the call is given says (rest is fp32: ln K is lost in it)."""
    z = logits(4, K, dtype, K, 2.0)
    t = torch.full((4, K), torch.finfo(dtype).min / 16).to(dtype)      # its quotient by 1/4 is still a fp32 number
    t[2, :1] = 1.0
    t[3] = -1e30
    for k in {1, 2, min(K, 6)}:
        v, i, rest = teacher_of(t, k, T)
        for reduction in ("mean", "none"):
            check_distill(z, v, i, rest, None, T, reduction, times=times)
            check_distill(z, v, i, None, None, T, reduction, times=times)


@pytest.mark.parametrize("rows, K", [(50, 6), (9000, 40), (50, 40), (5, 3000)])
@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_distill_slots_rewritten_before_the_backward(rows, K, itype):
    """A replayed graph's backward may meet other slots than its forward did: nothing is written for a class that is none,
    and the other rows' gradients are as they were."""
    from devis_amd import ops
    z, v, i, rest = pair(rows, K, 3, 1.0, torch.float32, K, itype)
    params, dev, shape, ts = ops.distill_params(z.cuda(), v.cuda(), i.cuda(), rest.cuda(), None, True, 1.0, False)
    _, scratch = ops.distill_fwd(params, dev, shape, ts[0], False, True)
    g = torch.ones((), device=dev)
    before = ops.distill_bwd(params, dev, ts[0], True, scratch, g, False)
    assert before.isfinite().all()
    ts[2][::7, 1] = K
    ts[2][1::7, 0] = -1
    after = ops.distill_bwd(params, dev, ts[0], True, scratch, g, False)
    same = torch.tensor([r % 7 > 1 for r in range(rows)])
    assert torch.equal(before[same.cuda()], after[same.cuda()])


def test_distill_layouts():
    first = lambda *sp: (False, lambda x: x.view(2, *sp, x.shape[1]).movedim(-1, 1).contiguous())
    view = lambda *sp: (False, lambda x: x.view(2, *sp, x.shape[1]).movedim(-1, 1))
    last = lambda *sp: (True, lambda x: x.view(2, *sp, x.shape[1]))
    odd = lambda *sp: (True, lambda x: torch.cat([x, x[:, :1]], 1).view(2, *sp, x.shape[1] + 1)[..., :-1])
    for K, k in ((4, 2), (10, 5), (21, 4), (300, 9)):
        for dtype in (torch.float32, torch.bfloat16):
            z, v, i, r = pair(2 * 3 * 4 * 5, K, k, 2.0, dtype, K)
            mask = torch.arange(z.shape[0]) % 7 != 3
            for layout in (first(3, 4, 5), view(3, 4, 5), last(3, 4, 5), odd(3, 4, 5), first(60), last(12, 5)):
                check_distill(z, v, i, r, mask, 2.0, "mean", layout)
            check_distill(z, v, i, None, None, 2.0, "none", first(4, 15))


def test_distill_gradient_against_differences():
    """Central differences of the kernel's own losses: h^2/6 of the third derivative (at most T^2/T^3 = 1/2 here) plus the
    losses' rounding over h."""
    from devis_amd import criterions
    z, v, i, r = pair(1, 9, 3, 2.0, torch.float32, 4)
    h = 2.0 ** -5
    for rest in (r, None):
        base = z.expand(18, 9).clone()
        for c in range(9):
            base[c, c] += h
            base[9 + c, c] -= h
        ex = lambda x: x.expand(18, *x.shape[1:]).cuda()
        losses = criterions.distill_top_loss(base.cuda(), ex(v), ex(i), None if rest is None else ex(rest), temperature=2.0,
                                             reduction="none").cpu().double()
        zd = z.cuda().requires_grad_(True)
        l = criterions.distill_top_loss(zd, v.cuda(), i.cuda(), None if rest is None else rest.cuda(), temperature=2.0, reduction="sum")
        l.backward()
        diff = (losses[:9] - losses[9:]) / (2 * h)
        tol = h * h / 6 * 0.5 + 4 * (2 * sum_error(base.numpy(), 2.0) + 100 * E) / h
        assert (zd.grad.cpu().double()[0] - diff).abs().max().item() <= tol


def test_distill_broadcast_and_shared_logits():
    """Logits expanded over rows: autograd adds the rows' gradients; logits used twice: the two gradients add up."""
    from devis_amd import criterions
    z, v, i, r = pair(6, 50, 5, 1.0, torch.float32, 8)
    one = z[:1].cuda().requires_grad_(True)
    criterions.distill_top_loss(one.expand(6, 50), v.cuda(), i.cuda(), r.cuda(), reduction="sum").backward()
    _, grad, _, scale, _ = oracle_rows(z[:1].expand(6, 50), v, i, r, None, 1.0)
    tol = scale.sum(0) * (2 * sum_error(z[0].numpy(), 1.0) + 24 * E) + E * 8
    assert np.all(np.abs(one.grad.cpu().double().numpy()[0] - grad.sum(0)) <= tol)
    zd = z.cuda().requires_grad_(True)
    a = criterions.distill_top_loss(zd, v.cuda(), i.cuda(), r.cuda(), reduction="sum")
    b = criterions.distill_top_loss(zd, v.cuda(), i.cuda(), r.cuda(), reduction="sum")
    (a + b).backward()
    ref = torch.autograd.grad(criterions.distill_top_loss(zd, v.cuda(), i.cuda(), r.cuda(), reduction="sum"), zd)[0]
    assert torch.equal(zd.grad, 2 * ref)


def test_distill_without_rows_and_without_gradient():
    from devis_amd import criterions
    z, v, i, r = pair(3, 20, 2, 1.0, torch.float32, 8)
    zd = z.cuda()[:0].requires_grad_(True)
    loss = criterions.distill_top_loss(zd, v.cuda()[:0], i.cuda()[:0])
    loss.backward()
    assert loss.item() == 0 and zd.grad.shape == (0, 20)
    with torch.no_grad():
        a = criterions.distill_top_loss(z.cuda().requires_grad_(True), v.cuda(), i.cuda())
    assert not a.requires_grad
    assert torch.equal(a, criterions.distill_top_loss(z.cuda(), v.cuda(), i.cuda()))


def test_distill_saved_tensors_moved_to_the_host_and_back():
    from devis_amd import criterions
    z, v, i, r = pair(7, 3001, 9, 1.0, torch.bfloat16, 8)
    wide = torch.cat([z, z[:, :2]], 1).cuda()
    want = None
    for moved in (False, True):
        zd = wide.clone().requires_grad_(True)
        if moved:
            with torch.autograd.graph.save_on_cpu():
                loss = criterions.distill_top_loss(zd[:, :3001], v.cuda(), i.cuda(), r.cuda())
        else:
            loss = criterions.distill_top_loss(zd[:, :3001], v.cuda(), i.cuda(), r.cuda())
        junk = torch.full((4_000_000,), 7.0, device="cuda")
        loss.backward()
        del junk
        if want is None:
            want = zd.grad
        else:
            assert torch.equal(want, zd.grad)


def test_distill_saved_tensors_come_back_far_apart():
    """Rows of few classes keep nothing for the backward; where hooks return them further apart than the kernels of few
    classes reach, they are brought together."""
    from devis_amd import criterions
    z, v, i, r = pair(5, 4, 2, 1.0, torch.float32, 11)
    dev = [x.cuda() for x in (z, v, i, r)]

    def back(t):
        if t.shape != z.shape:
            return t
        far = torch.zeros(5 * ((1 << 20) + 8), device="cuda", dtype=t.dtype).as_strided(t.shape, ((1 << 20) + 8, 1))
        return far.copy_(t)

    got = []
    for unpack in (lambda t: t, back):
        x = dev[0].clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            loss = criterions.distill_top_loss(x, dev[1], dev[2], dev[3])
        loss.backward()
        got.append(x.grad)
    assert torch.equal(*got)


def test_distill_refuses_a_second_derivative():
    from devis_amd import criterions
    z, v, i, r = pair(3, 20, 2, 1.0, torch.float32, 8)
    zd = z.cuda().requires_grad_(True)
    loss = criterions.distill_top_loss(zd, v.cuda(), i.cuda(), r.cuda())
    (g,) = torch.autograd.grad(loss, zd, create_graph=True)
    (plain,) = torch.autograd.grad(criterions.distill_top_loss(zd, v.cuda(), i.cuda(), r.cuda()), zd)
    assert torch.equal(g.detach(), plain)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_distill_is_reproducible():
    from devis_amd import criterions
    z, v, i, r = pair(300, 2000, 20, 1.0, torch.bfloat16, 8)
    runs = []
    for _ in range(3):
        zd = z.cuda().requires_grad_(True)
        loss = criterions.distill_top_loss(zd, v.cuda(), i.cuda(), r.cuda())
        loss.backward()
        runs.append((loss.detach(), zd.grad))
    assert all(torch.equal(runs[0][0], b[0]) and torch.equal(runs[0][1], b[1]) for b in runs[1:])


# ------------------------------------------------------------------ verification
def check_verify(tok, p, q, u, r, lengths=None, cuda=lambda x: x.cuda()):
    from devis_amd import ops
    got = ops.verify_drafts(tok.cuda(), cuda(p), None if q is None else cuda(q), u.cuda(), r.cuda(),
                            None if lengths is None else lengths.cuda())
    assert got["tokens"].dtype == tok.dtype and got["accepted"].dtype == tok.dtype
    have, acc = got["tokens"].cpu().numpy(), got["accepted"].cpu().numpy()
    pd, qd = p.double().numpy(), None if q is None else q.double().numpy()
    for b in range(tok.shape[0]):
        n = tok.shape[1] if lengths is None else int(lengths[b])
        want, a = O.verify_row(tok[b].numpy(), pd[b], None if qd is None else qd[b], u[b].double().numpy(), float(r[b]), n)
        assert acc[b] == a and np.array_equal(have[b], want), (b, have[b], want, acc[b], a)
    return got


def drafts(B, T, K, dtype, seed, bonus=True, tdt=torch.int64, near=0.7):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn((B, T + int(bonus), K), generator=g) * 2
    p = torch.softmax(z, -1).to(dtype)
    q = torch.softmax(z[:, :T] + near * torch.randn((B, T, K), generator=g), -1).to(dtype)
    tok = torch.multinomial(q.float().reshape(B * T, K), 1, generator=g).view(B, T).to(tdt) if T else torch.zeros((B, 0), dtype=tdt)
    return tok, p, q, torch.rand((B, T), generator=g), torch.rand((B,), generator=g)


@pytest.mark.parametrize("bonus", [True, False])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B, T, K", [(1, 1, 1), (3, 1, 2), (40, 1, 4), (40, 1, 7), (9, 3, 10), (7, 2, 31), (7, 2, 33), (5, 5, 64),
                                     (5, 4, 65), (6, 1, 257), (4, 3, 1000), (3, 2, 4097), (2, 70, 130), (2, 130, 9), (2, 2, 33001),
                                     (3, 1, 131072)])
def test_verify_sizes(B, T, K, dtype, bonus):
    for tdt in (torch.int64, torch.int32):
        tok, p, q, u, r = drafts(B, T, K, dtype, K + T, bonus, tdt)
        check_verify(tok, p, q, u, r)
        check_verify(tok, p, None, u, r)
        check_verify(tok, p, q, u * 0.01, r)                # nearly everything accepted
        lengths = torch.arange(B) % (T + 1)
        check_verify(tok, p, q, u, r, lengths)
        check_verify(tok, p, None, u * 0.01, r, lengths.to(torch.int32))


def many(x, times):
    return None if x is None else torch.cat([x] * times)


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("K", [4, 17, 40, 100, 256])
def test_verify_many_sequences(K, dtype, strided):
    """The same sequences many times over: a thread each; every copy as the first ones, and those as the oracle says."""
    from devis_amd import ops
    times = 200
    put = (lambda x: x.cuda().movedim(2, 0).contiguous().movedim(0, 2)) if strided else (lambda x: x.cuda())
    for bonus in (True, False):
        tok, p, q, u, r = drafts(41, 3, K, dtype, K, bonus, torch.int32)
        p[5] = 0.0
        p[8], q[8] = q[8, :1].expand(p.shape[1:]), p[8, :3]
        lengths = torch.arange(41) % 4
        for x, n in ((q, None), (q, lengths), (None, lengths)):
            one = check_verify(tok, p, x, u, r, n)
            out = ops.verify_drafts(many(tok, times).cuda(), put(many(p, times)), None if x is None else put(many(x, times)),
                                    many(u, times).cuda(), many(r, times).cuda(), None if n is None else many(n, times).cuda())
            assert torch.equal(out["tokens"], many(one["tokens"], times)) and torch.equal(out["accepted"], many(one["accepted"], times))


@pytest.mark.parametrize("K", [4, 40, 5000])
def test_verify_borders(K):
    tok, p, q, u, r = drafts(12, 2, K, torch.float32, K)
    r[0], r[1], r[2] = 0.0, 1.0 - 2.0 ** -24, 1.0            # the first class with weight, the last, and past the end
    u[3], u[4] = 0.0, 1.0
    p[5] = 0.0                                               # nothing to draw from
    tok[6, 0], tok[7, 0] = -1, K                             # not classes
    p[8] = q[8, :1].expand(3, K)                             # the same distribution: u < 1 is accepted
    q[8] = p[8, :2]
    p[9] = 0.0
    p[9, :, K - 1] = 1.0                                     # one class
    p[10, 0], u[10, 0] = q[10, 0] * 0.5, 0.9                 # the target below the drafter everywhere: nothing is left over
    p[11, 0, 1:] = math.nan
    for lengths in (None, torch.tensor([0, 1, 2, 0, 1, 2, 2, 2, 2, 1, 2, 2]), torch.full((12,), 99), torch.full((12,), -3)):
        for x in (q, None):
            check_verify(tok, p, x, u, r, lengths)


def test_verify_random_numbers_that_are_none():
    for K in (4, 900):
        tok, p, q, u, r = drafts(6, 2, K, torch.float32, K)
        u[0], r[1] = math.nan, math.nan                      # never accepted; the last class with weight
        q[2, 0, ::2] = math.nan
        check_verify(tok, p, q, u, r)
        check_verify(tok, p, None, u, r)


def test_verify_without_drafts_draws_from_the_target():
    tok, p, q, u, r = drafts(50, 0, 300, torch.float32, 3)
    check_verify(tok, p, q, u, r)
    check_verify(tok, p, None, u, r)


def test_verify_strides():
    tok, p, q, u, r = drafts(6, 3, 700, torch.bfloat16, 3)
    check_verify(tok, p, q, u, r, cuda=lambda x: x.cuda().movedim(1, 0).contiguous().movedim(0, 1))
    check_verify(tok, p, q, u, r, cuda=lambda x: x.cuda().movedim(2, 0).contiguous().movedim(0, 2))
    check_verify(tok, p, q, u, r, cuda=lambda x: torch.cat([x, x], -1).cuda()[..., :700])
    check_verify(tok, p[:, :, ::3].contiguous(), q[:, :, ::3].contiguous(), u, r)
    check_verify(tok % 233, p[:, :, 1::3], q[:, :, 1::3], u, r, cuda=lambda x: x.cuda())
    # a volume's classes first: voxels are sequences of one draft
    tok, p, q, u, r = drafts(60, 1, 4, torch.float32, 3, bonus=False)
    check_verify(tok, p, q, u, r, cuda=lambda x: x.cuda()[:, 0].t().contiguous().t().unsqueeze(1))
    # one row of probabilities for all sequences
    tok, p, q, u, r = drafts(6, 1, 40, torch.float32, 3, bonus=False)
    p, q = p[:1].expand(6, 1, 40), q[:1].expand(6, 1, 40)
    check_verify(tok, p, q, u, r, cuda=lambda x: x[:1].cuda().expand(6, 1, 40))


@pytest.mark.parametrize("K", [4, 40])
def test_verify_lengths_of_another_type_are_clamped_before_they_are_cast(K):
    from devis_amd import ops
    tok, p, q, u, r = drafts(5, 3, K, torch.float32, K, True, torch.int32)
    args = tok.cuda(), p.cuda(), q.cuda(), (u * 0.01).cuda(), r.cuda()
    far = ops.verify_drafts(*args, torch.tensor([2 ** 32, 2 ** 32 + 1, 2 ** 40, -2 ** 32 + 2, 2]).cuda())
    near = ops.verify_drafts(*args, torch.tensor([3, 3, 3, 0, 2], dtype=torch.int32).cuda())
    assert torch.equal(far["tokens"], near["tokens"]) and torch.equal(far["accepted"], near["accepted"])


def test_verify_no_sequences():
    from devis_amd import ops
    tok, p, q, u, r = [x.cuda()[:0] for x in drafts(2, 2, 5, torch.float32, 3)]
    out = ops.verify_drafts(tok, p, q, u, r)
    assert out["tokens"].shape == (0, 3) and out["accepted"].shape == (0,)


def test_verify_frequencies():
    """Drawn over a grid of both random numbers the answers follow the target: each class within a grid step."""
    from devis_amd import ops
    K, n = 5, 256
    g = torch.Generator().manual_seed(0)
    p, q = torch.softmax(torch.randn((2, K), generator=g), -1).double()
    u = (torch.arange(n).float() + 0.5) / n
    uu, rr = torch.meshgrid(u, u, indexing="ij")
    total = torch.zeros(K, dtype=torch.float64)
    pf, qf = p.float().cuda(), q.float().cuda()
    for d in range(K):
        tok = torch.full((n * n, 1), d, device="cuda")
        out = ops.verify_drafts(tok, pf.expand(n * n, 1, K), qf.expand(n * n, 1, K), uu.reshape(-1, 1).cuda(), rr.reshape(-1).cuda())
        total += q[d] * torch.bincount(out["tokens"][:, 0], minlength=K).cpu().double() / (n * n)
    assert (total - p).abs().max().item() < 2.0 / n


# ------------------------------------------------------------------ offsets past 32 bits
@pytest.mark.parametrize("first", [False, True])
def test_offsets_past_32_bits(first):
    """The last rows of arrays of more than 2^31 (volumes, channels first: 2^32) elements."""
    from devis_amd import criterions, ops
    if first:
        rows, K, k = 270_000_000, 8, 2                       # a lane a row
        z = torch.zeros((2, K, rows), dtype=torch.bfloat16, device="cuda")
        tail = lambda x: x[1, :, -5:].t() if x.dim() == 3 else x[1, -5:]
    else:
        rows, K, k = 34_000, 65_536, 9                       # a block a row
        z = torch.zeros((rows, K), dtype=torch.bfloat16, device="cuda")
        tail = lambda x: x[-5:]
    assert z.numel() > 2 ** 31
    want = logits(5, K, torch.bfloat16, 3)
    tail(z).copy_(want)
    out = ops.top_logits(z, k, channels_last=not first)
    v, i, r = teacher_of(want, k, 1.0)
    assert torch.equal(tail(out["indices"]).long().cpu(), i.long()) and torch.equal(tail(out["values"]).cpu(), v)
    assert (tail(out["rest"]).cpu().double() - r.double()).abs().max().item() < 2 * sum_error(want.double().numpy(), 1.0) + 32 * E
    z.requires_grad_(True)
    out["values"].mul_(0.5)
    per_row = criterions.distill_top_loss(z, out["values"], out["indices"], out["rest"], channels_last=not first, reduction="none")
    (dz,) = torch.autograd.grad(per_row, z, torch.ones_like(per_row))
    loss, grad, _, scale, err = oracle_rows(want, (v.float() * 0.5).to(v.dtype), i, tail(out["rest"]).cpu(), None, 1.0)
    assert np.all(np.abs(tail(per_row).detach().cpu().double().numpy() - loss) <= err)
    have = tail(dz).cpu().double().numpy()
    for a, b, c, row in zip(have, grad, scale, want):
        assert np.all(np.abs(a - b) <= c * (2 * sum_error(row.double().numpy(), 1.0) + 16 * E) + HALF[torch.bfloat16] * np.abs(b) + 1e-37)


def test_verify_offsets_past_32_bits():
    from devis_amd import ops
    B, K = 34_000, 65_536
    p = torch.zeros((B, 1, K), dtype=torch.bfloat16, device="cuda")
    tok, pw, q, u, r = drafts(4, 1, K, torch.bfloat16, 5, bonus=False)
    p[-4:] = pw.cuda()
    full = lambda x, n: torch.cat([torch.zeros((n,) + tuple(x.shape[1:]), dtype=x.dtype), x]).cuda()
    out = ops.verify_drafts(full(tok, B - 4), p, None, full(u, B - 4), full(r, B - 4))
    for j in range(4):
        want, a = O.verify_row(tok[j].numpy(), pw[j].double().numpy(), None, u[j].double().numpy(), float(r[j]), 1)
        assert out["accepted"][B - 4 + j].item() == a and np.array_equal(out["tokens"][B - 4 + j].cpu().numpy(), want)
    assert out["tokens"][0, 0].item() == -1                  # no class has weight


# ------------------------------------------------------------------ together, streams, graphs
def test_teacher_student_and_drafts_together():
    """As they are used: the teacher's top logits, some steps of a student towards them, and label maps drawn from the
    student and verified against the teacher."""
    from devis_amd import criterions, ops
    g = torch.Generator().manual_seed(1)
    teacher = (torch.randn((2, 8, 8, 8, 4), generator=g) * 3).cuda()
    top = ops.top_logits(teacher, 2, temperature=2.0)
    student = torch.zeros_like(teacher, requires_grad=True)
    kl = lambda: criterions.distill_top_loss(student, top["values"], top["indices"], top["rest"], temperature=2.0, reduction="sum")
    first = kl()
    for _ in range(50):
        loss = kl()
        (grad,) = torch.autograd.grad(loss, student)
        with torch.no_grad():
            student -= 0.3 * grad
    assert kl().item() < first.item()             # a descent on a convex function with a small step
    p, q = torch.softmax(teacher, -1).view(-1, 1, 4), torch.softmax(student.detach(), -1).view(-1, 1, 4)
    u = torch.rand((3, 1024, 1), generator=g)
    tok = (q.cpu()[:, 0].cumsum(-1) <= u[0]).sum(-1, keepdim=True).clamp_max(3)
    check_verify(tok, p.cpu(), q.cpu(), u[1], u[2][:, 0])


def run_all(x):
    from devis_amd import criterions, ops
    top = ops.top_logits(x["t"], x["k"], temperature=2.0)
    loss = criterions.distill_top_loss(x["z"], top["values"], top["indices"], top["rest"], temperature=2.0)
    (dz,) = torch.autograd.grad(loss, x["z"])
    ver = ops.verify_drafts(x["tok"], x["p"], x["q"], x["u"], x["r"])
    return [top["values"], top["indices"], top["rest"], loss.detach(), dz, ver["tokens"], ver["accepted"]]


def inputs(seed, rows=6, K=9000, k=12):
    tok, p, q, u, r = drafts(rows, 3, K, torch.float32, seed)
    x = dict(t=logits(rows, K, torch.bfloat16, seed), z=logits(rows, K, torch.bfloat16, seed + 50), tok=tok, p=p, q=q, u=u, r=r)
    x = {n: t.cuda() for n, t in x.items()}
    x["z"].requires_grad_(True)
    x["k"] = k
    return x


@pytest.mark.parametrize("rows, K, k", [(6, 9000, 12), (500, 4, 2), (300, 100, 5)])
def test_graphs_replayed_side_by_side(rows, K, k):
    """Two captured graphs, replayed on two streams at once with new inputs in the same buffers, several times, with eager
    work of the same calls between: every replay gives what the eager calls give."""
    xs = [inputs(s, rows, K, k) for s in (1, 2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            run_all(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run_all(x))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for rep in range(4):
        for j, x in enumerate(xs):
            new = inputs(10 + 2 * rep + j, rows, K, k)
            with torch.no_grad():
                for n in x:
                    if n != "k":
                        x[n].copy_(new[n])
        torch.cuda.synchronize()
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        for x, out in zip(xs, outs):
            for a, b in zip(run_all(x), out):
                assert torch.equal(a, b)


def test_two_streams_at_once_and_rows_behind_the_last():
    """Eager calls on two streams, and outputs that end where they should: the memory behind them keeps its value."""
    xs = [inputs(s) for s in (3, 4)]
    want = [run_all(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, x in zip(streams, xs):
            with torch.cuda.stream(st):
                got.append(run_all(x))
        torch.cuda.synchronize()
        for a, b in zip(want, got):
            assert all(torch.equal(c, d) for c, d in zip(a, b))


@pytest.mark.parametrize("K, dtype", [(4, torch.float32), (7, torch.bfloat16), (1001, torch.bfloat16), (5003, torch.float32)])
def test_outputs_end_where_they_should(K, dtype):
    from devis_amd import _lib, ops
    import ctypes as C
    lib = _lib.load()
    rows, k = 9, 3
    z, v, i, r = [x.cuda() for x in pair(rows, K, k, 1.0, dtype, K)]
    st = torch.cuda.current_stream().cuda_stream
    guard = lambda n, dt: torch.full((n + 64,), 77, dtype=dt, device="cuda")
    idt = torch.uint8 if K <= 256 else torch.int32
    gv, gi, gr = guard(rows * k, dtype), guard(rows * k, idt), guard(rows, torch.float32)
    lc = {torch.uint8: _lib.LABEL_U8, torch.int32: _lib.LABEL_I32}[idt]
    assert lib.devis_top_logits(z.data_ptr(), K, 0, 1, ops.dt_code(dtype), rows, 1, K, k, 1.0, gv.data_ptr(), gi.data_ptr(), lc,
                                k, 0, 1, gr.data_ptr(), st) == 0
    p = _lib.DistillParams(rows, 1, K, k, K, 0, 1, k, 0, 1, v.data_ptr(), i.data_ptr(), r.data_ptr(), None, 1.0, ops.dt_code(dtype),
                           ops.dt_code(v.dtype), _lib.LABEL_I32, 1)
    ns, nw = lib.devis_distill_stats_bytes(C.byref(p)), lib.devis_distill_workspace_bytes(C.byref(p))
    gl, g1, gs, gst, gw = (guard(n, d) for n, d in ((rows, torch.float32), (1, torch.float32), (2, torch.float32), (ns, torch.uint8),
                                                    (nw, torch.uint8)))
    assert lib.devis_distill_fwd(C.byref(p), z.data_ptr(), gl.data_ptr(), g1.data_ptr(), gs.data_ptr(), gst.data_ptr(), gw.data_ptr(),
                                 nw, st) == 0
    gd, one = guard(rows * K, dtype), torch.ones((), device="cuda")
    assert lib.devis_distill_bwd(C.byref(p), z.data_ptr(), gst.data_ptr(), gs.data_ptr(), one.data_ptr(), 0, gd.data_ptr(), K, 0, 1,
                                 st) == 0
    torch.cuda.synchronize()
    for t in (gv, gi, gr, gl, g1, gs, gst, gw, gd):
        assert (t[-64:] == 77).all()
    assert torch.isfinite(gd[:-64].float()).all()

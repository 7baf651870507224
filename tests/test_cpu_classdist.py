"""Operators on two models' class distributions: their oracle, and what the calls refuse (no GPU needed: a refused call
launches nothing)."""
import ctypes as C

import numpy as np
import pytest
import torch

from devis_amd import _lib, criterions, ops
from devis_amd._lib import DevisError
from oracle import classdist_oracle as O


def test_oracle_gradient_is_the_derivative_of_its_loss():
    rng = np.random.default_rng(0)
    z, v = rng.normal(size=9) * 2, rng.normal(size=3)
    idx = np.array([4, 1, 4])                     # a class in two slots
    for rest in (None, 0.3):
        _, g, _ = O.distill_row(z, v, idx, rest, 1.7)
        h = 1e-5
        for c in range(9):
            e = np.zeros(9)
            e[c] = h
            d = (O.distill_row(z + e, v, idx, rest, 1.7)[0] - O.distill_row(z - e, v, idx, rest, 1.7)[0]) / (2 * h)
            assert abs(d - g[c]) < 1e-8           # h^2 / 6 plus 1e-16 / h


def test_oracle_loss_of_a_full_list_is_the_kl_of_the_softmaxes():
    rng = np.random.default_rng(1)
    z, t = rng.normal(size=6), rng.normal(size=6)
    idx, rest = O.top_row(t, 6, 2.0)
    lz, lt = torch.log_softmax(torch.tensor(z) / 2, 0), torch.log_softmax(torch.tensor(t) / 2, 0)
    want = 4 * float((lt.exp() * (lt - lz)).sum())
    assert rest == -np.inf
    assert abs(O.distill_row(z, t[idx], idx, rest, 2.0)[0] - want) < 1e-12
    # four slots and the rest: the KL of the distributions with the rest put together
    idx, rest = O.top_row(t, 4, 2.0)
    p, q = lt.exp().numpy(), lz.exp().numpy()
    pr, qr = 1 - p[idx].sum(), 1 - q[idx].sum()
    want = 4 * float((p[idx] * np.log(p[idx] / q[idx])).sum() + pr * np.log(pr / qr))
    assert abs(O.distill_row(z, t[idx], idx, rest, 2.0)[0] - want) < 1e-10


def test_oracle_verification_is_distributed_as_the_target():
    """Accepting or redrawing leaves the target's distribution: exact, by integrating over both random numbers."""
    rng = np.random.default_rng(2)
    K = 4
    p, q = rng.dirichlet(np.ones(K)), rng.dirichlet(np.ones(K))
    n = 400
    for draft in (q[None], None):
        got = np.zeros(K)
        for d in range(K):
            u = (np.arange(n) + 0.5) / n
            pd = q[d] if draft is not None else 1.0 / K        # drafts without probabilities: any proposal, here uniform
            for ui in u:
                tok, a = O.verify_row([d], p[None], draft, [ui], 0.5, 1)
                if a:
                    got[d] += pd / n
                else:
                    w = np.maximum(p - q, 0) if draft is not None else np.where(np.arange(K) == d, 0, p)
                    got += pd / n * w / w.sum()
        if draft is not None:
            assert np.abs(got - p).max() < 2.0 / n             # one grid step of u for each class
        else:
            assert np.abs(got - p).max() < 2.0 / n             # accepted with p_d, else p without d: p again


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("call, text", [
    (lambda: ops.top_logits(t(3, 8), 0), "k must be in"),
    (lambda: ops.top_logits(t(3, 8), 9), "k must be in"),
    (lambda: ops.top_logits(t(3, 200), 129), "k must be in"),
    (lambda: ops.top_logits(t(3, 0), 1), "k must be in"),
    (lambda: ops.top_logits(t(3, 8), 2, temperature=0.0), "temperature"),
    (lambda: ops.top_logits(t(3, 8), 2, temperature=float("nan")), "temperature"),
    (lambda: ops.top_logits(t(3, 8), 2, temperature=float("inf")), "temperature"),
    (lambda: ops.top_logits(t(3, 8, dtype=torch.float64), 2), "dtype"),
    (lambda: ops.top_logits(t(8), 2, channels_last=False), "dimensions"),
    (lambda: ops.top_logits(t(3, 8), 2), "GPU tensors"),
])
def test_top_logits_refuses(call, text):
    with pytest.raises(DevisError, match=text):
        call()


def distill(z=(3, 8), v=(3, 2), i=(3, 2), idt=torch.int32, vdt=torch.float32, zdt=torch.float32, **kw):
    return criterions.distill_top_loss(t(*z, dtype=zdt), t(*v, dtype=vdt), t(*i, dtype=idt), **kw)


@pytest.mark.parametrize("kw, text", [
    (dict(v=(4, 2), i=(4, 2)), "do not go with"),
    (dict(v=(3, 1, 2), i=(3, 1, 2)), "do not go with"),
    (dict(i=(3, 3)), "differ in shape"),
    (dict(v=(3, 9), i=(3, 9)), "slots a row"),
    (dict(z=(3, 300), v=(3, 129), i=(3, 129)), "slots a row"),
    (dict(v=(3, 0), i=(3, 0)), "slots a row"),
    (dict(idt=torch.int16), "labels must be"),
    (dict(vdt=torch.float16), "dtype"),
    (dict(zdt=torch.float64), "dtype"),
    (dict(temperature=-1.0), "temperature"),
    (dict(rest=t(3, 1)), "rest must be"),
    (dict(rest=t(3, dtype=torch.bfloat16)), "rest must be"),
    (dict(row_mask=t(3)), "row_mask must be"),
    (dict(row_mask=t(2, dtype=torch.bool)), "row_mask must be"),
    (dict(z=(3, 8, 5), v=(3, 2, 4), i=(3, 2, 4), channels_last=False), "do not go with"),
    (dict(), "GPU tensors"),
])
def test_distill_refuses(kw, text):
    with pytest.raises(DevisError, match=text):
        distill(**kw)


def test_distill_refuses_reductions_and_teacher_gradients():
    with pytest.raises(ValueError, match="reduction"):
        distill(reduction="batchmean")
    z, v, i = t(3, 8), t(3, 2).requires_grad_(), t(3, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="teacher"):
        criterions.distill_top_loss(z, v, i)
    with pytest.raises(ValueError, match="teacher"):
        criterions.distill_top_loss(z, v.detach(), i, rest=t(3).requires_grad_())


def verify(tok=(2, 3), p=(2, 4, 8), q=(2, 3, 8), u=(2, 3), r=(2,), tdt=torch.int64, pdt=torch.float32, qdt=None, lengths=None):
    return ops.verify_drafts(t(*tok, dtype=tdt), t(*p, dtype=pdt), None if q is None else t(*q, dtype=qdt or pdt), t(*u), t(*r),
                             lengths=lengths)


@pytest.mark.parametrize("kw, text", [
    (dict(tok=(2,)), r"\(B, T\)"),
    (dict(p=(2, 8)), r"\(B, T\)"),
    (dict(tdt=torch.uint8), "tokens must be"),
    (dict(p=(2, 5, 8)), "do not go with"),
    (dict(p=(2, 2, 8)), "do not go with"),
    (dict(p=(3, 4, 8)), "do not go with"),
    (dict(p=(2, 4, 0), q=(2, 3, 0)), "do not go with"),
    (dict(tok=(2, 0), p=(2, 0, 8), q=None, u=(2, 0)), "do not go with"),
    (dict(q=(2, 4, 8)), "draft_probs must be"),
    (dict(qdt=torch.bfloat16), "draft_probs must be"),
    (dict(u=(2, 4)), "accept_u must be"),
    (dict(r=(3,)), "sample_u must be"),
    (dict(lengths=t(3, dtype=torch.int64)), "lengths must be"),
    (dict(lengths=t(2)), "lengths must be"),
    (dict(pdt=torch.float16), "dtype"),
    (dict(), "GPU tensors"),
])
def test_verify_refuses(kw, text):
    with pytest.raises(DevisError, match=text):
        verify(**kw)


def test_c_entries_refuse_bad_arguments_without_a_gpu():
    """Every refusal comes before the first launch, so placeholders stand for the device pointers."""
    lib = _lib.load()
    ph = 256
    top = lambda N=2, V=3, K=8, k=2, T=1.0, idt=_lib.LABEL_I32, z=ph, vals=ph, sK=1, dt=0: lib.devis_top_logits(
        z, V * K, K, sK, dt, N, V, K, k, T, vals, ph, idt, V * k, k, 1, None, None)
    for kw in (dict(N=0), dict(V=0), dict(K=0), dict(k=0), dict(k=9), dict(K=500, k=129), dict(T=0.0), dict(T=float("nan")),
               dict(T=float("inf")), dict(T=1e-45), dict(idt=_lib.LABEL_I64), dict(K=257, idt=_lib.LABEL_U8), dict(z=None),
               dict(vals=None), dict(sK=0), dict(sK=-1), dict(K=2 ** 30 + 1), dict(K=2 ** 31), dict(dt=2)):
        assert top(**kw) == -1, kw

    def params(**kw):
        d = dict(N=2, V=3, K=8, k=2, sN=24, sV=8, sK=1, oN=6, oV=2, oK=1, values=ph, indices=ph, rest=None, row_mask=None,
                 temperature=1.0, dtype=0, values_dtype=0, index_dtype=2, mean=1)
        d.update(kw)
        return _lib.DistillParams(**d)
    for kw in (dict(N=0), dict(K=0), dict(k=0), dict(k=9), dict(K=500, k=129), dict(sK=0), dict(oK=0), dict(values=None),
               dict(indices=None), dict(temperature=0.0), dict(temperature=float("nan")), dict(dtype=2), dict(values_dtype=7),
               dict(index_dtype=3), dict(K=2 ** 30 + 1), dict(K=2 ** 31)):
        assert lib.devis_distill_fwd(C.byref(params(**kw)), ph, ph, None, None, ph, None, 0, None) == -1, kw
        assert lib.devis_distill_bwd(C.byref(params(**kw)), ph, ph, ph, ph, 0, ph, 24, 8, 1, None) == -1, kw
    ok = params()
    nb = lib.devis_distill_workspace_bytes(C.byref(ok))
    assert lib.devis_distill_fwd(None, ph, ph, None, None, ph, None, 0, None) == -1
    assert lib.devis_distill_fwd(C.byref(ok), None, ph, None, None, ph, None, 0, None) == -1
    assert lib.devis_distill_fwd(C.byref(ok), ph, None, None, None, ph, ph, nb, None) == -1
    assert lib.devis_distill_fwd(C.byref(ok), ph, None, ph, None, ph, ph, nb, None) == -1
    assert lib.devis_distill_fwd(C.byref(ok), ph, None, ph, ph, ph, None, nb, None) == -1
    assert lib.devis_distill_fwd(C.byref(ok), ph, None, ph, ph, ph, ph, nb - 1, None) == -4
    assert lib.devis_distill_bwd(C.byref(ok), ph, ph, None, ph, 0, ph, 24, 8, 1, None) == -1
    assert lib.devis_distill_bwd(C.byref(ok), ph, ph, ph, None, 0, ph, 24, 8, 1, None) == -1
    assert lib.devis_distill_bwd(C.byref(ok), ph, ph, ph, ph, 0, None, 24, 8, 1, None) == -1
    assert lib.devis_distill_bwd(C.byref(ok), ph, ph, ph, ph, 0, ph, 24, 8, 0, None) == -1

    def vparams(**kw):
        d = dict(B=2, T=3, Tp=4, K=8, pB=32, pT=8, pK=1, qB=24, qT=8, qK=1, tokens=ph, accept_u=ph, sample_u=ph, lengths=None,
                 dtype=0, token_dtype=0)
        d.update(kw)
        return _lib.VerifyParams(**d)
    for kw in (dict(B=0), dict(T=-1), dict(Tp=5), dict(Tp=2), dict(T=0, Tp=0), dict(K=0), dict(K=2 ** 30 + 1), dict(K=2 ** 31), dict(tokens=None),
               dict(accept_u=None), dict(sample_u=None), dict(token_dtype=1), dict(dtype=2)):
        assert lib.devis_verify_drafts(C.byref(vparams(**kw)), ph, ph, ph, ph, None) == -1, kw
    v = vparams()
    for args in ((None, ph, ph, ph, ph), (C.byref(v), None, ph, ph, ph), (C.byref(v), ph, ph, None, ph), (C.byref(v), ph, ph, ph, None)):
        assert lib.devis_verify_drafts(*args, None) == -1


def test_rows_of_every_layout():
    x = torch.arange(2 * 5 * 4 * 3).view(2, 5, 4, 3)
    for y, last in ((x, True), (x, False), (x.movedim(1, -1), True), (x.transpose(2, 3), False), (x[:, :, ::2], False),
                    (x[:, ::2], True), (x[..., 1:], True), (x.expand(2, 5, 4, 3)[:1].expand(3, 5, 4, 3), True),
                    (x[..., :1].expand(2, 5, 4, 7), True), (x[0, 0, 0], True)):
        z, n, v, k, sn, sv, sk = ops.class_rows(y, last)
        rows = (y if last else y.movedim(1, -1)).reshape(n, v, k)
        assert sk >= 1
        flat = torch.as_strided(z, (n, v, k), (sn, sv, sk))
        assert torch.equal(flat, rows)

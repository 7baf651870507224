"""Training with a teacher over the models: volumes and images, each kind of net as the student, and the term with voxels left
out."""
import numpy as np
import pytest
import torch

from oracle import classdist_oracle as O
from tests.util import brats_args

pytestmark = pytest.mark.gpu

# dataset, classes, input channels, size, student, teacher
PAIRS = [("BraTS", 4, 4, (16, 16, 16), "AU", "U"), ("LiTS", 3, 1, (16, 32, 32), "V", "U"), ("ISIC", 2, 3, (32, 48), "U", "V"),
         ("DRIVE", 2, 3, (64, 64), "V", "U"), ("TOAR", 7, 1, (32, 32), "U", "U")]


def models(dataset, classes, student, teacher, dtype):
    from devis_amd import TMSU
    torch.manual_seed(0)
    make = lambda name: TMSU(brats_args(dataset=dataset, num_classes=classes, model_name=name, compute_dtype=dtype))
    return make(student).train(), make(teacher).eval().requires_grad_(False)


def batch(channels, classes, size, seed, n=2):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((n, channels) + size, generator=g).cuda(), torch.randint(0, classes, (n,) + size, generator=g).cuda()


@pytest.mark.parametrize("dataset, classes, channels, size, student, teacher", PAIRS)
def test_the_term_is_the_oracles(dataset, classes, channels, size, student, teacher):
    s, t = models(dataset, classes, student, teacher, torch.float32)
    x, y = batch(channels, classes, size, 1)
    with torch.no_grad():
        zs, zt = (m.backbone.forward_channels_last(x).reshape(-1, classes).double().cpu().numpy() for m in (s, t))
    for k in {1, classes}:
        want = 0.0
        for a, b in zip(zs, zt):
            idx, rest = O.top_row(b, k, 2.0)
            want += O.distill_row(a, b[idx], idx, rest, 2.0)[0] / len(zs)
        top = t.top_logits(x, k, 2.0)
        assert tuple(top["values"].shape) == (2,) + size + (k,)
        _, base = s(x, y, 5, 'train', dataset)
        _, both = s(x, y, 5, 'train', dataset, distill=(top, 2.0, 0.25))
        # logarithms are good to 32 x 2^-22 nats, T^2 = 4; two fp32 sums of the loss
        assert abs((both - base).item() - 0.25 * want) <= 0.25 * 4 * 32 * 2.0 ** -22 + 2 * 2.0 ** -23 * abs(both.item())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dataset, classes, channels, size, student, teacher", PAIRS)
def test_replayed_steps_give_the_eager_gradients(dataset, classes, channels, size, student, teacher, dtype, monkeypatch):
    from devis_amd import launch_plan
    grads = {}
    for plans in (False, True):
        monkeypatch.setattr(launch_plan, "ENABLED", plans)
        s, t = models(dataset, classes, student, teacher, dtype)
        out = []
        for step in range(4):
            x, y = batch(channels, classes, size, 10 + step)
            _, loss = s(x, y, 5, 'train', dataset, distill=(t.top_logits(x, classes, 2.0), 2.0, 0.5))
            s.zero_grad(set_to_none=True)
            loss.backward()
            out.append([loss.detach().clone()] + [p.grad.clone() for p in s.parameters()])
        grads[plans] = out
    # (two eager runs of a V net in bf16 differ in the last bits of its first block's gradients, with a teacher and without)
    repeats = dtype == torch.float32 or student != "V"
    for a, b in zip(grads[False], grads[True]):
        assert torch.equal(a[0], b[0])
        for p, q in zip(a[1:], b[1:]):
            assert torch.equal(p, q) if repeats else p.shape == q.shape
    assert all(torch.isfinite(p).all() for p in grads[True][-1])


@pytest.mark.parametrize("dataset, classes, channels, size, student, teacher", PAIRS[:1] + PAIRS[2:3])
def test_voxels_left_out_do_not_reach_the_weights(dataset, classes, channels, size, student, teacher):
    """A masked batch: what the teacher says of voxels that are left out changes no gradient, and the others' mean is the
    oracle's."""
    from devis_amd.criterions import distill_top_loss
    s, t = models(dataset, classes, student, teacher, torch.float32)
    x, _ = batch(channels, classes, size, 3)
    top = t.top_logits(x, classes - 1, 1.0)
    g = torch.Generator().manual_seed(4)
    mask = (torch.rand((2,) + size, generator=g) < 0.6).cuda()
    got = []
    for spoil in (False, True):
        values = top["values"].clone()
        if spoil:
            values[~mask] = float("nan")
        z = s.backbone.forward_channels_last(x)
        loss = distill_top_loss(z, values, top["indices"], top["rest"], row_mask=mask)
        s.zero_grad(set_to_none=True)
        loss.backward()
        got.append([loss.detach()] + [p.grad.clone() for p in s.parameters()])
    # the net's own step may differ from run to run in the last bits of its sums; what is left out would be NaN
    for a, b in zip(*got):
        assert torch.isfinite(b).all() and (a - b).abs().max().item() <= 1e-4 * a.abs().max().item()
    zs = z.detach().reshape(-1, classes).double().cpu().numpy()
    v, i, r = (top[n].reshape(len(zs), -1).cpu().numpy() for n in ("values", "indices", "rest"))
    keep = mask.reshape(-1).cpu().numpy()
    want = np.mean([O.distill_row(zs[n], v[n], i[n], r[n, 0], 1.0)[0] for n in np.nonzero(keep)[0]])
    assert abs(got[0][0].item() - want) <= 32 * 2.0 ** -22 + 2.0 ** -23 * want

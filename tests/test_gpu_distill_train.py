"""Training with a teacher: TMSU's distillation term against the oracle, through the launch plans' replayed steps, and the
`--teacher` flag of the training command."""
import argparse
import os

import numpy as np
import pytest
import torch

from oracle import classdist_oracle as O
from tests.util import brats_args

pytestmark = pytest.mark.gpu


def models(dtype=torch.float32):
    from devis_amd import TMSU
    torch.manual_seed(0)
    student = TMSU(brats_args(compute_dtype=dtype)).train()
    teacher = TMSU(brats_args(compute_dtype=dtype, model_name='V')).eval().requires_grad_(False)
    return student, teacher


def batch(seed, n=16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn((1, 4, n, n, n), generator=g).cuda(), torch.randint(0, 4, (1, n, n, n), generator=g).cuda()


def test_the_term_is_the_oracles_and_adds_to_the_loss():
    student, teacher = models()
    x, y = batch(1)
    top = teacher.top_logits(x, 2, 2.0)
    assert not teacher.training and top["values"].shape == (1, 16, 16, 16, 2) and top["indices"].dtype == torch.uint8
    with torch.no_grad():
        z = student.backbone.forward_channels_last(x).reshape(-1, 4).double().cpu().numpy()
        t = teacher.backbone.forward_channels_last(x).reshape(-1, 4).double().cpu().numpy()
    want = 0.0
    for a, b in zip(z, t):
        idx, rest = O.top_row(b, 2, 2.0)
        want += O.distill_row(a, b[idx], idx, rest, 2.0)[0] / len(z)
    _, base = student(x, y, 5, 'train', 'BraTS')
    _, both = student(x, y, 5, 'train', 'BraTS', distill=(top, 2.0, 0.25))
    # rest is fp32 (2^-24 of a few nats), a row's logarithms 2^-22 of a few nats, T^2 = 4; two fp32 sums of the loss
    tol = 0.25 * 4 * 32 * 2.0 ** -22 + 2 * 2.0 ** -23 * abs(both.item())
    assert abs((both - base).item() - 0.25 * want) <= tol


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_replayed_steps_give_the_eager_gradients(dtype, monkeypatch):
    """Two consumers of the logits feed one backward: recorded and replayed steps against eager ones, bit for bit."""
    from devis_amd import launch_plan
    grads = {}
    for plans in (False, True):
        monkeypatch.setattr(launch_plan, "ENABLED", plans)
        student, teacher = models(dtype)
        out = []
        for step in range(4):
            x, y = batch(10 + step, 32)
            top = teacher.top_logits(x, 2, 2.0)
            _, loss = student(x, y, 5, 'train', 'BraTS', distill=(top, 2.0, 0.5))
            student.zero_grad(set_to_none=True)
            loss.backward()
            out.append([loss.detach().clone()] + [p.grad.clone() for p in student.parameters()])
        grads[plans] = out
    for a, b in zip(grads[False], grads[True]):
        for p, q in zip(a, b):
            assert torch.equal(p, q)
    assert all(torch.isfinite(p).all() for p in grads[True][-1])


def test_a_teacher_equal_to_the_student_adds_nothing():
    """p = q: the term is zero to rounding (each row's logarithms differ by a few 2^-22 nats, T^2 = 1), and so is its pull."""
    from devis_amd import TMSU
    student, _ = models()
    student.eval()                                   # the same batch statistics on both sides
    x, y = batch(3)
    top = student.top_logits(x, 3, 1.0)
    from devis_amd.criterions import distill_top_loss
    z = student.backbone.forward_channels_last(x).detach().requires_grad_(True)
    loss = distill_top_loss(z, top["values"], top["indices"], top["rest"])
    loss.backward()
    assert abs(loss.item()) < 32 * 2.0 ** -22
    assert z.grad.abs().max().item() < 32 * 2.0 ** -22 / z[..., 0].numel()


def test_training_command_with_a_teacher(tmp_path):
    from devis_amd import TMSU, train as T
    torch.manual_seed(3)
    teacher = TMSU(brats_args(model_name='V', compute_dtype=torch.bfloat16))
    path = os.path.join(str(tmp_path), "teacher.pth")
    torch.save({'epoch': 1, 'state_dict': teacher.state_dict()}, path)
    argv = ['--dataset', 'BraTS', '--mode', 'train&test', '--synthetic', '2', '--crop_H', '32', '--crop_W', '32', '--crop_D', '32',
            '--start_epoch', '4', '--end_epochs', '4', '--save_dir', str(tmp_path), '--teacher', path, '--teacher_model', 'V']
    loaders = lambda a: (T.synthetic_loaders(a)[0], [], [])
    losses = {}
    for weight in ('0.0', '1.0'):
        out = T.run(T.getArgs(argv + ['--distill_weight', weight]), loaders=loaders, log=lambda *a: None)
        losses[weight] = out['loss_list'][0]
    plain = T.run(T.getArgs([a for a in argv if a not in ('--teacher', path, '--teacher_model', 'V')]), loaders=loaders,
                  log=lambda *a: None)['loss_list'][0]
    assert np.isfinite(losses['1.0'])
    assert losses['0.0'] == plain                    # nothing added: the step as it was
    assert losses['1.0'] > losses['0.0']             # a divergence is not negative, and these two models differ


@pytest.mark.parametrize("flags", [['--distill_top', '5'], ['--distill_top', '0'], ['--distill_weight', '-1'],
                                   ['--distill_temperature', '0']])
def test_training_command_refuses(flags, tmp_path):
    from devis_amd import train as T
    args = T.getArgs(['--dataset', 'BraTS', '--teacher', os.path.join(str(tmp_path), 'none.pth')] + flags)
    with pytest.raises(ValueError):
        T.load_teacher(args)


def test_the_term_belongs_to_training():
    student, teacher = models()
    x, y = batch(1)
    with pytest.raises(ValueError, match="train"):
        student(x, y, 5, 'val', 'LiTS', distill=(teacher.top_logits(x, 2), 1.0, 1.0))


def test_no_teacher_without_the_flag():
    from devis_amd import train as T
    assert T.load_teacher(T.getArgs(['--dataset', 'BraTS'])) is None
    assert T.load_teacher(argparse.Namespace()) is None

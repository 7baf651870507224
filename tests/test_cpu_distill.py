"""A model as a teacher: what needs no GPU."""
import pytest
import torch

from devis_amd import TMSU, ops
from tests.util import brats_args


@pytest.mark.parametrize("outer", [True, False])
@pytest.mark.parametrize("inner", [True, False])
def test_top_logits_leave_every_module_in_its_mode(outer, inner, monkeypatch):
    """In eval mode throughout, whatever mode the model and its parts were in, and in that mode again afterwards."""
    model = TMSU(brats_args())
    part = torch.nn.Dropout()
    model.backbone.add_module("part", part)
    model.train(outer)
    model.backbone.train(inner)
    part.train(not inner)
    seen = []
    monkeypatch.setattr(model.backbone, "forward_channels_last", lambda x: seen.append([m.training for m in model.modules()]) or x)
    monkeypatch.setattr(ops, "top_logits", lambda x, k, **kw: dict(grad=torch.is_grad_enabled(), k=k))
    before = [m.training for m in model.modules()]
    out = model.top_logits(torch.zeros(1), 2)
    assert not any(seen[0]) and out == dict(grad=False, k=2)
    assert [m.training for m in model.modules()] == before
    monkeypatch.setattr(ops, "top_logits", lambda *a, **kw: 1 / 0)
    with pytest.raises(ZeroDivisionError):
        model.top_logits(torch.zeros(1), 2)
    assert [m.training for m in model.modules()] == before


def test_the_command_keeps_every_class_of_a_live_teacher():
    """Nothing is stored of a teacher that runs beside the student, so by default nothing of it is left out."""
    from devis_amd import train as T
    for dataset, classes in (("BraTS", 4), ("LiTS", 3), ("HC", 10)):
        assert T.getArgs(['--dataset', dataset]).distill_top == classes
    assert T.getArgs(['--dataset', 'HC', '--distill_top', '2']).distill_top == 2

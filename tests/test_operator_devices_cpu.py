"""Tensors of a multi-axis rotary call on another device than q: refused on the
host, before any launch. CPU tensors and tensors of the meta device stand for
two GPUs."""
import pytest
import torch

from bloth_b200.kernels import mrope


def _q(device="cpu", heads=2):
    return torch.empty(1, 4, heads, 64, device=device)


POS, INV, AXES = torch.zeros(3, 1, 4).long(), torch.ones(32), (0,) * 32


def test_one_device_is_taken():
    mrope._check_pair(_q(), _q(heads=1))
    mrope._check_pair(_q(), None)
    mrope._source(_q(), POS, INV, AXES)
    mrope._weight(torch.ones(64), 64, torch.float32, torch.device("cpu"))


def test_another_device_is_refused():
    with pytest.raises(ValueError, match="k must be on cpu"):
        mrope._check_pair(_q(), _q("meta", 1))
    with pytest.raises(ValueError, match="position_ids must be on cpu"):
        mrope._source(_q(), POS.to("meta"), INV, AXES)
    with pytest.raises(ValueError, match="inv_freq must be on cpu"):
        mrope._source(_q(), POS, INV.to("meta"), AXES)
    with pytest.raises(ValueError, match="must be on cpu"):
        mrope._weight(torch.ones(64, device="meta"), 64, torch.float32, torch.device("cpu"))


@pytest.mark.parametrize("which", ["k", "wq", "wk", "position_ids", "inv_freq"])
def test_the_entry_points_check(monkeypatch, which):
    def fail(*args):
        raise AssertionError("launched")

    monkeypatch.setattr(mrope._lib, "require_cuda", lambda *tensors: None)
    monkeypatch.setattr(mrope._lib, "call", fail)
    a = dict(q=_q(), k=_q(heads=1), wq=torch.ones(64), wk=torch.ones(64), position_ids=POS,
             inv_freq=INV, axes=AXES)
    a[which] = a[which].to("meta")
    with pytest.raises(ValueError, match="must be on cpu"):
        mrope.fused_qk_norm_mrope(**a)
    if which not in ("wq", "wk"):
        del a["wq"], a["wk"]
        with pytest.raises(ValueError, match="must be on cpu"):
            mrope.apply_mrope_qk(**a)

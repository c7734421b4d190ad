"""Refusals and host parts of the incremental operators that need no GPU, beside those of
test_paged_host."""
import importlib.util

import pytest
import torch

import blt_burn_amd as pkg
from blt_burn_amd import _torch as T, fused_ops as F


@pytest.mark.parametrize("device", ["cpu", "cpu:0", "meta"])
def test_a_rotary_table_outside_the_gpu_is_refused(device):
    """Its index alone would pass for a GPU's, and a kernel would follow a host pointer."""
    with pytest.raises(pkg.BltError, match="GPU"):
        F.RotaryPlan(64, device=device)


@pytest.mark.parametrize("rot", [0, 1, 63, 514, -64, (1 << 32) + 64, -(1 << 32) + 64])
def test_rotary_dimensions_out_of_range_are_refused(rot):
    with pytest.raises(pkg.BltError, match="rotary_dim"):
        F.RotaryPlan(rot)


def test_rotary_of_something_else_than_tensors_is_a_type_error():
    x, pos = torch.zeros(1, 1, 1, 64), torch.zeros(1, dtype=torch.int32)
    plan = object.__new__(F.RotaryPlan)  # (no table: nothing of it is looked at)
    plan._index = 0
    for q, k, p in (([1.0], None, pos), (x, [1.0], pos), (x, None, [0]), (None, x, pos), (x, x, None)):
        with pytest.raises(TypeError, match="torch.Tensor"):
            F.fused_rotary(q, k, p, plan)
    with pytest.raises(pkg.BltError, match="GPU"):
        F.fused_rotary(x, x, pos, plan)


@pytest.mark.parametrize("missing", [["_cuda_getDevice"], ["_cuda_getCurrentRawStream"],
                                     ["_cuda_getDevice", "_cuda_getCurrentRawStream"]])
def test_a_torch_without_its_private_names_will_do(missing, monkeypatch):
    """The quick handles are private names of torch: without them the public calls serve."""
    for name in missing:
        monkeypatch.delattr(torch._C, name, raising=False)
    spec = importlib.util.spec_from_file_location("blt_burn_amd._torch_again", T.__file__)
    again = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(again)
    monkeypatch.setattr(again, "_current_device", lambda: 3)
    monkeypatch.setattr(again, "_raw_stream", lambda index: 77)
    got = []
    again.call_on(torch.device("cuda", 3), 3, lambda *a: got.append(a) or 0, "call", 1, 2)
    assert got == [(1, 2, 77)]

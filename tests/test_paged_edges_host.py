"""Refusals and host parts of the incremental operators that need no GPU, beside those of
test_paged_host."""
import pytest

import blt_burn_amd as pkg
from blt_burn_amd import fused_ops as F


@pytest.mark.parametrize("device", ["cpu", "cpu:0", "meta"])
def test_a_rotary_table_outside_the_gpu_is_refused(device):
    """Its index alone would pass for a GPU's, and a kernel would follow a host pointer."""
    with pytest.raises(pkg.BltError, match="GPU"):
        F.RotaryPlan(64, device=device)

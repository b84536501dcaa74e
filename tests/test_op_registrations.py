"""Each of the ops registered in C++ has one kernel a dispatch key."""

import pytest
import torch

import molnex_amd.molix.F  # noqa: F401


@pytest.mark.parametrize("name", ["layer_norm", "layer_norm_backward", "layer_norm_backward2", "grad_norm", "adamw_step",
                                  "adamw8_step", "adamw8_moments", "indexed_linear", "indexed_linear_wgrad",
                                  "orthogonalize", "muon_step"])
def test_no_kernel_hides_another(name):
    table = torch._C._dispatch_dump(f"molix::{name}")
    assert "CUDA:" in table and "(inactive)" not in table, table

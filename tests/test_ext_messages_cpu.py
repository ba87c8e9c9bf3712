"""The compiled op module's refusals format numbers into their messages (a build with the compiler of another
toolchain than the process's libstdc++ crashed there)."""
import pytest
import torch


def test_compiled_ops_refuse_other_ranks():
    from flashgmm_b200 import _ext
    ops = _ext.load()
    with pytest.raises(RuntimeError, match="X must be 2D"):
        ops.standard_m_step(torch.randn(8), torch.randn(8))
    with pytest.raises(RuntimeError, match="X must be 2D"):
        ops.flash_em_fused(torch.randn(8), torch.randn(2, 8), torch.randn(2, 8), torch.randn(2))

"""Which gates norm_after takes for one row (h of one dimension), on the host: past the argument checks a
call ends at the missing CPU path."""
import pytest
import torch


@pytest.mark.parametrize("h", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gate", [torch.float32, torch.bfloat16, torch.float16])
def test_one_row_and_a_gate_of_any_type(h, gate):
    from gatx import BlockNorm, norm_after
    with pytest.raises(RuntimeError, match="no CPU path"):
        norm_after(torch.zeros(8, dtype=h), torch.ones(8), gate=torch.zeros(8, dtype=gate))
    with pytest.raises(RuntimeError, match="no CPU path"):
        BlockNorm(8)(torch.zeros(8, dtype=h))
    with pytest.raises(ValueError, match="gate"):
        norm_after(torch.zeros(8, dtype=h), torch.ones(8), gate=torch.zeros(7, dtype=gate))
    with pytest.raises(ValueError, match="gate"):
        norm_after(torch.zeros(8, dtype=h), torch.ones(8), gate=torch.zeros(8, dtype=torch.int64))

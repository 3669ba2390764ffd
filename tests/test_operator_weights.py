"""The residual norm's wrapper refuses weights and gates that are not fp32, whose ends the kernel
would read past: on CPU tensors, where nothing is launched."""
import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64, torch.int32], ids=str)
@pytest.mark.parametrize("which", ["weight", "block_weight", "gate"])
def test_weights_are_fp32(dtype, which):
    import l2c
    x = torch.zeros(4, 64)
    w = {"weight": torch.ones(64), "block_weight": torch.ones(64), "gate": torch.ones(64)}
    with pytest.raises(ValueError, match="GPU tensors"):  # of fp32 the tensors' device is what is left to refuse
        l2c.residual_rmsnorm(x, x, x, x, w["weight"], 64, 4, block_weight=w["block_weight"], gate=w["gate"],
                             rows_per_gate=4)
    w[which] = w[which].to(dtype)
    with pytest.raises(ValueError, match="fp32 weights"):
        l2c.residual_rmsnorm(x, x, x, x, w["weight"], 64, 4, block_weight=w["block_weight"], gate=w["gate"],
                             rows_per_gate=4)

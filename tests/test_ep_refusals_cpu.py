"""What the expert-parallel layer does not do is refused, not passed over."""
import pytest
import torch
import torch.distributed as dist


@pytest.fixture
def layer():
    import __graft_entry__
    __graft_entry__.build()
    from momoe import ep
    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    yield ep.ExpertParallelMoE(16, 8, 4, 2, 0, Wg_DN=torch.zeros(16, 4), Wl1_ND2H=torch.zeros(4, 16, 16),
                               Wl2_NHD=torch.zeros(4, 8, 16), transport="nccl")
    dist.destroy_process_group()


@pytest.mark.parametrize("name,value", [("balance_coef", 0.01), ("z_coef", 0.001), ("experts_fp8", object())])
def test_single_gpu_settings_are_refused(layer, name, value):
    x = torch.zeros(1, 2, 16)
    setattr(layer, name, value)
    with pytest.raises(RuntimeError, match="ExpertParallelMoE"):
        layer(x)
    delattr(layer, name)
    with pytest.raises(RuntimeError, match="CUDA"):        # the layer itself, which has no CPU path
        layer(x)

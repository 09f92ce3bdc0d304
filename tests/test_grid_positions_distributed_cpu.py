"""The transformer on positions from the grid in place of tables, on gloo ranks with the CPU engine."""
import pytest
import torch
import torch.distributed as dist

from tests import _dist_workers as W
from tests.test_host_distributed_cpu import _spawn


def grid_dit_worker(rank, world, port, mode, ret):
    """Latents after two denoising steps, on tables and on the grid."""
    cfg_, ps = W._setup(rank, world, port)
    from tests import cpu_engine
    import ditango_b200.executor.cogvideox_dit as M
    M._engine = cpu_engine
    from ditango_b200.core.redundancy_map import init_redundancy_map
    cfg_.num_layers, cfg_.num_inference_steps = 2, 3
    init_redundancy_map(cfg_)
    out = []
    for rotary in ("tables", "grid"):
        dcfg = M.DiTConfig(num_layers=2, num_heads=4, head_dim=16, in_channels=4, patch_size=2, text_dim=32, time_dim=16, frames=2, height=8, width=8,
                           text_len=8, rotary=rotary)
        torch.manual_seed(0)
        model = M.CogVideoXDiT(dcfg, ps.get_isp_group(), mode=mode)
        g = torch.Generator().manual_seed(1)
        lat = torch.randn(1, 2, 4, 8, 8, generator=g)
        out.append(M.denoise(model, lat, torch.randn(1, 8, 32, generator=g), torch.randn(1, 8, 32, generator=g), num_steps=2))
    ret[rank] = out
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("mode", ["ditango", "ulysses"])
@pytest.mark.parametrize("world", [1, 2])
def test_grid_positions_give_the_latents_that_tables_give(world, mode):
    ret = _spawn(grid_dit_worker, world, mode)
    for r in range(world):
        tables, grid = ret[r]
        # (angles in 64 bits on one side, fp32 tables on the other; ulysses rounds its attention to bf16)
        assert torch.isfinite(grid).all() and (tables - grid).abs().max().item() < (2e-2 if mode == "ulysses" else 1e-4)

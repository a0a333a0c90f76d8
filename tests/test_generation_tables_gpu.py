"""The angle tables that generation keeps: page tables of many widths share a few."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_page_tables_of_any_width_share_angle_tables(cuda_device):
    from dscquant_b200.llama import LlamaConfig, LlamaW4A4

    model = LlamaW4A4(LlamaConfig(vocab=512, hidden=1024, heads=8, kv_heads=4, intermediate=2048, layers=1), cuda_device, seed=5)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    ids = torch.randint(0, 512, (20,), device=cuda_device, generator=g)
    start, length = (torch.tensor(x, dtype=torch.int32, device=cuda_device) for x in ([0, 20], [20]))
    first = None
    for width in range(2, 65):
        caches = model.caches(2, 16)
        table = torch.full((1, width), -1, dtype=torch.int32, device=cuda_device)
        table[0, :2] = torch.arange(2)
        logits = model.step(ids, caches, table, start, length)
        first = logits if first is None else first
        assert torch.equal(logits, first)
    # 32 to 1024 positions
    assert len(model._rope) <= 6
    assert sum(cos.shape[0] for cos, _ in model._rope.values()) <= 2 * 1024

"""token_logprobs on rows that hold NaN or +inf: the alternatives' ids are those of a stable sort with NaN above all."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V", [(5, 1), (5, 2), (5, 64), (5, 5000), (5, 40000), (700, 9000)])
def test_ids_with_nan(cuda_device, dtype, rows, V):
    """NaN first, last, everywhere; +inf; k up to the whole vocabulary; one block a row and rows in slices."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = (torch.randn(rows, V, generator=g, device=cuda_device) * 3).to(dtype)
    x[0, 0] = torch.nan
    x[1] = torch.nan
    x[2, -1] = torch.nan
    x[3, V // 2] = torch.inf
    x[4, 0], x[4, V // 2] = torch.nan, torch.nan
    t = torch.zeros(rows, dtype=torch.long, device=cuda_device)
    key = torch.where(torch.isnan(x), torch.inf, x.double())  # no row holds both NaN and +inf
    order = torch.sort(key, dim=-1, descending=True, stable=True)[1]
    for k in sorted({1, min(V, 2), min(V, 64)}):
        r = ops.token_logprobs(x, t, top_k=k)
        assert torch.equal(r.top_ids, order[:, :k])
        assert torch.isnan(r.logprobs[:5]).all() and torch.isnan(r.top_logprobs[:5]).all()

"""token_logprobs against log_softmax in 64 bits: log probabilities, entropy and the top alternatives."""
import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def check(x, targets, k, r):
    ref = torch.log_softmax(x.double(), -1)
    none = (x == -torch.inf).all(-1)
    ref = torch.where(none[:, None], -torch.inf, ref)
    V = x.shape[1]
    # 32-bit arithmetic: the difference from the maximum and its logarithm each round once, an exponential is
    # off by 2^-22 and the rounding of its argument, and a sum of V terms in 256 strands by V/256 + 16 roundings
    spread = torch.where(torch.isfinite(ref), ref.abs(), 0.0).amax(-1)
    tol = 2.0 ** -22 * (4 + spread) + 2.0 ** -24 * (V / 256 + 16)
    lp = torch.where(targets >= 0, ref.gather(-1, targets.clamp_min(0)[:, None])[:, 0], 0.0)

    def near(got, want, t):
        same = (got.double() == want) | (torch.isnan(got) & torch.isnan(want)) | ((got.double() - want).abs() <= t)
        assert bool(same.all()), f"{got[~same][:4]} for {want[~same][:4]}"

    near(r.logprobs, lp, tol)
    p = ref.exp()
    entropy = torch.where(none, 0.0, -torch.where(p > 0, p * ref, torch.where(torch.isnan(p), p, 0.0)).sum(-1))
    near(r.entropy, entropy, tol * (2 + spread))
    assert r.top_logprobs.shape == r.top_ids.shape == (x.shape[0], k)
    if k:
        key = torch.where(torch.isnan(x), torch.inf, x.double()) + 0.0  # NaN above all; here never beside +inf
        ids = torch.sort(key, dim=-1, descending=True, stable=True)[1][:, :k]
        assert torch.equal(r.top_ids, ids)
        near(r.top_logprobs, ref.gather(-1, ids), tol[:, None])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (3, 2, 2), (1, 32000, 5), (5, 1023, 20), (2, 50001, 64), (300, 4096, 1),
                                      (7, 129, 0), (33, 70007, 3), (2, 300001, 32)])
def test_random(cuda_device, dtype, rows, V, k):
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(V)
    x = (torch.randn(rows, V, generator=g, device=cuda_device) * 3).to(dtype)
    t = torch.randint(0, V, (rows,), generator=g, device=cuda_device)
    t[rows // 2] = -1
    r = ops.token_logprobs(x, t, top_k=k)
    check(x, t, k, r)
    again = ops.token_logprobs(x, t, top_k=k)
    for a, b in zip((r.logprobs, r.entropy, r.top_logprobs, r.top_ids),
                    (again.logprobs, again.entropy, again.top_logprobs, again.top_ids)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_masks_and_stripes(cuda_device, dtype):
    """Equal logits (all of them; both zeros), vocabularies masked to a few tokens or to none, the largest logits
    next to each other, all in one residue, ascending, descending."""
    from dscquant_b200 import ops

    V, k = 20011, 20
    i = torch.arange(V, device=cuda_device)
    base = torch.sin(i * 0.7)
    lo = torch.finfo(dtype).min
    rows = [torch.zeros(V, device=cuda_device), torch.where(i % 2 == 0, -0.0, 0.0), torch.full((V,), -torch.inf, device=cuda_device),
            torch.where(i % 7000 == 3, 1.0, -torch.inf), torch.where(i == V - 1, 2.0, -torch.inf),
            torch.full((V,), lo, device=cuda_device), torch.where(i == 5, 0.0, lo),
            torch.where((i >= 9000) & (i < 9200), 5.0 + base, base), torch.where(i % 2048 < 8, 5.0 + base, base),
            torch.where(i % 64 == 9, 5.0 + base, base), i / 1000.0, -i / 1000.0, base * 60, torch.where(i < 3, base, -torch.inf)]
    x = torch.stack([r.float() for r in rows]).to(dtype)
    t = torch.randint(0, V, (len(rows),), device=cuda_device)
    t[3], t[4], t[5] = 3, V - 1, 0
    for kk in (1, k, 64):
        check(x, t, kk, ops.token_logprobs(x, t, top_k=kk))
    check(x, t, 0, ops.token_logprobs(x, t))


@pytest.mark.parametrize("dtype", TYPES)
def test_not_finite(cuda_device, dtype):
    """NaN and +inf give NaN; NaN sorts above every number."""
    from dscquant_b200 import ops

    V = 5000
    x = torch.randn(3, V, device=cuda_device).to(dtype)
    x[0, 77] = torch.nan
    x[1, 4000] = torch.inf
    t = torch.tensor([5, 6, 7], device=cuda_device)
    r = ops.token_logprobs(x, t, top_k=4)
    assert torch.isnan(r.logprobs[:2]).all() and torch.isnan(r.entropy[:2]).all()
    assert r.top_ids[0, 0] == 77 and r.top_ids[1, 0] == 4000
    check(x[2:], t[2:], 4, type(r)(r.logprobs[2:], r.entropy[2:], r.top_logprobs[2:], r.top_ids[2:]))


def test_strides_and_alignment(cuda_device):
    """Rows with a stride, starting at any element; one row of a wider matrix."""
    from dscquant_b200 import ops

    for dtype in TYPES:
        big = torch.randn(9, 6007, device=cuda_device).to(dtype)
        for off in (0, 1, 3, 8):
            x = big[1:8, off:off + 5001]
            t = torch.arange(7, device=cuda_device) * 700
            check(x, t, 7, ops.token_logprobs(x, t, top_k=7))
        x = big[4:5, 1:]
        check(x, t[:1], 2, ops.token_logprobs(x, t[:1], top_k=2))
    e = ops.token_logprobs(big[:0], t[:0], top_k=3)
    assert e.logprobs.shape == (0,) and e.top_ids.shape == (0, 3)


def test_target_out_of_range(cuda_device):
    from dscquant_b200 import ops

    x = torch.randn(3, 100, device=cuda_device)
    r = ops.token_logprobs(x, torch.tensor([100, -100, 99], device=cuda_device))
    assert ops.device_status(cuda_device) == 4
    assert torch.isnan(r.logprobs[0]) and r.logprobs[1] == 0 and torch.isfinite(r.logprobs[2])


def test_captured(cuda_device):
    from dscquant_b200 import ops

    x = torch.randn(5, 3001, device=cuda_device).to(torch.bfloat16)
    t = torch.arange(5, device=cuda_device)
    ops.token_logprobs(x, t, top_k=5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ops.token_logprobs(x, t, top_k=5)
    for seed in range(2):
        x.copy_(torch.randn(5, 3001, device=cuda_device))
        t.add_(1)
        graph.replay()
        torch.cuda.synchronize()
        check(x, t, 5, r)
    del graph

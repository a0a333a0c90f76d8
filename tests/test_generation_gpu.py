"""The cache and scoring operators together, as the Llama harness uses them: prompts and single tokens through
4-bit caches, greedy decoding from a captured step, scoring; and what the operators refuse on CUDA tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda_device):
    from dscquant_b200.llama import LlamaConfig, LlamaW4A4

    cfg = LlamaConfig(vocab=512, hidden=1024, heads=8, kv_heads=4, intermediate=2048, layers=2)
    return LlamaW4A4(cfg, cuda_device, seed=5)


def ids(n, device, seed):
    return torch.randint(0, 512, (n,), device=device, generator=torch.Generator(device=device).manual_seed(seed))


def i32(values, device):
    return torch.tensor(values, dtype=torch.int32, device=device)


def test_step_in_chunks_fills_the_same_cache(model, cuda_device):
    """A prompt in one step or in chunks: the first layer's cache bit for bit, finite logits, and the first step close
    to the uncached prefill (whose keys and values are not rounded to 4 bits)."""
    n = 100
    x = ids(n, cuda_device, 0)
    table = i32([[3, 0, 2]], cuda_device)
    runs = []
    for cuts in ([0, n], [0, 37, 38, 99, n]):
        caches = model.caches(4)
        out = [model.step(x[a:b], caches, table, i32([0, b - a], cuda_device), i32([b], cuda_device), b - a)
               for a, b in zip(cuts, cuts[1:])]
        runs.append((caches, torch.cat(out)))
    (one, whole), (many, parts) = runs
    for a, b in ((one[0].k_codes, many[0].k_codes), (one[0].v_codes, many[0].v_codes)):
        assert torch.equal(a[table[0, :1].long()], b[table[0, :1].long()])
    assert bool(torch.isfinite(whole.float()).all()) and bool(torch.isfinite(parts.float()).all())
    assert torch.equal(whole, model.step(x, model.caches(4), table, i32([0, n], cuda_device), i32([n], cuda_device), n))
    assert torch.nn.functional.cosine_similarity(whole.float(), model(x).float(), dim=-1).median() > 0.8


def test_generate_follows_eager_steps(model, cuda_device):
    """Greedy decoding through the captured step equals eager steps, token for token and bit for bit."""
    from dscquant_b200 import ops

    prompts = [ids(70, cuda_device, 1), ids(1, cuda_device, 2), ids(129, cuda_device, 3)]
    new = 12
    got, lp = model.generate(prompts, new, page_size=16)
    again, lp2 = model.generate(prompts, new, page_size=16)
    assert torch.equal(got, again) and torch.equal(lp, lp2)
    assert got.shape == lp.shape == (3, new) and bool((lp <= 0).all())
    used = [-(-(len(p) + new) // 16) for p in prompts]
    table = torch.full((3, max(used)), -1, dtype=torch.int32)
    for b, n in enumerate(used):
        table[b, :n] = torch.arange(sum(used[:b]), sum(used[:b]) + n, dtype=torch.int32)
    table = table.to(cuda_device)
    caches = model.caches(sum(used), 16)
    counts = torch.tensor([len(p) for p in prompts], device=cuda_device)
    ends = counts.cumsum(0)
    logits = model.step(torch.cat(prompts), caches, table, torch.nn.functional.pad(ends, (1, 0)).int(), counts.int(), 129)
    nobody = torch.full((3,), -1, dtype=torch.long, device=cuda_device)
    rows = logits[ends - 1]
    for i in range(new):
        r = ops.token_logprobs(rows, nobody, top_k=1)
        assert torch.equal(r.top_ids[:, 0], got[:, i]) and torch.equal(r.top_logprobs[:, 0], lp[:, i])
        assert torch.equal(r.top_ids[:, 0], rows.float().argmax(-1))
        counts += 1
        rows = model.step(r.top_ids[:, 0], caches, table, torch.arange(4, device=cuda_device).int(), counts.int(), 1)


def test_generate_refusals(model, cuda_device):
    one = ids(3, cuda_device, 6)
    for prompts, new in (([one], 0), ([], 4), ([one, one[:0]], 4)):
        with pytest.raises(ValueError):
            model.generate(prompts, new)
    assert model.generate([one], 1)[0].shape == (1, 1)


def test_score(model, cuda_device):
    x = ids(90, cuda_device, 4)
    r = model.score(x, top_k=3)
    ref = torch.log_softmax(model(x).double(), -1)[:-1]
    want = ref.gather(-1, x[1:, None])[:, 0]
    # 32-bit arithmetic on logits of a few units: differences, exponentials and sums round by 2^-22 of them
    assert bool(((r.logprobs.double() - want).abs() <= 2.0 ** -20 * (4 + want.abs())).all())
    assert r.top_ids.shape == (89, 3) and r.entropy.shape == (89,)


def test_refusals(cuda_device):
    from dscquant_b200 import PagedKV4, ops

    bf, dev = torch.bfloat16, cuda_device
    cache = PagedKV4.allocate(4, 2, 64, 16, bf, dev)
    q, kv = torch.zeros(3, 4, 64, dtype=bf, device=dev), torch.zeros(3, 2, 64, dtype=bf, device=dev)
    tab = torch.zeros(64, 64, dtype=bf, device=dev)
    table, start, length = i32([[0, 1, 2]], dev), i32([0, 3], dev), i32([40], dev)
    good = dict(cache=cache, q=q, k=kv, v=kv, cos=tab, sin=tab, page_table=table, q_start=start, lengths=length)
    ops.kv4_append(**good)
    wide = torch.zeros(3, 4, 72, dtype=bf, device=dev)
    for change in (dict(q=q.half()), dict(q=q[0]), dict(q=q[..., :32]), dict(k=q), dict(v=kv[:2]), dict(k=kv.cpu()),
                   dict(q=wide[..., 4:68]), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(cos=tab[:, :32]),
                   dict(cos=tab.half()), dict(sin=tab[:32]), dict(cos=tab.t()), dict(sin=tab.float()),
                   dict(page_table=table.long()), dict(page_table=table[0]), dict(page_table=table.repeat(2, 1)),
                   dict(q_start=start[:1]), dict(lengths=length.long()), dict(lengths=length.cpu()),
                   dict(page_table=i32([[0, 0], [1, 1]], dev).t(), q_start=i32([0, 1, 3], dev), lengths=i32([4, 4], dev)),
                   dict(q=q.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            ops.kv4_append(**{**good, **change})
    good = dict(cache=cache, q=q, page_table=table, q_start=start, lengths=length)
    ops.kv4_attention(**good, max_q=3)
    for change in (dict(q=q[:, :3]), dict(q=q.half()), dict(max_q=-1), dict(scale=float("nan")), dict(lengths=length.float()),
                   dict(q=q.clone().requires_grad_())):
        with pytest.raises(RuntimeError):
            ops.kv4_attention(**{**good, **change})
    with torch.no_grad():
        ops.kv4_attention(**{**good, "q": q.clone().requires_grad_()})
    with pytest.raises(RuntimeError):
        ops.kv4_read(cache, table, start, length, rows=-1)
    with pytest.raises(AttributeError):
        cache.k_codes = cache.v_codes
    for bad in (dict(k_codes=cache.k_codes[:, :1]), dict(k_affine=cache.k_affine.float()), dict(v_codes=cache.v_codes.cpu()),
                dict(v_codes=cache.v_codes.transpose(0, 1)), dict(v_affine=cache.v_affine.half())):
        t = {n: getattr(cache, n) for n in ("k_codes", "k_affine", "v_codes", "v_affine")}
        with pytest.raises(RuntimeError):
            PagedKV4(**{**t, **bad})
    x, t = torch.zeros(3, 50, device=dev), torch.zeros(3, dtype=torch.long, device=dev)
    for args in ((x.double(), t), (x[0], t), (x, t[:2]), (x, t.int()), (x, t.cpu()), (x.t(), torch.zeros(50, dtype=torch.long, device=dev)),
                 (x[:1].expand(3, 50), t), (x, t, 65), (x, t, -1), (x[:, :4], t, 5), (x.clone().requires_grad_(), t)):
        with pytest.raises(RuntimeError):
            ops.token_logprobs(*args)

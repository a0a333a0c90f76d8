"""The 4-bit paged cache on the GPU: kv4_append, kv4_read and kv4_attention against their definitions in 64 bits
(kv4_reference.py), alone and together, over lengths, heads, pages, strides and masks; codes and their step and
low bit for bit, attention within the roundings it may make."""
import pytest
import torch

from kv4_reference import Batch, pack, quantise, rotate, round16, values

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


def tables(positions, D, dtype, device):
    rate = 10000.0 ** -(torch.arange(0, D, 2, dtype=torch.float64, device=device) / D)
    a = torch.outer(torch.arange(positions, dtype=torch.float64, device=device), rate).repeat(1, 2)
    return a.cos().to(dtype), a.sin().to(dtype)


def randn(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale).to(dtype)


def check_append(bt, q, k, v, cos, sin, q_out, before):
    """Queries within one rounding; the cache's new rows equal the definition's bits, its other rows untouched."""
    eps = torch.finfo(bt.dtype).eps
    want = [t.clone() for t in before]
    ref = torch.zeros_like(q_out, dtype=torch.float64)
    tol = torch.zeros_like(ref)
    for b in range(len(bt.seqs)):
        rows, pos = bt.rows(b)
        if len(pos) == 0:
            continue
        c, s = cos[pos.start:pos.stop].double()[:, None], sin[pos.start:pos.stop].double()[:, None]
        x = q[rows].double()
        ref[rows] = rotate(x, c, s)
        h = x.shape[-1] // 2
        size = (x * c).abs() + (torch.cat((x[..., h:], x[..., :h]), -1) * s).abs()
        tol[rows] = eps / 2 * ref[rows].abs() + 2.0 ** -22 * size + torch.finfo(bt.dtype).tiny * eps
        pages, off = bt.slots(b, pos.start, pos.stop)
        for y, codes, affine in ((rotate(k[rows].double(), c, s), want[0], want[1]), (v[rows].double(), want[2], want[3])):
            code, step, low = quantise(y, bt.dtype)
            codes[pages, :, off] = pack(code)
            affine[pages, :, off] = torch.cat((step, low), -1).float().to(bt.dtype)
    assert bool(((q_out.double() - ref).abs() <= tol).all())
    c = bt.cache
    for got, w in zip((c.k_codes, c.k_affine, c.v_codes, c.v_affine), want):
        if got.dtype == torch.uint8:
            assert torch.equal(got, w)
        else:
            assert torch.equal(torch.isnan(got), torch.isnan(w))
            assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(w))


def snapshot(bt):
    c = bt.cache
    return [t.clone() for t in (c.k_codes, c.k_affine, c.v_codes, c.v_affine)]


MIXES = {
    "one": [(1, 1)],
    "single": [(1, 17), (1, 64), (0, 50), (1, 65), (1, 1), (0, 0), (1, 700)],
    "ragged": [(5, 5), (3, 200), (130, 130), (70, 333), (1, 129)],
    "many": [(1, 1 + 7 * i) for i in range(70)],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,heads,kv_heads,ps", [(128, 8, 8, 64), (128, 14, 2, 16), (64, 6, 3, 32), (64, 1, 1, 128)])
@pytest.mark.parametrize("mix", MIXES)
def test_append(cuda_device, dtype, D, heads, kv_heads, ps, mix):
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(1)
    bt = Batch(MIXES[mix], kv_heads, D, ps, dtype, cuda_device, pad=3)
    q = randn((bt.T, heads, D), g, dtype)
    k, v = randn((bt.T, kv_heads, D), g, dtype, 3), randn((bt.T, kv_heads, D), g, dtype)
    k[..., 5] *= 9
    for tab in (dtype, torch.float32):
        cos, sin = tables(800, D, tab, cuda_device)
        before = snapshot(bt)
        out = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
        check_append(bt, q, k, v, cos, sin, out, before)
        assert not out[bt.starts[-1]:].any()


def test_append_strided_views(cuda_device):
    """q, k and v as slices of one fused projection, and heads-major."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(2)
    D, dtype = 128, torch.bfloat16
    cos, sin = tables(300, D, dtype, cuda_device)
    bt = Batch([(4, 100), (9, 9)], 2, D, 64, dtype, cuda_device)
    fused = randn((bt.T, 10, D), g, dtype)
    q, k, v = fused[:, :6], fused[:, 6:8], fused[:, 8:]
    before = snapshot(bt)
    out = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
    check_append(bt, q, k, v, cos, sin, out, before)
    flipped = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    after = snapshot(bt)
    assert torch.equal(ops.kv4_append(bt.cache, *flipped, cos, sin, *bt.where), out)
    for a, b in zip(snapshot(bt), after):
        assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


@pytest.mark.parametrize("dtype", TYPES)
def test_append_awkward_rows(cuda_device, dtype):
    """Constant rows, ties between codes, tiny and huge ranges, subnormals, infinities and NaN."""
    from dscquant_b200 import ops

    D = 64
    fin = torch.finfo(dtype)
    ramp = torch.arange(D, dtype=torch.float64)
    rows = [torch.full((D,), 2.5), torch.zeros(D), ramp * 0.5, -ramp, (ramp % 16) + 0.5, torch.where(ramp < 1, 0.0, 7.5),
            ramp * fin.tiny, ramp * fin.smallest_normal * 2 ** -4, (ramp - 30) * (fin.max / 64), ramp * 1e-3 + 100,
            torch.where(ramp == 3, torch.inf, ramp), torch.where(ramp == 60, -torch.inf, ramp),
            torch.where(ramp == 33, torch.nan, ramp), torch.full((D,), torch.nan), (ramp % 31) / 2]
    x = torch.stack([r.double() for r in rows]).to(dtype).to(cuda_device)
    n = len(rows)
    bt = Batch([(n, n)], 1, D, 16, dtype, cuda_device)
    cos, sin = torch.ones(n, D, dtype=dtype, device=cuda_device), torch.zeros(n, D, dtype=dtype, device=cuda_device)
    before = snapshot(bt)
    q = torch.zeros(n, 1, D, dtype=dtype, device=cuda_device)
    kv = x[:, None].contiguous()
    k = torch.where(torch.isfinite(kv), kv, torch.zeros_like(kv))  # sin = 0 times infinity is no number
    out = ops.kv4_append(bt.cache, q, k, kv, cos, sin, *bt.where)
    check_append(bt, q, k, kv, cos, sin, out, before)
    kh, vh = ops.kv4_read(bt.cache, *bt.where, rows=n)
    assert torch.equal(torch.isnan(vh).all(-1)[:, 0], ~torch.isfinite(x).all(-1))
    step = bt.cache.k_affine[bt.table[0, :1].long(), 0, :n, 0].double().reshape(n, 1)
    assert bool(((kh[:, 0].double() - k[:, 0].double()).abs() <= step * 0.75 + fin.eps * k[:, 0].double().abs().amax(-1, keepdim=True)).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
def test_read(cuda_device, dtype, D):
    """kv4_read gives code * step + low rounded once, of the newest rows or of whole sequences."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(3)
    bt = Batch([(2, 77), (0, 5), (40, 40)], 3, D, 32, dtype, cuda_device, pad=2)
    bt.fill(g)
    for whole in (False, True):
        counts = [L if whole else n for n, L in bt.seqs]
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        k, v = ops.kv4_read(bt.cache, bt.table, torch.tensor(starts, dtype=torch.int32, device=cuda_device), bt.lengths,
                            rows=starts[-1] + 2)
        for b, (_, L) in enumerate(bt.seqs):
            pages, off = bt.slots(b, L - counts[b], L)
            for got, codes, affine in ((k, bt.cache.k_codes, bt.cache.k_affine), (v, bt.cache.v_codes, bt.cache.v_affine)):
                want = round16(values(codes[pages, :, off], affine[pages, :, off]), dtype)
                assert torch.equal(got[starts[b]:starts[b + 1]].double(), want)
        assert not k[starts[-1]:].any() and not v[starts[-1]:].any()


def check_attention(bt, q, out, scale=None):
    ref, bound = bt.attention(q, scale)
    tol = bound + torch.finfo(bt.dtype).eps / 2 * (ref.abs() + bound) + torch.finfo(bt.dtype).tiny
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of what is allowed"


ATTEND = {
    "one": [(1, 1)],
    "single": [(1, 17), (1, 64), (0, 50), (1, 65), (1, 1), (0, 0), (1, 700), (1, 128)],
    "drafts": [(4, 4), (3, 90), (2, 65), (6, 1000)],
    "prompts": [(130, 130), (70, 333), (1, 129), (257, 257)],
    "empty rows": [(5, 3), (4, 0), (140, 100), (2, 2)],
    "many": [(1, 1 + 9 * i) for i in range(70)],
    "long": [(1, 9000), (2, 5001)],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,heads,kv_heads,ps", [(128, 4, 4, 64), (128, 16, 2, 64), (128, 7, 1, 16), (64, 24, 2, 16),
                                                 (64, 2, 2, 128), (128, 40, 1, 32)])
@pytest.mark.parametrize("mix", ATTEND)
def test_attention(cuda_device, dtype, D, heads, kv_heads, ps, mix):
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(4)
    bt = Batch(ATTEND[mix], kv_heads, D, ps, dtype, cuda_device, pad=2)
    bt.fill(g, v_offset=0.5)
    q = randn((bt.T, heads, D), g, dtype, 1.5)
    most = max(n for n, _ in bt.seqs)
    out = ops.kv4_attention(bt.cache, q, *bt.where, max_q=most)
    check_attention(bt, q, out)
    assert torch.equal(out, ops.kv4_attention(bt.cache, q, *bt.where, max_q=most))  # no order of arrival in the bits
    assert not out[bt.starts[-1]:].any()


PROMPTS = {
    "whole": [(300, 300), (129, 129), (257, 257)],
    "chunks": [(200, 1000), (65, 3000), (1, 50), (300, 437)],
    "empty rows": [(300, 170), (200, 0), (130, 1), (128, 128)],
    "mixed": [(1, 700), (400, 400), (0, 9), (3, 90), (70, 71)],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,heads,kv_heads,ps", [(128, 32, 32, 64), (128, 64, 8, 16), (64, 48, 16, 128), (64, 33, 11, 32)])
@pytest.mark.parametrize("mix", PROMPTS)
def test_attention_prompts(cuda_device, dtype, D, heads, kv_heads, ps, mix):
    """Enough rows and heads for the tensor-core kernel, single tokens and drafts among them."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(11)
    bt = Batch(PROMPTS[mix], kv_heads, D, ps, dtype, cuda_device, pad=3)
    bt.fill(g, k_scale=1.5, v_offset=0.3)
    q = randn((bt.T, heads, D), g, dtype, 1.5)
    out = ops.kv4_attention(bt.cache, q, *bt.where)
    check_attention(bt, q, out)
    assert torch.equal(out, ops.kv4_attention(bt.cache, q, *bt.where))
    assert not out[bt.starts[-1]:].any()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_prompts_with_awkward_cache(cuda_device, dtype):
    """The tensor-core kernel on rows that are no numbers, seen or not, pages out of range, values that grow by
    orders of magnitude along the keys, constant rows, and keys of very different sizes."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(12)
    hk, D = 32, 64
    bt = Batch([(300, 400), (260, 260)], hk, D, 16, dtype, cuda_device)
    bt.fill(g)
    grow = torch.logspace(-3, 3, 400, base=10 if dtype is torch.bfloat16 else 4, device=cuda_device)
    pages, off = bt.slots(0, 0, 400)
    bt.cache.v_affine[pages, :, off] = (bt.cache.v_affine[pages, :, off].float() * grow[:, None, None]).to(dtype)
    flat, foff = bt.slots(1, 30, 60)
    bt.cache.v_affine[flat, :, foff, 0] = 0  # constant rows
    bt.cache.k_affine[flat, :, foff, 0] = 0
    q = randn((bt.T, hk, D), g, dtype)
    check_attention(bt, q, ops.kv4_attention(bt.cache, q, *bt.where))
    for side in ("k_affine", "v_affine"):
        affine = getattr(bt.cache, side)
        kept = affine.clone()
        pages, off = bt.slots(1, 200, 201)
        affine[pages, :, off] = torch.nan
        out = ops.kv4_attention(bt.cache, q, *bt.where)
        seen = torch.zeros(bt.T, dtype=torch.bool, device=cuda_device)
        seen[300 + 200:] = True
        assert torch.equal(torch.isnan(out).all(-1).all(-1), seen) and torch.equal(torch.isnan(out).any(-1).any(-1), seen)
        affine.copy_(kept)
    want = ops.kv4_attention(bt.cache, q, *bt.where)
    bt.table[0, 5] = bt.pages + 3
    out = ops.kv4_attention(bt.cache, q, *bt.where)
    assert ops.device_status(cuda_device) == 4
    assert torch.equal(out[300:], want[300:]) and torch.isfinite(out).all()


@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (96, 2)])
def test_crowd(cuda_device, heads, kv_heads):
    """More sequences than a warp or a CTA adds up at once, idle ones and a few prompts among them."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(13)
    seqs = [(i % 3 != 0, 1 + i % 37) for i in range(1300)]
    seqs[5], seqs[700], seqs[1290] = (150, 170), (90, 90), (70, 300)
    bt = Batch([(int(n), L) for n, L in seqs], kv_heads, 64, 16, torch.bfloat16, cuda_device, pad=4)
    bt.fill(g)
    q = randn((bt.T, heads, 64), g, torch.bfloat16)
    k, v = randn((bt.T, kv_heads, 64), g, torch.bfloat16), randn((bt.T, kv_heads, 64), g, torch.bfloat16)
    cos, sin = tables(400, 64, torch.bfloat16, cuda_device)
    before = snapshot(bt)
    out = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
    check_append(bt, q, k, v, cos, sin, out, before)
    a = ops.kv4_attention(bt.cache, out, *bt.where)
    check_attention(bt, out, a)
    assert not a[bt.starts[-1]:].any()


def test_attention_scale_strides_and_sharp_softmax(cuda_device):
    """Another scale, queries as a strided view, weights on single keys, keys far from zero."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(5)
    for dtype in TYPES:
        bt = Batch([(1, 300), (3, 400), (150, 200)], 2, 128, 64, dtype, cuda_device)
        bt.fill(g, k_scale=4.0, v_offset=-3.0)
        q = randn((bt.T, 10, 128), g, dtype, 4)[:, 1:9]
        check_attention(bt, q, ops.kv4_attention(bt.cache, q, *bt.where, scale=0.3), 0.3)
        check_attention(bt, q, ops.kv4_attention(bt.cache, q, *bt.where, scale=0.0), 0.0)
        check_attention(bt, q, ops.kv4_attention(bt.cache, q, *bt.where, scale=-0.2), -0.2)
        big = Batch([(150, 200), (300, 300)], 16, 128, 64, dtype, cuda_device)
        big.fill(g, k_scale=4.0, v_offset=-3.0)
        q = randn((big.T, 18, 128), g, dtype, 4)[:, 1:17]
        for scale in (0.3, 0.0, -0.2):
            check_attention(big, q, ops.kv4_attention(big.cache, q, *big.where, scale=scale), scale)


def test_attention_shared_pages_and_wide_table(cuda_device):
    """Two sequences reading the same prefix pages, in a table far wider than they use and with a row stride."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(6)
    bt = Batch([(1, 200), (2, 190)], 2, 128, 64, torch.bfloat16, cuda_device, wide=500)
    bt.table[1, :3] = bt.table[0, :3]
    bt.fill(g)
    big = torch.full((2, 700), -7, dtype=torch.int32, device=cuda_device)
    big[:, :500] = bt.table
    bt.table = big[:, :500]
    q = randn((bt.T, 4, 128), g, torch.bfloat16)
    check_attention(bt, q, ops.kv4_attention(bt.cache, q, *bt.where))


def test_attention_poisoned_keys_show(cuda_device):
    """A visible cached row of NaN reaches exactly the rows that see it."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(7)
    bt = Batch([(4, 70), (1, 90), (140, 140)], 1, 64, 16, torch.bfloat16, cuda_device)
    bt.fill(g)
    for b, at in ((0, 68), (2, 100)):
        pages, off = bt.slots(b, at, at + 1)
        bt.cache.v_affine[pages, :, off] = torch.nan
    q = randn((bt.T, 2, 64), g, torch.bfloat16)
    out = ops.kv4_attention(bt.cache, q, *bt.where)
    seen = torch.zeros(bt.T, dtype=torch.bool, device=cuda_device)
    seen[2:4] = True
    seen[5 + 100:5 + 140] = True
    assert torch.equal(torch.isnan(out).all(-1).all(-1), seen) and torch.equal(torch.isnan(out).any(-1).any(-1), seen)


def test_out_of_range_pages_are_left_out(cuda_device):
    """Page ids, positions and lengths outside the batch: nothing is touched, the status word says so."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(8)
    dtype, D = torch.bfloat16, 64
    cos, sin = tables(100, D, dtype, cuda_device)
    for spoil in ("page", "negative page", "length", "table rows", "before the first"):
        bt = Batch([(1, 40), (1, 50)], 1, D, 16, dtype, cuda_device)
        bt.fill(g)
        q, kv = randn((2, 2, D), g, dtype), randn((2, 1, D), g, dtype)
        c, s = cos, sin
        if spoil == "page":
            bt.table[0, 2] = bt.pages
        elif spoil == "negative page":
            bt.table[0, 2] = -1
        elif spoil == "length":
            bt.lengths[0] = 16 * bt.table.shape[1] + 1
        elif spoil == "table rows":
            c, s = cos[:30], sin[:30]
        else:
            bt.lengths[0] = 0
        before = snapshot(bt)
        out = ops.kv4_append(bt.cache, q, kv, kv, c, s, *bt.where)
        assert ops.device_status(cuda_device) == 4, spoil
        for got, was in zip(snapshot(bt), before):
            pages, off = bt.slots(1, 49, 50)
            got[pages, :, off] = was[pages, :, off]
            assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(was.float())) or spoil == "table rows"
        assert not out[0].any()
        if spoil in ("page", "negative page", "length"):
            a = ops.kv4_attention(bt.cache, q, *bt.where)
            assert ops.device_status(cuda_device) == 4
            ops.kv4_read(bt.cache, *bt.where, rows=2)
            assert ops.device_status(cuda_device) == 4
            assert torch.isfinite(a[1]).all()


def test_nothing_to_do(cuda_device):
    from dscquant_b200 import ops

    bt = Batch([(0, 20)], 1, 64, 16, torch.bfloat16, cuda_device)
    e = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    cos, sin = tables(30, 64, torch.bfloat16, cuda_device)
    assert ops.kv4_append(bt.cache, e, e[:, :1], e[:, :1], cos, sin, *bt.where).shape == (0, 2, 64)
    assert ops.kv4_attention(bt.cache, e, *bt.where).shape == (0, 2, 64)
    none = (bt.table[:0], bt.q_start[:1], bt.lengths[:0])
    q = torch.ones((3, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    assert not ops.kv4_attention(bt.cache, q, *none).any()
    assert not ops.kv4_append(bt.cache, q, q[:, :1], q[:, :1], cos, sin, *none).any()


def test_append_then_attend_token_by_token(cuda_device):
    """A prompt appended and attended at once, then token by token: the same cache and, row by row, the same
    attention as the whole sequence in one call allows; on a stream of its own."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(9)
    D, hq, hk, dtype, n = 128, 8, 2, torch.bfloat16, 150
    cos, sin = tables(n, D, dtype, cuda_device)
    q, k, v = randn((n, hq, D), g, dtype), randn((n, hk, D), g, dtype), randn((n, hk, D), g, dtype)
    whole = Batch([(n, n)], hk, D, 64, dtype, cuda_device)
    steps = Batch([(n, n)], hk, D, 64, dtype, cuda_device)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream(cuda_device)):
        qr = ops.kv4_append(whole.cache, q, k, v, cos, sin, *whole.where)
        out = ops.kv4_attention(whole.cache, qr, *whole.where)
        torch.cuda.current_stream().synchronize()
        for lo, hi in [(0, 137)] + [(i, i + 1) for i in range(137, n)]:
            start = torch.tensor([0, hi - lo], dtype=torch.int32, device=cuda_device)
            length = torch.tensor([hi], dtype=torch.int32, device=cuda_device)
            r = ops.kv4_append(steps.cache, q[lo:hi], k[lo:hi], v[lo:hi], cos, sin, steps.table, start, length)
            assert torch.equal(r, qr[lo:hi])
            a = ops.kv4_attention(steps.cache, r, steps.table, start, length, max_q=hi - lo)
            ref, bound = whole.attention(qr)
            tol = bound + torch.finfo(dtype).eps / 2 * (ref.abs() + bound)
            assert bool(((a.double() - ref[lo:hi]).abs() <= tol[lo:hi]).all())
        torch.cuda.current_stream().synchronize()
    check_attention(whole, qr, out)
    for a, b in zip(snapshot(whole), snapshot(steps)):
        assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(b.float()))


def test_captured_step_follows_its_arrays(cuda_device):
    """One captured append + attention replayed while lengths, pages and rows change, next to a second captured
    step; padded rows stay zero."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(10)
    D, hq, hk, dtype = 128, 8, 2, torch.float16
    cos, sin = tables(1000, D, dtype, cuda_device)

    def step(seqs, seed):
        bt = Batch(seqs, hk, D, 64, dtype, cuda_device, seed=seed, pad=1, wide=16)
        bt.fill(g)
        q, k, v = randn((bt.T, hq, D), g, dtype), randn((bt.T, hk, D), g, dtype), randn((bt.T, hk, D), g, dtype)
        return bt, q, k, v

    def run(bt, q, k, v):
        r = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
        return r, ops.kv4_attention(bt.cache, r, *bt.where, max_q=1)

    held = [step([(1, 10), (1, 900), (1, 333)], 0), step([(1, 700), (1, 1), (1, 64)], 1)]
    graphs, outs = [], []
    for st in held:
        run(*st)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(*st))
        graphs.append(graph)
    for lengths in ([11, 901, 334], [1000, 1, 65]):
        for (bt, q, k, v), graph in zip(held, graphs):
            fresh = Batch([(1, n) for n in lengths], hk, D, 64, dtype, cuda_device, seed=7, pad=1, wide=16,
                          spare=0)
            if fresh.pages > bt.pages:
                continue
            bt.table.copy_(fresh.table)
            bt.lengths.copy_(fresh.lengths)
            bt.seqs = fresh.seqs
            bt.fill(g)
            q.copy_(randn(q.shape, g, dtype))
        side = torch.cuda.Stream(cuda_device)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for (bt, q, k, v), (r, a) in zip(held, outs):
            check_attention(bt, r, a)
            assert not a[bt.starts[-1]:].any()
    del graphs

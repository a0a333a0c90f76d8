"""4-bit cache attention where cached rows differ by orders of magnitude or carry unusual numbers: rows a query does not
see, or hardly weighs, must not cost it precision. Compared in 64 bits with bounds taken over the keys each row sees."""
import pytest
import torch

from kv4_reference import Batch, pack, quantise, values

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]

# (rows, cached tokens) of the sequences, heads, key heads: the few-row kernel, then the tensor-core one
FEW = ([(4, 90), (1, 300), (6, 700)], 8, 2)
MANY = ([(300, 300), (260, 400)], 32, 32)


def randn(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=gen.device) * scale).to(dtype)


def reference(bt, q, scale=None):
    """(out, tolerance) in float64. Per row and over the keys j it sees, p_j their weights: scores are off by 32-bit sums of
    D products of |q| (15 |step| + |low|) and a rounding of each key to 11 bits, weights by that on both sides of their
    normalisation; a weight (times up to 15 steps) and a value each round to 11 bits; weights under 2^-31 of the largest
    contribution and elements under 2^-27 of their row may go."""
    T, hq, D = q.shape
    group, scale = hq // bt.kv_heads, D ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    for b, (n, L) in enumerate(bt.seqs):
        if n == 0 or L <= 0:
            continue
        rows, pos = bt.rows(b)
        pages, off = bt.slots(b, 0, L)
        seen = torch.arange(L, device=q.device)[None] <= torch.tensor(list(pos), device=q.device)[:, None]
        for h in range(bt.kv_heads):
            ka, va = bt.cache.k_affine[pages, h, off].double(), bt.cache.v_affine[pages, h, off].double()
            k = values(bt.cache.k_codes[pages, h, off], ka)
            v = values(bt.cache.v_codes[pages, h, off], va)
            for g in range(h * group, (h + 1) * group):
                x = q[rows, g].double()
                p = torch.softmax((x @ k.T * scale).masked_fill(~seen, -torch.inf), -1)
                p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                out[rows, g] = p @ v
                size = x.abs().sum(-1, keepdim=True) * (15 * ka[:, 0].abs() + ka[:, 1].abs())
                off_s = torch.where(seen, abs(scale) * (2.0 ** -23 * D * size + 2.0 ** -12 * (x.abs() @ k.abs().T)), 0.0)
                off_s = off_s.amax(-1, keepdim=True) + 2.0 ** -20
                row = v.abs().amax(-1)
                tol[rows, g] = (2.1 * off_s + 2.0 ** -12) * (p @ v.abs()) + 2.0 ** -11 * (p @ (15 * va[:, :1].abs())) + \
                    2.0 ** -27 * (p @ row)[:, None] + L * 2.0 ** -31 * (p * row).amax(-1, keepdim=True)
    return out, tol + torch.finfo(bt.dtype).eps / 2 * (out.abs() + tol) + torch.finfo(bt.dtype).tiny


def check(bt, q, out, scale=None):
    ref, tol = reference(bt, q, scale)
    err = (out.double() - ref).abs()
    assert bool((err <= tol).all()), f"off by {float((err / tol).max()):.2f} of what is allowed"


def put(bt, b, at, side, y):
    """Cached rows of position `at` of sequence b: the quantised rows y [kv_heads, D]."""
    pages, off = bt.slots(b, at, at + 1)
    code, step, low = quantise(y[None].double(), bt.dtype)
    getattr(bt.cache, side + "_codes")[pages, :, off] = pack(code)
    getattr(bt.cache, side + "_affine")[pages, :, off] = torch.cat((step, low), -1).to(bt.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mix", [FEW, MANY], ids=["few", "many"])
def test_steps_of_either_sign(cuda_device, dtype, D, mix):
    """element = code * step + low holds for any pair: negative steps alone, and beside positive ones sixteen times smaller."""
    from dscquant_b200 import ops

    seqs, heads, kv_heads = mix
    g = torch.Generator(device=cuda_device).manual_seed(21)
    for signs in ("negative", "both"):
        bt = Batch(seqs, kv_heads, D, 16, dtype, cuda_device)
        bt.fill(g, v_offset=0.5)
        for affine in (bt.cache.k_affine, bt.cache.v_affine):
            a = torch.nan_to_num(affine.float())
            flip = torch.ones_like(a[..., 0]) if signs == "negative" else \
                (torch.rand(a[..., 0].shape, generator=g, device=cuda_device) < 0.3).float()
            size = 1.0 if signs == "negative" else 1 + 15 * flip
            # the row upside down: low becomes its largest element
            affine[..., 1] = torch.where(flip > 0, a[..., 1] + 15 * a[..., 0] * size, a[..., 1]).to(dtype)
            affine[..., 0] = torch.where(flip > 0, -a[..., 0] * size, a[..., 0]).to(dtype)
        q = randn((bt.T, heads, D), g, dtype, 0.3)
        check(bt, q, ops.kv4_attention(bt.cache, q, *bt.where))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mix", [FEW, MANY], ids=["few", "many"])
def test_tiny_queries_keys_and_scales(cuda_device, dtype, mix):
    """Scores that all but vanish weigh every visible key alike: zero or tiny keys, tiny queries, a tiny scale."""
    from dscquant_b200 import ops

    seqs, heads, kv_heads = mix
    g = torch.Generator(device=cuda_device).manual_seed(22)
    D = 64
    small = 2.0 ** -60 if dtype is torch.bfloat16 else 2.0 ** -14
    for keys, size, scale in ((0.0, small, None), (small, small, None), (1.0, 1.0, 1e-38), (1.0, small, 1e-30), (0.0, 1.0, -1e-38)):
        bt = Batch(seqs, kv_heads, D, 16, dtype, cuda_device)
        bt.fill(g, v_offset=0.5)
        bt.cache.k_affine.copy_((torch.nan_to_num(bt.cache.k_affine.float()) * keys).to(dtype))
        q = randn((bt.T, heads, D), g, dtype, size)
        check(bt, q, ops.kv4_attention(bt.cache, q, *bt.where, scale=scale), scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mix", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("log2", [12, 14, 40, 100])
@pytest.mark.parametrize("side", ["k", "v"])
def test_rows_do_not_feel_what_they_cannot_see(cuda_device, dtype, mix, log2, side):
    """The newest tokens of each sequence far larger than all others: the rows before them are as exact as without them."""
    from dscquant_b200 import ops

    if dtype is torch.float16 and log2 > 14:
        pytest.skip("beyond fp16")
    seqs, heads, kv_heads = mix
    g = torch.Generator(device=cuda_device).manual_seed(23)
    D = 64
    bt = Batch(seqs, kv_heads, D, 16, dtype, cuda_device)
    bt.fill(g)
    for b, (n, L) in enumerate(seqs):
        # the largest of a sequence of many rows stands inside a block of keys that earlier rows see
        for at in ({L - 1} if n < 64 else {L - 1, L - 70}):
            put(bt, b, at, side, torch.randn(kv_heads, D, generator=g, device=cuda_device) * 2.0 ** log2)
    q = randn((bt.T, heads, D), g, dtype)
    out = ops.kv4_attention(bt.cache, q, *bt.where)
    ref, tol = reference(bt, q)
    before = torch.zeros(bt.T, dtype=torch.bool, device=cuda_device)
    for b, (n, L) in enumerate(seqs):
        last = L - 1 if n < 64 else L - 70
        before[[bt.starts[b] + i for i, p in enumerate(range(L - n, L)) if p < last]] = True
    assert int(before.sum()) > 5
    err = (out.double() - ref).abs()[before] / tol[before]
    assert bool((err <= 1).all()), f"off by {float(err.max()):.2f} of what is allowed"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mix", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("log2", [12, 14, 60])
def test_large_values_of_no_weight(cuda_device, dtype, mix, log2):
    """The first key's value is far larger than all others and its score far lower: it counts as much as its weight says."""
    from dscquant_b200 import ops

    if dtype is torch.float16 and log2 > 14:
        pytest.skip("beyond fp16")
    seqs, heads, kv_heads = mix
    g = torch.Generator(device=cuda_device).manual_seed(24)
    D = 64
    bt = Batch(seqs, kv_heads, D, 16, dtype, cuda_device)
    bt.fill(g)
    low = torch.zeros(kv_heads, D, device=cuda_device)
    low[:, 0] = -32.0 if log2 < 60 else -240.0
    for b in range(len(seqs)):
        put(bt, b, 0, "k", low)
        put(bt, b, 0, "v", torch.randn(kv_heads, D, generator=g, device=cuda_device) * 2.0 ** log2)
    q = randn((bt.T, heads, D), g, dtype)
    q[..., 0] = 8
    # the rows that see the first key alone have nothing else to be exact about
    check(bt, q, ops.kv4_attention(bt.cache, q, *bt.where))


@pytest.mark.parametrize("D", [64, 128])
def test_f16_prompts_are_exact_but_for_two_roundings(cuda_device, D):
    """f16 prompts and chunks over keys with channels seven times the others. The output and the weights round to 11 bits, by
    at most 2^-11 / sqrt(3) each in the mean square; independent, they add up to 2^-11 sqrt(2/3). All else is 32-bit."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(25)
    bt = Batch([(300, 1500), (257, 2100)], 16, D, 64, torch.float16, cuda_device)
    for b, (_, L) in enumerate(bt.seqs):
        pages, off = bt.slots(b, 0, L)
        loud = 1 + 6 * (torch.rand(1, 16, D, generator=g, device=cuda_device) < 0.03)
        for side, by in (("k", loud), ("v", 1)):
            y = torch.randn(L, 16, D, generator=g, device=cuda_device, dtype=torch.float64) * by
            code, step, low = quantise(y, torch.float16)
            getattr(bt.cache, side + "_codes")[pages, :, off] = pack(code)
            getattr(bt.cache, side + "_affine")[pages, :, off] = torch.cat((step, low), -1).half()
    q = randn((bt.T, 32, D), g, torch.float16)
    ref = reference(bt, q)[0]
    for max_q in (None, 300):
        out = ops.kv4_attention(bt.cache, q, *bt.where, max_q=max_q).double()
        assert float((out - ref).norm() / ref.norm()) <= 2.0 ** -11 * (2 / 3) ** 0.5 * 1.01


@pytest.mark.parametrize("mix", [FEW, MANY], ids=["few", "many"])
def test_rows_behind_the_page_table_are_zero(cuda_device, mix):
    """A length beyond what the page table holds: rows at positions behind it are left out (zero), the others stay."""
    from dscquant_b200 import ops

    seqs, heads, kv_heads = mix
    g = torch.Generator(device=cuda_device).manual_seed(26)
    bt = Batch(seqs, kv_heads, 64, 16, torch.bfloat16, cuda_device)
    bt.fill(g)
    q = randn((bt.T, heads, 64), g, torch.bfloat16)
    n, L = seqs[-1]
    room = 16 * bt.table.shape[1]
    assert room - L < n or L == room
    # the last sequence moves up until only its first two rows are inside
    over = room - 2 + n
    bt.table[-1, L // 16:] = bt.table[-1, 0]
    bt.lengths[-1] = over
    out = ops.kv4_attention(bt.cache, q, *bt.where)
    assert ops.device_status(cuda_device) == 4
    lo = bt.starts[-2]
    assert not out[lo + 2:].any()
    bt.lengths[-1] = room
    bt.q_start[-1] = lo + 2
    want = ops.kv4_attention(bt.cache, q[:lo + 2].contiguous(), *bt.where)
    assert bool(out[lo:lo + 2].any())
    err = (out[:lo + 2].float() - want.float()).abs()
    assert bool((err <= 2.0 ** -6 * want.float().abs() + 2.0 ** -8).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("mix", [FEW, MANY], ids=["few", "many"])
def test_rows_of_every_size(cuda_device, dtype, D, mix):
    """Each cached row of a size of its own (keys smaller than the queries' units, values either way), zero and constant rows
    among them, then a value row that is no number and a page out of range."""
    from dscquant_b200 import ops

    seqs, heads, kv_heads = mix
    g = torch.Generator(device=cuda_device).manual_seed(27)
    bt = Batch(seqs, kv_heads, D, 16, dtype, cuda_device)
    bt.fill(g, v_offset=0.3)
    wide = 40 if dtype is torch.bfloat16 else 8

    def exponents(lo, hi):
        return torch.randint(lo, hi + 1, bt.cache.k_affine.shape[:3], generator=g, device=cuda_device)

    for affine, by in ((bt.cache.k_affine, exponents(-wide, 0)), (bt.cache.v_affine, exponents(-wide, wide))):
        a = torch.nan_to_num(affine.float()) * 2.0 ** by[..., None]
        kind = exponents(0, 15)
        a[..., 0] = torch.where(kind < 2, 0.0, a[..., 0])
        a[..., 1] = torch.where(kind == 0, 0.0, a[..., 1])
        affine.copy_(a.to(dtype))
    q = randn((bt.T, heads, D), g, dtype)
    want = ops.kv4_attention(bt.cache, q, *bt.where)
    check(bt, q, want)
    assert torch.equal(want, ops.kv4_attention(bt.cache, q, *bt.where))
    n, L = seqs[-1]
    pages, off = bt.slots(len(seqs) - 1, L - 2, L - 1)
    kept = bt.cache.v_affine.clone()
    bt.cache.v_affine[pages, :, off] = torch.nan
    out = ops.kv4_attention(bt.cache, q, *bt.where)
    sees = torch.zeros(bt.T, dtype=torch.bool, device=cuda_device)
    sees[bt.starts[-1] - 2:] = True
    assert torch.isnan(out[sees]).all() and torch.equal(out[~sees], want[~sees])
    bt.cache.v_affine.copy_(kept)
    bt.table[0, 1] = bt.pages
    out = ops.kv4_attention(bt.cache, q, *bt.where)
    assert ops.device_status(cuda_device) == 4
    assert torch.isfinite(out).all() and torch.equal(out[bt.starts[1]:], want[bt.starts[1]:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mix", [FEW, MANY], ids=["few", "many"])
@pytest.mark.parametrize("key", [-8.0, 8.0, -250.0, 250.0])
def test_scores_far_from_zero(cuda_device, dtype, mix, key):
    """Scores of thousands, of either sign and all alike: every row is the mean of the values it sees."""
    from dscquant_b200 import ops

    seqs, heads, kv_heads = mix
    g = torch.Generator(device=cuda_device).manual_seed(28)
    bt = Batch(seqs, kv_heads, 64, 16, dtype, cuda_device)
    bt.fill(g, v_offset=0.5)
    bt.cache.k_affine[..., 0] = 0
    bt.cache.k_affine[..., 1] = key
    q = torch.full((bt.T, heads, 64), 31.0, dtype=dtype, device=cuda_device)
    for scale in (None, 1.0):
        out = ops.kv4_attention(bt.cache, q, *bt.where, scale=scale).double()
        ref = reference(bt, q, scale)[0]
        # equal weights, 11-bit values and a rounded output: elements of at most 5 by 2^-12 of the terms and half a step
        assert bool(((out - ref).abs() <= 2.0 ** -11 * 5 + torch.finfo(dtype).eps / 2 * ref.abs()).all())

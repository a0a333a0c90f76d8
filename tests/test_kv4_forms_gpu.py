"""Forms of the 4-bit cache operators that long calls take: tokens enough for a thread to append several rows, contexts
cut over more thread blocks than one joining step reads, pages up to the largest, captured steps whose arrays change."""
import pytest
import torch

from kv4_reference import Batch
from test_kv4_gpu import check_append, check_attention, randn, snapshot, tables

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("table_f32", [False, True])
@pytest.mark.parametrize("D,heads,kv_heads", [(128, 32, 32), (128, 14, 2), (64, 33, 11), (64, 3, 1), (128, 40, 5)])
def test_append_of_many_tokens(cuda_device, dtype, table_f32, D, heads, kv_heads):
    """More than eight tokens an SM (a block takes a token with all its rows): several rounds a thread, the last one
    ragged, rows that need 64 bits in late rounds, rows of no sequence, one on a page out of range."""
    from dscquant_b200 import ops

    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    g = torch.Generator(device=cuda_device).manual_seed(31)
    seqs = [(700, 700), (1, 90), (0, 40), (8 * sms - 500, 8 * sms - 400), (33, 64)]
    bt = Batch(seqs, kv_heads, D, 32, dtype, cuda_device, pad=5)
    assert bt.T > 8 * sms
    q = randn((bt.T, heads, D), g, dtype)
    k, v = randn((bt.T, kv_heads, D), g, dtype, 3), randn((bt.T, kv_heads, D), g, dtype)
    k[..., 5] *= 9
    # ties between codes, constant rows and subnormals in the last heads, whose rows come in the last rounds
    ramp = torch.arange(D, device=cuda_device)
    v[::3, -1] = ((ramp % 16) + 0.5).to(dtype)
    v[1::3, -1] = 2.5
    v[2::9, -1] = (ramp * torch.finfo(dtype).smallest_normal * 2 ** -4).to(dtype)
    k[::5, -1] = 0
    k[1::5, -1] = 1.5
    tab = torch.float32 if table_f32 else dtype
    cos, sin = tables(max(L for _, L in seqs), D, tab, cuda_device)
    before = snapshot(bt)
    out = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
    check_append(bt, q, k, v, cos, sin, out, before)
    assert not out[bt.starts[-1]:].any()
    # the same with the page of 32 of the first sequence's tokens out of range: nothing else changes
    full = snapshot(bt)
    for t in (bt.cache.k_codes, bt.cache.v_codes, bt.cache.k_affine, bt.cache.v_affine):
        t.fill_(0)
    lost = bt.table[0, 3].clone()
    bt.table[0, 3] = bt.pages
    again = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
    assert ops.device_status(cuda_device) == 4
    assert not again[96:128].any()
    keep = torch.ones(bt.T, dtype=torch.bool, device=cuda_device)
    keep[96:128] = False
    assert torch.equal(again[keep], out[keep])
    bt.table[0, 3] = lost
    for b, (n, L) in enumerate(seqs):
        for lo, hi in ((L - n, L),) if b else ((0, 96), (128, 700)):
            pages, off = bt.slots(b, lo, hi)
            for got, want in zip(snapshot(bt), full):
                assert torch.equal(torch.nan_to_num(got[pages, :, off].float()), torch.nan_to_num(want[pages, :, off].float()))
    for t in snapshot(bt):
        assert not t[lost.long()].any()


@pytest.mark.parametrize("rows,heads", [(1, 1), (1, 8), (3, 4), (2, 16)])
@pytest.mark.parametrize("dtype", TYPES)
def test_one_context_over_many_blocks(cuda_device, dtype, rows, heads):
    """One key head, one long context: its tiles go over all SMs, pieces of more than 32 blocks are joined; runs that end
    next to a border of 32 blocks."""
    from dscquant_b200 import ops

    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    warps = 12 if rows * heads <= 8 else 8
    g = torch.Generator(device=cuda_device).manual_seed(32)
    # one tile of 64 keys a warp up to `warps` x SMs tiles: a run of 32 n blocks' tiles, one less and one more
    for tiles in (32 * warps - 1, 32 * warps, 32 * warps + 1, 64 * warps, 64 * warps + 1, sms * warps, 2 * sms * warps + 3):
        L = 64 * tiles - 5
        bt = Batch([(rows, L)], 1, 64, 64, dtype, cuda_device)
        bt.fill(g, v_offset=0.5)
        q = randn((bt.T, heads, 64), g, dtype, 1.5)
        out = ops.kv4_attention(bt.cache, q, *bt.where)
        check_attention(bt, q, out)
        assert torch.equal(out, ops.kv4_attention(bt.cache, q, *bt.where))


def test_two_contexts_over_many_blocks(cuda_device):
    """A run that begins inside a block and crosses more than 32 others, with short ones around it."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(33)
    for dtype in TYPES:
        bt = Batch([(1, 2000), (2, 60001), (1, 1), (1, 30000), (0, 9), (1, 777)], 1, 64, 128, dtype, cuda_device)
        bt.fill(g, v_offset=0.5)
        q = randn((bt.T, 4, 64), g, dtype, 1.5)
        for max_q in (None, 2):
            check_attention(bt, q, ops.kv4_attention(bt.cache, q, *bt.where, max_q=max_q))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ps", [256, 512, 1024])
def test_large_pages(cuda_device, dtype, ps):
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(34)
    for seqs, heads, kv_heads in (([(1, 17), (3, 1030), (1, 2048), (0, 5)], 4, 2), ([(300, 1400), (1, 3), (257, 257)], 32, 32)):
        bt = Batch(seqs, kv_heads, 64, ps, dtype, cuda_device, pad=2)
        assert bt.cache.nbytes() == bt.pages * kv_heads * ps * 2 * (32 + 4)
        bt.fill(g, v_offset=0.5)
        q = randn((bt.T, heads, 64), g, dtype)
        k, v = randn((bt.T, kv_heads, 64), g, dtype, 3), randn((bt.T, kv_heads, 64), g, dtype)
        cos, sin = tables(3000, 64, dtype, cuda_device)
        before = snapshot(bt)
        out = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
        check_append(bt, q, k, v, cos, sin, out, before)
        check_attention(bt, out, ops.kv4_attention(bt.cache, out, *bt.where))


def test_positions_behind_the_angles_touch_nothing(cuda_device):
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(35)
    cos, sin = tables(40, 64, torch.bfloat16, cuda_device)
    bt = Batch([(1, 41), (2, 40), (1, 90)], 1, 64, 16, torch.bfloat16, cuda_device)
    bt.fill(g)
    q, kv = randn((bt.T, 2, 64), g, torch.bfloat16), randn((bt.T, 1, 64), g, torch.bfloat16)
    before = snapshot(bt)
    out = ops.kv4_append(bt.cache, q, kv, kv, cos, sin, *bt.where)
    assert ops.device_status(cuda_device) == 4
    assert not out[0].any() and not out[3].any() and bool(out[1:3].any())
    inside = [(bt.slots(1, 38, 40))]
    for got, was in zip(snapshot(bt), before):
        for pages, off in inside:
            assert not torch.equal(got[pages, :, off], was[pages, :, off])
            got[pages, :, off] = was[pages, :, off]
        assert torch.equal(torch.nan_to_num(got.float()), torch.nan_to_num(was.float()))


def test_two_captured_steps_follow_their_arrays(cuda_device):
    """Two captured append + attention steps replayed on two streams at once while lengths and page tables of both change."""
    from dscquant_b200 import ops

    g = torch.Generator(device=cuda_device).manual_seed(36)
    D, hq, hk, dtype = 128, 8, 2, torch.bfloat16
    cos, sin = tables(1100, D, dtype, cuda_device)

    def step(lengths, seed):
        bt = Batch([(1, n) for n in lengths], hk, D, 64, dtype, cuda_device, seed=seed, pad=1, wide=17, spare=20)
        bt.fill(g)
        return bt, randn((bt.T, hq, D), g, dtype), randn((bt.T, hk, D), g, dtype), randn((bt.T, hk, D), g, dtype)

    def run(bt, q, k, v):
        r = ops.kv4_append(bt.cache, q, k, v, cos, sin, *bt.where)
        return r, ops.kv4_attention(bt.cache, r, *bt.where, max_q=1)

    held = [step([10, 900, 333], 0), step([700, 1, 64], 1)]
    graphs, outs = [], []
    for st in held:
        run(*st)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(*st))
        graphs.append(graph)
    for turn, lengths in enumerate(([11, 901, 334], [1000, 1, 65], [64, 1088, 2])):
        for i, ((bt, q, k, v), _) in enumerate(zip(held, graphs)):
            own = lengths if i == 0 else lengths[::-1]
            fresh = Batch([(1, n) for n in own], hk, D, 64, dtype, cuda_device, seed=40 + 2 * turn + i, pad=1, wide=17, spare=0)
            assert fresh.pages <= bt.pages and not torch.equal(fresh.lengths, bt.lengths) and not torch.equal(fresh.table, bt.table)
            bt.table.copy_(fresh.table)
            bt.lengths.copy_(fresh.lengths)
            bt.seqs = fresh.seqs
            bt.fill(g)
            for t in (q, k, v):
                t.copy_(randn(t.shape, g, dtype))
        before = [snapshot(st[0]) for st in held]
        side = torch.cuda.Stream(cuda_device)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        torch.cuda.synchronize()
        for (bt, q, k, v), (r, a), was in zip(held, outs, before):
            check_append(bt, q, k, v, cos, sin, r, was)
            check_attention(bt, r, a)
            assert not a[bt.starts[-1]:].any()
    del graphs

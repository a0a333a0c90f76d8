"""The 4-bit paged cache's operators in 64 bits, straight from their definitions, and batches to try them on."""
import torch


def round16(y, dtype):
    """Float64 -> the 16-bit type (through 32 bits, as the kernels round) -> float64."""
    return y.float().to(dtype).double()


def rotate(x, cos, sin):
    """x [..., D] float64 with tables of the same last dimension (rotate-half form)."""
    h = x.shape[-1] // 2
    return x * cos + torch.cat((-x[..., h:], x[..., :h]), -1) * sin


def quantise(y, dtype):
    """Rows [..., D] float64 -> codes, step, low (float64; the last two [..., 1])."""
    low = round16(y.amin(-1, keepdim=True), dtype)
    step = round16((y.amax(-1, keepdim=True) - low) / 15, dtype)
    bad = ~(torch.isfinite(low) & torch.isfinite(step))
    code = torch.where(bad | (step == 0), 0.0, ((y - low) / step).round().clamp(0, 15))
    return code, torch.where(bad, torch.nan, step), torch.where(bad, torch.nan, low)


def pack(code):
    c = code.to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def values(codes, affine):
    """Cached rows -> float64 values [..., D]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double()
    return c * affine[..., :1].double() + affine[..., 1:].double()


class Batch:
    """Sequences given as (rows, cached tokens) pairs over a pool with a shuffled page table; -1 where unmapped."""

    def __init__(self, seqs, kv_heads, D, page_size, dtype, device, seed=0, pad=0, spare=2, wide=None):
        from dscquant_b200 import PagedKV4

        g = torch.Generator(device="cpu").manual_seed(seed)
        self.seqs, self.D, self.ps, self.dtype, self.kv_heads = seqs, D, page_size, dtype, kv_heads
        used = [-(-max(L, 0) // page_size) for _, L in seqs]
        self.pages = sum(used) + spare
        order = torch.randperm(self.pages, generator=g).to(torch.int32)
        P = max(used + [1]) if wide is None else wide
        table = torch.full((len(seqs), P), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            table[b, :n] = order[at:at + n]
            at += n
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.T = starts[-1] + pad
        self.table = table.to(device)
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=device)
        self.lengths = torch.tensor([L for _, L in seqs], dtype=torch.int32, device=device)
        self.cache = PagedKV4.allocate(self.pages, kv_heads, D, page_size, dtype, device)
        for t in (self.cache.k_codes, self.cache.v_codes):
            t.fill_(0xA7)
        for t in (self.cache.k_affine, self.cache.v_affine):
            t.fill_(torch.nan)  # what no append wrote must not be read

    @property
    def where(self):
        return self.table, self.q_start, self.lengths

    def slots(self, b, lo, hi):
        """(pages, offsets) of positions lo .. hi-1 of sequence b."""
        pos = torch.arange(lo, hi, device=self.table.device)
        return self.table[b, pos // self.ps].long(), pos % self.ps

    def fill(self, gen, k_scale=1.0, v_offset=0.0):
        """Quantised normal rows in every cached position."""
        for b, (_, L) in enumerate(self.seqs):
            if L <= 0:
                continue
            pages, off = self.slots(b, 0, L)
            for codes, affine, s, o in ((self.cache.k_codes, self.cache.k_affine, k_scale, 0.0),
                                        (self.cache.v_codes, self.cache.v_affine, 1.0, v_offset)):
                y = torch.randn(L, self.kv_heads, self.D, generator=gen, device=codes.device, dtype=torch.float64) * s + o
                code, step, low = quantise(y, self.dtype)
                codes[pages, :, off] = pack(code)
                affine[pages, :, off] = torch.cat((step, low), -1).to(self.dtype)

    def rows(self, b):
        """Token-axis slice and positions of sequence b's rows."""
        n, L = self.seqs[b]
        return slice(self.starts[b], self.starts[b + 1]), range(L - n, L)

    def attention(self, q, scale=None):
        """(out, bound) in float64. `bound`: how far a kernel may be off before its last rounding, when it keeps
        scores and sums in 32 bits, rounds each softmax weight to the cache's type or better once, and may
        take keys, values and weights as fp16 scaled by powers of two (11 bits, 2^-18 of the largest at least,
        weights 2^-25 at least)."""
        T, hq, D = q.shape
        group = hq // self.kv_heads
        scale = D ** -0.5 if scale is None else scale
        half = torch.finfo(self.dtype).eps / 2
        out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
        bound = torch.zeros_like(out)
        for b, (n, L) in enumerate(self.seqs):
            if n == 0 or L <= 0:
                continue
            rows, pos = self.rows(b)
            pages, off = self.slots(b, 0, L)
            seen = torch.arange(L, device=q.device)[None] <= torch.tensor(list(pos), device=q.device)[:, None]
            for h in range(self.kv_heads):
                ka, va = self.cache.k_affine[pages, h, off].double(), self.cache.v_affine[pages, h, off].double()
                k = values(self.cache.k_codes[pages, h, off], ka)
                v = values(self.cache.v_codes[pages, h, off], va)
                for g in range(h * group, (h + 1) * group):
                    x = q[rows, g].double()
                    s = (x @ k.T * scale).masked_fill(~seen, -torch.inf)
                    p = torch.softmax(s, -1)
                    p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                    out[rows, g] = p @ v
                    # scores: D products of |q| times up to 32 steps (codes as 16..31 sixteenths) and the low
                    # part, each accumulation off by 2^-23, and keys rounded to 11 bits; weights follow as exp of
                    # that error, on both sides of the normalisation; the exponential and the sums add 2^-20
                    size = x.abs().sum(-1, keepdim=True) * (32 * ka[:, 0].abs().max() + ka[:, 1].abs().max())
                    rounded = torch.where(seen, x.abs() @ k.abs().T, 0.0).amax(-1, keepdim=True) * 2.0 ** -12 + \
                        x.abs().sum(-1, keepdim=True) * k.abs().max() * 2.0 ** -18
                    off_s = abs(scale) * (2.0 ** -23 * D * size + rounded) + 2.0 ** -20
                    bound[rows, g] = half * 1.01 * (p @ (v - va[:, 1:]).abs()) + 2.1 * off_s * (p @ v.abs()) + \
                        2.0 ** -11 * (p @ v.abs()) + (2.0 ** -18 + L * 2.0 ** -25) * v.abs().max()
        return out, bound

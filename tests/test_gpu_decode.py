"""The text decoder's operators on the B200 (include/ppocr_b200_decode.h)
against their restatements in 64 bits (oracle/decode.py).

Tolerances of the attention, per output value, from the roundings it makes:
u is the unit roundoff of the cache's 16-bit type (2^-11 fp16, 2^-8 bf16).
Probabilities, restored values and the output are each rounded to it, at most
3 u sum(p |v|) together to first order; scores carry an error e of their own,
which changes each probability by at most a factor exp(2 e). Where keys are
restored to the 16-bit type, e is u scale sum|q k|; where they are multiplied
as codes, only fp32 sums round (2^-20 scale sum|q k| covers 128 channels)."""

import itertools
import math

import numpy as np
import pytest
import torch

from oracle import decode as O

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def gen(seed):
    return torch.Generator().manual_seed(20261206 + seed)


def fault(native):
    torch.cuda.synchronize()
    return native.ppocr_b200_device_error()


class Scene:
    """A pool with shuffled pages, what it should hold, and its tokens."""

    def __init__(self, lengths, new, kv, dim, page, dtype, seed=0, spare=3, stale="nan", width=None):
        from ppocr_b200 import decode

        g = gen(seed)
        self.lengths, self.new, self.kv, self.dim, self.page, self.dtype = lengths, new, kv, dim, page, dtype
        batch = len(lengths)
        self.width = width or max(1, -(-max(lengths) // page))
        pages = batch * self.width + spare
        self.table = torch.randperm(pages, generator=g)[: batch * self.width].view(batch, self.width).int()
        block = O.block_bytes(page, dim)
        if stale == "nan":  # 0xFF: NaN scales and minimums in both types
            self.pool = torch.full((pages, kv, block), 255, dtype=torch.uint8)
        else:
            self.pool = torch.randint(0, 256, (pages, kv, block), generator=g, dtype=torch.uint8)
        wide = torch.exp(0.5 * torch.randn(kv, dim, generator=g))
        self.k, self.v = [], []
        for length in lengths:
            self.k.append((torch.randn(length, kv, dim, generator=g) * wide).to(dtype))
            self.v.append(torch.randn(length, kv, dim, generator=g).to(dtype))
        self.starts = torch.tensor([0] + list(itertools.accumulate(new)), dtype=torch.int32)
        self.decode = decode

    def fill(self, upto):
        """Writes each sequence's first upto[b] tokens into the host pool."""
        for b, n in enumerate(upto):
            pos = torch.arange(n)
            page, slot = self.table[b].long()[pos // self.page], pos % self.page
            views = O.views(self.pool, self.page, self.dim, self.dtype)
            for which, x in ((0, self.k[b]), (1, self.v[b])):
                codes, scale, low = O.quantise(x[:n])
                views[which][page, :, slot] = codes[..., 0::2] | (codes[..., 1::2] << 4)
                views[2 + which][page, :, slot] = torch.stack([scale, low], -1)

    def cache(self):
        return self.decode.KvCache4(self.pool.shape[0], self.page, self.kv, self.dim, dtype=self.dtype,
                                    pool=self.pool.cuda())

    def places(self):
        return self.table.cuda(), torch.tensor(self.lengths, dtype=torch.int32).cuda()

    def tail(self, xs):
        return torch.cat([x[len(x) - n:] for x, n in zip(xs, self.new)])


# ------------------------------------------------------- writing and reading
CACHE_CASES = [
    # lengths, new, kv heads, dim, page, type
    ([1], [1], 1, 32, 16, F16),
    ([1, 16, 17, 33], [1, 1, 1, 1], 4, 64, 16, F16),
    ([5, 0, 64, 129], [5, 0, 3, 129], 2, 128, 64, BF16),
    ([300, 31, 128], [300, 30, 1], 3, 64, 32, BF16),
    ([127, 128, 129, 257], [127, 2, 129, 100], 8, 128, 128, F16),
    ([77], [77], 5, 32, 32, BF16),
    ([15, 16, 17], [15, 16, 17], 1, 128, 16, F16),
]


@pytest.mark.parametrize("lengths,new,kv,dim,page,dtype", CACHE_CASES)
@pytest.mark.parametrize("strided", [False, True])
def test_append_and_read(native, cuda, lengths, new, kv, dim, page, dtype, strided):
    s = Scene(lengths, new, kv, dim, page, dtype, seed=sum(lengths) + dim, stale="random")
    s.fill([a - b for a, b in zip(lengths, new)])
    cache = s.cache()
    k, v = s.tail(s.k), s.tail(s.v)
    tokens = k.shape[0]
    if strided:  # slices of a wider projection
        both = torch.zeros(tokens, 2 * kv * dim + 24, dtype=dtype)
        both[:, 8:8 + kv * dim] = k.flatten(1)
        both[:, 16 + kv * dim:16 + 2 * kv * dim] = v.flatten(1)
        both = both.cuda()
        dk = both[:, 8:8 + kv * dim].unflatten(1, (kv, dim))
        dv = both[:, 16 + kv * dim:16 + 2 * kv * dim].unflatten(1, (kv, dim))
    else:
        dk, dv = k.cuda(), v.cuda()
    table, lens = s.places()
    cache.append(dk, dv, table, lens, starts=s.starts.cuda(), max_new=max(new))
    rk, rv = cache.read(table, lens, tokens, starts=s.starts.cuda(), max_new=max(new) + 2)
    assert fault(native) == 0
    s.fill(lengths)
    # Every byte: the new tokens as the definition has them, the rest as it was.
    assert torch.equal(cache.pool.cpu(), s.pool)
    for got, xs, which in ((rk, s.k, 0), (rv, s.v, 1)):
        want = torch.cat([O.held(s.pool, page, dim, dtype, s.table[b], lengths[b], which)[lengths[b] - new[b]:]
                          for b in range(len(lengths))])
        assert torch.equal(got.cpu(), want.to(dtype))
    # The whole of each sequence reads back through the same call.
    whole = torch.tensor([0] + list(itertools.accumulate(lengths)), dtype=torch.int32).cuda()
    rk, _ = cache.read(table, lens, sum(lengths), starts=whole, max_new=max(lengths))
    want = torch.cat([O.held(s.pool, page, dim, dtype, s.table[b], lengths[b], 0) for b in range(len(lengths))])
    assert torch.equal(rk.cpu(), want.to(dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_unusual_values(native, cuda, dtype):
    """Constant groups, zeros, NaN, infinities, the type's extremes and tiny values."""
    big = float(torch.finfo(dtype).max)
    tiny = float(torch.finfo(dtype).tiny)
    rows = torch.zeros(8, 2, 64)
    rows[0] = 3.25
    rows[1, 0, 5] = math.nan
    rows[1, 1] = torch.linspace(-4, 4, 64)
    rows[1, 1, 7] = math.inf
    rows[2] = torch.linspace(-1, 1, 128).view(2, 64)
    rows[2, 0, 3] = -math.inf
    rows[3, 0, 0], rows[3, 0, 1] = big, -big
    rows[4] = math.nan
    rows[5] = tiny * torch.arange(128).view(2, 64).float()
    rows[6] = tiny / 4
    rows[7, 1, 63] = -big
    s = Scene([8], [8], 2, 64, 16, dtype, stale="random")
    s.k, s.v = [rows.to(dtype)], [rows.flip(0).to(dtype)]
    cache = s.cache()
    table, lens = s.places()
    cache.append(s.k[0].cuda(), s.v[0].cuda(), table, lens)
    rk, rv = cache.read(table, lens, 8)
    assert fault(native) == 0
    s.fill([8])
    assert torch.equal(cache.pool.cpu(), s.pool)
    assert torch.isfinite(rk.float()).all() and torch.isfinite(rv.float()).all()
    want = O.held(s.pool, 16, 64, dtype, s.table[0], 8, 0)
    assert torch.equal(rk.cpu(), want.to(dtype))


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_append_scales_on_rounding_boundaries(native, cuda, dtype):
    """Groups whose range is 15 times a midpoint of the 16-bit type: the scale
    is what the fp32 product with 1/15 rounds to, not the quotient."""
    digits = 11 if dtype == F16 else 8
    steps = torch.arange(2 ** (digits - 1), 2 ** digits).double() + 0.5  # midpoints
    high = 15 * steps * 2.0 ** -digits
    rows = torch.zeros(len(steps), 1, 32)
    # The range, split over the ends so that both are representable.
    top = high.to(dtype)
    rest = (high - top.double()).to(dtype)
    keep = (top.double() + rest.double() == high)
    rows[:, 0, 0], rows[:, 0, 1] = top.float(), -rest.float()
    rows[:, 0, 2:] = (torch.rand(len(steps), 30, generator=gen(50)) * 0.9 + 0.05) * top.float()[:, None]
    x = rows[keep & (rest.double() >= 0)].to(dtype)
    assert len(x) >= 16
    s = Scene([len(x)], [len(x)], 1, 32, 64, dtype, stale="random")
    s.k, s.v = [x], [x.flip(0)]
    cache = s.cache()
    table, lens = s.places()
    cache.append(x.cuda(), s.v[0].cuda(), table, lens)
    assert fault(native) == 0
    s.fill([len(x)])
    assert torch.equal(cache.pool.cpu(), s.pool)


def test_cache_error_of_quantisation(native, cuda):
    """What reads back is within half a step (plus the scale's and the
    output's own rounding) of what was written."""
    s = Scene([200], [200], 4, 128, 32, F16, seed=5)
    cache = s.cache()
    table, lens = s.places()
    cache.append(s.k[0].cuda(), s.v[0].cuda(), table, lens)
    rk, _ = cache.read(table, lens, 200)
    x = s.k[0].double().unflatten(-1, (-1, 32))
    step = (x.amax(-1) - x.amin(-1)) / 15
    err = (rk.cpu().double().unflatten(-1, (-1, 32)) - x).abs().amax(-1)
    # scale rounds by 2^-11: up to 15 * 2^-11 steps at the top code; values by 2^-11
    bound = step * (0.5 + 15 * 2.0 ** -11) + x.abs().amax(-1) * 2.0 ** -11 + 1e-6
    assert (err <= bound).all()


def test_more_new_tokens_than_length(native, cuda):
    """Rows whose position would be negative: not written, read as zero, see nothing."""
    s = Scene([3, 0], [5, 2], 2, 32, 16, F16, stale="nan")
    cache = s.cache()
    table, lens = s.places()
    x = torch.randn(7, 2, 32, generator=gen(1)).half().cuda()
    cache.append(x, x, table, lens, starts=s.starts.cuda(), max_new=5)
    k, v = cache.read(table, lens, 7, starts=s.starts.cuda(), max_new=5)
    o = cache.attention(x, table, lens, starts=s.starts.cuda(), max_new=5)
    assert fault(native) == 0
    for y in (k, v, o):
        assert torch.isfinite(y.float()).all()
        assert (y[:2] == 0).all() and (y[5:] == 0).all()
        assert (y[2:5] != 0).any()
    # The written positions are 0..2 of sequence 0 alone.
    touched = (cache.pool.cpu() != 255).any(-1).any(-1).nonzero().flatten().tolist()
    assert touched == [int(s.table[0, 0])]


# ------------------------------------------------------------------ attention
def check_attention(native, s, heads, window=0, sinks=0, scale=None, strided=True, keys_rounded=False, seed=9,
                    rows=None, cache=None):
    s.fill(s.lengths)
    cache = cache or s.cache()
    table, lens = s.places()
    tokens = sum(s.new)
    g = gen(seed)
    q = (torch.randn(tokens, heads, s.dim, generator=g) * torch.exp(torch.randn(tokens, 1, 1, generator=g) / 2)).to(s.dtype)
    if strided:
        wide = torch.full((tokens, heads * s.dim + 16), math.nan, dtype=s.dtype)
        wide[:, 8:8 + heads * s.dim] = q.flatten(1)
        dq = wide.cuda()[:, 8:8 + heads * s.dim].unflatten(1, (heads, s.dim))
    else:
        dq = q.cuda()
    args = dict(starts=s.starts.cuda(), max_new=max(s.new), window=window, sinks=sinks, scale=scale)
    got = cache.attention(dq, table, lens, **args)
    again = cache.attention(dq, table, lens, **args)
    assert fault(native) == 0
    assert torch.equal(got, again), "two runs differ"
    got = got.cpu().double()
    scale = s.dim ** -0.5 if scale is None else scale
    u = U[s.dtype]
    at = 0
    for b, n in enumerate(s.new):
        k = O.held(s.pool, s.page, s.dim, s.dtype, s.table[b], s.lengths[b], 0)
        v = O.held(s.pool, s.page, s.dim, s.dtype, s.table[b], s.lengths[b], 1)
        pick = range(n) if rows is None else sorted({i for i in rows if i < n} | ({n - 1} if n else set()))
        for i in pick:
            want, mag, most = O.attention(q[at + i:at + i + 1], k, v, s.lengths[b] - n + i, scale, window, sinks)
            e = (u if keys_rounded else 2.0 ** -20) * most
            tol = mag * (3.2 * u + torch.expm1(2.2 * e)[..., None]) + 2.0 ** -24
            err = (got[at + i:at + i + 1] - want).abs()
            assert (err <= tol).all(), (
                f"sequence {b} token {i}: worst {float((err - tol).max()):.3g} over the bound "
                f"(error {float(err.max()):.3g})")
        at += n
    return cache


STEP_CASES = [
    # lengths, heads, kv heads, dim, page, type
    ([1], 1, 1, 32, 16, F16),
    ([1, 2, 15, 16, 17], 4, 4, 64, 16, F16),
    ([31, 32, 33, 127, 128, 129], 8, 2, 128, 32, BF16),
    ([255, 256, 257, 0, 640], 8, 1, 128, 64, F16),
    ([1000, 3, 511], 6, 2, 64, 128, BF16),
    ([700, 64], 16, 2, 32, 32, BF16),
    ([513, 90], 16, 1, 128, 128, F16),       # 16 rows a unit
    ([300, 129], 24, 2, 64, 64, BF16),       # 12 rows a unit
    ([200], 40, 2, 128, 16, BF16),           # 20 rows: two row groups
    ([5000, 17, 2600], 4, 4, 128, 64, F16),  # units split over CTAs
    ([9001], 8, 8, 64, 32, BF16),
    ([4100], 16, 1, 32, 128, F16),
]


@pytest.mark.parametrize("lengths,heads,kv,dim,page,dtype", STEP_CASES)
def test_attention_single_token(native, cuda, lengths, heads, kv, dim, page, dtype):
    s = Scene(lengths, [1 if n else 0 for n in lengths], kv, dim, page, dtype, seed=sum(lengths))
    check_attention(native, s, heads)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (64, 0), (128, 4), (200, 17), (5000, 3), (333, 400)])
@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_window_and_sinks(native, cuda, window, sinks, dtype):
    s = Scene([1, 130, 900, 1500, 4000], [1, 1, 1, 1, 1], 2, 64, 32, dtype, seed=window + sinks)
    check_attention(native, s, 8, window=window, sinks=sinks)


@pytest.mark.parametrize("new,lengths,heads,kv,dim,page,dtype", [
    ([2, 3, 4], [2, 300, 1000], 2, 2, 64, 16, F16),
    ([4, 4], [700, 129], 16, 4, 128, 64, BF16),
    ([8, 1, 0], [8, 2000, 5], 8, 2, 128, 32, F16),
    ([5], [260], 3, 1, 32, 16, BF16),
])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 5)])
def test_attention_few_tokens(native, cuda, new, lengths, heads, kv, dim, page, dtype, window, sinks):
    s = Scene(lengths, new, kv, dim, page, dtype, seed=sum(lengths))
    check_attention(native, s, heads, window=window, sinks=sinks, keys_rounded=True)


PROMPT_CASES = [
    # new, lengths, heads, kv heads, dim, page, type
    ([33], [33], 1, 1, 64, 16, F16),
    ([128], [128], 1, 1, 128, 128, F16),
    ([129], [129], 1, 1, 128, 64, BF16),
    ([1, 64, 0, 127], [1, 64, 0, 127], 2, 2, 32, 16, F16),
    ([256, 257, 90], [256, 257, 400], 4, 4, 64, 32, BF16),
    ([70, 300], [700, 1500], 8, 2, 128, 64, F16),
    ([100], [1000], 16, 1, 32, 128, BF16),
    ([65, 8], [2000, 9], 12, 4, 128, 16, BF16),
    ([700], [700], 6, 2, 64, 64, F16),
]


@pytest.mark.parametrize("new,lengths,heads,kv,dim,page,dtype", PROMPT_CASES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 0), (300, 9)])
def test_attention_prompt(native, cuda, new, lengths, heads, kv, dim, page, dtype, window, sinks):
    s = Scene(lengths, new, kv, dim, page, dtype, seed=sum(lengths) + dim)
    some = {0, 1, 15, 16, 31, 32, 63, 64, 65, 127, 128, 129, 255, 256, 300}
    check_attention(native, s, heads, window=window, sinks=sinks, keys_rounded=True, rows=some)


@pytest.mark.parametrize("scale", [4.0, -0.1, 0.0])
def test_attention_prompt_scales(native, cuda, scale):
    s = Scene([400], [200], 2, 128, 32, F16, seed=41)
    check_attention(native, s, 4, scale=scale, keys_rounded=True, rows={0, 100, 150})


def test_attention_prompt_nan_stays_in_its_row(native, cuda):
    s = Scene([300], [100], 2, 64, 16, F16, seed=42)
    s.fill([300])
    cache = s.cache()
    table, lens = s.places()
    q = torch.randn(100, 4, 64, generator=gen(3)).half()
    clean = cache.attention(q.cuda(), table, lens)
    q[40, 1, 7] = math.nan
    got = cache.attention(q.cuda(), table, lens)
    assert fault(native) == 0
    assert torch.isnan(got[40, 1].float()).all()
    keep = torch.ones(100, 4, dtype=torch.bool)
    keep[40, 1] = False
    assert torch.equal(got.cpu()[keep], clean.cpu()[keep])


def test_attention_large_scores(native, cuda):
    """Scores far beyond exp's range: the running maximum carries them."""
    s = Scene([600, 70], [1, 1], 2, 128, 32, F16, seed=3)
    check_attention(native, s, 4, scale=3.0)


def test_attention_zero_scale_is_the_mean(native, cuda):
    s = Scene([300], [1], 1, 64, 64, F16, seed=4)
    check_attention(native, s, 2, scale=0.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_small_and_large_queries(native, cuda, dtype):
    """Query rows are scaled by powers of two inside: rows of very different
    size, all-zero rows and the type's extremes give what they should."""
    s = Scene([260], [6], 1, 64, 32, dtype, seed=8)
    s.fill([260])
    cache = s.cache()
    table, lens = s.places()
    q = torch.randn(6, 1, 64, generator=gen(2))
    size = torch.tensor([0.0, 2.0 ** -14, 1e-3, 1.0, 300.0, 2.0 ** 9])
    q = (q * size[:, None, None]).to(dtype)
    o = cache.attention(q.cuda(), table, lens, scale=2.0 ** -9).cpu().double()
    assert fault(native) == 0
    k, v = (O.held(s.pool, 32, 64, dtype, s.table[0], 260, w) for w in (0, 1))
    want, mag, most = O.attention(q, k, v, 254, 2.0 ** -9)
    tol = mag * (3.2 * U[dtype] + torch.expm1(2.2 * U[dtype] * most)[..., None]) + 2.0 ** -24
    assert ((o - want).abs() <= tol).all()


@pytest.mark.parametrize("new", [1, 80])
@pytest.mark.parametrize("sizes", [[1e-30, 1e-3, 1.0, 1e15, 1e30], [1e30, 1.0, 1e-30], [0.0, 0.0, 1e-35], [3e37, 3e37]])
def test_attention_bf16_values_of_any_size(native, cuda, new, sizes):
    """bf16 values far beyond fp16's range, growing and shrinking along the cache."""
    s = Scene([900], [new], 2, 64, 64, BF16, seed=13)
    each = -(-900 // len(sizes))
    s.v[0] = (s.v[0].float().clamp(-2, 2) * torch.tensor(sizes).repeat_interleave(each)[:900, None, None]).to(BF16)
    check_attention(native, s, 4, keys_rounded=new > 1, rows={0, 40})


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_many_light_keys(native, cuda, dtype):
    """One key far above thousands of light ones, whose shares together count."""
    n = 6000
    s = Scene([n], [1], 1, 32, 128, dtype, seed=14)
    s.k[0] = torch.zeros(n, 1, 32).to(dtype)
    s.k[0][7] = 1.0
    s.v[0] = (torch.ones(n, 1, 32) + 0.25 * torch.randn(n, 1, 32, generator=gen(15))).to(dtype)
    s.fill([n])
    cache = s.cache()
    q = torch.full((1, 1, 32), 14 / 32, dtype=dtype)
    got = cache.attention(q.cuda(), *s.places(), scale=1.0).cpu().double()
    assert fault(native) == 0
    k, v = (O.held(s.pool, 128, 32, dtype, s.table[0], n, w) for w in (0, 1))
    want, mag, most = O.attention(q, k, v, n - 1, 1.0)
    assert ((got - want).abs() <= mag * (3.2 * U[dtype] + math.expm1(2.2 * 2.0 ** -20 * float(most.max())))).all()


def test_attention_nan_query_stays_in_its_row(native, cuda):
    s = Scene([100, 50], [1, 1], 2, 64, 16, F16, seed=6)
    s.fill([100, 50])
    cache = s.cache()
    table, lens = s.places()
    q = torch.randn(2, 4, 64, generator=gen(3)).half()
    clean = cache.attention(q.cuda(), table, lens)
    q[0, 1, 7] = math.nan
    q[1, 2, 0] = math.inf
    got = cache.attention(q.cuda(), table, lens)
    assert fault(native) == 0
    bad = torch.zeros(2, 4, dtype=torch.bool)
    bad[0, 1] = bad[1, 2] = True
    assert torch.isnan(got.cpu().float()[bad]).all()
    assert torch.equal(got.cpu()[~bad], clean.cpu()[~bad])


def test_attention_cache_past_32_bit_offsets(native, cuda):
    """A pool of more than 2^32 bytes, the sequence in its last pages."""
    from ppocr_b200 import decode

    kv, dim, page = 8, 128, 128
    block = O.block_bytes(page, dim)
    pages = (2 ** 32 + 2 ** 28) // (block * kv)
    s = Scene([1000], [1], kv, dim, page, F16, seed=12, spare=0)
    s.fill([1000])
    width = s.width
    pool = torch.zeros(pages, kv, block, dtype=torch.uint8, device="cuda")
    high = torch.arange(pages - width, pages)
    pool[pages - width:] = s.pool[s.table[0].long()].cuda()
    cache = decode.KvCache4(pages, page, kv, dim, pool=pool)
    table = high.int().view(1, -1).cuda()
    lens = torch.tensor([1000], dtype=torch.int32).cuda()
    q = torch.randn(1, 16, dim, generator=gen(4)).half()
    got = cache.attention(q.cuda(), table, lens)
    small = s.cache().attention(q.cuda(), *s.places())
    assert torch.equal(got, small)
    x = torch.randn(1, kv, dim, generator=gen(5)).half().cuda()
    cache.append(x, x, table, lens)
    k, v = cache.read(table, lens, 1)
    assert fault(native) == 0
    want = O.restore(*O.quantise(x.cpu())).half()
    assert torch.equal(k.cpu(), want) and torch.equal(v.cpu(), want)


def test_attention_on_a_side_stream_and_reused_workspace(native, cuda):
    """Different shapes through one workspace, in turn, on another stream."""
    a = Scene([5000, 40], [1, 1], 1, 128, 64, F16, seed=21)
    b = Scene([900], [3], 1, 128, 64, F16, seed=22)
    a.fill(a.lengths)
    b.fill(b.lengths)
    ca, cb = a.cache(), b.cache()
    cb.workspace = ca.workspace
    qa = torch.randn(2, 8, 128, generator=gen(6)).half().cuda()
    qb = torch.randn(3, 4, 128, generator=gen(7)).half().cuda()
    first = ca.attention(qa, *a.places()), cb.attention(qb, *b.places())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    pa, pb = a.places(), b.places()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [(ca.attention(qa, *pa), cb.attention(qb, *pb)) for _ in range(5)]
    side.synchronize()
    assert fault(native) == 0
    for x, y in outs:
        assert torch.equal(x, first[0]) and torch.equal(y, first[1])


def test_attention_of_thousands_of_sequences(native, cuda):
    """More (sequence, row group) entries than one launch's prefix holds."""
    lengths = [1 + (i * 7) % 40 for i in range(2600)]
    s = Scene(lengths, [1] * 2600, 1, 32, 16, F16, seed=33, width=3)
    s.fill(lengths)
    cache = s.cache()
    q = torch.randn(2600, 2, 32, generator=gen(34)).half()
    got = cache.attention(q.cuda(), *s.places()).cpu().double()
    assert fault(native) == 0
    for b in (0, 1, 1023, 2047, 2048, 2049, 2599):
        k, v = (O.held(s.pool, 16, 32, F16, s.table[b], lengths[b], w) for w in (0, 1))
        want, mag, most = O.attention(q[b:b + 1], k, v, lengths[b] - 1, 32 ** -0.5)
        tol = mag * (3.2 * U[F16] + torch.expm1(2.2 * 2.0 ** -20 * most)[..., None]) + 2.0 ** -24
        assert ((got[b:b + 1] - want).abs() <= tol).all(), b


@pytest.mark.parametrize("new,length,heads,kv", [(40, 6000, 2, 1), (130, 3000, 4, 2), (33, 2047, 1, 1)])
def test_attention_prompt_over_a_long_cache(native, cuda, new, length, heads, kv):
    """Few row blocks: several CTAs share a block's key tiles."""
    s = Scene([length], [new], kv, 64, 64, F16, seed=length)
    check_attention(native, s, heads, keys_rounded=True, rows={0, 1, 31, 39, 64, 128})
    check_attention(native, s, heads, keys_rounded=True, window=900, sinks=3, rows={0, 39})


def test_append_then_attention_then_append(native, cuda):
    """Token by token through the cache equals the whole prompt at once."""
    s = Scene([70], [70], 2, 64, 16, F16, seed=30)
    cache = s.cache()
    table, _ = s.places()
    q = torch.randn(70, 4, 64, generator=gen(8)).half().cuda()
    k, v = s.k[0].cuda(), s.v[0].cuda()
    steps = []
    for i in range(70):
        lens = torch.tensor([i + 1], dtype=torch.int32).cuda()
        cache.append(k[i:i + 1], v[i:i + 1], table, lens)
        steps.append(cache.attention(q[i:i + 1], table, lens))
    steps = torch.cat(steps)
    prompt = s.cache()
    lens = torch.tensor([70], dtype=torch.int32).cuda()
    prompt.append(k, v, table, lens)
    whole = prompt.attention(q, table, lens)
    assert fault(native) == 0
    assert torch.equal(cache.pool, prompt.pool)
    kk, vv = (O.held(cache.pool.cpu(), 16, 64, F16, s.table[0], 70, w) for w in (0, 1))
    _, mag, most = O.attention(q.cpu(), kk, vv, 0, 0.125)
    tol = mag * (6.4 * U[F16] + torch.expm1(4.4 * U[F16] * most)[..., None]) + 2.0 ** -23
    assert ((whole.cpu().double() - steps.cpu().double()).abs() <= tol).all()


def test_device_reports_bad_pages_and_lengths(native, cuda):
    """What the host cannot see: kept in bounds and reported."""
    s = Scene([40], [1], 1, 32, 16, F16, seed=31)
    s.fill([40])
    cache = s.cache()
    table, lens = s.places()
    q = torch.randn(1, 1, 32).half().cuda()
    assert fault(native) == 0
    bad = table.clone()
    bad[0, 1] = 10 ** 6
    cache.attention(q, bad, lens)
    assert fault(native) == 61
    bad[0, 1] = -1
    cache.append(q, q, bad, torch.tensor([20], dtype=torch.int32).cuda())
    assert fault(native) == 61
    cache.attention(q, table, torch.tensor([49], dtype=torch.int32).cuda())  # the table has 48 positions
    assert fault(native) == 62
    cache.read(table, lens, 1, starts=torch.tensor([0, 9], dtype=torch.int32).cuda(), max_new=4)
    assert fault(native) == 62
    ok = cache.attention(q, table, lens)
    assert fault(native) == 0 and torch.isfinite(ok.float()).all()


# ------------------------------------------------------------------- sampling
def draw(logits, uniform, **kw):
    from ppocr_b200 import decode

    rows = logits.shape[0]
    dev = {}
    for name, v in kw.items():
        t = torch.int32 if name == "top_k" else torch.float32
        dev[name] = torch.as_tensor(v, dtype=t).expand(rows).contiguous().cuda()
    ids, prob, kept = decode.sample(logits if logits.is_cuda else logits.cuda(), uniform.cuda(), **dev)
    torch.cuda.synchronize()
    return ids.cpu().long(), prob.cpu().double(), kept.cpu().long()


def check_sample(logits, uniform, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Each id is one that the uniform number may pick, each count one that
    the masses allow: masses are floor(e 2^32) of fp32 e (relative error of
    the exponent's argument 2^-23 |d| / T and of e 2^-22, absolute 2^-32)."""
    ids, prob, kept = draw(logits, uniform, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    host = logits.cpu()
    V = host.shape[1]
    for r in range(host.shape[0]):
        order, ps, n = O.sample_row(host[r].float(), temperature, top_k, top_p, min_p)
        t = temperature if temperature > 0 else 1.0
        rel = 2.0 ** -21 * (1 + 25 / max(t, 1.0) + 25)
        eps = rel + V * 2.0 ** -32 / float((ps / ps[0]).sum()) + 2.0 ** -23
        total = float(ps[: (top_k if 0 < top_k < V else V)].sum())
        got = int(kept[r])
        if got != n:  # allowed only when a threshold lies within the error
            a, b = sorted((got, n))
            near_p = top_p < 1 and abs(float(ps[:a].sum()) - top_p * total) <= 2 * eps * total + float(ps[a:b - 1].sum())
            near_m = min_p > 0 and abs(float(ps[b - 1] / ps[0]) - min_p) <= 2 * eps
            assert near_p or near_m, f"row {r}: kept {got}, expected {n}"
        ranked = order[:got]
        assert int(ids[r]) in set(ranked.tolist()), f"row {r}: id {int(ids[r])} is not among the {got} kept"
        stay = torch.zeros(V, dtype=torch.float64)
        stay[ranked] = ps[:got]
        cum = stay.cumsum(0) / stay.sum()
        i, u = int(ids[r]), float(uniform[r])
        before = float(cum[i - 1]) if i else 0.0
        assert before - 2 * eps <= u <= float(cum[i]) + 2 * eps, f"row {r}: {before} <= {u} <= {float(cum[i])}"
        p = float(ps[(order == i).nonzero()[0, 0]])
        assert abs(float(prob[r]) - p) <= eps * p + 2.0 ** -32


def logits_of(rows, vocab, seed, dtype=torch.float32, std=2.0):
    g = gen(seed)
    x = torch.randn(rows, vocab, generator=g) * std
    at = torch.randint(0, vocab, (rows, 8), generator=g)
    x.scatter_add_(1, at, 6 + 4 * torch.rand(rows, 8, generator=g))
    return x.to(dtype), torch.rand(rows, generator=g)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 31), (5, 33), (4, 1000), (3, 1025), (6, 18385), (2, 50001),
                                        (1, 131072), (1, 200003)])
@pytest.mark.parametrize("kw", [
    {}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 7}, {"top_k": 50, "top_p": 0.9}, {"top_p": 0.5},
    {"top_p": 0.97, "temperature": 1.5}, {"min_p": 0.05}, {"temperature": 0.0}, {"top_p": 0.0},
    {"temperature": 3.0, "top_k": 600, "top_p": 0.95, "min_p": 0.001}])
def test_sample(native, cuda, rows, vocab, kw):
    dtype = [torch.float32, F16, BF16][(rows + vocab) % 3]
    x, u = logits_of(rows, vocab, rows * 7 + vocab, dtype)
    check_sample(x, u, **kw)
    assert fault(native) == 0


def test_sample_extreme_uniforms(native, cuda):
    x, _ = logits_of(4, 777, 3)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 0.5])
    ids, _, kept = draw(x, u, top_k=20)
    first = torch.sort(x, 1, descending=True).indices[:, :20]
    assert int(ids[0]) == int(first[0].min())
    assert int(ids[1]) == int(first[1].max()) and int(ids[2]) == int(first[2].max())
    assert (kept == 20).all()


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
def test_sample_ties_go_to_the_lowest_index(native, cuda, dtype):
    x = torch.zeros(5, 4096, dtype=dtype)
    x[1, 4000:] = 2.0
    x[2, ::2] = -0.0
    x[3] = -5.0
    x[3, [77, 1033, 4095]] = 1.0
    x[4, 10:] = -math.inf
    u = torch.tensor([0.999, 0.0, 0.49, 0.5, 0.95])
    ids, prob, kept = draw(x, u, top_k=[10, 10, 10, 2, 100])
    assert ids.tolist() == [9, 4000, 4, 1033, 9]
    assert kept.tolist() == [10, 10, 10, 2, 100]
    # Equal logits, no limit: the id follows the uniform number.
    ids, prob, kept = draw(torch.zeros(3, 4096, dtype=dtype), torch.tensor([0.0, 0.5, 0.75]))
    assert ids.tolist() == [0, 2048, 3072] and kept.tolist() == [4096] * 3
    assert torch.allclose(prob, torch.full((3,), 1 / 4096, dtype=torch.float64), rtol=1e-6)
    # Half of the mass of equal logits is the first half.
    ids, _, kept = draw(torch.zeros(2, 4096, dtype=dtype), torch.tensor([0.0, 0.9999999]), top_p=0.5)
    assert kept.tolist() == [2048, 2048] and ids.tolist() == [0, 2047]


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
def test_sample_infinite_and_missing_logits(native, cuda, dtype):
    x = torch.full((6, 300), -math.inf, dtype=dtype)
    x[1] = math.nan
    x[2, 299] = -3.0
    x[3, [5, 9]] = math.inf
    x[3, 100] = 4.0
    x[4, 7] = math.nan
    x[4, 8] = 1.0
    x[5] = torch.finfo(dtype).min
    x[5, 17] = torch.finfo(dtype).max
    ids, prob, kept = draw(x, torch.tensor([0.5, 0.5, 0.999, 0.6, 0.0, 0.99]), top_p=0.9)
    assert ids.tolist() == [-1, -1, 299, 9, 8, 17]
    assert kept.tolist() == [0, 0, 1, 2, 1, 1]
    assert prob.tolist() == [0, 0, 1, 0.5, 1, 1]
    greedy, _, kept = draw(x, torch.full((6,), 0.9), temperature=0.0)
    assert greedy.tolist() == [-1, -1, 299, 5, 8, 17] and kept.tolist() == [0, 0, 1, 1, 1, 1]


def test_sample_per_row_parameters_and_strides(native, cuda):
    x, u = logits_of(6, 900, 11)
    wide = torch.full((6, 1003), 50.0)
    wide[:, 3:903] = x
    t = [1.0, 0.0, 0.5, 2.0, -1.0, 1.0]
    k = [0, 5, 3, 900, 7, 1]
    p = [0.9, 1.0, 1.0, 0.3, 0.5, 1.0]
    m = [0.0, 0.0, 0.2, 0.0, 0.0, 0.5]
    ids, prob, kept = draw(wide.cuda()[:, 3:903], u, temperature=t, top_k=k, top_p=p, min_p=m)
    for r in range(6):
        one = draw(x[r:r + 1], u[r:r + 1], temperature=t[r], top_k=k[r], top_p=p[r], min_p=m[r])
        assert (int(one[0][0]), float(one[1][0]), int(one[2][0])) == (int(ids[r]), float(prob[r]), int(kept[r]))


@pytest.mark.parametrize("vocab", [300, 9000, 60000, 170000])
@pytest.mark.parametrize("kw", [{"top_p": 0.99}, {"top_p": 0.7, "temperature": 4.0}, {"top_k": 5000},
                                {"top_k": 5000, "top_p": 0.9}, {"top_p": 0.9999, "min_p": 1e-4}])
def test_sample_flat_distributions(native, cuda, vocab, kw):
    """Prefixes of thousands of tokens: beyond what is sorted at once."""
    x, u = logits_of(4, vocab, vocab, F16 if vocab < 1000 else torch.float32, std=1.0)
    x[1] = torch.randn(vocab, generator=gen(77)).to(x.dtype) * 0.01
    x[2] = torch.round(x[2].float() * 2).to(x.dtype) / 2      # few distinct values
    x[3, : vocab // 2] = -math.inf
    check_sample(x, u, **kw)
    assert fault(native) == 0


@pytest.mark.parametrize("dtype", [torch.float32, F16, BF16])
@pytest.mark.parametrize("kw", [{}, {"top_k": 60, "top_p": 0.9, "temperature": 0.7}, {"top_p": 0.8, "min_p": 0.001},
                                {"temperature": 0.0}])
def test_sample_rows_longer_than_a_cluster_holds(native, cuda, dtype, kw):
    x, u = logits_of(2, 500001, 91, dtype)
    check_sample(x, u, **kw)
    assert fault(native) == 0


def test_sample_many_rows(native, cuda):
    """More rows than a grid's second dimension holds."""
    x = torch.zeros(70000, 24)
    at = torch.arange(70000) % 24
    x[torch.arange(70000), at] = 30.0
    ids, _, kept = draw(x, torch.full((70000,), 0.5), top_p=0.9)
    assert torch.equal(ids, at) and (kept == 1).all()


def test_sample_frequencies(native, cuda):
    """Evenly spread uniform numbers hit every token as often as its share."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 3.0]]).expand(4096, 5).contiguous()
    u = (torch.arange(4096).float() + 0.5) / 4096
    ids, _, _ = draw(x, u, temperature=1.3)
    want = torch.softmax(x[0].double() / 1.3, 0) * 4096
    got = torch.bincount(ids, minlength=5).double()
    assert (got - want).abs().max() <= 1.0

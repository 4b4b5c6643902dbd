"""Serving from a paged KV cache: torch.ops.spyre.{paged_append, paged_attention,
sample} on the CPU (their formulas) and on spyre, and their C entry points.

Expected values come from plain 64-bit arithmetic here.  Tolerances, with h = half a
step of the element type (finfo.eps / 2):

  * paged_append: one rounding at the end, h of the value; before it some ten fp32
    roundings of the two products' magnitudes and, with a norm, of the mean (at most
    128 squares, a depth of 11 additions): 2^-19 of those magnitudes.
  * paged_attention: probabilities round to the element type (h each, so h A with A = sum p
    |v|), the result once more (h |o|).  Scores are fp32 sums of at most 128
    products, each step off by 2^-24: at most 2^-17 of sum |q k| scale, which is below
    2^5 for the inputs here: 2^-12 of A.  fp16 probabilities below 2^-14
    of the largest have a step of 2^-24: at most 2^-25 of the largest |v| a key.
  * sample: whole numbers, equal.
"""

import math

import numpy as np
import pytest
import torch

import torch_spyre  # noqa: F401
from torch_spyre import _capi

DEVICES = ["cpu", pytest.param("spyre", marks=pytest.mark.gpu)]
DTYPES = [torch.float16, torch.bfloat16]
ops = torch.ops.spyre
NAN, INF = float("nan"), float("inf")


def rand(shape, k=0, scale=1.0, dtype=torch.float16):
    g = torch.Generator().manual_seed(0x5E + k)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def new_cache(pages, kv, page, d, dtype, layout="head", fill=None, k=0):
    """[pages, kv, page, d] on the CPU, as a view of the layout's buffer."""
    shape = {"head": (pages, kv, page, d), "token": (pages, page, kv, d),
             "wide": (pages, kv, page, d + 24)}[layout]
    x = rand(shape, 50 + k, dtype=dtype) if fill is None else torch.full(shape, fill, dtype=dtype)
    return cache_view(x, layout, d)


def cache_view(x, layout, d):
    return x.transpose(1, 2) if layout == "token" else x[..., 5:5 + d] if layout == "wide" else x


def on(device, cache, layout):
    """The cache on `device` with the strides it has here."""
    base = cache._base if cache._base is not None else cache
    return cache_view(base.to(device), layout, cache.shape[3])


# ---- paged_append ------------------------------------------------------------

def tables(n, d, dtype):
    inv = 1e4 ** (-torch.arange(0, d, 2).double() / d)
    a = (torch.arange(n).double()[:, None] * inv).repeat(1, 2)
    return a.cos().to(dtype), a.sin().to(dtype)


def turned64(x, w, eps, cos, sin):
    """(value, magnitude of its two products) for heads x [T, h, d]."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    d = x.shape[-1]
    rot = torch.cat([-x[..., d // 2:], x[..., :d // 2]], -1)
    a, b = x * cos.double()[:, None], rot * sin.double()[:, None]
    return a + b, a.abs() + b.abs()


def check_turned(got, want, dtype):
    v, m = want
    bound = v.abs() * half(dtype) + m * 2.0 ** -19 + 2.0 ** -25
    off = (got.cpu().double() - v).abs()
    assert bool((off <= bound).all()), (off / bound).max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", [None, "same", "fp32", "k only"])
@pytest.mark.parametrize("t,h,kv,d,page,layout,tab", [
    (1, 4, 2, 128, 16, "head", "same"), (7, 32, 8, 128, 5, "token", "fp32"),
    (33, 3, 1, 64, 1, "wide", "same"), (130, 6, 6, 64, 48, "head", "fp32"),
    (5, 17, 17, 128, 64, "token", "same")])
def test_append(t, h, kv, d, page, layout, tab, norm, dtype, device):
    pages = -(-t // page) + 2
    kc, vc = (new_cache(pages, kv, page, d, dtype, layout, k=i) for i in (0, 1))
    cos, sin = tables(100, d, dtype if tab == "same" else torch.float32)
    qkv = rand((t, (h + 2 * kv) * d), 1, dtype=dtype)
    g = torch.Generator().manual_seed(t)
    pos = torch.randint(0, 100, (t,), generator=g)
    slots = torch.randperm(pages * page, generator=g)[:t]
    if t > 5:
        slots[3] = -1
        pos[3] = 10 ** 12  # (a padding row's position is not looked at)
    wt = torch.float32 if norm == "fp32" else dtype
    qn = rand((d,), 2, 0.2, wt) + 1 if norm in ("same", "fp32") else None
    kn = rand((d,), 3, 0.2, wt) + 1 if norm else None
    eps = 1e-3
    kd, vd = on(device, kc, layout), on(device, vc, layout)
    q = ops.paged_append(*(x.to(device) for x in (qkv, cos, sin, pos, slots)), kd, vd, h,
                         None if qn is None else qn.to(device),
                         None if kn is None else kn.to(device), eps)
    assert q.shape == (t, h, d) and q.dtype == dtype and q.is_contiguous()
    rows = slots >= 0
    x = qkv.view(t, h + 2 * kv, d)[rows]
    c, s = cos[pos[rows]], sin[pos[rows]]
    check_turned(q.cpu()[rows], turned64(x[:, :h], qn, eps, c, s), dtype)
    assert not q.cpu()[~rows].any()
    page_of, at = slots[rows] // page, slots[rows] % page
    kd, vd = kd.cpu(), vd.cpu()
    check_turned(kd[page_of, :, at], turned64(x[:, h:h + kv], kn, eps, c, s), dtype)
    assert torch.equal(vd[page_of, :, at], x[:, h + kv:])
    # nothing else of the caches is touched
    kc[page_of, :, at], vc[page_of, :, at] = kd[page_of, :, at], vd[page_of, :, at]
    assert torch.equal(kd, kc) and torch.equal(vd, vc)


@pytest.mark.parametrize("device", DEVICES)
def test_append_rows_inside_wider_ones_and_special_values(device):
    t, h, kv, d = 4, 2, 1, 128
    base = rand((t, 3 + (h + 2 * kv) * d + 10), 4)
    base[1, 3 + 5] = NAN
    base[2, 3 + 7] = INF
    cos, sin = (x[:, 1:] for x in tables(9, d, torch.float16))
    cos, sin = (torch.cat([x[:, :1], x], 1)[:, 1:] for x in tables(9, d, torch.float16))
    kc = new_cache(2, kv, 16, d, torch.float16)
    vc = kc.clone()
    pos, slots = torch.tensor([0, 8, 3, 3]), torch.tensor([31, 0, 16, 15])
    qkv = base[:, 3:3 + (h + 2 * kv) * d]
    w = torch.ones(d, dtype=torch.float16)
    out = []
    for strided in (True, False):
        kd, vd = kc.to(device), vc.to(device)
        x = base.to(device)[:, 3:3 + (h + 2 * kv) * d] if strided else qkv.contiguous().to(device)
        tab = [torch.stack([y, y], 2).to(device)[..., 0] if strided else y.contiguous().to(device)
               for y in (cos, sin)]
        q = ops.paged_append(x, *tab, pos.to(device), slots.to(device), kd, vd, h, w.to(device),
                             w.to(device), 0.0)
        out.append([y.cpu() for y in (q, kd, vd)])
    for a, b in zip(*out):
        torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
    q = out[0][0]
    assert q[1, 0].isnan().all() and not q[1, 1].isnan().any() and not q[0].isnan().any()
    assert q[2, 0, 7].isnan()  # inf / inf
    assert torch.equal(out[0][2][1, :, 15], qkv[0, (h + kv) * d:].view(kv, d))


@pytest.mark.parametrize("device", DEVICES)
def test_append_nothing(device):
    kc = new_cache(2, 1, 16, 64, torch.float16).to(device)
    vc, cos = kc.clone(), torch.zeros(4, 64, dtype=torch.float16, device=device)
    none = torch.zeros(0, dtype=torch.int64, device=device)
    q = ops.paged_append(torch.zeros(0, 6 * 64, dtype=torch.float16, device=device), cos, cos, none,
                         none, kc, vc, 4)
    assert q.shape == (0, 4, 64)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("slot,pos", [(32, 0), (2 ** 62, 0), (3, -1), (3, 4)])
def test_append_out_of_range(slot, pos, device):
    kc = new_cache(2, 1, 16, 64, torch.float16)
    kd, vd = kc.to(device), kc.clone().to(device)
    cos, sin = (x.to(device) for x in tables(4, 64, torch.float16))
    qkv = rand((2, 3 * 64), 5).to(device)
    with pytest.raises(IndexError):
        ops.paged_append(qkv, cos, sin, torch.tensor([1, pos]).to(device),
                         torch.tensor([0, slot]).to(device), kd, vd, 1)
        torch.spyre.synchronize()
    if device == "spyre":  # the other row is appended, this one is not
        assert torch.equal(vd.cpu()[0, 0, 0], qkv.cpu()[0, 128:])
        assert torch.equal(kd.cpu()[1], kc[1]) and torch.equal(kd.cpu()[0, :, 1:], kc[0, :, 1:])


# ---- paged_attention ---------------------------------------------------------

class Step:
    """A step of ragged sequences on the CPU: news new tokens behind lens - news others."""

    def __init__(self, news, lens, h, kv, d, page, dtype, layout="head", mask=None, pad=0, lead=0,
                 k=0, extra=1, fill=None):
        g = torch.Generator().manual_seed(99 + k)
        self.news, self.lens, self.h, self.kv, self.d, self.page = news, lens, h, kv, d, page
        self.dtype, self.layout = dtype, layout
        need = [-(-m // page) for m in lens]
        pages = sum(need) + 2
        self.k_cache, self.v_cache = (new_cache(pages, kv, page, d, dtype, layout, fill, k=k + 2 * i)
                                      for i in (1, 2))
        perm = torch.randperm(pages, generator=g).tolist()
        self.table = torch.full((len(lens), max(need + [0]) + extra), -5, dtype=torch.int64)
        for row, n in zip(self.table, need):
            row[:n] = torch.tensor(perm[:n], dtype=torch.int64)
            perm = perm[n:]
        if fill is not None:  # only the sequences' own keys hold values
            for b, m in enumerate(lens):
                for x in range(m):
                    pg, at = int(self.table[b, x // page]), x % page
                    self.k_cache[pg, :, at] = torch.randn(kv, d, generator=g).to(dtype)
                    self.v_cache[pg, :, at] = torch.randn(kv, d, generator=g).to(dtype)
        self.starts = torch.tensor([lead] + news).cumsum(0)
        self.lens_t = torch.tensor(lens, dtype=torch.int64)
        self.q = rand((lead + sum(news) + pad, h, d), 60 + k, dtype=dtype)
        self.scale = 1 / math.sqrt(d)
        self.mask = mask

    def run(self, device, q=None):
        return ops.paged_attention(
            (self.q if q is None else q).to(device), on(device, self.k_cache, self.layout),
            on(device, self.v_cache, self.layout), self.table.to(device), self.lens_t.to(device),
            self.starts.to(device), self.scale, None if self.mask is None else self.mask.to(device))

    def keys(self, b):
        m = self.lens[b]
        x = torch.arange(m)
        pg = self.table[b, x // self.page] if m else x
        return self.k_cache[pg, :, x % self.page], self.v_cache[pg, :, x % self.page]

    def seen(self, b):
        n, m = self.news[b], self.lens[b]
        s = torch.ones(n, m, dtype=torch.bool)
        if self.mask is None:
            return s.tril(m - n)
        s[:, m - n:] = self.mask[self.starts[b]:self.starts[b] + n, :n]
        return s

    def want(self):
        """(result, bound) in 64 bits; NaN where a row sees a value that is not finite."""
        o = torch.zeros(self.q.shape, dtype=torch.float64)
        bound = torch.zeros_like(o)
        h = half(self.dtype)
        for b, n in enumerate(self.news):
            k, v = (x.double() for x in self.keys(b))
            seen, r0 = self.seen(b), int(self.starts[b])
            for j in range(self.h):
                q, kj, vj = (self.q[r0:r0 + n, j].double(), k[:, j * self.kv // self.h],
                             v[:, j * self.kv // self.h])
                p = (q @ kj.t() * self.scale).masked_fill(~seen, -INF)
                p = torch.softmax(p, -1)
                p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
                # (0 times what is not seen is 0, whatever it is)
                terms = torch.where(seen[:, :, None], p[:, :, None] * vj, 0.0)
                o[r0:r0 + n, j] = terms.sum(1)
                a = terms.abs().sum(1)
                most = vj.abs().nan_to_num(0, 0, 0).max() if vj.numel() else 0.0
                bound[r0:r0 + n, j] = (h * (a + terms.sum(1).abs()) * (1 + 2.0 ** -4)
                                       + 2.0 ** -12 * a + len(vj) * 2.0 ** -25 * most)
        return o, bound

    def check(self, device, q=None):
        got = self.run(device, q)
        assert got.shape == self.q.shape and got.dtype == self.dtype and got.is_contiguous()
        got = got.cpu().double()
        want, bound = self.want()
        fine = want.isfinite()
        assert torch.equal(got.isfinite(), fine)
        off = (got - want).abs()[fine]
        assert bool((off <= bound[fine]).all()), (off / bound[fine].clamp(min=1e-30)).max()
        used = torch.zeros(len(got), dtype=torch.bool)
        used[int(self.starts[0]):int(self.starts[-1])] = True
        assert not got[~used].any()
        return got


def tree(news, width, seed, pad=0, lead=0):
    g = torch.Generator().manual_seed(seed)
    rows = [torch.ones(lead, width, dtype=torch.bool)]
    for n in news:
        m = torch.eye(n, width, dtype=torch.bool)
        for i in range(1, n):
            m[i] |= m[int(torch.randint(0, i, (1,), generator=g))]
        rows.append(m)
    return torch.cat(rows + [torch.ones(pad, width, dtype=torch.bool)])


STEPS = [
    # (new tokens, lengths, query heads, KV heads, head dim, page, layout)
    ([1], [1], 4, 1, 128, 16, "head"),
    ([1], [33], 8, 2, 64, 16, "token"),
    ([1, 1, 1, 1], [7, 128, 129, 700], 8, 2, 128, 16, "head"),
    ([1, 0, 1], [257, 90, 31], 4, 4, 128, 5, "wide"),
    ([1] * 5, [1, 2, 40, 300, 131], 16, 1, 64, 1, "head"),
    ([1, 1], [2300, 1500], 8, 2, 128, 64, "head"),
    ([3, 17, 9], [3, 200, 129], 8, 2, 128, 48, "token"),
    ([16], [1300], 28, 4, 64, 16, "head"),
    ([5, 64, 1, 33], [500, 64, 800, 97], 6, 2, 128, 16, "head"),
    ([40, 70], [333, 70], 4, 2, 64, 7, "wide"),
    ([150], [290], 8, 2, 128, 32, "head"),
    ([130, 1, 200], [130, 512, 411], 3, 1, 128, 16, "token"),
    ([2] * 300, [2 + i % 40 for i in range(300)], 2, 1, 64, 16, "head"),
    ([37] + [0] * 20 + [1] * 9 + [0] * 30, [340] + [9] * 20 + list(range(60, 150, 10)) + [0] * 30,
     8, 2, 128, 16, "head"),
    ([1] * 30 + [70], [200 + 7 * i for i in range(30)] + [500], 4, 2, 128, 16, "token"),
    ([1, 4], [70, 300], 24, 1, 64, 16, "head"),
    ([1, 1, 1], [70, 300, 9], 24, 1, 128, 16, "head"),
]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("step", range(len(STEPS)))
def test_attention(step, masked, dtype, device):
    news, lens, h, kv, d, page, layout = STEPS[step]
    lead, pad = (2, 3) if step % 2 else (0, 0)
    mask = tree(news, max(news) + step % 3, step, pad, lead) if masked else None
    Step(news, lens, h, kv, d, page, dtype, layout, mask, pad, lead, k=step).check(device)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("news,lens,h,kv,page,masked", [
    ([1], [4100], 8, 2, 16, False), ([1, 1], [2177, 9000], 3, 1, 5, False),
    ([16], [4100], 8, 2, 16, True), ([3, 1], [7000, 40], 6, 2, 20, False),
    ([40], [4300], 6, 1, 16, False), ([40], [4300], 6, 1, 16, True), ([33, 5], [300, 5000], 4, 4, 32, True)])
def test_attention_of_many_parts(news, lens, h, kv, page, masked, d, dtype):
    """Keys of one tile of rows over more than 16 workgroups (each has 128 of them), whose parts
    are merged by all groups of lanes together; tiles with few and with all rows.  Results
    do not change from call to call."""
    assert max(lens) > 16 * 128
    s = Step(news, lens, h, kv, d, page, dtype, mask=tree(news, max(news), 5) if masked else None, k=31)
    got = s.check("spyre")
    for _ in range(3):
        junk = torch.full((64, 1000), NAN, device="spyre")
        assert torch.equal(s.run("spyre").cpu().double(), got)
        del junk


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,m,h,kv,d", [(4097, 4097, 4, 2, 128), (2500, 6001, 3, 1, 64)])
def test_attention_of_long_pieces(n, m, h, kv, d, dtype):
    """Whole prompts and pieces of many tiles, beside a single token."""
    s = Step([1, n], [77, m], h, kv, d, 16, dtype, k=33)
    got = s.run("spyre").cpu().double()[1:]
    k, v = (x.double() for x in s.keys(1))
    half_step = half(dtype)
    for j in range(h):
        kj, vj = k[:, j * kv // h], v[:, j * kv // h]
        p = torch.softmax((s.q[1:, j].double() @ kj.t() * s.scale)
                          .masked_fill(~s.seen(1), -INF), -1)
        want, a = p @ vj, p @ vj.abs()
        bound = (half_step * (a + want.abs()) * (1 + 2.0 ** -4) + 2.0 ** -12 * a
                 + m * 2.0 ** -32 * vj.abs().max())
        off = (got[:, j] - want).abs()
        assert bool((off <= bound).all()), (off / bound).max()


@pytest.mark.gpu
@pytest.mark.parametrize("last", [1, 2])
@pytest.mark.parametrize("d", [64, 128])
def test_attention_of_as_many_sequences_as_it_takes(d, last):
    """4096 of them: one token each, and one more (the form of 128-row tiles)."""
    n = 4096
    Step([1] * (n - 1) + [last], [2 + i % 40 for i in range(n)], 2, 1, d, 16, torch.float16,
         k=32).check("spyre")


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 6])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (12, 2)])
def test_attention_ignores_what_is_not_seen(heads, page, dtype, device):
    """Slots past the sequences' ends, pages of nobody, and new tokens that only some
    rows see hold NaN and infinities.  (13 tokens on average: 13, 54 and 81 rows.)"""
    news, lens = [9, 4, 40, 1], [50, 4, 300, 77]
    mask = torch.rand(sum(news), 40, generator=torch.Generator().manual_seed(3)) < 0.4
    mask[0:3, [2, 5, 8]] = False
    s = Step(news, lens, *heads, 128, page, dtype, mask=mask, k=7, fill=NAN)
    clean = s.check(device)
    # poisoned new tokens: three of sequence 0, one of sequence 2
    for b, j, bad in ((0, 2, NAN), (0, 5, INF), (0, 8, -INF), (2, 31, NAN)):
        x = lens[b] - news[b] + j
        where = (int(s.table[b, x // page]), slice(None), x % page)
        if j % 2:
            s.v_cache[where] = bad
        else:
            s.k_cache[where] = NAN
            s.v_cache[where] = bad
    got = s.run(device).cpu().double()
    want, _ = s.want()
    # rows that see one of them are NaN or infinite as the formula's are, others as before
    hit = torch.zeros(sum(news), dtype=torch.bool)
    hit[0:9] = mask[0:9, 2] | mask[0:9, 5] | mask[0:9, 8]
    hit[13:53] = mask[13:53, 31]
    assert bool(hit.any()) and bool((~hit[:9]).any())
    torch.testing.assert_close(got[~hit], clean[~hit], rtol=0, atol=0)
    assert not got[hit].isfinite().any() and not want[hit].isfinite().any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_causal_ignores_later_values(dtype, device):
    """Pieces of prompts whose later tokens hold infinities in V."""
    news, lens = [50], [90]
    s = Step(news, lens, 4, 2, 64, 16, dtype, k=8)
    clean = s.check(device)
    for j, bad in ((20, INF), (33, NAN)):
        x = 40 + j
        s.v_cache[int(s.table[0, x // 16]), 0, x % 16] = bad
    got = s.run(device).cpu().double()
    torch.testing.assert_close(got[:20], clean[:20], rtol=0, atol=0)
    torch.testing.assert_close(got[:, 2:], clean[:, 2:], rtol=0, atol=0)  # the other KV head
    assert bool((got[20:33, :2] == INF).all()) and got[33:, :2].isnan().all()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_rows_that_see_nothing(device):
    news, lens = [4, 20], [4, 20]
    mask = torch.zeros(24, 20, dtype=torch.bool)
    mask[1, 0] = mask[3, 2] = mask[10, 6] = True
    s = Step(news, lens, 4, 2, 128, 16, torch.float16, mask=mask, k=9)
    got = s.check(device)
    rows = mask.any(1)
    assert not got[~rows].any() and bool(got[rows].any(-1).all())
    # a key alone has weight 1: its value comes back
    assert torch.equal(got[1, 0], s.keys(0)[1][0, 0].double())


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_large_scores(dtype, device):
    """Scores far apart and far from 0: no overflow, the largest wins."""
    s = Step([1, 6], [70, 400], 4, 2, 128, 16, dtype, k=10)
    s.q = s.q * 60
    want, bound = s.want()
    got = s.run(device).cpu().double()
    # scores of some hundreds: fp32 sums are off by 2^-17 of sum |q k| scale, about 500
    # here, so probabilities by 2^-8 of themselves
    off = (got - want).abs()
    a = (bound / half(dtype)).clamp(min=1e-6)
    assert bool((off <= bound + a * 2.0 ** -8).all()), (off / bound).max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("gap", [0.0, 9.0, 15.0, 17.0, 17.5, 20.0, 22.0])
@pytest.mark.parametrize("new", [1, 2])
def test_attention_one_key_far_above_many(new, gap, dtype, device):
    """The first key has no value and weighs e^gap times as much as every other: what
    thousands of small weights add up to is kept.  With n others of value 1 the result is
    n / (n + e^gap).  It may be off by half a step of every weight and of itself, 2^-12 of
    it through exp (an exponent of 32 at most, as a product in fp32), and in fp16 by 2^-32 for
    each weight below 2^-21, whose step is coarser.  (300 sequences share the pages, so that one
    workgroup has all keys of a row, or most of them.)"""
    b, m, kv, d, page = 300, 4096, 2, 64, 16
    k = torch.zeros(m // page, kv, page, d, dtype=dtype)
    v = torch.ones_like(k)
    k[0, :, 0, 0] = gap
    v[0, :, 0] = 0
    q = torch.zeros(b * new, kv, d, dtype=dtype)
    q[..., 0] = 1
    got = ops.paged_attention(*(x.to(device) for x in (
        q, k, v, torch.arange(m // page).expand(b, -1).contiguous(), torch.full((b,), m),
        torch.arange(0, b * new + 1, new))), 1.0).cpu().double().view(b, new, kv, d)
    n = torch.arange(m - new, m).double()[:, None, None]
    want = n / (n + math.exp(gap))
    tail = n * 2.0 ** -32 if dtype == torch.float16 else 0.0
    bound = want * (2 * half(dtype) * (1 + 2.0 ** -4) + 2.0 ** -12) + tail
    off = (got - want).abs()
    assert bool((off <= bound).all()), (off / bound).max()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_strided_queries_tables_and_masks(device):
    news, lens = [5, 2], [60, 33]
    mask = tree(news, 6, 4)
    s = Step(news, lens, 6, 3, 64, 16, torch.bfloat16, mask=mask, k=11)
    want = s.run(device).cpu()
    n = sum(news)
    wide = torch.zeros(n, 10, 6, 70, dtype=torch.bfloat16)
    wide[:, 3, :, 1:65] = s.q
    q = wide.to(device)[:, 3, :, 1:65]
    table = torch.stack([s.table, s.table], 2).to(device)[..., 1]
    m = torch.zeros(n, 11, dtype=torch.bool)
    m[:, 4:10] = mask
    lens2 = torch.stack([s.lens_t, s.lens_t], 1).to(device)[:, 0]
    for mk in (m.to(device)[:, 4:10], mask.t().contiguous().to(device).t()):
        got = ops.paged_attention(q, s.k_cache.to(device), s.v_cache.to(device), table, lens2,
                                  s.starts.to(device), s.scale, mk)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("device", DEVICES)
def test_attention_empty_calls(device):
    kc = new_cache(2, 1, 16, 64, torch.float16).to(device)

    def call(t, b, width, lens, starts):
        return ops.paged_attention(
            torch.ones(t, 2, 64, dtype=torch.float16, device=device), kc, kc,
            torch.zeros(b, width, dtype=torch.int64, device=device),
            torch.tensor(lens, dtype=torch.int64).to(device),
            torch.tensor(starts, dtype=torch.int64).to(device), 0.1).cpu()

    assert call(0, 0, 0, [], [0]).shape == (0, 2, 64)
    assert call(0, 2, 1, [5, 0], [0, 0, 0]).shape == (0, 2, 64)
    assert not call(3, 0, 4, [], [0]).any()
    assert not call(3, 2, 1, [16, 0], [1, 1, 1]).any()


BAD = [  # lengths, starts, table entry: which is wrong
    ([17, 5], [0, 1, 3], None), ([9, 1], [0, 1, 3], None), ([9, -1], [0, 1, 1], None),
    ([9, 5], [0, 1, 4], None), ([9, 5], [1, 0, 3], None), ([9, 5], [-1, 1, 3], None),
    ([9, 5], [0, 1, 3], 2), ([9, 5], [0, 1, 3], -1), ([9, 5], [0, 1, 3], 2 ** 40)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("bad", range(len(BAD)))
def test_attention_out_of_range(bad, page, device):
    lens, starts, entry = BAD[bad]
    if lens[0] == 17:
        lens = [page + 1, 5]
    if lens[1] == -1 and device == "cpu":
        pytest.skip("a sequence without new tokens is not looked at")
    kc = new_cache(2, 2, page, 128, torch.float16).to(device)
    table = torch.tensor([[0], [1 if entry is None else entry]]).to(device)
    with pytest.raises(IndexError):
        ops.paged_attention(rand((3, 4, 128), 12).to(device), kc, kc, table,
                            torch.tensor(lens).to(device), torch.tensor(starts).to(device), 0.1)
        torch.spyre.synchronize()


@pytest.mark.parametrize("device", DEVICES)
def test_attention_more_new_tokens_than_the_mask_has_columns(device):
    kc = new_cache(2, 2, 16, 128, torch.float16).to(device)
    for width in (0, 2):
        with pytest.raises(IndexError):
            ops.paged_attention(rand((3, 4, 128), 12).to(device), kc, kc,
                                torch.tensor([[0]]).to(device), torch.tensor([9]).to(device),
                                torch.tensor([0, 3]).to(device), 0.1,
                                torch.ones(3, width, dtype=torch.bool, device=device))
            torch.spyre.synchronize()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("news", [[1], [1, 0, 1], [9], [1, 130, 0, 2]])
def test_attention_new_tokens_without_pages(news, page, masked, device):
    """A block table of no columns holds no keys, new ones neither: the call is refused and the
    table, which has no memory, not read."""
    n = sum(news)
    kc = new_cache(2, 2, page, 128, torch.float16).to(device)
    mask = torch.ones(n, max(news), dtype=torch.bool, device=device) if masked else None
    for lens in (news, [0] * len(news), [x + 5 for x in news]):
        with pytest.raises(IndexError):
            ops.paged_attention(rand((n, 4, 128), 12).to(device), kc, kc,
                                torch.zeros(len(news), 0, dtype=torch.int64, device=device),
                                torch.tensor(lens).to(device),
                                torch.tensor([0] + news).cumsum(0).to(device), 0.1, mask)
            torch.spyre.synchronize()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("page", [16, 20])
def test_attention_sequences_without_new_tokens(page, device):
    """Their lengths have to be in range as the others', their pages are not looked at."""
    kc = new_cache(2, 2, page, 128, torch.float16).to(device)
    q = rand((3, 4, 128), 13).to(device)

    def call(lens, starts, table, caches=kc):
        out = ops.paged_attention(q, caches, caches, torch.tensor(table).to(device),
                                  torch.tensor(lens).to(device), torch.tensor(starts).to(device), 0.1)
        torch.spyre.synchronize()
        return out.cpu()

    want = call([9], [0, 3], [[1]])
    for other in (0, 1, page):
        for entry in (-1, 0, 2 ** 40):
            assert torch.equal(call([9, other], [0, 3, 3], [[1], [entry]]), want)
            assert torch.equal(call([other, 9], [0, 0, 3], [[entry], [1]]), want)
    for other in (-1, page + 1, 2 ** 40, -2 ** 40):
        with pytest.raises(IndexError):
            call([9, other], [0, 3, 3], [[1], [0]])
    # no pages at all: nothing is appended, nothing asked
    assert not call([page, 0], [3, 3, 3], [[0], [0]], kc[:0]).any()
    with pytest.raises(IndexError):
        call([9], [0, 3], [[0]], kc[:0])


# ---- sample ------------------------------------------------------------------

def token64(l, u, t=1.0, k=0, p=1.0, m=0.0):
    """One row (numpy, 64 bits) by the definition, written out."""
    l = l.astype(np.float64)
    l[np.isnan(l)] = -np.inf
    top = l.max()
    if top == -np.inf:
        return -1
    if not t > 0:
        return int(np.argmax(l))
    if top == np.inf:
        l, top = np.where(l == np.inf, 0.0, -np.inf), 0.0
    order = np.argsort(-l, kind="stable")
    w = np.exp((l[order] - top) / t)
    if k > 0:
        order, w = order[:k], w[:k]
    if p < 1:
        want, run, n = max(p, 0.0) * math.fsum(w), 0.0, 0
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < want).sum()))
        order, w = order[:n], w[:n]
    stay = w >= min(m, 1.0)
    order, w = order[stay], w[stay]
    by = np.argsort(order)
    order, run = order[by], np.cumsum(w[by])
    at = int(np.searchsorted(run, max(u, 0.0) * run[-1], side="right"))
    last = int(np.searchsorted(run, run[-1], side="left"))
    return int(order[min(at, last)])


def check_sample(logits, device, u, t=None, k=None, p=None, m=None):
    rows = logits.shape[0]

    def each(v, dtype):
        return None if v is None else torch.as_tensor(v, dtype=dtype).expand(rows).contiguous()

    u, t, k, p, m = (each(v, y) for v, y in ((u, torch.float32), (t, torch.float32),
                                             (k, torch.int64), (p, torch.float32),
                                             (m, torch.float32)))
    got = ops.sample(logits.to(device), *(None if v is None else v.to(device)
                                          for v in (u, t, k, p, m)))
    assert got.dtype == torch.int64 and got.shape == (rows,)
    want = [token64(logits[i].double().numpy().copy(), float(u[i]),
                    1.0 if t is None else float(t[i]), 0 if k is None else int(k[i]),
                    1.0 if p is None else float(p[i]), 0.0 if m is None else float(m[i]))
            for i in range(rows)]
    assert got.tolist() == want
    return want


def uniforms(n, seed=0):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 64, 511, 4099, 49155])
def test_sample(vocab, dtype, device):
    rows = 24 if vocab < 40000 else 8
    l = rand((rows, vocab), vocab, 2.5, dtype)
    u = uniforms(rows, vocab)
    check_sample(l, device, u)
    check_sample(l, device, u, t=0.7)
    check_sample(l, device, u, t=0.7, k=5)
    check_sample(l, device, u, t=1.5, k=1000)
    check_sample(l, device, u, p=0.9)
    check_sample(l, device, u, t=3.0, p=0.5, k=max(1, vocab // 2))
    check_sample(l, device, u, m=0.1)
    check_sample(l, device, u, t=0.9, k=300, p=0.95, m=0.01)
    assert check_sample(l, device, u, t=0.0) == l.float().argmax(1).tolist()


@pytest.mark.parametrize("device", DEVICES)
def test_sample_parameters_of_every_row(device):
    rows = 40
    l = rand((rows, 3001), 7, 2.0, torch.bfloat16)
    g = torch.Generator().manual_seed(1)
    t = torch.rand(rows, generator=g) * 2
    t[::7] = 0
    t[3] = -1.0
    t[4] = INF
    t[5] = 1e-40
    t[6] = 1e30
    k = torch.randint(-2, 60, (rows,), generator=g)
    k[1], k[2] = 3001, 10 ** 15
    p = torch.rand(rows, generator=g) * 1.2
    p[8], p[9], p[10] = 0.0, -1.0, 1.0
    m = torch.rand(rows, generator=g) * 0.2
    m[11], m[12], m[13] = 1.0, 2.0, -1.0
    u = uniforms(rows, 3)
    u[14], u[15] = 0.0, 1 - 2.0 ** -24
    check_sample(l, device, u, t, k, p, m)
    check_sample(l, device, u, t, None, p, None)
    check_sample(l, device, u, None, k, None, m)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("vocab", [5, 3000, 20000])
def test_sample_ties_go_to_the_lowest_index(vocab, device):
    """Few values: every cut falls into tokens that are alike."""
    g = torch.Generator().manual_seed(vocab)
    l = torch.randint(-1, 2, (30, vocab), generator=g).half()
    l[0] = 0.0
    l[1] = -3.0
    l[2] = torch.where(torch.arange(vocab) % 2 == 0, 0.0, -0.0)
    u = uniforms(30, 4)
    for k, p in ((1, None), (3, None), (vocab // 2 + 1, None), (None, 0.3), (None, 0.75),
                 (vocab // 2 + 1, 0.5), (vocab - 1, 0.99)):
        check_sample(l, device, u, k=k, p=p)
    # top-k of equal logits: the first k
    assert max(check_sample(l[:3], device, u[:3], k=2)) <= 1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", DTYPES + [torch.float32])
def test_sample_special_values(dtype, device):
    v = 9000
    l = rand((12, v), 8, 2.0, dtype)
    l[0] = -INF
    l[1] = NAN
    l[2, ::2] = NAN
    l[3, 5:8000] = -INF
    l[4, 17] = INF
    l[5, [3, 8000, 8999]] = INF
    l[6] = torch.finfo(dtype).min
    l[7, 1:] = torch.finfo(dtype).min
    l[8, :7] = torch.finfo(dtype).max
    l[9] = torch.finfo(dtype).max
    l[9, 100] = torch.finfo(dtype).min
    l[10, 0] = INF
    l[10, 1] = NAN
    l[11, :-1] = -INF
    u = uniforms(12, 5)
    for kw in ({}, {"t": 0.0}, {"k": 3}, {"p": 0.8}, {"t": 0.5, "k": 50, "p": 0.9, "m": 0.05},
               {"m": 1.0}, {"t": 1e20}, {"t": 1e20, "k": 7, "p": 0.5}, {"t": 3e37},
               {"t": 1e38, "p": 0.3}, {"t": 3e38, "k": 2000, "m": 0.9}):
        got = check_sample(l, device, u, **kw)
        assert got[:2] == [-1, -1] and got[4] == 17 and got[10] == 0 and got[11] == v - 1
        assert got[5] in (3, 8000, 8999)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("vocab", [40, 4097, 20000])
def test_sample_borders_of_the_filters(vocab, device):
    """min-p through 0, logits far from 0 beside a small temperature, k around the number of
    threads, filters that meet at one value."""
    l = rand((16, vocab), vocab, 1.0, torch.float32)
    l[:, 3] = 0.0
    l[:, 5] = -0.0
    l[0:4, 7] = 3.0
    l[4:8] = 1e6 + torch.round(l[4:8])
    l[8:12] = torch.round(l[8:12] * 2) / 2
    l[12:] = -1e-30 * torch.rand(4, vocab)
    u = uniforms(16, vocab)
    exact = torch.full((16,), math.exp(-3.0))  # (float: 0 passes or not by its last bit)
    for m in (exact, torch.nextafter(exact, torch.tensor(1.0)), torch.full((16,), 0.3)):
        check_sample(l, device, u, m=m)
        check_sample(l, device, u, m=m, k=30, p=0.9)
        check_sample(l, device, u, m=m, p=0.7, t=0.5)
    for t in (1e-3, 1e-10, 30.0):
        check_sample(l, device, u, t=t)
        check_sample(l, device, u, t=t, p=0.6)
        check_sample(l, device, u, t=t, k=700, p=0.8)
    for k in (39, 512, 1023, 1024, 1025, 4096):
        check_sample(l, device, u, k=k)
        check_sample(l, device, u, k=k, p=0.97, m=0.02)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("vocab", [5, 3000, 20000])
@pytest.mark.parametrize("t", [1e-45, 1e-40, 1.3e-37, 1.4e-37, 1e-36])
def test_sample_smallest_temperatures_and_shares(t, vocab, device):
    """A row has a token however small its temperature and top-p are."""
    l = rand((6, vocab), vocab, 2.0, torch.float32)
    l[3:] = torch.round(l[3:])
    u = uniforms(6, 1)
    for p in (None, 0.0, -1.0, 1e-30, 0.5):
        for k in (None, 3, 2000):
            check_sample(l, device, u, t=t, p=p, k=k)
            check_sample(l.half(), device, u, t=t, p=p, k=k, m=0.5)


@pytest.mark.parametrize("device", DEVICES)
def test_sample_bounds_of_the_random_number(device):
    l = torch.tensor([[0.0, 1.0, -INF, 2.0, -INF]]).expand(5, 5).contiguous()
    u = torch.tensor([0.0, 1.0, 5.0, -3.0, NAN])
    got = ops.sample(l.to(device), u.to(device))
    assert got.tolist() == [0, 3, 3, 0, 0]


@pytest.mark.parametrize("device", DEVICES)
def test_sample_strided_rows(device):
    base = rand((6, 2, 5000), 9, 2.0, torch.float16)
    u = uniforms(6, 6)
    want = check_sample(base[:, 1, 3:4900], device, u, k=20)
    dev = base.to(device)
    assert ops.sample(dev[:, 1, 3:4900], u.to(device), None,
                      torch.full((6,), 20).to(device)).tolist() == want
    wide = torch.stack([base[:, 1, 3:4900], base[:, 0, 3:4900]], 2).to(device)[..., 0]
    two = torch.stack([u, u], 1).to(device)[:, 1]
    assert ops.sample(wide, two, None, torch.full((6,), 20).to(device)).tolist() == want
    same = check_sample(base[:1, 1].expand(6, 5000), device, u, p=0.9)
    assert ops.sample(dev[:1, 1].expand(6, 5000), u.to(device), None, None,
                      torch.full((6,), 0.9).to(device)).tolist() == same
    assert ops.sample(dev[:0, 1], u[:0].to(device)).shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [131072, 151936 + 1, 1 << 20])
def test_sample_large_vocabularies(vocab):
    for dtype in DTYPES + [torch.float32]:
        l = rand((3, vocab), 10, 2.0, dtype)
        l[1, 1000:] = -INF
        l[2] = l[2] * 1e-3  # nearly flat
        u = uniforms(3, 7)
        check_sample(l, "spyre", u)
        check_sample(l, "spyre", u, t=0.8, p=0.9)
        check_sample(l, "spyre", u, k=5000, p=0.99, m=1e-4)


# ---- large buffers, several streams ---------------------------------------------

@pytest.mark.gpu
def test_caches_past_32_bits():
    """Pages at both ends of caches of more than 2^32 elements give what pages of small ones
    give, to the last bit."""
    page, kv, d, n = 16, 2, 128, 61
    pages = 2 ** 32 // (kv * page * d) + 8
    places = torch.tensor([pages - 1, 0, pages // 2 + 1, pages - 7])
    qkv = rand((n, 8 * d), 60, 1.0).to("spyre")
    cos, sin = (x.to("spyre") for x in tables(n, d, torch.float32))
    at = torch.arange(n)
    got = []
    for count, where in ((4, torch.arange(4)), (pages, places)):
        k, v = (torch.empty(count, kv, page, d, dtype=torch.float16, device="spyre")
                for _ in range(2))
        q = ops.paged_append(qkv, cos, sin, at.to("spyre"),
                             (where[at // page] * page + at % page).to("spyre"), k, v, 4)
        table, lens = where[None].to("spyre"), torch.tensor([n]).to("spyre")
        for new in (1, 16, n):
            starts = torch.tensor([0, new]).to("spyre")
            got.append(ops.paged_attention(q[n - new:], k, v, table, lens, starts, 0.09).cpu())
        del k, v
    for small, large in zip(got[:3], got[3:]):
        assert torch.isfinite(small).all() and torch.equal(small, large)


@pytest.mark.gpu
def test_logits_past_32_bits():
    rows, vocab = 2052, 1 << 20
    l = torch.empty(rows, vocab, dtype=torch.float16, device="spyre")
    last = rand((3, vocab), 61, 2.0)
    l[rows - 3:].copy_(last)
    u = uniforms(rows, 61)
    got = ops.sample(l, u.to("spyre"), None, None, torch.full((rows,), 0.9).to("spyre"))
    want = check_sample(last, "spyre", u[rows - 3:], p=0.9)
    assert got[rows - 3:].tolist() == want


@pytest.mark.parametrize("device", DEVICES)
def test_append_one_slot_twice(device):
    """Each element is one of the two rows'; nothing else changes."""
    a = _append_args(device, slots=torch.tensor([5, 20, 5]))
    before = [a["k_cache"].cpu().clone(), a["v_cache"].cpu().clone()]
    ops.paged_append(**a)
    rows = []
    for keep in ([5, 20, -1], [-1, 20, 5]):
        b = _append_args(device, slots=torch.tensor(keep))
        ops.paged_append(**b)
        rows.append([b["k_cache"].cpu(), b["v_cache"].cpu()])
    for i, name in enumerate(("k_cache", "v_cache")):
        got = a[name].cpu()
        assert ((got == rows[0][i]) | (got == rows[1][i])).all()
        seen = torch.ones(2, 16, dtype=torch.bool)
        seen.view(-1)[[5, 20]] = False
        assert torch.equal(got[:, 0][seen], before[i][:, 0][seen])


@pytest.mark.gpu
def test_c_entries_on_two_streams():
    """Calls on two streams at once, each with its own workspace and output."""
    lib, dev = _capi.lib(), "cuda"
    h, kv, d, page, b, n = 8, 2, 128, 16, 3, 700
    pages = b * (n // page + 1)
    k, v = (rand((pages, kv, page, d), 62 + i).to(dev) for i in range(2))
    q = rand((b, h, d), 64).to(dev)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).view(b, -1).to(dev)
    lens = torch.tensor([n, n - 333, 1], device=dev)
    starts = torch.arange(b + 1, device=dev)
    logits, u = rand((b, 49155), 65, 2.0).to(dev), uniforms(b, 65).to(dev)
    share = torch.full((b,), 0.9, device=dev)
    bytes_ = lib.sph_paged_attention_workspace_bytes(b, b, h, kv, d, table.shape[1] * page)
    runs = []
    for i in range(2):
        runs.append((torch.cuda.Stream(), torch.empty(bytes_, dtype=torch.uint8, device=dev),
                     torch.zeros(b, h, d, dtype=torch.float16, device=dev),
                     torch.zeros(b, dtype=torch.int64, device=dev)))
    torch.cuda.synchronize()
    for _ in range(10):
        for stream, ws, out, tokens in runs:
            s = stream.cuda_stream
            assert lib.sph_paged_attention(
                _capi.F16, b, b, h, kv, d, q.data_ptr(), h * d, d, k.data_ptr(), *k.stride()[:3],
                v.data_ptr(), *v.stride()[:3], pages, page, table.data_ptr(), table.shape[1],
                table.shape[1], lens.data_ptr(), starts.data_ptr(), None, 0, 0, 0.09,
                out.data_ptr(), ws.data_ptr(), bytes_, None, s) == 0
            assert lib.sph_sample(_capi.F16, b, 49155, logits.data_ptr(), 49155, u.data_ptr(), None,
                                  None, share.data_ptr(), None, tokens.data_ptr(), s) == 0
    torch.cuda.synchronize()
    want = ops.paged_attention(*(x.cpu().to("spyre") for x in (q, k, v, table, lens, starts)), 0.09)
    drawn = ops.sample(logits.cpu().to("spyre"), u.cpu().to("spyre"), None, None,
                       share.cpu().to("spyre"))
    for _, _, out, tokens in runs:
        assert torch.equal(out.cpu(), want.cpu()) and torch.equal(tokens.cpu(), drawn.cpu())


# ---- refusals ----------------------------------------------------------------

def _append_args(device, **kw):
    a = dict(qkv=rand((3, 4 * 64), 1), cos=rand((9, 64), 2), sin=rand((9, 64), 3),
             positions=torch.zeros(3, dtype=torch.int64), slots=torch.arange(3),
             k_cache=rand((2, 1, 16, 64), 4), v_cache=rand((2, 1, 16, 64), 5), n_heads=2)
    a.update(kw)
    return {n: x.to(device) if isinstance(x, torch.Tensor) else x for n, x in a.items()}


@pytest.mark.parametrize("device", DEVICES)
def test_append_refusals(device):
    bad = [dict(qkv=rand((3, 4 * 64), 1, dtype=torch.float32)), dict(qkv=rand((3, 250), 1)),
           dict(qkv=rand((256,), 1)), dict(n_heads=3), dict(n_heads=0), dict(cos=rand((9, 32), 2)),
           dict(sin=rand((8, 64), 2)), dict(cos=rand((9, 64), 2, dtype=torch.bfloat16)),
           dict(positions=torch.zeros(2, dtype=torch.int64)),
           dict(positions=torch.zeros(3, dtype=torch.int32)),
           dict(slots=torch.zeros(3)), dict(slots=torch.zeros(1, 3, dtype=torch.int64)),
           dict(k_cache=rand((2, 1, 16, 64), 4, dtype=torch.bfloat16)),
           dict(v_cache=rand((2, 1, 8, 64), 4)), dict(k_cache=rand((2, 16, 64), 4)),
           dict(q_norm=rand((32,), 6)), dict(k_norm=rand((64,), 6, dtype=torch.bfloat16)),
           dict(q_norm=rand((64,), 6), k_norm=rand((64,), 6, dtype=torch.float32))]
    for kw in bad:
        with pytest.raises(RuntimeError, match="paged_append"):
            ops.paged_append(**_append_args(device, **kw))
    ops.paged_append(**_append_args(device))


def _attention_args(device, **kw):
    a = dict(q=rand((3, 4, 64), 1), k_cache=rand((2, 2, 16, 64), 4), v_cache=rand((2, 2, 16, 64), 5),
             block_table=torch.tensor([[0], [1]]), seq_lens=torch.tensor([5, 9]),
             q_starts=torch.tensor([0, 1, 3]), scale=0.125)
    a.update(kw)
    return {n: x.to(device) if isinstance(x, torch.Tensor) else x for n, x in a.items()}


@pytest.mark.parametrize("device", DEVICES)
def test_attention_refusals(device):
    bad = [dict(q=rand((3, 4, 64), 1, dtype=torch.float32)), dict(q=rand((3, 256), 1)),
           dict(q=rand((3, 3, 64), 1)), dict(q=rand((3, 4, 32), 1)),
           dict(k_cache=rand((2, 2, 16, 64), 4, dtype=torch.bfloat16)),
           dict(v_cache=rand((2, 2, 8, 64), 4)), dict(block_table=torch.tensor([0, 1])),
           dict(block_table=torch.tensor([[0], [1]], dtype=torch.int32)),
           dict(seq_lens=torch.tensor([5])), dict(seq_lens=torch.tensor([5.0, 9.0])),
           dict(q_starts=torch.tensor([0, 3])), dict(scale=0.0), dict(scale=-1.0),
           dict(scale=INF), dict(scale=NAN), dict(mask=torch.ones(2, 2, dtype=torch.bool)),
           dict(mask=torch.ones(3, 2)), dict(mask=torch.ones(3, dtype=torch.bool))]
    for kw in bad:
        with pytest.raises(RuntimeError, match="paged_attention"):
            ops.paged_attention(**_attention_args(device, **kw))
    ops.paged_attention(**_attention_args(device))


@pytest.mark.parametrize("device", DEVICES)
def test_sample_refusals(device):
    l, u = rand((3, 50), 1).to(device), torch.rand(3).to(device)
    f, i = torch.ones(3, device=device), torch.ones(3, dtype=torch.int64, device=device)
    for args in [(l.double(), u), (l[0], u), (l[:, :0], u), (l, u[:2]), (l, u.half()), (l, u, i),
                 (l, u, f[:1]), (l, u, f, f), (l, u, f, i[:, None]), (l, u, f, i, i),
                 (l, u, f, i, f, f[:2])]:
        with pytest.raises(RuntimeError, match="sample"):
            ops.sample(*args)
    ops.sample(l, u, f, i, f, f)


@pytest.mark.gpu
def test_refusals_of_the_device():
    with pytest.raises(RuntimeError, match="head_dim must be 64 or 128"):
        ops.paged_attention(**_attention_args("spyre", q=rand((3, 4, 96), 1),
                                              k_cache=rand((2, 2, 16, 96), 1),
                                              v_cache=rand((2, 2, 16, 96), 1)))
    with pytest.raises(RuntimeError, match="head_dim must be 64 or 128"):
        ops.paged_append(**_append_args("spyre", qkv=rand((3, 4 * 32), 1), cos=rand((9, 32), 2),
                                        sin=rand((9, 32), 3), k_cache=rand((2, 1, 16, 32), 4),
                                        v_cache=rand((2, 1, 16, 32), 4)))
    a = _attention_args("spyre")
    with pytest.raises(RuntimeError, match="seq_lens is on cpu"):
        ops.paged_attention(**dict(a, seq_lens=torch.tensor([5, 9])))
    with pytest.raises(RuntimeError, match="stride 1"):
        ops.paged_attention(**dict(a, k_cache=rand((2, 2, 64, 16), 1).to("spyre").transpose(2, 3)))
    with pytest.raises(RuntimeError, match="2\\^20"):
        ops.sample(torch.zeros(1, (1 << 20) + 1, dtype=torch.float16, device="spyre"),
                   torch.zeros(1, device="spyre"))
    # caches that overlap themselves or each other cannot be written
    c = rand((2, 1, 16, 64), 4).to("spyre")
    with pytest.raises(RuntimeError):
        ops.paged_append(**dict(_append_args("spyre"), k_cache=c[:1].expand(2, 1, 16, 64)))
    with pytest.raises(RuntimeError):
        ops.paged_append(**dict(_append_args("spyre"), k_cache=c, v_cache=c))
    with pytest.raises(RuntimeError, match="4096"):
        ops.paged_attention(**dict(a, block_table=torch.zeros(5000, 1, dtype=torch.int64).to("spyre"),
                                   seq_lens=torch.zeros(5000, dtype=torch.int64).to("spyre"),
                                   q_starts=torch.zeros(5001, dtype=torch.int64).to("spyre")))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["qkv", "cos", "sin", "q_norm", "k_norm", "positions", "slots"])
@pytest.mark.parametrize("cache", ["k_cache", "v_cache"])
def test_append_refuses_inputs_in_the_caches(cache, name):
    """Rows, tables, weights and indices that lie in a cache would be read while it is written."""
    a = _append_args("spyre", q_norm=rand((64,), 6), k_norm=rand((64,), 7))
    before = a[cache].cpu()
    flat = a[cache].view(-1)
    if a[name].dtype == torch.int64:
        flat = flat.view(torch.int64)
    with pytest.raises(RuntimeError, match="overlap|memory location"):
        ops.paged_append(**dict(a, **{name: flat[:a[name].numel()].view(a[name].shape)}))
    assert torch.equal(a[cache].cpu(), before)


@pytest.mark.parametrize("device", DEVICES)
def test_no_gradients(device):
    for call, args, name in ((ops.paged_append, _append_args(device), "qkv"),
                             (ops.paged_attention, _attention_args(device), "q")):
        leaf = args[name].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            call(**dict(args, **{name: leaf}))
        with torch.no_grad():
            call(**dict(args, **{name: leaf}))
    l = rand((3, 50), 1, dtype=torch.float32).to(device).requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.sample(l, torch.rand(3).to(device))
    assert not ops.sample(l.detach(), torch.rand(3).to(device)).requires_grad


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tokens", [3, 0])
def test_append_raises_the_versions_of_the_caches(tokens, device):
    """A backward pass that saved a cache raises once the cache has been written."""
    a = _append_args(device)
    if tokens == 0:
        a.update({n: a[n][:0] for n in ("qkv", "positions", "slots")})
    names = ("k_cache", "v_cache")
    for name in names:
        before = [a[n]._version for n in names]
        # (read through a view: it has its base's version)
        w = torch.ones(1, 16, 64, dtype=torch.float16).to(device).requires_grad_()
        y = (w * a[name][1]).sum()
        with torch.no_grad():
            ops.paged_append(**a)
        assert all(a[n]._version > x for n, x in zip(names, before))
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("device", DEVICES)
def test_append_to_inference_tensors(device):
    want = _append_args(device)
    q = ops.paged_append(**want)
    with torch.inference_mode():
        a = {n: x.clone() if isinstance(x, torch.Tensor) else x
             for n, x in _append_args(device).items()}
        assert torch.equal(ops.paged_append(**a).cpu(), q.cpu())
        for n in ("k_cache", "v_cache"):
            assert a[n].is_inference() and torch.equal(a[n].cpu(), want[n].cpu())


def test_fakes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode() as mode:
        def fake(args):
            return {n: mode.from_tensor(x) if isinstance(x, torch.Tensor) else x
                    for n, x in args.items()}

        q = ops.paged_append(**fake(_append_args("cpu")))
        assert q.shape == (3, 2, 64) and q.dtype == torch.float16
        assert ops.paged_attention(**fake(_attention_args("cpu"))).shape == (3, 4, 64)
        t = ops.sample(torch.empty(3, 50), torch.empty(3))
        assert t.shape == (3,) and t.dtype == torch.int64
        with pytest.raises(RuntimeError, match="paged_append"):
            ops.paged_append(**fake(_append_args("cpu", n_heads=5)))


# ---- the C entry points ------------------------------------------------------

def test_c_entries_refuse_before_any_launch():
    lib = _capi.lib()
    one = torch.zeros(64, dtype=torch.int64)
    x = one.data_ptr()

    def attn(**kw):
        a = dict(dtype=_capi.F16, tokens=4, batch=2, heads=4, kv=2, dim=128, q=x, q_t=512, q_h=128,
                 k=x, kp=1, kh=1, ks=1, v=x, vp=1, vh=1, vs=1, pages=3, page=16, table=x, ldt=1,
                 width=1, lens=x, starts=x, mask=None, ldm=0, mw=0, scale=0.1, o=x, ws=x,
                 bytes=1 << 40, err=None, stream=None)
        a.update(kw)
        return lib.sph_paged_attention(*a.values())

    for kw in (dict(dtype=_capi.F32), dict(dim=96), dict(kv=3), dict(scale=0.0), dict(scale=INF),
               dict(q=None), dict(lens=None), dict(batch=5000), dict(tokens=-1), dict(batch=0),
               dict(page=0), dict(width=1 << 29), dict(bytes=16), dict(ws=None), dict(ws=x + 4),
               dict(tokens=1 << 24), dict(mask=x, ldm=2, mw=3), dict(k=None), dict(table=None)):
        assert attn(**kw) >= 1001, kw
    assert attn(tokens=0) == 0
    assert lib.sph_paged_attention_workspace_bytes(0, 1, 4, 2, 128, 100) == 0
    few = lib.sph_paged_attention_workspace_bytes(1, 1, 4, 1, 128, 100)
    many = lib.sph_paged_attention_workspace_bytes(1, 1, 4, 1, 128, 1 << 29)
    assert 0 < few < many == lib.sph_paged_attention_workspace_bytes(1, 1, 4, 1, 128, 1 << 30)

    def append(**kw):
        a = dict(dtype=_capi.F16, table=_capi.F16, norm=_capi.F16, tokens=2, heads=2, kv=1, dim=64,
                 qkv=x, ld=256, cos=x, ldc=64, sin=x, lds=64, n=4, pos=x, slots=x, qn=None, kn=None,
                 eps=1e-5, k=x, kp=1, kh=1, ks=1, v=x, vp=1, vh=1, vs=1, pages=1, page=16, q=x,
                 err=None, stream=None)
        a.update(kw)
        return lib.sph_paged_append(*a.values())

    for kw in (dict(dtype=_capi.F32), dict(table=_capi.BF16), dict(norm=_capi.I32), dict(dim=32),
               dict(heads=0), dict(tokens=-1), dict(qkv=None), dict(ld=255), dict(pos=None),
               dict(page=0), dict(tokens=1 << 24), dict(cos=None), dict(v=None), dict(q=None)):
        assert append(**kw) >= 1001, kw
    assert append(tokens=0) == 0
    ok = [_capi.F16, 2, 50, x, 50, x, None, None, None, None, x, None]
    for i, v in ((0, _capi.I32), (1, -1), (1, 1 << 22), (2, 0), (2, (1 << 20) + 1), (3, None),
                 (4, -1), (5, None), (10, None)):
        assert lib.sph_sample(*(ok[:i] + [v] + ok[i + 1:])) >= 1001, (i, v)
    assert lib.sph_sample(*(ok[:1] + [0] + ok[2:])) == 0

"""The 8-bit serving operators (e4m3 codes, one fp32 scale per group of 128):
torch.ops.spyre.{quantize_fp8, rms_norm_fp8, add_rms_norm_fp8, silu_mul_fp8,
mm_fp8} on the CPU (their formulas) and on spyre, and their C entry points.

Expected values come from plain 64-bit arithmetic here.  Tolerances:

  * A code is off its exact value v = y * 448 / amax by half an e4m3 step:
    2^-4 of |v|, at least 2^-10 (half of the subnormal step), plus the few
    fp32 roundings before it (2^-18 of |v| covers them).
  * Scales of plain values are one division: equal to torch's fp32 result.
    Those of silu(g) * u take about ten roundings of 2^-24: 2^-20.  Those of a
    norm hold a sum of squares, at most 128 additions deep in a thread and ten
    levels of lanes above it, whose relative error the root halves: 2^-16.
  * A product's inner sums come from the 8-bit matrix instruction.  Codes that
    are small integers with scales that are powers of two make every partial
    sum a small multiple of one power of two, so the result is exact.  For
    other codes the instruction drops low bits of its terms, measured as at
    most 1.6e-4 of the terms' magnitudes over random bytes: 2^-12 of the sum
    of magnitudes, plus half a step of the result's type.
"""

import ctypes
import math

import pytest
import torch

import torch_spyre  # noqa: F401
from torch_spyre import _capi

E4M3 = torch.float8_e4m3fn
DEVICES = ["cpu", pytest.param("spyre", marks=pytest.mark.gpu)]
ops = torch.ops.spyre


def rand(shape, k=0, scale=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(0xF8 + k)
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def codes64(q):
    return q.cpu().float().double()


def group_amax(y, block_rows=1):
    """[R / block_rows, ceil(C / 128)] largest magnitudes of y [R, C]."""
    r, c = y.shape
    p = torch.zeros(-(-r // block_rows) * block_rows, -(-c // 128) * 128, dtype=y.dtype)
    p[:r, :c] = y.abs()
    return p.view(-1, block_rows, p.shape[1] // 128, 128).amax((1, 3))


def spread(s, shape, block_rows=1):
    """Scales [R / block_rows, groups] for every element of `shape`."""
    return s.repeat_interleave(block_rows, 0)[:shape[0]].repeat_interleave(128, 1)[:, :shape[1]]


def check_codes(q, y, block_rows=1):
    """q [R, C] rounds y (64 bits) scaled so that its group's largest is 448."""
    v = y * 448 / spread(group_amax(y, block_rows).clamp(min=2.0 ** -100), y.shape, block_rows)
    off = (codes64(q) - v).abs()
    bound = torch.clamp(v.abs() * 2.0 ** -4, min=2.0 ** -10) + v.abs() * 2.0 ** -18
    assert bool((off <= bound).all()), (off / bound).max()


def check_scales(s, want, rel):
    torch.testing.assert_close(s.cpu().double(), want, rtol=rel, atol=0)


# ---- quantize_fp8 ------------------------------------------------------------

SHAPES = [(1, 1), (1, 128), (3, 130), (17, 512), (2, 15), (5, 4100), (130, 384), (257, 96)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(shape, dtype, block_rows, device):
    x = rand(shape, 1, 3.0, dtype)
    q, s = ops.quantize_fp8(x.to(device), block_rows)
    assert q.dtype == E4M3 and tuple(q.shape) == shape
    assert q.device.type == device and q.stride(0) % 16 == 0 or shape[0] == 1
    amax = group_amax(x.float(), block_rows)
    assert torch.equal(s.cpu(), amax / 448)
    check_codes(q, x.double(), block_rows)
    # bit for bit the fp32 formula (448 / tensor would be a reciprocal times 448)
    r = spread(torch.full_like(amax, 448) / amax, shape, block_rows)
    assert torch.equal(codes64(q), (x.float() * r).to(E4M3).double())


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_strides_and_dims(device):
    base = rand((4, 9, 300), 2, dtype=torch.float16)
    dev = base.to(device)
    for pick in (lambda t: t[:, :, 3:291], lambda t: t[1], lambda t: t[:, 4], lambda t: t[0, 0],
                 lambda t: t.transpose(0, 1), lambda t: t[:, ::2, :128], lambda t: t[..., ::2],
                 lambda t: t[:1].expand(3, 9, 300), lambda t: t[2:2], lambda t: t[..., :0]):
        x = pick(base)
        q, s = ops.quantize_fp8(pick(dev))
        wq, ws = ops.quantize_fp8(x.contiguous())
        assert q.shape == x.shape and s.shape == (*x.shape[:-1], -(-x.shape[-1] // 128))
        assert torch.equal(codes64(q), codes64(wq)) and torch.equal(s.cpu(), ws)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_quantize_special_values(dtype, device):
    x = rand((9, 256), 3, dtype=dtype)
    x[0, 5] = float("inf")
    x[1, 200] = float("nan")
    x[2] = 0
    x[3, :128] = -0.0
    x[4, 7] = -float("inf")
    x[5] = torch.finfo(dtype).max
    x[6] = torch.finfo(dtype).tiny / 4 if dtype != torch.float16 else 2.0 ** -24
    x[7, 0] = torch.finfo(dtype).max
    x[8, 3], x[8, 4] = float("nan"), float("inf")
    q, s = ops.quantize_fp8(x.to(device))
    q, s = codes64(q), s.cpu()
    amax = x.float().abs().view(9, 2, 128).amax(2).clamp(min=2.0 ** -100)
    assert torch.equal(s.isnan(), amax.isnan())
    assert torch.equal(s[~s.isnan()], (amax / 448)[~s.isnan()])
    assert q[0, 5].isnan() and not q[0, :5].any() and not q[0, 128:].isnan().any()
    assert q[1, 128:].isnan().all() and not q[1, :128].isnan().any()
    assert not q[2].any() and q[4, 7].isnan() and bool((q[5] == 448).all())
    assert q[7, 0] == 448 and q[8, :128].isnan().all()
    assert not q[6].isnan().any()
    if dtype == torch.float16:  # subnormals are values like others
        assert bool((q[6] == 448).all())


@pytest.mark.parametrize("device", DEVICES)
def test_quantize_ties_and_halves(device):
    # every fp16 value from 448 down through the codes' subnormals, scaled by 1
    x = torch.arange(0x6000, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[x <= 448]
    n = x.numel() // 127 * 127
    x = torch.cat([torch.full((n // 127, 1), 448.0, dtype=torch.float16), x[:n].view(-1, 127)], 1)
    q, s = ops.quantize_fp8(x.to(device))
    assert bool((s.cpu() == 1).all())
    assert torch.equal(codes64(q), x.float().to(E4M3).double())
    q, s = ops.quantize_fp8((-x).to(device))
    assert torch.equal(codes64(q), (-x).float().to(E4M3).double())


# ---- norms -------------------------------------------------------------------

def norm64(h, w, eps):
    y = h * torch.rsqrt((h * h).mean(-1, keepdim=True) + eps)
    return y if w is None else y * w


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("weight", ["same", "fp32", None])
@pytest.mark.parametrize("shape", [(1, 1), (1, 4096), (3, 130), (7, 2048), (33, 2049), (2, 8200),
                                   (5, 96), (19, 512), (1, 40001)])
def test_norms(shape, weight, dtype, device):
    x, r = rand(shape, 4, 2.0, dtype), rand(shape, 5, 1.0, dtype)
    w = None if weight is None else (1 + rand(shape[1:], 6, 0.2, torch.float32))
    w = w.to(dtype) if weight == "same" else w
    w64, wd = (None, None) if w is None else (w.double(), w.to(device))
    eps = 1e-5
    q, s = ops.rms_norm_fp8(x.to(device), wd, eps)
    y = norm64(x.double(), w64, eps)
    check_codes(q, y)
    check_scales(s, group_amax(y) / 448, 2.0 ** -16)
    q, s, h = ops.add_rms_norm_fp8(x.to(device), r.to(device), wd, eps)
    assert torch.equal(h.cpu(), x + r) and h.is_contiguous()
    y = norm64((x + r).double(), w64, eps)
    check_codes(q, y)
    check_scales(s, group_amax(y) / 448, 2.0 ** -16)


@pytest.mark.parametrize("device", DEVICES)
def test_norms_strided_rows_and_special_values(device):
    base, res = rand((6, 700), 7, dtype=torch.float16), rand((6, 900), 8, dtype=torch.float16)
    x, r = base[:, 5:605], res[:, 300:900]
    w = 1 + rand((600,), 9, 0.1, torch.float16)
    base[1] = 0
    res[1] = 0
    base[2, 50] = float("nan")
    base[3, 40] = float("inf")
    q, s, h = ops.add_rms_norm_fp8(base.to(device)[:, 5:605], res.to(device)[:, 300:900],
                                   w.to(device), 1e-5)
    q, s = codes64(q), s.cpu().double()
    torch.testing.assert_close(h.cpu(), x + r, rtol=0, atol=0, equal_nan=True)
    ok = [0, 4, 5]
    y = norm64((x + r).double(), w.double(), 1e-5)
    check_codes(q[ok], y[ok])
    check_scales(s[ok], group_amax(y[ok]) / 448, 2.0 ** -16)
    # a row of zeros: zero codes, finite scales
    assert not q[1].any() and bool((s[1] > 0).all() and s[1].isfinite().all())
    # NaN: every value of the row is NaN; infinity: its group is, the others are 0
    v = q * spread(s, q.shape)
    assert v[2].isnan().all() and v[3, 35].isnan()
    assert not v[3, 128:].any() and not v[3, 128:].isnan().any()


# ---- silu_mul_fp8 ------------------------------------------------------------

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 131), (24, 12800), (18, 1000), (130, 64)])
def test_silu_mul(shape, dtype, device):
    gu = rand((shape[0], 2 * shape[1]), 10, 3.0, dtype)
    gu[:, :1] = -30.0  # far into the tails
    gu[0, 0] = 30.0
    q, s = ops.silu_mul_fp8(gu.to(device))
    g, u = gu.double().chunk(2, 1)
    y = g / (1 + torch.exp(-g)) * u
    check_codes(q, y)
    check_scales(s, group_amax(y).clamp(min=2.0 ** -100) / 448, 2.0 ** -20)
    wide = torch.zeros(shape[0], 2 * shape[1] + 37, dtype=dtype)
    wide[:, 5:5 + 2 * shape[1]] = gu
    q2, s2 = ops.silu_mul_fp8(wide.to(device)[:, 5:5 + 2 * shape[1]])
    assert torch.equal(codes64(q2), codes64(q)) and torch.equal(s2.cpu(), s.cpu())


@pytest.mark.parametrize("device", DEVICES)
def test_silu_mul_extremes(device):
    big = torch.finfo(torch.bfloat16).max
    g = torch.tensor([0.0, -0.0, big, -big, float("inf"), -float("inf"), float("nan"), 1.0, -90.0])
    gu = torch.zeros(9, 256, dtype=torch.bfloat16)
    gu[:, 3] = g.bfloat16()
    gu[:, 131] = 2.0
    q, s = ops.silu_mul_fp8(gu.to(device))
    q, s = codes64(q)[:, 3], s.cpu()[:, 0]
    assert q[0] == 0 and q[1] == 0 and s[2] == float("inf") and q[3] == 0
    assert s[4] == float("inf") and q[5].isnan() and q[6].isnan() and q[7] == 448
    # 2 silu(-90) = -1.5e-37, under the least magnitude: -8e-5 in code units
    assert q[8] == 0


@pytest.mark.parametrize("device", DEVICES)
def test_silu_mul_deep_in_the_negative_tail(device):
    """Gates at which exp(-g) is near the end of fp32's range, with up values that
    bring the product back into it."""
    g = torch.tensor([-80.0, -85.0, -86.5, -87.0, -87.5, -88.0, -88.5])
    gu = torch.cat([g[:, None].expand(7, 128), torch.full((7, 128), 2.0 ** 110)], 1).bfloat16()
    q, s = ops.silu_mul_fp8(gu.to(device))
    g, u = gu.double().chunk(2, 1)
    y = g / (1 + torch.exp(-g)) * u
    check_codes(q, y)
    check_scales(s, group_amax(y) / 448, 2.0 ** -20)


# ---- mm_fp8 ------------------------------------------------------------------

def whole_operands(m, n, k, seed=0):
    """Codes that are integers up to 3, scales that are powers of two."""
    g = torch.Generator().manual_seed(77 + seed)
    kb = -(-k // 128)
    x = torch.randint(-3, 4, (m, k), generator=g).float().to(E4M3)
    w = torch.randint(-3, 4, (n, k), generator=g).float().to(E4M3)
    xs = torch.ldexp(torch.ones(m, kb), torch.randint(-1, 1, (m, kb), generator=g))
    ws = torch.ldexp(torch.ones(-(-n // 128), kb),
                     torch.randint(-1, 1, (-(-n // 128), kb), generator=g))
    return x, xs, w, ws


def mm64(x, xs, w, ws, mags=False):
    """The product in 64 bits; with mags, that of the magnitudes."""
    a = codes64(x) * spread(xs.double(), x.shape)
    b = codes64(w) * spread(ws.double(), w.shape, 128)
    return a.abs() @ b.abs().t() if mags else a @ b.t()


MM_SHAPES = [(1, 1, 1), (1, 128, 128), (1, 6144, 4096), (2, 16, 64), (3, 130, 257), (4, 4100, 1040),
             (8, 256, 12800), (9, 300, 384), (16, 129, 130), (17, 640, 2048), (24, 515, 4096),
             (33, 1000, 512), (64, 256, 1024), (65, 96, 48), (100, 384, 4096), (128, 512, 640),
             (130, 257, 1300), (200, 1024, 2048), (256, 256, 128), (257, 513, 384),
             (333, 640, 4096), (512, 768, 1024), (777, 1100, 272), (300, 2048, 16),
             (24, 4096, 12800), (70, 5000, 1024), (600, 3200, 1920), (1030, 2000, 1310),
             (777, 6144, 1045), (651, 1033, 5539), (73, 7747, 5376), (333, 4096, 6500), (116, 6117, 5199), (1800, 10300, 256),
             (2040, 6100, 2048), (3000, 5000, 1536), (4000, 6200, 2048),
             (2313, 5123, 1152), (3459, 4616, 896), (2591, 6357, 1152)]


def plan(m, n, k, workspace=None):
    """((kernel, rows of X, rows of W, workgroups per CU), K slices, "", "columns"
    or "rows": what is split off for a second product) that the library runs a
    product on (host only)."""
    lib, out = _capi.lib(), (ctypes.c_int32 * 7)()
    if workspace is None:
        workspace = lib.sph_gemm_fp8_workspace_bytes(m, n, k)
    assert lib.sph_gemm_fp8_plan(m, n, k, workspace, ctypes.addressof(out)) == 0
    return ({1: "stream", 2: "ring", 3: "tiles"}[out[0]], out[1], out[2], out[4]), out[3], ("", "columns",
            "rows")[out[6]]


def test_mm_shapes_cover_every_kernel():
    assert {plan(*s)[0] for s in MM_SHAPES} == {
        ("stream", 16, 16, 4), ("ring", 32, 64, 3), ("ring", 64, 128, 2),
        ("ring", 128, 128, 1), ("ring", 128, 128, 2), ("tiles", 256, 192, 1),
        ("tiles", 256, 256, 1)}
    assert {plan(*s)[1] > 1 for s in MM_SHAPES} == {True, False}
    assert {plan(*s)[2] for s in MM_SHAPES} == {"", "columns", "rows"}
    # without a workspace nothing is split
    assert all(plan(*s, 0)[1] == 1 for s in MM_SHAPES)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", MM_SHAPES)
def test_mm_whole_numbers(m, n, k):
    x, xs, w, ws = whole_operands(m, n, k, m + n + k)
    want = mm64(x, xs, w, ws)
    # |sums| <= 9 * 12800 in quarters: exact in fp32; rounded once to the type
    dev = [t.to("spyre") for t in (x, xs.t().contiguous().t(), w, ws)]
    for dtype in (torch.bfloat16, torch.float16):
        y = ops.mm_fp8(*dev, dtype).cpu()
        assert y.dtype == dtype and torch.equal(y, want.float().to(dtype)), (
            (y.double() - want).abs().max())
    bias = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(5)).half()
    y = ops.mm_fp8(*dev, torch.float16, bias.to("spyre")).cpu()
    assert torch.equal(y, (want + bias.double()).float().half())


# Streamed products of more than one pass of 32 blocks of K, whole and partial last
# blocks, few rows and few columns.
STREAMED = [(1, 2048, 5376), (4, 4096, 12800), (8, 4096, 14336), (5, 3001, 9001), (1, 245, 4192),
            (1, 9152, 1664), (3226, 16, 4210)]


def test_streaming_follows_its_fitted_time():
    for s in STREAMED:
        assert plan(*s)[0][0] == "stream", s
    for m in (1, 2, 4, 8):  # a down projection of the decoder, and longer rows
        for k in (4096, 8192, 12800, 13312, 14336, 16384):
            assert plan(m, 4096, k)[0][0] == "stream", (m, k)
        # a 257th workgroup begins a second round
        assert plan(m, 4097, 12800)[0][0] == "ring", m
    for m in (16, 24, 32):  # bytes of X beside W's
        assert plan(m, 4096, 12800)[0][0] == "ring" and plan(m, 4096, 12800)[1] > 1, m
    assert plan(1, 6144, 4096)[0][0] == plan(1, 4096, 4096)[0][0] == "stream"


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", STREAMED)
def test_mm_streamed_over_long_rows(m, n, k):
    x, xs, w, ws = whole_operands(m, n, k, m + n + k)
    bias = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(7)).half()
    want = mm64(x, xs, w, ws) + bias.double()
    dev = [t.to("spyre") for t in (x, xs.t().contiguous().t(), w, ws)]
    y = ops.mm_fp8(*dev, torch.float16, bias.to("spyre")).cpu()
    assert torch.equal(y, want.float().half()), (y.double() - want).abs().max()


# Products on 256 rows of X by 256 or 192 of W with several tiles per workgroup, so
# that the loads of one tile run on behind the stores of the one before: rows of
# the result on cache lines (streaming stores) and off them, whole and ragged
# tiles, 192-row tiles that begin in the middle of a block of W.
TILE_SHAPES = [(3428, 6144, 1024), (3000, 12288, 896), (1501, 15509, 1024), (8192, 6144, 512),
               (2600, 16384, 512), (2000, 13000, 640)]


def test_tile_shapes_cover_both_stores_and_second_tiles():
    found = set()
    for m, n, k in TILE_SHAPES:
        (kernel, tm, tn, _), _, split = plan(m, n, k)
        assert kernel == "tiles" and not split and -(-m // tm) * -(-n // tn) > 256
        found.add((tn, n % 64 == 0))
    assert found == {(256, True), (256, False), (192, True), (192, False)}
    assert any(-(-m // 256) * -(-n // 192) > 512 for m, n, k in TILE_SHAPES
               if plan(m, n, k)[0][2] == 192)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", TILE_SHAPES)
def test_mm_several_tiles_per_workgroup(m, n, k):
    x, xs, w, ws = whole_operands(m, n, k, m + n + k)
    want = mm64(x, xs, w, ws)
    bias = torch.randint(-8, 9, (n,), generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    dev = [t.to("spyre") for t in (x, xs.t().contiguous().t(), w, ws)]
    for dtype, b in ((torch.bfloat16, bias), (torch.float16, None), (torch.float16, bias.half())):
        y = ops.mm_fp8(*dev, dtype, None if b is None else b.to("spyre")).cpu()
        y64 = want if b is None else want + b.double()
        assert torch.equal(y, y64.float().to(dtype)), (y.double() - y64).abs().max()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", [(1, 640, 4096), (5, 130, 300), (24, 257, 1000), (130, 384, 640),
                                   (300, 512, 2064)])
def test_mm_random(m, n, k, dtype, device):
    xq, xs = ops.quantize_fp8(rand((m, k), 11, 2.0).to(device))
    wq, ws = ops.quantize_fp8(rand((n, k), 12, 0.05).to(device), 128)
    bias = rand((n,), 13, 0.5, dtype)
    y = ops.mm_fp8(xq, xs, wq, ws, dtype, bias.to(device)).cpu().double()
    parts = [t.cpu() for t in (xq, xs, wq, ws)]
    want, mags = mm64(*parts) + bias.double(), mm64(*parts, mags=True)
    half = torch.finfo(dtype).eps / 2
    bound = mags * 2.0 ** -12 + want.abs() * half * (1 + 2.0 ** -8) + 2.0 ** -24
    assert bool(((y - want).abs() <= bound).all()), ((y - want).abs() / bound).max()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 3, 16, 40, 130, 300])
def test_mm_layouts(m):
    """Operands in wider rows whose other bytes are NaN codes, off 16 bytes and
    not, scales in every order, inputs of more dimensions."""
    n, k = 260, 200
    x, xs, w, ws = whole_operands(m, n, k, m)
    want = mm64(x, xs, w, ws).float().half()

    def inside(t, left, right):
        base = torch.full((t.shape[0] + 2, left + t.shape[1] + right), 0x7F, dtype=torch.uint8)
        base[1:-1, left:left + t.shape[1]] = t.view(torch.uint8)
        return base.view(E4M3).to("spyre")[1:-1, left:left + t.shape[1]]

    for left, right in ((0, 24), (16, 8), (48, 40), (3, 5)):
        for sx in (xs.to("spyre"), xs.t().contiguous().to("spyre").t(),
                   torch.stack([xs, xs], 2).to("spyre")[..., 0]):
            sw = ws.t().contiguous().to("spyre").t()
            y = ops.mm_fp8(inside(x, left, right), sx, inside(w, left, right), sw, torch.float16)
            assert torch.equal(y.cpu(), want)
    y = ops.mm_fp8(x.to("spyre").view(1, m, k), xs.to("spyre").view(1, m, 2), w.to("spyre"),
                   ws.to("spyre"), torch.float16)
    assert y.shape == (1, m, n) and torch.equal(y.cpu()[0], want)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2, 300, 512), (70, 300, 512), (300, 300, 512), (2040, 6100, 1024)])
def test_mm_nan_stays_in_its_row_and_column(m, n, k):
    x, xs, w, ws = whole_operands(m, n, k)
    want = mm64(x, xs, w, ws).float().half()
    x.view(torch.uint8)[1, 300] = 0x7F
    w.view(torch.uint8)[131, 17] = 0xFF
    y = ops.mm_fp8(x.to("spyre"), xs.to("spyre"), w.to("spyre"), ws.to("spyre"),
                   torch.float16).cpu()
    nan = torch.zeros(m, n, dtype=torch.bool)
    nan[1], nan[:, 131] = True, True
    assert torch.equal(y.isnan(), nan) and torch.equal(y[~nan], want[~nan])


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(2, 1100, 512), (40, 1100, 600), (300, 1100, 640), (2040, 6100, 1024)])
def test_mm_rows_far_apart(m, n, k):
    """Rows of W (and, from 1030 rows on, X) that reach past 2^32 bytes."""
    x, xs, w, ws = whole_operands(m, n, k, m)

    def apart(t):
        ld = 4194288  # the largest stride of whole chunks
        base = torch.empty(t.shape[0] * ld, dtype=torch.uint8, device="spyre").view(E4M3)
        view = base.as_strided(t.shape, (ld, 1))
        view.copy_(t.to("spyre"))
        return view

    y = ops.mm_fp8(apart(x), xs.to("spyre"), apart(w), ws.to("spyre"), torch.float16)
    assert torch.equal(y.cpu(), mm64(x, xs, w, ws).float().half())


@pytest.mark.gpu
def test_mm_rows_further_apart_than_the_entry_takes():
    """The last position of 1024 x 4096 codes a sequence (4194304 bytes apart), one
    row of such a tensor, and W laid out that way."""
    x, xs, w, ws = whole_operands(4, 300, 4096, 9)
    base = torch.zeros(4, 1024, 4096, dtype=torch.uint8, device="spyre").view(E4M3)
    base[:, -1] = x.to("spyre")
    xs, w, ws = xs.to("spyre"), w.to("spyre"), ws.to("spyre")
    want = mm64(x, *(t.cpu() for t in (xs, w, ws))).float().half()
    assert torch.equal(ops.mm_fp8(base[:, -1], xs, w, ws, torch.float16).cpu(), want)
    assert torch.equal(ops.mm_fp8(base[2:3, -1], xs[2:3], w, ws, torch.float16).cpu(), want[2:3])
    assert torch.equal(ops.mm_fp8(base[2, -1], xs[2], w, ws, torch.float16).cpu(), want[2])
    wide = ops.mm_fp8(x.to("spyre"), xs, base[:, -1], xs[:1], torch.float16).cpu()
    assert torch.equal(wide, mm64(x, xs.cpu(), x, xs[:1].cpu()).float().half())


@pytest.mark.gpu
def test_mm_result_past_32_bits():
    """50000 x 49152 results are 4.9 GB; the last rows against a product of their own."""
    m, n, k = 50000, 49152, 128
    x, xs, w, ws = (t.to("spyre") for t in whole_operands(m, n, k))
    y = ops.mm_fp8(x, xs, w, ws, torch.bfloat16)
    for rows in (slice(0, 70), slice(43690, 43760), slice(m - 70, m)):
        want = mm64(*(t.cpu() for t in (x[rows], xs[rows], w, ws)))
        assert torch.equal(y[rows].cpu(), want.float().to(torch.bfloat16))


@pytest.mark.gpu
def test_rows_past_32_bits():
    """Row kernels on 70000 x 32768 values (4.6 GB): the last rows as on their own."""
    x = torch.empty(70000, 32768, dtype=torch.bfloat16, device="spyre")
    tail = rand((40, 32768), 21).to("spyre")
    x[-40:] = tail
    x[:40] = tail
    runs = [lambda t: ops.quantize_fp8(t), lambda t: ops.quantize_fp8(t[:, :4160]),
            lambda t: ops.silu_mul_fp8(t), lambda t: ops.rms_norm_fp8(t, None, 1e-5),
            lambda t: ops.rms_norm_fp8(t[:, :4096], None, 1e-5),
            lambda t: ops.add_rms_norm_fp8(t[:, :1024], t[:, 1024:2048], None, 1e-5)]
    for run in runs:
        for big, alone in zip(run(x), run(tail)):
            for part in (big[-40:], big[:40]):
                assert torch.equal(part.cpu().float(), alone.cpu().float())


@pytest.mark.gpu
def test_mm_on_two_streams_at_once():
    """Two products with K slices, each with a workspace of its own, through the C
    entry on two streams."""
    lib = _capi.lib()
    jobs = []
    for m, n, k in ((16, 300, 6400), (70, 900, 4096)):
        host = whole_operands(m, n, k, m)
        dev = [t.cuda() for t in host]
        nws = lib.sph_gemm_fp8_workspace_bytes(m, n, k)
        assert nws > 0
        jobs.append((m, n, k, host, dev, torch.empty(nws, dtype=torch.uint8, device="cuda"),
                     torch.zeros(m, n, dtype=torch.float16, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for m, n, k, _, (x, xs, w, ws), wsp, y, st in jobs:
            _capi.call("sph_gemm_fp8", _capi.F16, m, n, k, x.data_ptr(), k, xs.data_ptr(),
                       *xs.stride(), w.data_ptr(), k, ws.data_ptr(), *ws.stride(), None,
                       y.data_ptr(), n, wsp.data_ptr(), wsp.numel(), st.cuda_stream)
    torch.cuda.synchronize()
    for *_, host, _, _, y, _ in jobs:
        assert torch.equal(y.cpu(), mm64(*host).float().half())


@pytest.mark.parametrize("device", DEVICES)
def test_mm_empty(device):
    e = lambda *s: torch.zeros(*s, device=device)  # noqa: E731
    q = lambda *s: torch.zeros(*s).to(E4M3).to(device)  # noqa: E731
    assert ops.mm_fp8(q(0, 64), e(0, 1), q(8, 64), e(1, 1), torch.float16).shape == (0, 8)
    assert ops.mm_fp8(q(4, 64), e(4, 1), q(0, 64), e(0, 1), torch.float16).shape == (4, 0)
    y = ops.mm_fp8(q(4, 0), e(4, 0), q(8, 0), e(1, 0), torch.float16,
                   torch.ones(8, dtype=torch.float16, device=device))
    assert torch.equal(y.cpu(), torch.ones(4, 8, dtype=torch.float16))
    x, s = ops.quantize_fp8(torch.zeros(3, 0, dtype=torch.float16, device=device))
    assert x.shape == (3, 0) and s.shape == (3, 0)


# ---- refusals ----------------------------------------------------------------

@pytest.mark.parametrize("device", DEVICES)
def test_refusals(device):
    x = rand((4, 256)).to(device)
    q, s = ops.quantize_fp8(x)
    w, ws = ops.quantize_fp8(rand((130, 256)).to(device), 128)
    f16 = torch.float16

    def refuse(match, call, *args):
        with pytest.raises(RuntimeError, match=match):
            call(*args)

    refuse("block_rows must be 1 or 128", ops.quantize_fp8, x, 64)
    refuse("2-dimensional", ops.quantize_fp8, x[None], 128)
    refuse("fp16, bf16 or fp32", ops.quantize_fp8, x.to(torch.int32))
    refuse("fp16 or bf16", ops.rms_norm_fp8, x.float(), None, 1e-5)
    refuse("x's shape and type", ops.add_rms_norm_fp8, x, x[:2], None, 1e-5)
    refuse("x's shape and type", ops.add_rms_norm_fp8, x, x.half(), None, 1e-5)
    refuse("weight must be", ops.rms_norm_fp8, x, x[0, :8], 1e-5)
    refuse("weight must have", ops.rms_norm_fp8, x, x[0].half(), 1e-5)
    refuse("must be even", ops.silu_mul_fp8, x[:, :7])
    refuse("fp16 or bf16", ops.silu_mul_fp8, x.float())
    refuse("float8_e4m3fn", ops.mm_fp8, x, s, w, ws, f16)
    refuse("result must be", ops.mm_fp8, q, s, w, ws, torch.float32)
    refuse("scales must be fp32", ops.mm_fp8, q, s.half(), w, ws, f16)
    refuse("x_scale must be", ops.mm_fp8, q, s[:, :1], w, ws, f16)
    refuse("w_scale must be", ops.mm_fp8, q, s, w, ws[:1], f16)
    refuse(r"\[\.\.\., K\]", ops.mm_fp8, q[:, :128], s, w, ws, f16)
    refuse("bias must be", ops.mm_fp8, q, s, w, ws, f16, x[0])
    leaf = x[0].detach().clone().requires_grad_()
    refuse("no gradient", ops.rms_norm_fp8, x, leaf, 1e-5)
    with torch.no_grad():
        ops.rms_norm_fp8(x, leaf, 1e-5)
    if device == "spyre":
        refuse("is on cpu", ops.mm_fp8, q, s, w, ws.cpu(), f16)
        refuse("is on cpu", ops.rms_norm_fp8, x, leaf.detach().cpu(), 1e-5)


def test_c_entry_refusals():
    """Host checks only: every call fails before a launch."""
    lib, F16, F32, I8 = _capi.lib(), _capi.F16, _capi.F32, _capi.I8
    P = 0x10000  # never read

    def quant(dtype=F16, x=P, ldx=256, rows=4, cols=256, block=1, q=P, ldq=256, s=P, sr=1, sg=4):
        return lib.sph_quantize_fp8(dtype, x, ldx, rows, cols, block, q, ldq, s, sr, sg, None)

    assert quant(rows=-1) == 1001 and quant(block=2) == 1001 and quant(ldx=8) == 1001
    assert quant(ldq=8) == 1001 and quant(q=None) == 1001 and quant(x=None) == 1001
    assert quant(dtype=I8) == 1002 and quant(sr=-1) == 1001 and quant(cols=1 << 40, ldx=1 << 40,
                                                                      ldq=1 << 40) == 1003
    assert quant(block=128, rows=128 * 65535 + 1) == 1003
    assert quant(rows=0, x=None, q=None, s=None) == 0

    def silu(dtype=F16, ld=512, rows=4, cols=256, gu=P):
        return lib.sph_silu_mul_fp8(dtype, gu, ld, rows, cols, P, 256, P, 1, 4, None)

    assert silu(dtype=F32) == 1002 and silu(ld=511) == 1001 and silu(gu=None) == 1001

    def norm(dtype=F16, wd=F16, x=P, res=None, h=None, ldr=256, ldh=256, cols=256, w=P):
        return lib.sph_rmsnorm_fp8(dtype, wd, x, max(cols, 256), res, ldr, w, h, ldh, 4, cols, 1e-5,
                                   P, max(cols, 256), P, 1, 4, None)

    assert norm(dtype=F32) == 1002 and norm(wd=_capi.BF16) == 1002 and norm(x=None) == 1001
    assert norm(res=P) == 1001 and norm(res=P, h=P, ldr=1) == 1001
    assert norm(res=P, h=P, ldh=1) == 1001 and norm(cols=1048577) == 1003

    def gemm(dtype=F16, m=4, n=8, k=256, x=P, ldx=256, xs=P, w=P, ldw=256, ws=P, d=P, ldd=8, sg=1):
        return lib.sph_gemm_fp8(dtype, m, n, k, x, ldx, xs, 1, sg, w, ldw, ws, 1, 1, None, d, ldd,
                                None, 0, None)

    assert gemm(m=-1) == 1001 and gemm(dtype=F32) == 1002 and gemm(d=None) == 1001
    assert gemm(ldd=7) == 1001 and gemm(x=None) == 1001 and gemm(ws=None) == 1001
    assert gemm(ldx=255) == 1001 and gemm(ldw=240) == 1001 and gemm(sg=-1) == 1001
    assert gemm(x=P + 8) == 1002 and gemm(w=P + 1) == 1002 and gemm(ldx=264) == 1002
    assert gemm(k=1 << 30, ldx=1 << 30, ldw=1 << 30) == 1003
    assert gemm(m=0, x=None, d=None) == 0


def test_c_entry_limits():
    """More workgroups than a launch holds, sizes past the limits and a workspace
    off 16 bytes: refused on the host."""
    lib, F16 = _capi.lib(), _capi.F16
    P = 0x10000  # never read

    def gemm(m, n, k, ld=4096, wsp=None, nws=0):
        return lib.sph_gemm_fp8(F16, m, n, k, P, ld, P, 1, 1, P, ld, P, 1, 1, None, P, n, wsp, nws,
                                None)

    assert gemm(1, 134217713, 16) == 1003 and gemm(1, 1 << 31, 16) == 1003
    assert gemm(20, 1 << 30, 256) == 1003 and gemm(1048561, 8, 16) == 1003
    assert gemm(1 << 20, 1 << 21, 16) == 1003 and gemm(4, 8, 256, wsp=P + 4, nws=64) == 1002
    out = (ctypes.c_int32 * 7)()
    for m, n, k in ((1 << 40, 1 << 40, 1 << 40), (1, 1 << 31, 16), (8, 8, 1 << 22)):
        assert lib.sph_gemm_fp8_workspace_bytes(m, n, k) == 0
        assert lib.sph_gemm_fp8_plan(m, n, k, 0, ctypes.addressof(out)) == 1003
    big = 1 << 29  # rows of one column (or two)
    assert lib.sph_silu_mul_fp8(F16, P, 2, big, 1, P, 1, P, 1, big, None) == 1003
    assert lib.sph_rmsnorm_fp8(F16, F16, P, 1, None, 0, None, None, 0, big, 1, 1e-5, P, 1, P, 1, big,
                               None) == 1003
    assert lib.sph_rmsnorm_fp8(F16, F16, P, 16384, None, 0, None, None, 0, 1 << 22, 16384, 1e-5, P,
                               16384, P, 1, 1 << 22, None) == 1003
    for rows in (1 << 60, (1 << 63) - 1):
        assert lib.sph_quantize_fp8(F16, P, 8, rows, 8, 1, P, 8, P, 1, 1, None) == 1003


def test_fakes_match_the_formulas():
    from torch._subclasses.fake_tensor import FakeTensorMode

    def meta(f):
        return [(t.shape, t.dtype, t.stride()) for t in f()]

    for shape in ((5, 384), (2, 3, 130), (7,), (4, 15)):
        x, r, w = rand(shape, 1), rand(shape, 2), rand(shape[-1:], 3)
        gu = rand((*shape[:-1], 2 * shape[-1]), 4)
        real = [meta(lambda: ops.quantize_fp8(x)), meta(lambda: ops.rms_norm_fp8(x, w, 1e-5)),
                meta(lambda: ops.add_rms_norm_fp8(x, r, w, 1e-5)),
                meta(lambda: ops.silu_mul_fp8(gu))]
        with FakeTensorMode() as mode:
            x, r, w, gu = (mode.from_tensor(t) for t in (x, r, w, gu))
            fake = [meta(lambda: ops.quantize_fp8(x)), meta(lambda: ops.rms_norm_fp8(x, w, 1e-5)),
                    meta(lambda: ops.add_rms_norm_fp8(x, r, w, 1e-5)),
                    meta(lambda: ops.silu_mul_fp8(gu))]
        assert real == fake
    assert math.isclose(2.0 ** -100 / 448, ops.quantize_fp8(torch.zeros(1, 8))[1].item(),
                        rel_tol=2.0 ** -24)  # half an fp32 step


# ---- derivatives ---------------------------------------------------------------

def _float_calls(device):
    """Every operator as a function of one tensor that a derivative could be
    taken by, and that tensor."""
    f16 = torch.float16
    x = rand((4, 256), 30).to(device)
    q, s = ops.quantize_fp8(x)
    w, ws = ops.quantize_fp8(rand((130, 256), 31).to(device), 128)
    return {
        "quantize": (lambda t: ops.quantize_fp8(t)[1], x),
        "rms_norm": (lambda t: ops.rms_norm_fp8(t, None, 1e-5)[1], x),
        "rms_norm weight": (lambda t: ops.rms_norm_fp8(x, t, 1e-5)[1], x[0]),
        "add_rms_norm": (lambda t: ops.add_rms_norm_fp8(x, t, None, 1e-5)[2], x),
        "silu": (lambda t: ops.silu_mul_fp8(t)[1], x),
        "mm x_scale": (lambda t: ops.mm_fp8(q, t, w, ws, f16), s),
        "mm w_scale": (lambda t: ops.mm_fp8(q, s, w, t, f16), ws),
        "mm bias": (lambda t: ops.mm_fp8(q, s, w, ws, f16, t), rand((130,), 32, 1.0, f16).to(device)),
    }


@pytest.mark.parametrize("device", DEVICES)
def test_derivatives_are_refused(device):
    """A leaf that requires a gradient and a dual tensor; the same calls without
    either run, also while a dual level is open."""
    from torch.autograd import forward_ad

    for name, (call, t) in _float_calls(device).items():
        with pytest.raises(RuntimeError, match="no gradient"):
            call(t.detach().clone().requires_grad_())
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.detach(), torch.ones_like(t))
            with pytest.raises(RuntimeError, match="without tangents"):
                call(dual)
            with torch.no_grad(), pytest.raises(RuntimeError, match="without tangents"):
                call(dual)
            call(t)
        with torch.no_grad():
            call(t.detach().clone().requires_grad_())


def test_transforms_and_compile_refuse_derivatives():
    for name, (call, t) in _float_calls("cpu").items():
        with pytest.raises(RuntimeError, match="no gradient"):
            torch.func.vjp(call, t)
        with pytest.raises(RuntimeError, match="no gradient"):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
        leaf = t.detach().clone().requires_grad_()
        run = torch.compile(lambda v, call=call: call(v) * 2, backend="aot_eager")
        with pytest.raises(RuntimeError, match="no gradient"):
            run(leaf)
        with torch.no_grad():
            assert torch.equal(run(leaf), call(t) * 2)


# ---- devices, layouts and fakes ------------------------------------------------

@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("shape", [(1, 130), (1, 15), (1, 256), (3, 130), (2, 3, 40)])
def test_results_stay_on_the_device_in_padded_rows(shape, device):
    x, w = rand(shape, 33).to(device), rand(shape[-1:], 34).to(device)
    gu = rand((*shape[:-1], 2 * shape[-1]), 35).to(device)
    for q, s, *h in (ops.quantize_fp8(x), ops.rms_norm_fp8(x, w, 1e-5),
                     ops.add_rms_norm_fp8(x, x, w, 1e-5), ops.silu_mul_fp8(gu)):
        pitch = -(-shape[-1] // 16) * 16
        rows = math.prod(shape[:-1])
        strides = (shape[1] * pitch, pitch, 1) if len(shape) == 3 else (pitch, 1)
        assert all(t.device.type == device for t in (q, s, *h))
        assert q.stride() == strides
        # (of one row's scales the row stride says nothing)
        assert s.stride()[-2:] == (1, rows) or rows == 1 and s.stride(-1) == 1
        assert q.shape == shape and s.shape == (*shape[:-1], -(-shape[-1] // 128))
    if len(shape) == 2:
        q, s = ops.quantize_fp8(x, 128)
        assert q.device.type == s.device.type == device and q.stride() == (pitch, 1)
        assert s.is_contiguous() and s.shape == (1, -(-shape[1] // 128))


def test_fakes_of_products_and_weights_match():
    from torch._subclasses.fake_tensor import FakeTensorMode

    def meta(*tensors):
        return [(t.shape, t.dtype, t.stride(), t.device) for t in tensors]

    for m, n, k in ((5, 130, 384), (1, 7, 100), (0, 16, 64), (4, 3, 0)):
        x, w = rand((m, k), 36), rand((n, k), 37)
        lead = (1, m, k)
        bias = rand((n,), 38, 1.0, torch.float16)

        def results(x, w, bias):
            q, s = ops.quantize_fp8(x.view(lead))
            wq, ws = ops.quantize_fp8(w, 128)
            y = ops.mm_fp8(q, s, wq, ws, torch.float16, bias)
            return meta(q, s, wq, ws, y, ops.mm_fp8(q[0], s[0], wq, ws, torch.bfloat16))

        real = results(x, w, bias)
        with FakeTensorMode() as mode:
            assert results(*(mode.from_tensor(t) for t in (x, w, bias))) == real


@pytest.mark.gpu
def test_operands_on_another_device_than_the_current_one():
    """Strided operands are copied first, on their own device too."""
    if torch.spyre.device_count() < 2:
        pytest.skip("needs two GPUs")
    x, w = rand((40, 512), 39), rand((130, 256), 40)
    q, s = ops.quantize_fp8(x[:, ::2])
    wq, ws = ops.quantize_fp8(w, 128)
    assert torch.spyre.current_device() == 0
    x1, w1 = x.to("spyre:1"), w.to("spyre:1")
    q1, s1 = ops.quantize_fp8(x1[:, ::2])
    w1q, w1s = ops.quantize_fp8(w1, 128)
    assert torch.equal(codes64(q1), codes64(q)) and torch.equal(s1.cpu(), s)
    y = ops.mm_fp8(q1, s1, w1q, w1s, torch.float16)
    assert y.device.index == 1 and torch.spyre.current_device() == 0
    want, mags = mm64(q, s, wq, ws), mm64(q, s, wq, ws, mags=True)
    assert bool(((y.cpu().double() - want).abs() <= mags * 2.0 ** -12 + want.abs() * 2.0 ** -10).all())

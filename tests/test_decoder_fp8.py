"""The decoder with 8-bit projections (examples.decoder.quantize_params): its
operators one after another as prefill and decode run them, eagerly, compiled
and in a captured graph.

Tolerances (relative 2-norms).  A code is off its value by at most 2^-4, 2^-4 /
sqrt(3) in the mean square at worst, so a product of codes on both sides is off
by about 5 % of its own size; the two layers' eight products and the head add
up in squares to 15 %, with the residual stream's share of earlier ones less
than 20 %: the bound against the 16-bit model is 25 %.

Two runs of the 8-bit model that round differently anywhere do not stay
together: a difference d turns over the codes that lie that near to a border, d /
2^-3 of them, each by a step of 2^-3, and leaves sqrt(d 2^-3).  From one fp16
rounding, d = 2^-11, that is 2^-7, then 2^-5, 2^-4: it grows until it is the
codes' own error in both runs, 5 % sqrt(2) a product, sqrt(9) times that over
all: 21 %.  (On the CPU alone, 2^-12 of noise on the embedding moves the logits
by 8 %.)  So whole runs are held to 25 % of each other too, and the operators
to their own roundings stage by stage.
"""

import pytest
import torch

import torch_spyre  # noqa: F401
from torch_spyre.examples import decoder as D

CFG = D.DecoderConfig(hidden=512, n_heads=4, n_kv_heads=2, head_dim=128, intermediate=640,
                      vocab=515, n_layers=2)
BOUND = 0.25


def _params(dtype=torch.float16):
    return D.init_params(CFG, "cpu", dtype=dtype, seed=11, std=0.05)


def _to(v, device):
    if isinstance(v, torch.Tensor):
        return v.to(device)
    if isinstance(v, dict):
        return {k: _to(x, device) for k, x in v.items()}
    return type(v)(_to(x, device) for x in v)


def _tokens(b, s, seed=3):
    return torch.randint(0, CFG.vocab, (b, s), generator=torch.Generator().manual_seed(seed))


def _rel(a, b):
    a, b = a.cpu().double(), b.cpu().double()
    return float((a - b).norm() / b.norm())


def _flow(params, device, b=2, s=9, steps=3, **kw):
    p = _to(params, device)
    teacher = _tokens(b, steps, 4).to(device)
    with torch.no_grad():
        return D.generate(_tokens(b, s).to(device), p, CFG, steps, device, teacher=teacher, **kw)[1]


def test_weights_are_half_the_bytes():
    p = _params()
    q = D.quantize_params(p)
    for w, w8 in zip(p["layers"], q["layers"]):
        assert set(w8) == {"attn_norm", "mlp_norm", "wqkv_fp8", "wo_fp8", "wgu_fp8", "wd_fp8"}
        for name in ("wqkv", "wo", "wgu", "wd"):
            codes, scales = w8[name + "_fp8"]
            assert codes.dtype == torch.float8_e4m3fn and codes.shape == w[name].shape
            assert scales.shape == tuple(-(-n // 128) for n in w[name].shape)
    # layers that hold their projections apart give the same codes
    apart = {"wq": None, "wk": None, "wv": None, "wg": None, "wu": None}
    split = dict(p, layers=[{k: v for k, v in w.items() if k not in ("wqkv", "wgu")}
                            for w in p["layers"]])
    assert set(apart) <= set(split["layers"][0])
    again = D.quantize_params(split)
    assert torch.equal(again["layers"][1]["wqkv_fp8"][0].view(torch.uint8),
                       q["layers"][1]["wqkv_fp8"][0].view(torch.uint8))


def test_cpu_flow_against_the_16_bit_model_and_itself():
    p = _params(torch.bfloat16)
    q = D.quantize_params(p)
    plain, eight = _flow(p, "cpu"), _flow(q, "cpu")
    assert _rel(eight, plain) < BOUND
    assert _rel(_flow(q, "cpu", decode_fn=D.decode_step_static), eight) < BOUND


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_flow_on_the_device(dtype):
    p = _params(dtype)
    q = D.quantize_params(p)
    plain, want = _flow(p, "cpu"), _flow(q, "cpu")
    got = _flow(q, "spyre")
    static = _flow(q, "spyre", decode_fn=D.decode_step_static)
    for run in (got, static):
        assert _rel(run, plain) < BOUND and _rel(run, want) < BOUND
    graph = _flow(q, "spyre", decode_fn=D.decode_step_static, use_graph=True)
    assert torch.equal(graph.cpu(), static.cpu())


@pytest.mark.gpu
def test_quantized_on_the_device_are_the_same_weights():
    p = _params()
    a, b = D.quantize_params(p), D.quantize_params(_to(p, "spyre"))
    for x, y in zip(a["layers"], b["layers"]):
        for name in ("wqkv_fp8", "wo_fp8", "wgu_fp8", "wd_fp8"):
            assert torch.equal(x[name][0].view(torch.uint8), y[name][0].cpu().view(torch.uint8))
            assert torch.equal(x[name][1], y[name][1].cpu())


@pytest.mark.gpu
def test_layer_stage_by_stage():
    """Every operator of a layer on what the one before it left on the device,
    against its formula on the same inputs."""
    ops, dt = torch.ops.spyre, torch.float16
    w = _to(D.quantize_params(_params()), "spyre")["layers"][0]
    g = torch.Generator().manual_seed(6)
    h = torch.randn(3, 37, CFG.hidden, generator=g).half().to("spyre")
    a = torch.randn(111, 512, generator=g).half().to("spyre")

    def both(call, *args):
        got = call(*args)
        want = call(*(t.cpu() if isinstance(t, torch.Tensor) else t for t in args))
        if isinstance(got, torch.Tensor):
            got, want = (got,), (want,)
        for x, y in zip(got, want):
            assert x.shape == y.shape and x.dtype == y.dtype and x.stride() == y.stride()
            if x.dtype == torch.float8_e4m3fn:  # a step of the code at most, and rarely
                x, y = x.cpu().float(), y.float()
                off = (x - y).abs()
                assert bool((off <= torch.clamp(y.abs() * 0.125, min=2.0 ** -9)).all())
                assert int((off > 0).sum()) <= 1 + x.numel() // 1000
            else:  # fp32 scales of a norm: 2^-16; fp16 sums in other orders: two steps
                assert _rel(x, y) < (2.0 ** -16 if x.dtype == torch.float32 else 2.0 ** -9)
        return got if len(got) > 1 else got[0]

    x = both(ops.rms_norm_fp8, h, w["attn_norm"], CFG.eps)
    qkv = both(ops.mm_fp8, *x, *w["wqkv_fp8"], dt)
    assert qkv.shape == (3, 37, 1024)
    o = both(ops.mm_fp8, *both(ops.quantize_fp8, a, 1), *w["wo_fp8"], dt).view(h.shape)
    xq, xs, h = both(ops.add_rms_norm_fp8, o, h, w["mlp_norm"], CFG.eps)
    gu = both(ops.mm_fp8, xq, xs, *w["wgu_fp8"], dt)
    both(ops.mm_fp8, *both(ops.silu_mul_fp8, gu), *w["wd_fp8"], dt)


@pytest.mark.gpu
def test_compiled_flow():
    q = D.quantize_params(_params())
    want = _flow(q, "spyre", decode_fn=D.decode_step_static)
    layer = torch.compile(D.layer_forward, dynamic=False)
    step = torch.compile(D.decode_step_static, dynamic=False)
    got = _flow(q, "spyre", layer_fn=layer, decode_fn=step)
    assert _rel(got, want) < BOUND
    graph = _flow(q, "spyre", layer_fn=layer, decode_fn=step, use_graph=True)
    assert torch.equal(graph.cpu(), got.cpu())


@pytest.mark.gpu
def test_graph_replays_with_new_inputs_and_eager_work_between():
    """One captured run of the operators, split product among them, replayed on
    changing inputs with eager calls of the same shapes and synchronisations
    between, against eager results; two graphs of the same work at once."""
    ops = torch.ops.spyre
    k, n, m = 4096, 512, 40
    w = ops.quantize_fp8((torch.randn(n, k, generator=torch.Generator().manual_seed(1)) * 0.05)
                         .half().to("spyre"), 128)
    norm = torch.ones(k, dtype=torch.float16, device="spyre")
    x, r = (torch.zeros(m, k, dtype=torch.float16, device="spyre") for _ in range(2))

    def work():
        q, s, h = ops.add_rms_norm_fp8(x, r, norm, 1e-5)
        y = ops.mm_fp8(q, s, *w, torch.float16)
        return h, y, ops.mm_fp8(*ops.silu_mul_fp8(torch.cat([h, h], 1)), *w, torch.float16)

    work()
    graphs = [torch.spyre.SpyreGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.spyre.graph(g):
            outs.append(work())
    for t in range(4):
        gen = torch.Generator().manual_seed(20 + t)
        x.copy_(torch.randn(m, k, generator=gen).half())
        r.copy_(torch.randn(m, k, generator=gen).half())
        for g in graphs:
            g.replay()
        eager = work()
        if t % 2:
            torch.spyre.synchronize()
        for out in outs:
            for a, b in zip(out, eager):
                assert torch.equal(a.cpu(), b.cpu())
    for g in graphs:
        g.reset()

"""The decoder over a paged cache (examples.decoder.step_paged and what is built on it):
prompts of different lengths, decoded and drafted tokens, sampling, 8-bit weights,
compiled and captured steps.

Tolerances.  Two runs of the model that differ in the order of sums differ by roundings of
2^-11 (fp16): a layer rounds its norms, projections, attention and sums some 12 times,
two layers and the head 26 times, and roundings of different places add up at worst:
26 / 2048 = 1.3 % of the logits' norm, with the scores that the op-by-op chain rounds
too less than 2 %.  8-bit weights: 25 %, as derived in test_decoder_fp8.py.
"""

import pytest
import torch

import torch_spyre  # noqa: F401
from torch_spyre.examples import decoder as D

CFG = D.DecoderConfig(hidden=512, n_heads=4, n_kv_heads=2, head_dim=128, intermediate=640,
                      vocab=515, n_layers=2)
DEVICES = ["cpu", pytest.param("spyre", marks=pytest.mark.gpu)]
BOUND = 0.02


def _params(seed=11):
    return D.init_params(CFG, "cpu", dtype=torch.float16, seed=seed, std=0.05)


def _to(v, device):
    if isinstance(v, torch.Tensor):
        return v.to(device)
    if isinstance(v, dict):
        return {k: _to(x, device) for k, x in v.items()}
    return type(v)(_to(x, device) for x in v)


def _tokens(*shape, seed=3):
    return torch.randint(0, CFG.vocab, shape, generator=torch.Generator().manual_seed(seed))


def _rel(a, b):
    a, b = a.cpu().double(), b.cpu().double()
    return float((a - b).norm() / b.norm())


PROMPTS = [_tokens(n, seed=n) for n in (9, 1, 30, 17)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("page_size", [16, 5])
def test_equal_prompts_as_with_the_contiguous_cache(page_size, device):
    p = _params()
    prompt, teacher = _tokens(3, 21), _tokens(3, 4, seed=4)
    want = D.generate(prompt, p, CFG, 4, "cpu", teacher=teacher)[1]
    with torch.no_grad():
        got = D.generate_paged(list(prompt), _to(p, device), CFG, 4, device, page_size,
                               teacher=teacher.to(device))[1]
    assert _rel(got, want) < BOUND


@pytest.mark.parametrize("device", DEVICES)
def test_ragged_prompts_as_one_by_one(device):
    p = _to(_params(), device)
    teacher = _tokens(4, 3, seed=5)
    got = D.generate_paged(PROMPTS, p, CFG, 3, device, teacher=teacher.to(device))[1].cpu()
    for b, prompt in enumerate(PROMPTS):
        one = D.generate_paged([prompt], p, CFG, 3, device, 64, teacher=teacher[b:b + 1].to(device))
        assert _rel(got[:, b], one[1][:, 0]) < BOUND


@pytest.mark.parametrize("device", DEVICES)
def test_drafted_trees_as_their_paths(device):
    """Logits of a tree's nodes equal those of decoding each path on its own."""
    p = _to(_params(), device)
    plan = D.PagedPlan([40, 40], 16)
    cos, sin = D.rope_tables(CFG, 64, device, torch.float32)
    tokens = [_tokens(7, seed=20).tolist(), _tokens(3, seed=21).tolist()]
    parents = [[-1, 0, 0, 1, 1, 2, 5], [-1, 0, 1]]
    prompts = [PROMPTS[0], PROMPTS[3]]
    cache = D.new_paged_cache(CFG, plan.pages, 16, device)
    lens = [len(x) for x in prompts]

    def dev(x):
        return torch.as_tensor(x).to(device)

    starts = torch.tensor([0] + lens).cumsum(0)
    D.step_paged(dev(torch.cat(prompts)), dev(torch.cat([torch.arange(n) for n in lens])),
                 dev(torch.cat([plan.slots(b, 0, n) for b, n in enumerate(lens)])),
                 dev(plan.table), dev(lens), dev(starts), p, cos, sin, cache, CFG)
    depth = [[0, 1, 1, 2, 2, 2, 3], [0, 1, 2]]
    mask = torch.zeros(11, 7, dtype=torch.bool)  # (the last row is padding)
    mask[:7] = D.tree_mask(parents[0])
    mask[7:10, :3] = D.tree_mask(parents[1])
    got = D.step_paged(dev(tokens[0] + tokens[1] + [0]),
                       dev([lens[0] + d for d in depth[0]] + [lens[1] + d for d in depth[1]] + [-7]),
                       dev(torch.cat([plan.slots(0, lens[0], 7), plan.slots(1, lens[1], 3),
                                      torch.tensor([-1])])),
                       dev(plan.table), dev([lens[0] + 7, lens[1] + 3]), dev([0, 7, 10]), p, cos,
                       sin, cache, CFG, dev(mask)).cpu()
    assert got.shape == (11, CFG.vocab) and bool(got.isfinite().all())
    row = 0
    for b in range(2):
        for i in range(len(tokens[b])):
            path, j = [], i
            while j >= 0:
                path.insert(0, tokens[b][j])
                j = parents[b][j]
            alone = D.generate_paged([torch.cat([prompts[b], torch.tensor(path)])], p, CFG, 0,
                                     device)[1][0, 0]
            assert _rel(got[row], alone) < BOUND, (b, i)
            row += 1


def test_speculation_gives_the_greedy_tokens():
    p, steps = _params(), 10
    want = D.generate_paged([PROMPTS[0]], p, CFG, steps, "cpu")[0][0].tolist()
    n = len(PROMPTS[0])

    def good(seq):  # the right tokens among wrong ones, as second children
        at = len(seq) - n
        right = want[at:at + 3]
        tokens, parents, last = [], [], -1
        for t in right:
            tokens += [(t + 1) % CFG.vocab, t]
            parents += [last, last]
            last = len(tokens) - 1
        return tokens, parents

    for draft, most in ((good, 3), (lambda s: ([], []), steps), (lambda s: ([1, 2], [-1, 0]), steps)):
        got, rounds = D.generate_speculative(PROMPTS[0], p, CFG, steps, "cpu", draft)
        assert got.tolist() == want and rounds <= most


@pytest.mark.gpu
def test_speculation_on_the_device():
    p = _to(_params(), "spyre")
    calls = []

    def draft(seq):
        calls.append(len(seq))
        return _tokens(9, seed=len(seq)).tolist(), [-1, -1, 0, 0, 1, 2, 2, 5, 7]

    got, rounds = D.generate_speculative(PROMPTS[0], p, CFG, 6, "spyre", draft)
    assert got.shape == (6,) and rounds == len(calls) >= 1
    assert bool(((got >= 0) & (got < CFG.vocab)).all())


@pytest.mark.parametrize("device", DEVICES)
def test_norms_of_heads(device):
    p = _params()
    g = torch.Generator().manual_seed(1)
    for w in p["layers"]:
        w["q_norm"] = (1 + 0.2 * torch.randn(128, generator=g)).half()
        w["k_norm"] = (1 + 0.2 * torch.randn(128, generator=g)).half()
    want = D.generate_paged(PROMPTS, p, CFG, 0, "cpu")[1]
    got = D.generate_paged(PROMPTS, _to(p, device), CFG, 0, device)[1]
    plain = D.generate_paged(PROMPTS, _params(), CFG, 0, "cpu")[1]
    assert _rel(got, want) < BOUND < _rel(plain, want)


@pytest.mark.parametrize("device", DEVICES)
def test_8_bit_weights(device):
    p = _params()
    want = D.generate_paged(PROMPTS, p, CFG, 2, "cpu", teacher=_tokens(4, 2))[1]
    with torch.no_grad():
        got = D.generate_paged(PROMPTS, _to(D.quantize_params(p), device), CFG, 2, device,
                               teacher=_tokens(4, 2).to(device))[1]
    assert _rel(got, want) < 0.25


@pytest.mark.parametrize("device", DEVICES)
def test_sampled_tokens_are_those_of_their_logits(device):
    g = torch.Generator().manual_seed(8)
    u = torch.rand(5, 4, generator=g)
    how = dict(temperature=torch.tensor([0.7, 1.0, 0.0, 1.5]), top_k=torch.tensor([40, 0, 3, 7]),
               top_p=torch.tensor([0.9, 0.8, 1.0, 0.95]), min_p=torch.tensor([0.0, 0.05, 0.0, 0.1]))
    tokens, logits = D.generate_paged(PROMPTS, _to(_params(), device), CFG, 5, device, uniform=u, **how)
    for t in range(5):
        want = torch.ops.spyre.sample(logits[t].cpu(), u[t], *how.values())
        assert torch.equal(tokens[:, t].cpu(), want)
    assert tokens[2].tolist() == logits[:5, 2].cpu().float().argmax(1).tolist()


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [False, True])
def test_captured_steps_equal_eager_ones(compiled):
    p = _to(_params(), "spyre")
    torch._dynamo.reset()
    step = torch.compile(D.step_paged) if compiled else None
    g = torch.Generator().manual_seed(9)
    how = dict(uniform=torch.rand(7, 4, generator=g), temperature=torch.full((4,), 0.8),
               top_k=torch.full((4,), 20), top_p=torch.full((4,), 0.9))
    with torch.no_grad():
        eager = D.generate_paged(PROMPTS, p, CFG, 7, "spyre", step_fn=step, **how)
        graph = D.generate_paged(PROMPTS, p, CFG, 7, "spyre", step_fn=step, use_graph=True, **how)
    assert torch.equal(eager[0].cpu(), graph[0].cpu())
    assert torch.equal(eager[1].cpu(), graph[1].cpu())


@pytest.mark.gpu
def test_compiled_steps_are_near_eager_ones():
    p = _to(_params(), "spyre")
    torch._dynamo.reset()
    teacher = _tokens(4, 3, seed=5).to("spyre")
    with torch.no_grad():
        a = D.generate_paged(PROMPTS, p, CFG, 3, "spyre", teacher=teacher)[1]
        b = D.generate_paged(PROMPTS, p, CFG, 3, "spyre", teacher=teacher,
                             step_fn=torch.compile(D.step_paged))[1]
    assert _rel(b, a) < BOUND


@pytest.mark.gpu
def test_two_graphs_of_one_cache():
    """Two captured calls with workspaces of their own over the same caches, replayed in
    turn with other lengths, tables and eager work between them."""
    ops = torch.ops.spyre
    g = torch.Generator().manual_seed(10)
    kc, vc = (torch.randn(60, 2, 16, 128, generator=g).half().to("spyre") for _ in range(2))
    table = torch.randperm(60, generator=g).view(4, 15).to("spyre")
    q = [torch.randn(n, 8, 128, generator=g).half().to("spyre") for n in (4, 40)]
    lens = [torch.tensor([240, 3, 100, 17]).to("spyre"), torch.tensor([30, 240, 11, 90]).to("spyre")]
    starts = [torch.tensor([0, 1, 2, 3, 4]).to("spyre"), torch.tensor([0, 10, 20, 30, 40]).to("spyre")]

    def call(i):
        return ops.paged_attention(q[i], kc, vc, table, lens[i], starts[i], 0.1)

    for i in (0, 1):
        call(i)
    torch.spyre.synchronize()
    graphs, outs = [], []
    for i in (0, 1):
        graphs.append(torch.spyre.SpyreGraph())
        with torch.spyre.graph(graphs[i]):
            outs.append(call(i))
    for r in range(5):
        lens[0].copy_(torch.tensor([[240, 3, 100, 17], [1, 240, 16, 200], [64, 65, 128, 129],
                                    [1, 1, 1, 1], [239, 240, 238, 17]][r]).to("spyre"))
        lens[1].copy_(torch.tensor([30 + r, 240 - r, 11 + 7 * r, 90]).to("spyre"))
        table.copy_(torch.randperm(60, generator=g).view(4, 15).to("spyre"))
        for i in ((0, 1), (1, 0))[r % 2]:
            graphs[i].replay()
        torch.spyre.synchronize()
        junk = [torch.full((64, 200), 7.0, device="spyre") for _ in range(3)]
        for i in (0, 1):
            assert torch.equal(outs[i].cpu(), call(i).cpu()), (r, i)
        del junk
    for x in graphs:
        x.reset()


def test_plan_gives_no_slots_of_other_sequences():
    plan = D.PagedPlan([40, 5, 0], 16)
    assert plan.pages == 4 and plan.room == [48, 16, 0]
    mine = [plan.slots(b, 0, n).tolist() for b, n in enumerate(plan.room)]
    assert sorted(sum(mine, [])) == list(range(64))
    assert plan.slots(1, 16, 0).numel() == 0
    for b, first, n in ((0, 0, 49), (0, 48, 1), (1, 16, 1), (1, 7, 10), (2, 0, 1), (0, -1, 2)):
        with pytest.raises(IndexError):
            plan.slots(b, first, n)


def test_prompts_have_a_token():
    """An empty prompt has no last row to go on from (the one before it is another's)."""
    p, none = _params(), torch.zeros(0, dtype=torch.int64)
    for prompts in ([none], [PROMPTS[0], none], [none, PROMPTS[0]]):
        with pytest.raises(ValueError, match="at least one token"):
            D.generate_paged(prompts, p, CFG, 2, "cpu")
    with pytest.raises(ValueError, match="at least one token"):
        D.generate_speculative(none, p, CFG, 2, "cpu", lambda s: ([], []))


@pytest.mark.parametrize("name", ["q_norm", "k_norm"])
@pytest.mark.parametrize("eight_bit", [False, True])
def test_norms_of_heads_are_refused_over_the_contiguous_cache(name, eight_bit):
    """Left out there, they would give another model's logits."""
    p = _params()
    p["layers"][1][name] = torch.full((128,), 2.0, dtype=torch.float16)
    if eight_bit:
        p = D.quantize_params(p)
    with pytest.raises(ValueError, match="step_paged"):
        D.generate(_tokens(2, 5), p, CFG, 2, "cpu")
    cos, sin = D.rope_tables(CFG, 8, "cpu")
    for step in (D.decode_step, D.decode_step_static):
        at = 3 if step is D.decode_step else torch.tensor([3])
        with pytest.raises(ValueError, match="step_paged"):
            step(_tokens(2), at, p, cos, sin, D.new_cache(CFG, 2, 8, "cpu"), CFG)


def _second_children(want, n, vocab):
    """A draft that names up to three of the tokens `want`, which follow the prompt's n, each
    behind a wrong one: the accepted nodes are never the first ones of their tree."""
    def draft(seq):
        tokens, parents, last = [], [], -1
        for t in want[len(seq) - n:len(seq) - n + 3]:
            tokens += [(t + 1) % vocab, t]
            parents += [last, last]
            last = len(tokens) - 1
        return tokens, parents
    return draft


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("page_size", [16, 5])
def test_speculation_moves_accepted_nodes(page_size, device, monkeypatch):
    """Tokens, and keys and values in the cache, are those of decoding one by one.  (This
    prompt's two largest logits are 0.14 apart at every step, six times 2 % of the logits' root
    mean square.)"""
    caches, make = [], D.new_paged_cache
    monkeypatch.setattr(D, "new_paged_cache",
                        lambda *a, **kw: caches.append(make(*a, **kw)) or caches[-1])
    p, prompt, steps = _to(_params(), device), _tokens(20, seed=111), 10
    n = len(prompt)
    want = D.generate_paged([prompt], p, CFG, steps, device, page_size)[0][0].tolist()
    got, rounds = D.generate_speculative(prompt, p, CFG, steps, device,
                                         _second_children(want, n, CFG.vocab), page_size)
    assert got.tolist() == want and rounds == 3  # (one token, then four a round)
    for one, tree in zip(*caches):
        for a, b in zip(one, tree):
            a, b = (x.cpu().transpose(1, 2).reshape(-1, 2, 128)[:n + steps - 1].double()
                    for x in (a, b))
            assert bool(((a - b).norm(dim=(1, 2)) < BOUND * a.norm(dim=(1, 2))).all())


def test_speculation_copies_no_cache():
    """Moving a few rows takes no tensor of a whole cache's size."""
    from torch.utils._python_dispatch import TorchDispatchMode

    large = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            out = func(*args, **(kwargs or {}))
            new = all(r.alias_info is None for r in func._schema.returns)
            if new and isinstance(out, torch.Tensor) and out.numel() >= 2000 * 256:
                large.append(str(func))
            return out

    p, prompt, steps = _params(), _tokens(20, seed=111), 10
    want = D.generate_paged([prompt], p, CFG, steps, "cpu")[0][0].tolist()
    with Watch():
        got, _ = D.generate_speculative(prompt, p, CFG, steps, "cpu",
                                        _second_children(want, 20, CFG.vocab), most=2000)
    assert got.tolist() == want
    assert large == ["aten.zeros.default"] * (2 * CFG.n_layers), large


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("compiled", [False, pytest.param(True, marks=pytest.mark.gpu)])
@pytest.mark.parametrize("eight_bit", [False, True])
def test_logits_of_some_rows(eight_bit, compiled, device, monkeypatch):
    """step_paged's `rows` gives the logits that all rows' would hold there, from an LM head
    of those rows alone."""
    if compiled and device == "cpu":
        pytest.skip("compiled for spyre")
    p = D.quantize_params(_params()) if eight_bit else _params()
    p, heads, head = _to(p, device), [], D.lm_logits
    if not compiled:
        monkeypatch.setattr(D, "lm_logits", lambda h, p, c, x=None: heads.append(
            (h if x is None else x[0]).shape[0]) or head(h, p, c, x))
    torch._dynamo.reset()
    step = torch.compile(D.step_paged) if compiled else D.step_paged
    plan, n = D.PagedPlan([30], 16), 30
    cos, sin = D.rope_tables(CFG, n, device, torch.float32)
    at = torch.arange(n)

    def call(rows):
        cache = D.new_paged_cache(CFG, plan.pages, 16, device)
        with torch.no_grad():
            return step(PROMPTS[2].to(device), at.to(device), plan.slots(0, 0, n).to(device),
                        plan.table.to(device), torch.tensor([n]).to(device),
                        torch.tensor([0, n]).to(device), p, cos, sin, cache, CFG, None,
                        None if rows is None else rows.to(device)).cpu()

    rows = torch.tensor([29, 3, 3, 0])
    some, every = call(rows), call(None)
    assert some.shape == (4, CFG.vocab) and every.shape == (n, CFG.vocab)
    assert _rel(some, every[rows]) < BOUND
    assert compiled or heads == [4, n]

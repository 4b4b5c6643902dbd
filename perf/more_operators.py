"""Serving a batch from a paged cache, as cases that can be timed.

Several sequences share one cache of pages; a step brings each of them some new
tokens (one decoded token, the tree of drafted tokens of speculative decoding, or
a piece of a prompt) and ends in drawing the tokens that follow.  The operators
are

  paged_append     the step's projection rows [T, (H + 2 Hkv) D] (queries, keys,
                   values): an RMSNorm of every query and key head (optional),
                   the position rotation, keys and values written to their slots
                   of the paged cache; returns the queries
  paged_attention  attention of the new tokens over their sequences' pages:
                   everything committed before the step, and of the step's own
                   tokens those that a tree mask allows (without one: causal)
  sample           tokens drawn from logits with temperature, top-k, top-p and
                   min-p, from random numbers that are given

Sizes are those of the repository's decoder (32 query heads on 8 key / value
heads of 128, 1024-token prompts with 128 decoded tokens, a vocabulary of 49155)
and generic ones around them.  The framework serves (it registers no gradients of
these), so the directions are prompts, drafts and decoded tokens.
"""

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
VOCAB = 49155


def listed():
    return [
        # one decoded token of one sequence: launch latency
        _append("append_1", 1, 32, 8, 128, 16, "bf16"),
        # a decode batch of 24 drafting 5 tokens each, heads normalised
        _append("append_120_norm", 120, 32, 8, 128, 16, "fp16", norm=True),
        # three prompts of 777 tokens; rotation tables in fp32, heads normalised
        _append("append_2331_norm", 2331, 32, 8, 128, 64, "bf16", norm=True, tables="fp32"),
        # long prompts, cache laid out page by token by head
        _append("append_8192", 8192, 32, 8, 128, 32, "fp16", layout="token"),
        # decoding 4 sequences of a 1024-token prompt, 128 tokens on at most
        _attend("decode_4x1152", 4, 1, 1, 1025, 1152, 32, 8, 128, 16, "fp16"),
        # decoding a full batch of sequences of very different lengths
        _attend("decode_64_ragged", 64, 1, 1, 37, 4000, 32, 8, 128, 16, "bf16"),
        # one long document, a tree of 16 drafts
        _attend("tree16_1x131072", 1, 16, 16, 131072, 131072, 32, 8, 128, 64, "bf16", tree=True),
        # eight sequences, trees of up to 48 drafts
        _attend("tree48_8x6000", 8, 30, 48, 1500, 6000, 32, 8, 128, 16, "fp16", tree=True),
        # three prompts' 777-token pieces behind 2048 cached tokens each
        _attend("chunk777_3x2825", 3, 777, 777, 2825, 2825, 32, 8, 128, 32, "bf16"),
        # one decoded token with every filter: latency
        _draws("sample_1_all", 1, VOCAB, "bf16", temperature=0.8, top_k=50, top_p=0.95, min_p=0.02),
        # a decode batch, nucleus sampling over the whole vocabulary
        _draws("sample_24_top_p", 24, VOCAB, "fp16", temperature=1.0, top_p=0.9),
        # a large batch and vocabulary in fp32, temperature alone; a quarter of the rows greedy
        _draws("sample_256_plain", 256, 131072, "fp32", temperature=0.9, greedy=True),
    ]


def _append(name, tokens, heads, kv, dim, page, dtype, norm=False, tables="same", layout="head"):
    return {"name": name, "kind": "append", "tokens": tokens, "heads": heads, "kv": kv, "dim": dim,
            "page": page, "dtype": dtype, "norm": norm, "tables": tables, "layout": layout}


def _attend(name, batch, new_lo, new_hi, len_lo, len_hi, heads, kv, dim, page, dtype, tree=False,
            layout="head", pad=0):
    return {"name": name, "kind": "attend", "batch": batch, "new_lo": new_lo, "new_hi": new_hi,
            "len_lo": len_lo, "len_hi": len_hi, "heads": heads, "kv": kv, "dim": dim, "page": page,
            "dtype": dtype, "tree": tree, "layout": layout, "pad": pad}


def _draws(name, rows, vocab, dtype, temperature=0.0, top_k=0, top_p=0.0, min_p=0.0, greedy=False,
           banned=False):
    return {"name": name, "kind": "sample", "rows": rows, "vocab": vocab, "dtype": dtype,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "greedy": greedy, "banned": banned}


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8), (32, 8), (16, 16), (8, 1), (40, 8), (28, 4), (12, 2)]
PAGES = [16, 16, 32, 64, 128, 256, 48, 5, 1]


def draw(rng):
    kind = rng.choice(["append", "append", "attend", "attend", "attend", "sample", "sample"])
    dtype, dim = rng.choice(["fp16", "bf16"]), rng.choice([128, 128, 64])
    (heads, kv), page = rng.choice(HEADS), rng.choice(PAGES)
    layout = rng.choice(["head", "head", "token"])
    if kind == "append":
        tokens = _log_int(rng, 1, 8192 * 48 * 128 // ((heads + 2 * kv) * dim))
        c = _append("", tokens, heads, kv, dim, page, dtype, rng.random() < 0.5,
                    rng.choice(["same", "fp32"]), layout)
    elif kind == "attend":
        form = rng.choice(["decode", "decode", "tree", "tree", "chunk"])
        new = 1 if form == "decode" else _log_int(rng, 2, 64) if form == "tree" else \
            _log_int(rng, 65, 777)
        # keys in all, and pairs of rows and keys, no more than the largest cases have
        longest = _log_int(rng, new, 32768)
        most = min((1 << 27) // (longest * kv * dim), 3 * 777 * 2400 * 32 // (new * longest * heads))
        batch = _log_int(rng, 1, max(1, min(256, most)))
        longest = min(longest, (1 << 27) // (batch * kv * dim),
                      3 * 777 * 2400 * 32 // (batch * new * heads))
        longest = max(longest, new)
        c = _attend("", batch, rng.randint(max(1, new // 2), new), new,
                    _log_int(rng, new, longest), longest, heads, kv, dim, page, dtype,
                    form == "tree", layout, rng.choice([0, 0, 0, 7]))
    else:
        vocab = rng.choice([VOCAB, 131072, _log_int(rng, 100, 200000)])
        rows = _log_int(rng, 1, min(256, 256 * 131072 // vocab))
        filters = {"top_k": rng.choice([0, 1, 20, 50, 1000]),
                   "top_p": rng.choice([0.0, 0.5, 0.9, 0.95, 0.99]),
                   "min_p": rng.choice([0.0, 0.0, 0.05, 0.1])}
        c = _draws("", rows, vocab, rng.choice([dtype, "fp32"]),
                   rng.choice([0.6, 0.8, 1.0, 1.0, 1.3]), greedy=rng.random() < 0.3,
                   banned=rng.random() < 0.3, **filters)
    del c["name"]
    return c


# ---- the plain forms --------------------------------------------------------

def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight.float()


def _rotate(x, cos, sin):
    """x [T, heads, D], cos / sin [T, D]: x cos + rot(x) sin, rot(x) = (-x2, x1)."""
    half = x.shape[-1] // 2
    rot = torch.cat([-x[..., half:], x[..., :half]], -1)
    return x * cos[:, None] + rot * sin[:, None]


def _plain_append(s):
    kc, vc = s["k_cache"], s["v_cache"]
    h, kv, d = s["heads"], kc.shape[1], kc.shape[3]
    x = s["qkv"].float().view(-1, h + 2 * kv, d)
    q, k = x[:, :h], x[:, h:h + kv]
    if "q_norm" in s:
        q, k = _rms(q, s["q_norm"]), _rms(k, s["k_norm"])
    cos, sin = s["cos"][s["positions"]].float(), s["sin"][s["positions"]].float()
    page, at = s["slots"] // kc.shape[2], s["slots"] % kc.shape[2]
    kc[page, :, at] = _rotate(k, cos, sin).to(kc.dtype)
    vc[page, :, at] = s["qkv"].view(-1, h + 2 * kv, d)[:, h + kv:]
    return _rotate(q, cos, sin).to(s["qkv"].dtype), kc, vc


def _plain_attend(s):
    q, kc, vc, table = s["q"], s["k_cache"], s["v_cache"], s["block_table"]
    (t, h, d), kv, page = q.shape, kc.shape[1], kc.shape[2]
    dev, b, n, length = q.device, table.shape[0], s["new_hi"], s["len_hi"]
    starts, lens = s["q_starts"], s["seq_lens"]
    new = starts[1:] - starts[:-1]
    # keys and values of every sequence side by side: [B, kv, L, D]
    at = torch.arange(length, device=dev)
    pages = table[:, at // page]
    k = kc[pages, :, at % page].float().transpose(1, 2)
    v = vc[pages, :, at % page].float().transpose(1, 2)
    # rows of every sequence, padded to the most new tokens: [B, kv, (H / kv) n, D]
    i = torch.arange(n, device=dev)
    live = i < new[:, None]
    rows = torch.where(live, starts[:-1, None] + i, 0)
    qs = q[rows].float().view(b, n, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    score = (qs @ k.transpose(2, 3)).mul_(s["scale"]).view(b, h, n, length)
    # what a row sees: committed keys, and of the step's own those the mask allows
    draft = at - (lens - new)[:, None]
    if "mask" in s:
        seen = torch.gather(s["mask"][rows], 2,
                            draft.clamp(0, s["mask"].shape[1] - 1)[:, None].expand(b, n, length))
    else:
        seen = draft[:, None] <= i[:, None]
    seen = ((draft < 0)[:, None] | seen) & (at < lens[:, None])[:, None]
    score.masked_fill_(~seen[:, None], float("-inf"))
    score -= score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = score.exp_()
    p /= p.sum(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).tiny)
    o = (p.view(b, kv, -1, length) @ v).view(b, h, n, d).transpose(1, 2)
    out = torch.zeros_like(q)
    out[rows[live]] = o[live].to(q.dtype)
    return out


def _plain_sample(s):
    l = s["logits"].double()
    r, v = l.shape
    t = s["temperature"].double()[:, None]
    top, order = l.sort(dim=-1, descending=True, stable=True)
    w = ((top - top[:, :1]) / t.clamp(min=torch.finfo(torch.float64).tiny)).exp()
    rank = torch.arange(v, device=l.device)
    keep = torch.ones_like(w, dtype=torch.bool)
    if "top_k" in s:
        k = s["top_k"][:, None]
        keep &= (rank < k) | (k <= 0)
    if "top_p" in s:
        kept = w * keep
        before = kept.cumsum(-1) - kept
        keep &= (before < s["top_p"].double()[:, None] * kept.sum(-1, keepdim=True)) | (rank == 0)
    if "min_p" in s:
        keep &= w >= s["min_p"].double()[:, None].clamp(max=1)
    mass = torch.zeros_like(w).scatter_(1, order, w * keep).cumsum(-1)
    token = (mass <= s["uniform"].double()[:, None] * mass[:, -1:]).sum(-1)
    return torch.where(t[:, 0] > 0, token, order[:, 0])


def _plain(s):
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[s["kind"]](s)


# ---- the framework's calls --------------------------------------------------

def _spyre():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "torch-spyre_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import torch_spyre  # noqa: F401  (registers the device and torch.ops.spyre)


def _framework(s):
    ops = torch.ops.spyre
    if s["kind"] == "append":
        q = ops.paged_append(s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"],
                             s["k_cache"], s["v_cache"], s["heads"], s.get("q_norm"),
                             s.get("k_norm"), EPS)
        return q, s["k_cache"], s["v_cache"]
    if s["kind"] == "attend":
        return ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"],
                                   s["seq_lens"], s["q_starts"], s["scale"], s.get("mask"))
    return ops.sample(s["logits"], s["uniform"], s["temperature"], s.get("top_k"), s.get("top_p"),
                      s.get("min_p"))


# ---- cases ------------------------------------------------------------------

def _lengths(case):
    """(new tokens, length) of every sequence: spread over the case's ranges, in
    an order of their own.  They belong to the case, not to the seed."""
    b, r = case["batch"], random.Random(case["batch"] * 1000003 + case["len_hi"])

    def spread(lo, hi):
        x = [hi if b == 1 else round(lo + (hi - lo) * i / (b - 1)) for i in range(b)]
        r.shuffle(x)
        return x

    new = spread(case["new_lo"], case["new_hi"])
    return new, [max(n, m) for n, m in zip(new, spread(case["len_lo"], case["len_hi"]))]


def _paged(g, case, pages):
    """A cache of `pages` pages [pages, kv, page, D] in the case's layout."""
    kv, page, d = case["kv"], case["page"], case["dim"]
    shape = (pages, page, kv, d) if case["layout"] == "token" else (pages, kv, page, d)
    x = torch.randn(shape, generator=g, device="cuda", dtype=DTYPES[case["dtype"]])
    return x.transpose(1, 2) if case["layout"] == "token" else x


def _inputs_append(case, g):
    t, h, kv, d, dt = (case[n] for n in ("tokens", "heads", "kv", "dim", "dtype"))
    dt = DTYPES[dt]
    pages = -(-t // case["page"]) + 3
    most = max(1152, t)
    inv = 1e4 ** (-torch.arange(0, d, 2, device="cuda").double() / d)
    angle = (torch.arange(most, device="cuda").double()[:, None] * inv).repeat(1, 2)
    tables = dt if case["tables"] == "same" else torch.float32
    s = {"qkv": torch.randn(t, (h + 2 * kv) * d, generator=g, device="cuda").to(dt),
         "cos": angle.cos().to(tables), "sin": angle.sin().to(tables),
         "positions": torch.randint(0, most, (t,), generator=g, device="cuda"),
         "slots": torch.randperm(pages * case["page"], generator=g, device="cuda")[:t],
         "k_cache": _paged(g, case, pages), "v_cache": _paged(g, case, pages)}
    if case["norm"]:
        s["q_norm"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
        s["k_norm"] = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(dt)
    return s


def _tree_mask(rng, new, width, pad):
    """Each draft sees itself and its ancestors: rows of [T, width]."""
    rows = []
    for n in new:
        m = torch.eye(n, width, dtype=torch.bool)
        for i in range(1, n):
            m[i] |= m[rng.randint(max(0, i - 6), i - 1)]
        rows.append(m)
    return torch.cat(rows + [torch.zeros(pad, width, dtype=torch.bool)])


def _inputs_attend(case, g, seed):
    new, lens = _lengths(case)
    d, page, dt = case["dim"], case["page"], DTYPES[case["dtype"]]
    need = [-(-n // page) for n in lens]
    pages, width = sum(need) + 2, max(need) + 1
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(int(seed))).tolist()
    table = torch.zeros(case["batch"], width, dtype=torch.int64)
    for row, n in zip(table, need):
        row[:n] = torch.tensor(free[:n])
        del free[:n]
    starts = torch.tensor([0] + new).cumsum(0)
    s = {"q": torch.randn(int(starts[-1]) + case["pad"], case["heads"], d, generator=g,
                          device="cuda").to(dt),
         "k_cache": _paged(g, case, pages), "v_cache": _paged(g, case, pages),
         "block_table": table.cuda(), "seq_lens": torch.tensor(lens).cuda(),
         "q_starts": starts.cuda()}
    if case["tree"]:
        s["mask"] = _tree_mask(random.Random(int(seed)), new, case["new_hi"], case["pad"]).cuda()
    return s


def _inputs_sample(case, g):
    r, v, dt = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    # logits as a model leaves them: a broad body and a few candidates that stand out
    l = torch.randn(r, v, generator=g, device="cuda") * 2
    l += 6 * torch.rand(r, v, generator=g, device="cuda") * (
        torch.rand(r, v, generator=g, device="cuda") < 20 / v)
    if case["banned"]:  # tokens that a grammar rules out
        l[torch.rand(r, v, generator=g, device="cuda") < 0.3] = float("-inf")

    def each(value, dtype=torch.float32):
        return torch.full((r,), value, dtype=dtype, device="cuda")

    s = {"logits": l.to(dt), "uniform": torch.rand(r, generator=g, device="cuda"),
         "temperature": each(case["temperature"])}
    if case["greedy"]:
        s["temperature"][::4] = 0
    if case["top_k"]:
        s["top_k"] = each(case["top_k"], torch.int64)
    if case["top_p"]:
        s["top_p"] = each(case["top_p"])
    if case["min_p"]:
        s["min_p"] = each(case["min_p"])
    return s


def _inputs(case, seed):
    """The case's inputs on the GPU, from the seed alone."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["kind"] == "append":
        return _inputs_append(case, g)
    return _inputs_attend(case, g, seed) if case["kind"] == "attend" else _inputs_sample(case, g)


def prepare(case, seed):
    # The same values by the same way through host memory for both sides; a
    # program that uses the framework holds its tensors on the "spyre" device.
    device = "cuda"
    if own:
        _spyre()
        device = "spyre"
    s = {}
    for name, t in _inputs(case, seed).items():
        if name.endswith("_cache") and case["layout"] == "token":
            s[name] = t.transpose(1, 2).cpu().to(device).transpose(1, 2)
        else:
            s[name] = t.cpu().to(device)
    s["kind"] = case["kind"]
    if case["kind"] == "append":
        s["heads"] = case["heads"]
    elif case["kind"] == "attend":
        s.update(scale=1 / math.sqrt(case["dim"]), new_hi=case["new_hi"],
                 len_hi=max(_lengths(case)[1]))
    return s


def run(s):
    return _framework(s) if own else _plain(s)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "append":
        t, d = case["tokens"], case["dim"]
        tables = 2 * d * (4 if case["tables"] == "fp32" else e)
        return {"bytes": t * (2 * e * (case["heads"] + 2 * case["kv"]) * d + tables + 16)
                + (2 * e * d if case["norm"] else 0), "flops": 0}
    if case["kind"] == "attend":
        new, lens = _lengths(case)
        h, d = case["heads"], case["dim"]
        # of the step's own tokens a tree's drafts see themselves at least
        pairs = sum(n * (m - n) + (n if case["tree"] else n * (n + 1) // 2)
                    for n, m in zip(new, lens))
        return {"bytes": 2 * e * d * (case["kv"] * sum(lens) + h * (sum(new) + case["pad"] / 2))
                + 8 * sum(-(-m // case["page"]) for m in lens), "flops": 4 * d * h * pairs}
    r = case["rows"]
    return {"bytes": e * r * case["vocab"] + 16 * r, "flops": 0}


# ---- the definition in 64 bits ----------------------------------------------

def _exact_append(case, d):
    h, kv, dim = case["heads"], case["kv"], case["dim"]
    x = d["qkv"].double().view(-1, h + 2 * kv, dim)
    turned = []
    for i, name in ((0, "q_norm"), (1, "k_norm")):
        y = x[:, :h] if i == 0 else x[:, h:h + kv]
        if case["norm"]:
            y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / dim + EPS) * d[name].double()
        c = d["cos"].double()[d["positions"]][:, None]
        sn = d["sin"].double()[d["positions"]][:, None]
        half = dim // 2
        lo, hi = y[..., :half], y[..., half:]
        turned.append(torch.cat([lo * c[..., :half] - hi * sn[..., :half],
                                 hi * c[..., half:] + lo * sn[..., half:]], -1))
    # the cache as one row per slot
    caches = []
    for old, rows in ((d["k_cache"], turned[1]), (d["v_cache"], x[:, h + kv:])):
        flat = old.double().transpose(1, 2).reshape(-1, kv, dim)
        flat[d["slots"]] = rows
        caches.append(flat.view(-1, case["page"], kv, dim).transpose(1, 2))
    return turned[0], caches[0], caches[1]


def _exact_attend(case, d):
    h, kv, dim = case["heads"], case["kv"], case["dim"]
    out = torch.zeros(d["q"].shape, dtype=torch.float64, device="cuda")
    first = 0
    for b, (n, m) in enumerate(zip(*_lengths(case))):
        mine = d["block_table"][b, :-(-m // case["page"])]
        k, v = (d[c][mine].transpose(1, 2).reshape(-1, kv, dim)[:m].double()
                for c in ("k_cache", "v_cache"))
        hidden = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        hidden[:, m - n:] = ~(d["mask"][first:first + n, :n] if case["tree"] else
                              torch.ones(n, n, dtype=torch.bool, device="cuda").tril())
        for j in range(h):
            a = d["q"][first:first + n, j].double() @ k[:, j * kv // h].t().contiguous()
            a = (a / math.sqrt(dim)).masked_fill(hidden, float("-inf"))
            out[first:first + n, j] = torch.softmax(a, -1) @ v[:, j * kv // h].contiguous()
        first += n
    return out


def _exact_sample(case, d):
    """Row by row: cut the candidates off one filter after another, then walk the
    remaining ones in the order of their tokens."""
    tokens = []
    for i in range(case["rows"]):
        l = d["logits"][i].double()
        t = float(d["temperature"][i])
        best = int(torch.nonzero(l == l.max())[0])
        if t <= 0:
            tokens.append(best)
            continue
        ids = torch.argsort(l, descending=True, stable=True)
        if case["top_k"]:
            ids = ids[:case["top_k"]]
        w = torch.exp((l[ids] - l[best]) / t)
        if case["top_p"]:
            most = float(d["top_p"][i]) * float(w.sum())
            ids = ids[:max(1, int(torch.searchsorted(torch.cumsum(w, 0), most)) + 1)]
            w = w[:ids.numel()]
        if case["min_p"]:
            ids = ids[w >= float(d["min_p"][i])]
        ids = ids.sort().values
        total = torch.cumsum(torch.exp((l[ids] - l[best]) / t), 0)
        at = int(torch.searchsorted(total, float(d["uniform"][i]) * float(total[-1]), right=True))
        tokens.append(int(ids[min(at, ids.numel() - 1)]))
    return torch.tensor(tokens, device="cuda")


def exact(case, seed):
    d = _inputs(case, seed)
    return {"append": _exact_append, "attend": _exact_attend,
            "sample": _exact_sample}[case["kind"]](case, d)

"""Serving from a paged KV cache: torch.ops.spyre.{paged_append, paged_attention,
sample}.

Several sequences share one cache of pages, k_cache and v_cache [pages, n_kv_heads,
page_size, head_dim] (any strides, the last 1), and a step brings each of them
some new tokens: one decoded token, the tree of tokens that speculative decoding
drafts, or a piece of a prompt.  A layer's step is

    q = ops.paged_append(qkv, cos, sin, positions, slots, k_cache, v_cache, n_heads)
    a = ops.paged_attention(q, k_cache, v_cache, block_table, seq_lens, q_starts, scale, mask)

and the model's ends in

    tokens = ops.sample(logits, uniform, temperature, top_k, top_p, min_p)

Everything that changes from step to step is a tensor of a fixed shape, so a step can be
captured in a graph: padding rows have slot -1, and rows behind the last
sequence's come back as zeros.

The operators are defined without the custom_op wrapper and their spyre kernels
registered in C++ (torch_spyre/_C, ops_serving.cpp), for the host time of a call;
elsewhere they run as the formulas below.  The reference has neither a KV cache nor
sampling; what a user of it writes for the same layer is its composite RMSNorm
(codegen/inputs/Metadata.yaml:236-253), mul / add (base.jinja2:16-241) and
spyre__bmm_default (spyre_torch_ops.cpp:297-377) over copied caches.
"""

from __future__ import annotations

from typing import Optional

import torch

from .customops import _fp8_check as _check
from .customops import _fp8_refuse_gradients as _refuse_gradients

_SCHEMAS = {
    "paged_append": "(Tensor qkv, Tensor cos, Tensor sin, Tensor positions, Tensor slots, "
                    "Tensor(a!) k_cache, Tensor(b!) v_cache, int n_heads, Tensor? q_norm=None, "
                    "Tensor? k_norm=None, float eps=1e-5) -> Tensor",
    "paged_attention": "(Tensor q, Tensor k_cache, Tensor v_cache, Tensor block_table, "
                       "Tensor seq_lens, Tensor q_starts, float scale, Tensor? mask=None) -> Tensor",
    "sample": "(Tensor logits, Tensor uniform, Tensor? temperature=None, Tensor? top_k=None, "
              "Tensor? top_p=None, Tensor? min_p=None) -> Tensor",
}
for _name, _schema in _SCHEMAS.items():
    torch.library.define(f"spyre::{_name}", _schema)

_lib = torch.library.Library("spyre", "FRAGMENT")
for _name in _SCHEMAS:
    _lib.impl(_name, _refuse_gradients(getattr(torch.ops.spyre, _name).default), "Autograd",
              with_keyset=True)


def _vec(op, name, t, n, dtype):
    _check(t.dim() == 1 and t.shape[0] == n and t.dtype == dtype,
           f"{op}: {name} must be [{n}] of {dtype}, got {list(t.shape)} of {t.dtype}")


def _check_caches(op, x, k_cache, v_cache):
    _check(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and k_cache.shape[1] > 0
           and k_cache.shape[2] > 0,
           f"{op}: k_cache and v_cache must be [pages, n_kv_heads, page_size, head_dim], got "
           f"{list(k_cache.shape)} and {list(v_cache.shape)}")
    _check(k_cache.dtype == v_cache.dtype == x.dtype, f"{op}: the caches must have the type {x.dtype}")


def _index(cond, op, what):
    if bool(cond.any()):
        raise IndexError(f"{op}: {what} out of range")


# ---- paged_append ------------------------------------------------------------

def _paged_append_check(qkv, cos, sin, positions, slots, k_cache, v_cache, n_heads, q_norm, k_norm):
    op = "paged_append"
    _check(qkv.dtype in (torch.float16, torch.bfloat16),
           f"{op}: qkv must be fp16 or bf16, got {qkv.dtype}")
    _check_caches(op, qkv, k_cache, v_cache)
    kv, d = k_cache.shape[1], k_cache.shape[3]
    _check(n_heads > 0 and qkv.dim() == 2 and qkv.shape[1] == (n_heads + 2 * kv) * d,
           f"{op}: qkv must be [tokens, (n_heads + 2 n_kv_heads) * head_dim] = [tokens, "
           f"{(n_heads + 2 * kv) * d}], got {list(qkv.shape)}")
    _check(cos.dim() == 2 and cos.shape[1] == d and sin.shape == cos.shape
           and sin.dtype == cos.dtype and cos.dtype in (qkv.dtype, torch.float32),
           f"{op}: cos and sin must be [positions, {d}] of qkv's type or fp32")
    _vec(op, "positions", positions, qkv.shape[0], torch.int64)
    _vec(op, "slots", slots, qkv.shape[0], torch.int64)
    for name, w in (("q_norm", q_norm), ("k_norm", k_norm)):
        if w is not None:
            _check(w.dtype in (qkv.dtype, torch.float32),
                   f"{op}: norm weights must have qkv's type or fp32, got {w.dtype}")
            _vec(op, name, w, d, w.dtype)
    _check(q_norm is None or k_norm is None or q_norm.dtype == k_norm.dtype,
           f"{op}: q_norm and k_norm must have one type")


def _norm_rotate(x, w, eps, cos, sin):
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.float()
    half = x.shape[-1] // 2
    return x * cos[:, None] + torch.cat([-x[..., half:], x[..., :half]], -1) * sin[:, None]


@torch.library.impl("spyre::paged_append", "CompositeExplicitAutograd")
def paged_append(qkv, cos, sin, positions, slots, k_cache, v_cache, n_heads: int,
                 q_norm: Optional[torch.Tensor] = None, k_norm: Optional[torch.Tensor] = None,
                 eps: float = 1e-5):
    """Appends a step's keys and values to the paged caches, in place, and returns its
    queries [tokens, n_heads, head_dim].  qkv [tokens, (n_heads + 2 n_kv_heads) *
    head_dim] holds a token's query heads, then its key heads, then its value heads.
    Query (key) heads are normalised where q_norm (k_norm) [head_dim] is given,
    x / sqrt(mean(x^2) + eps) * w, and rotated to positions[token]: y cos + rot(y) sin
    with rot(y) = (-y2, y1) for the halves y1, y2 and rows of cos / sin [positions,
    head_dim].  slots[token] = page * page_size + offset says where the token's key
    and value go; below 0 the token is padding, its queries are zeros.  fp32 inside,
    rounded once.  Slots have to differ: of one named twice each element is either row's."""
    _paged_append_check(qkv, cos, sin, positions, slots, k_cache, v_cache, n_heads, q_norm, k_norm)
    pages, kv, page, d = k_cache.shape
    rows = (slots >= 0).nonzero()[:, 0]
    slot, pos = slots[rows], positions[rows]
    _index(slot >= pages * page, "paged_append", "slot")
    _index((pos < 0) | (pos >= cos.shape[0]), "paged_append", "position")
    x = qkv[rows].reshape(-1, n_heads + 2 * kv, d)
    c, s = cos[pos].float(), sin[pos].float()
    q = qkv.new_zeros(qkv.shape[0], n_heads, d)
    q[rows] = _norm_rotate(x[:, :n_heads].float(), q_norm, eps, c, s).to(qkv.dtype)
    k = _norm_rotate(x[:, n_heads:n_heads + kv].float(), k_norm, eps, c, s)
    k_cache[slot // page, :, slot % page] = k.to(qkv.dtype)
    v_cache[slot // page, :, slot % page] = x[:, n_heads + kv:]
    return q


@torch.library.register_fake("spyre::paged_append")
def _(qkv, cos, sin, positions, slots, k_cache, v_cache, n_heads, q_norm=None, k_norm=None,
      eps=1e-5):
    _paged_append_check(qkv, cos, sin, positions, slots, k_cache, v_cache, n_heads, q_norm, k_norm)
    return qkv.new_empty((qkv.shape[0], n_heads, k_cache.shape[3]))


# ---- paged_attention ---------------------------------------------------------

def _paged_attention_check(q, k_cache, v_cache, block_table, seq_lens, q_starts, scale, mask):
    op = "paged_attention"
    _check(q.dtype in (torch.float16, torch.bfloat16),
           f"{op}: q must be fp16 or bf16, got {q.dtype}")
    _check(q.dim() == 3, f"{op}: q must be [tokens, n_heads, head_dim], got {list(q.shape)}")
    _check_caches(op, q, k_cache, v_cache)
    kv = k_cache.shape[1]
    _check(k_cache.shape[3] == q.shape[2],
           f"{op}: the caches' head_dim must be {q.shape[2]}, got {k_cache.shape[3]}")
    _check(q.shape[1] > 0 and q.shape[1] % kv == 0,
           f"{op}: {q.shape[1]} query heads are no multiple of {kv} KV heads")
    _check(0 < scale < float("inf"), f"{op}: scale must be positive and finite, got {scale}")
    _check(block_table.dim() == 2 and block_table.dtype == torch.int64,
           f"{op}: block_table must be [sequences, pages] of int64, got "
           f"{list(block_table.shape)} of {block_table.dtype}")
    _vec(op, "seq_lens", seq_lens, block_table.shape[0], torch.int64)
    _vec(op, "q_starts", q_starts, block_table.shape[0] + 1, torch.int64)
    _check(mask is None or (mask.dim() == 2 and mask.shape[0] == q.shape[0]
                            and mask.dtype == torch.bool),
           f"{op}: mask must be [{q.shape[0]}, new tokens] of bool")


def _attend(q, k, v, seen, scale):
    """q [n, H, d] over k / v [m, Hkv, d] where seen [n, m], in fp32; what a row does
    not see has no effect on it, whatever it holds."""
    g = q.shape[1] // k.shape[1]
    k, v = (x.float().repeat_interleave(g, 1).transpose(0, 1) for x in (k, v))
    score = torch.matmul(q.float().transpose(0, 1), k.transpose(1, 2).contiguous()) * scale
    p = torch.softmax(score.masked_fill(~seen, float("-inf")), -1)
    p = p.masked_fill(~seen.any(-1, keepdim=True), 0.0)  # (rows that see nothing)
    odd = ~v.isfinite().all(-1)  # [H, m]
    o = torch.matmul(p, v.masked_fill(odd[..., None], 0.0))
    for j in odd.any(0).nonzero()[:, 0].tolist():
        o = torch.where(odd[:, j, None, None] & seen[:, j, None],
                        o + p[:, :, j, None] * v[:, None, j], o)
    return o.transpose(0, 1)


@torch.library.impl("spyre::paged_attention", "CompositeExplicitAutograd")
def paged_attention(q, k_cache, v_cache, block_table, seq_lens, q_starts, scale: float,
                    mask: Optional[torch.Tensor] = None):
    """Attention of a step's new tokens over their sequences' pages: sequence b has
    seq_lens[b] keys, key x in page block_table[b, x // page_size] at x % page_size;
    the last n = q_starts[b + 1] - q_starts[b] of them are its new tokens, whose
    queries are rows q_starts[b] .. of q [tokens, n_heads, head_dim].  New token i
    sees every key before the new ones and, of the new ones, those j with
    mask[q_starts[b] + i, j] (a tree's ancestors and itself, say), or without a
    mask j <= i.  Returns softmax(scale q k^T) v over what is seen, like q; rows that see
    nothing, and rows before the first and behind the last sequence's, are zeros.  Of a
    sequence without new tokens only the length is looked at: it has to be one that the block
    table holds (0, say), its pages may be anything."""
    _paged_attention_check(q, k_cache, v_cache, block_table, seq_lens, q_starts, scale, mask)
    op, page = "paged_attention", k_cache.shape[2]
    out = q.new_zeros(q.shape)
    starts, lens = q_starts.tolist(), seq_lens.tolist()
    for b, m in enumerate(lens):
        first, n = starts[b], starts[b + 1] - starts[b]
        if first < 0 or n < 0 or starts[b + 1] > q.shape[0]:
            raise IndexError(f"{op}: q_starts out of range")
        if m < n or m > block_table.shape[1] * page or (mask is not None and n > mask.shape[1]):
            raise IndexError(f"{op}: length out of range")
        if n == 0:
            continue
        pages = block_table[b, :-(-m // page)]
        _index((pages < 0) | (pages >= k_cache.shape[0]), op, "page")
        k, v = (c[pages].transpose(1, 2).reshape(-1, c.shape[1], c.shape[3])[:m]
                for c in (k_cache, v_cache))
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if mask is None:
            seen = seen.tril(m - n)
        else:
            seen[:, m - n:] = mask[first:first + n, :n]
        out[first:first + n] = _attend(q[first:first + n], k, v, seen, scale).to(q.dtype)
    return out


@torch.library.register_fake("spyre::paged_attention")
def _(q, k_cache, v_cache, block_table, seq_lens, q_starts, scale, mask=None):
    _paged_attention_check(q, k_cache, v_cache, block_table, seq_lens, q_starts, scale, mask)
    return q.new_empty(q.shape)


# ---- sample ------------------------------------------------------------------

def _sample_check(logits, uniform, temperature, top_k, top_p, min_p):
    op = "sample"
    _check(logits.dtype in (torch.float16, torch.bfloat16, torch.float32),
           f"{op}: logits must be fp16, bf16 or fp32, got {logits.dtype}")
    _check(logits.dim() == 2 and logits.shape[1] > 0,
           f"{op}: logits must be [rows, vocabulary], got {list(logits.shape)}")
    rows = logits.shape[0]
    for name, t, dtype in (("uniform", uniform, torch.float32),
                           ("temperature", temperature, torch.float32),
                           ("top_k", top_k, torch.int64), ("top_p", top_p, torch.float32),
                           ("min_p", min_p, torch.float32)):
        if t is not None:
            _vec(op, name, t, rows, dtype)


@torch.library.impl("spyre::sample", "CompositeExplicitAutograd")
def sample(logits, uniform, temperature: Optional[torch.Tensor] = None,
           top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
           min_p: Optional[torch.Tensor] = None):
    """Tokens [rows] (int64) drawn from logits [rows, vocabulary] by the random numbers
    uniform [rows] in [0, 1), each row with its own parameters.  A token weighs
    exp((logit - largest) / temperature); in the order of falling logits, equal ones by
    index, top_k > 0 keeps the first so many, top_p < 1 of those the shortest run from
    the first that holds this share of their weight (one at least), and min_p those that
    weigh at least so much (at most 1).  The token is the first by index at which the kept
    weights, added by index, exceed uniform times their sum.  A temperature not above
    0 takes the largest logit (the lowest index first).  NaN counts as -inf; a row without any
    logit above -inf gives -1; beside +inf only +inf counts.  Weights are held in 64 bits."""
    _sample_check(logits, uniform, temperature, top_k, top_p, min_p)
    x = logits.double()
    x = torch.where(x.isnan(), float("-inf"), x)
    most = x.amax(1, keepdim=True)
    x = torch.where(most == float("inf"), torch.where(x == float("inf"), 0.0, float("-inf")), x)
    val, order = x.sort(dim=1, descending=True, stable=True)
    t = torch.ones_like(x[:, :1]) if temperature is None else temperature.double()[:, None]
    w = torch.where(val > float("-inf"), ((val - val[:, :1]) / torch.where(t > 0, t, 1.0)).exp(), 0.0)
    rank = torch.arange(x.shape[1], device=x.device)
    keep = torch.ones_like(w, dtype=torch.bool)
    if top_k is not None:
        keep &= (rank < top_k[:, None]) | (top_k[:, None] <= 0)
    if top_p is not None:
        kept = w * keep
        want = top_p.double()[:, None] * kept.sum(1, keepdim=True)
        keep &= (kept.cumsum(1) - kept < want) | (rank == 0) | ~(top_p[:, None] < 1)
    if min_p is not None:
        keep &= ~(w < min_p.double()[:, None].clamp(max=1.0))
    mass = torch.zeros_like(w).scatter_(1, order, w * keep).cumsum(1)
    u = uniform.double()[:, None]
    target = torch.where(u > 0, u.clamp(max=1.0), 0.0) * mass[:, -1:]
    # (a number of 1 or rounding at the end: the last token that has weight)
    last = (mass < mass[:, -1:]).sum(1)
    token = torch.minimum((mass <= target).sum(1), last)
    token = torch.where(t[:, 0] > 0, token, order[:, 0])
    return torch.where(most[:, 0] > float("-inf"), token, -1)


@torch.library.register_fake("spyre::sample")
def _(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    _sample_check(logits, uniform, temperature, top_k, top_p, min_p)
    return logits.new_empty((logits.shape[0],), dtype=torch.int64)

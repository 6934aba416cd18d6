"""Performance cases of three operators that a decoding step is made of: the
projections over 4-bit weights, the rotary embedding of their query and key
heads, and the attention of a batch whose sequences share a long prefix.

Shapes are the Qwen3-0.6B / 8B / 32B geometries that the rest of this
repository measures (head counts, projection widths, 256-token pages), with
batches and contexts of a serving program.

``own`` chooses between the plain form of an operator (elementary torch
operations in float32, angles in float64, one rounding at the end) and the
calls that a user makes of ``nanovllm_amd.kernels``.  ``exact`` computes the
same outputs in float64 from the operators' definitions.
"""
from __future__ import annotations

import math
import os
import random
import sys
import zlib
from types import SimpleNamespace

import torch

own = False

BF16 = torch.bfloat16
FP8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
D = 128                     # head_dim of the attention cases
THETA = 1000000.0
TRAINED = 40960             # positions a model was trained on, before scaling


def _kernels():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "extend-nano-vllm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from nanovllm_amd import kernels

    return kernels


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one request's decode step, the output projection of the 8B model: the
        # smallest product that matters, all latency
        dict(name="w4-o-1", kind="w4", rows=1, n=4096, k=4096, group=128, zeros=False, bias=False),
        # gate and up of the 8B model for the verified rows of one request
        dict(name="w4-gate-up-6", kind="w4", rows=6, n=24576, k=4096, group=128, zeros=False,
             bias=False),
        # down of the 32B model at a small batch, asymmetric weights in small
        # groups
        dict(name="w4-down-16", kind="w4", rows=16, n=5120, k=25600, group=64, zeros=True,
             bias=False),
        # q/k/v with a bias at an odd batch, the smallest groups
        dict(name="w4-qkv-61", kind="w4", rows=61, n=6144, k=4096, group=32, zeros=True,
             bias=True),
        # one new token: the head counts of the smallest model
        dict(name="rope-1", kind="rope", tokens=1, hq=16, hkv=8, d=128, rot=128,
             interleaved=False, scaling=1.0, dtype="bf16", far=TRAINED, packed=True),
        # the verified rows of a serving batch, scaled to long contexts
        dict(name="rope-verify", kind="rope", tokens=384, hq=32, hkv=8, d=128, rot=128,
             interleaved=False, scaling=4.0, dtype="bf16", far=4 * TRAINED, packed=True),
        # a prefill step's packed prompts, rotated in interleaved pairs
        dict(name="rope-prefill", kind="rope", tokens=16384, hq=32, hkv=8, d=128, rot=128,
             interleaved=True, scaling=1.0, dtype="bf16", far=TRAINED, packed=True),
        # a ragged prompt whose heads rotate in their first half only, half
        # precision, heads of their own tensors
        dict(name="rope-part", kind="rope", tokens=5003, hq=24, hkv=4, d=128, rot=64,
             interleaved=False, scaling=32.0, dtype="fp16", far=32 * 4096, packed=False),
        # a few requests over one short system prompt
        dict(name="prefix-few", kind="prefix", batch=8, q=1, ragged=False, hq=16, hkv=8, block=256,
             prefix=768, lo=1, hi=200, kv="bf16"),
        # decode of a serving batch over one long system prompt
        dict(name="prefix-decode", kind="prefix", batch=64, q=1, ragged=False, hq=32, hkv=8,
             block=256, prefix=8192, lo=64, hi=1024, kv="bf16"),
        # verification of drafts at the largest model and batch, a prefix that
        # ends inside a page
        dict(name="prefix-verify", kind="prefix", batch=128, q=8, ragged=True, hq=64, hkv=8,
             block=256, prefix=4111, lo=8, hi=1500, kv="bf16"),
        # FP8 pages, a long document that every request asks about
        dict(name="prefix-fp8", kind="prefix", batch=100, q=5, ragged=False, hq=16, hkv=8,
             block=256, prefix=16384, lo=5, hi=512, kv="fp8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        case = _draw(rng)
        w = work(case)
        if all(w[key] <= max(m[key] for m in most) for key in w):
            return case


def _draw(rng):
    kind = rng.choice(["w4", "w4", "rope", "rope", "prefix", "prefix", "prefix"])
    if kind == "w4":
        group = rng.choice([32, 64, 128])
        return dict(kind=kind, rows=_log_int(rng, 1, 96), n=_log_int(rng, 64, 25600),
                    k=group * _log_int(rng, max(1, 256 // group), 25600 // group), group=group,
                    zeros=rng.random() < 0.5, bias=rng.random() < 0.3)
    if kind == "rope":
        d = rng.choice([64, 80, 96, 128, 128, 128, 192, 256])
        rot = rng.choice([d, d, d // 2, d // 4])
        scaling = rng.choice([1.0, 2.0, 4.0, 8.0, 32.0])
        hkv = rng.choice([1, 2, 4, 8, 8])
        return dict(kind=kind, tokens=_log_int(rng, 1, 16384), hq=hkv * rng.choice([1, 2, 4, 5, 8]),
                    hkv=hkv, d=d, rot=rot, interleaved=rng.random() < 0.5, scaling=scaling,
                    dtype=rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"]),
                    far=int(scaling * _log_int(rng, 2048, TRAINED)), packed=rng.random() < 0.6)
    hkv = rng.choice([1, 2, 4, 8, 8, 8])
    hi = _log_int(rng, 8, 2048)
    q = rng.choice([1, 1, 1, 2, 4, 5, 6, 8, 9, _log_int(rng, 10, 100)])
    prefix = _log_int(rng, 32, 16384)
    lo = max(1, q - prefix, hi // rng.randint(1, 16))    # a row is one of its sequence's keys
    return dict(kind=kind, batch=_log_int(rng, 2, 160), q=q, ragged=q > 1 and rng.random() < 0.5,
                hq=hkv * rng.choice([1, 2, 4, 4, 5, 8]), hkv=hkv,
                block=rng.choice([32, 64, 256, 256, 256]), prefix=prefix, lo=lo, hi=max(lo, hi),
                kv=rng.choice(["bf16", "bf16", "fp8"]))


# ---------------------------------------------------------------- lengths

def _lengths(case):
    """(query rows, keys) of every sequence, from the case alone; a sequence's
    query rows are its last keys."""
    text = repr(sorted((key, v) for key, v in case.items() if key != "name"))
    rng = random.Random(zlib.crc32(text.encode()))
    n = case["batch"]
    rows = [rng.randint(1, case["q"]) if case["ragged"] else case["q"] for _ in range(n)]
    return rows, [case["prefix"] + rng.randint(case["lo"], case["hi"]) for _ in range(n)]


def _pairs(rows, keys):
    """(query row, visible key) pairs under the bottom-right causal mask."""
    return sum(r * k - r * (r - 1) // 2 for r, k in zip(rows, keys))


def _cu(values):
    out = [0]
    for v in values:
        out.append(out[-1] + v)
    return out


def work(case):
    kind = case["kind"]
    if kind == "w4":
        m, n, k, g = case["rows"], case["n"], case["k"], k_groups(case)
        scales = g * n * (2 + (1 if case["zeros"] else 0)) + (2 * n if case["bias"] else 0)
        return {"bytes": n * k // 2 + scales + 2 * m * (n + k), "flops": 2 * m * n * k}
    if kind == "rope":
        size = DTYPES[case["dtype"]].itemsize
        elems = case["tokens"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 2 * elems * size + case["tokens"] * 8 + case["rot"] * 4,
                "flops": 3 * case["tokens"] * (case["hq"] + case["hkv"]) * case["rot"]}
    rows, keys = _lengths(case)
    size = 1 if case["kv"] == "fp8" else 2
    stored = case["prefix"] + sum(k - case["prefix"] for k in keys)
    return {"bytes": stored * case["hkv"] * D * size * 2 + sum(rows) * case["hq"] * D * 4,
            "flops": 4 * D * case["hq"] * _pairs(rows, keys)}


def k_groups(case):
    return case["k"] // case["group"]


# ---------------------------------------------------------------- inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _i32(values):
    return torch.tensor(values, dtype=torch.int32).to("cuda")


def _normal(shape, gen, std=1.0, dtype=BF16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _frequencies(case):
    """(angle per position of each pair, factor on cos and sin): frequencies
    that turn less than once over the trained positions are slowed by
    ``scaling``, those that turn 32 times stay, with a ramp between."""
    rot, factor = case["rot"], case["scaling"]
    i = torch.arange(0, rot, 2, dtype=torch.float64)
    freq = THETA ** (-i / rot)
    if factor == 1.0:
        return freq.to("cuda"), 1.0
    turns = case["far"] / factor * freq / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return (freq * keep + freq / factor * (1.0 - keep)).to("cuda"), 0.1 * math.log(factor) + 1.0


def _pages(case, rows, keys, seed, gen):
    """A paged cache whose sequences all list the same pages for the whole
    pages of the prefix; a page in which the prefix ends is every sequence's
    own, with the prefix's last keys copied into each."""
    block, hkv = case["block"], case["hkv"]
    shared, rest = divmod(case["prefix"], block)
    blocks = [-(-k // block) for k in keys]
    total = shared + sum(b - shared for b in blocks)
    order = list(range(total))
    random.Random(seed).shuffle(order)
    table, at = [], shared
    for b in blocks:
        table.append(order[:shared] + order[at:at + b - shared] + [-1] * (max(blocks) - b))
        at += b - shared
    shape = (total, hkv, 2, block, D)
    if case["kv"] == "fp8":
        pages = torch.empty(shape, dtype=FP8, device="cuda")
        step = max(1, (1 << 28) // (hkv * 2 * block * D))
        for b in range(0, total, step):
            part = pages[b:b + step]
            part.copy_(_normal(part.shape, gen))
    else:
        pages = _normal(shape, gen)
    if rest:
        raw = pages.view(torch.uint8) if case["kv"] == "fp8" else pages
        own_pages = torch.tensor([t[shared] for t in table], device="cuda")
        raw[own_pages, :, :, :rest] = raw[own_pages[0], :, :, :rest].clone()
    view = pages.permute(2, 0, 3, 1, 4)
    return view[0], view[1], _i32(table)


def prepare(case, seed):
    gen = _gen(seed)
    s = SimpleNamespace(case=case, kind=case["kind"])
    if s.kind == "w4":
        m, n, k, groups = case["rows"], case["n"], case["k"], k_groups(case)
        # the activations behind a norm; 4-bit codes and scales as a quantizer
        # leaves them, [groups, n] as checkpoints store them
        s.x = _normal((m, k), gen)
        s.qweight = torch.randint(0, 256, (n, k // 2), generator=gen, device="cuda",
                                  dtype=torch.uint8)
        s.scales = (torch.rand((groups, n), generator=gen, device="cuda") * 0.008 + 0.002).to(BF16)
        s.zeros = torch.randint(4, 12, (groups, n), generator=gen, device="cuda",
                                dtype=torch.uint8) if case["zeros"] else None
        s.bias = _normal((n,), gen) if case["bias"] else None
        return s
    if s.kind == "rope":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["d"]
        dtype = DTYPES[case["dtype"]]
        if case["packed"]:      # the rows of a fused q/k/v projection
            qkv = _normal((t, (hq + 2 * hkv) * d), gen, 1.0, dtype)
            s.q = qkv[:, :hq * d].view(t, hq, d)
            s.k = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
        else:
            s.q, s.k = _normal((t, hq, d), gen, 1.0, dtype), _normal((t, hkv, d), gen, 1.0, dtype)
        s.positions = torch.randint(0, case["far"], (t,), generator=gen, device="cuda")
        s.freq, s.factor = _frequencies(case)
        return s
    rows, keys = _lengths(case)
    s.rows, s.keys = rows, keys
    s.k_cache, s.v_cache, s.table = _pages(case, rows, keys, seed, gen)
    s.q = _normal((sum(rows), case["hq"], D), gen)
    s.cu_q, s.cu_k, s.lens = _i32(_cu(rows)), _i32(_cu(keys)), _i32(keys)
    s.max_q, s.max_k = case["q"], case["prefix"] + case["hi"]
    fp8 = case["kv"] == "fp8"
    s.k_scale = torch.tensor([0.75 if fp8 else 1.0], device="cuda")
    s.v_scale = torch.tensor([1.25 if fp8 else 1.0], device="cuda")
    s.scale = D ** -0.5
    # where each query row stands in its sequence
    s.seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows)).to("cuda")
    s.nth = torch.cat([torch.arange(r) for r in rows]).to("cuda")
    return s


# ---------------------------------------------------------------- one pass

def run(s):
    return {"w4": _run_w4, "rope": _run_rope, "prefix": _run_prefix}[s.kind](s)


def _run_w4(s):
    if own:
        return _kernels().linear_w4(s.x, s.qweight, s.scales, s.zeros, s.bias)
    n, half = s.qweight.shape
    groups = s.scales.shape[0]
    codes = torch.stack((s.qweight & 15, s.qweight >> 4), dim=-1).float().view(n, groups, -1)
    zeros = 8.0 if s.zeros is None else s.zeros.t().float()[:, :, None]
    w = ((codes - zeros) * s.scales.t().float()[:, :, None]).view(n, 2 * half)
    y = s.x.float() @ w.t()
    if s.bias is not None:
        y = y + s.bias.float()
    return y.to(BF16)


def _run_rope(s):
    if own:
        return _kernels().rotary_embedding(s.positions, s.q, s.k, s.freq,
                                           interleaved=s.case["interleaved"], factor=s.factor)
    angle = s.positions.double()[:, None, None] * s.freq
    cos, sin = (angle.cos() * s.factor).float(), (angle.sin() * s.factor).float()
    return (_turn(s.q, cos, sin, s.case["interleaved"]),
            _turn(s.k, cos, sin, s.case["interleaved"]))


def _turn(x, cos, sin, interleaved):
    half = cos.shape[-1]
    y = x.float()
    part = y[..., :2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half],
                                                                   part[..., half:])
    u, v = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((u, v), dim=-1).flatten(-2) if interleaved else torch.cat((u, v), dim=-1)
    return torch.cat((part, y[..., 2 * half:]), dim=-1).to(x.dtype)


def _run_prefix(s):
    c = s.case
    if own:
        kernels = _kernels()
        if c["q"] == 1:
            return kernels.shared_prefix_attention_decode(
                s.q, s.k_cache, s.v_cache, s.lens, s.table, c["prefix"], s.scale,
                max_seqlen_k=s.max_k, k_scale=s.k_scale, v_scale=s.v_scale)
        return kernels.shared_prefix_attention_varlen(
            s.q, s.k_cache, s.v_cache, s.cu_q, s.cu_k, s.max_q, s.max_k, c["prefix"], s.scale,
            s.table, k_scale=s.k_scale, v_scale=s.v_scale)
    block, prefix, hkv = c["block"], c["prefix"], c["hkv"]
    t, hq, _ = s.q.shape
    g = hq // hkv
    batch = s.table.shape[0]
    q = s.q.float() * s.scale
    last = s.lens[s.seq] - (s.cu_q[1:] - s.cu_q[:-1])[s.seq] + s.nth     # the last visible key

    # the prefix's keys, once for every row
    pages = s.table[0, :-(-prefix // block)].long()
    k1 = (s.k_cache[pages].float() * s.k_scale).flatten(0, 1)[:prefix].permute(1, 2, 0)
    v1 = (s.v_cache[pages].float() * s.v_scale).flatten(0, 1)[:prefix].transpose(0, 1)
    s1 = torch.matmul(q.view(t, hkv, g, D).transpose(0, 1).reshape(hkv, t * g, D), k1)
    s1 = s1.view(hkv, t, g, prefix)
    s1 = s1.masked_fill((torch.arange(prefix, device="cuda") > last[:, None])[None, :, None],
                        float("-inf"))

    # each sequence's own keys, padded to the longest
    first = prefix // block
    ids = s.table[:, first:].clamp(min=0).long()
    at = prefix - first * block
    k2 = (s.k_cache[ids].float() * s.k_scale).flatten(1, 2)[:, at:].permute(0, 2, 3, 1)
    v2 = (s.v_cache[ids].float() * s.v_scale).flatten(1, 2)[:, at:].transpose(1, 2)
    n2 = k2.shape[3]
    padded = torch.zeros(batch, c["q"], hq, D, device="cuda")
    padded[s.seq, s.nth] = q
    s2 = torch.matmul(padded.view(batch, c["q"], hkv, g, D).transpose(1, 2).reshape(
        batch, hkv, c["q"] * g, D), k2).view(batch, hkv, c["q"], g, n2)
    ends = torch.full((batch, c["q"]), -1, dtype=torch.int64, device="cuda")
    ends[s.seq, s.nth] = last.long()
    hidden = prefix + torch.arange(n2, device="cuda") > ends[:, :, None]
    s2 = s2.masked_fill(hidden[:, None, :, None, :], float("-inf"))

    # one softmax over both; every row sees its own key
    m2 = s2.amax(-1)[s.seq, :, s.nth].transpose(0, 1)                    # [hkv, t, g]
    m = torch.maximum(s1.amax(-1), m2)
    p1 = (s1 - m[..., None]).exp()
    top = torch.zeros(batch, hkv, c["q"], g, device="cuda")
    top[s.seq, :, s.nth] = m.transpose(0, 1)
    p2 = (s2 - top[..., None]).exp()
    total = p1.sum(-1) + p2.sum(-1)[s.seq, :, s.nth].transpose(0, 1)
    o2 = torch.matmul(p2.view(batch, hkv, c["q"] * g, n2), v2).view(batch, hkv, c["q"], g, D)
    o = torch.matmul(p1.view(hkv, t * g, prefix), v1).view(hkv, t, g, D)
    o = (o + o2[s.seq, :, s.nth].transpose(0, 1)) / total[..., None]
    return o.transpose(0, 1).reshape(t, hq, D).to(BF16)


# ---------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "w4":
        n, groups = case["n"], k_groups(case)
        w = torch.empty(n, case["k"], dtype=torch.float64, device="cuda")
        w[:, 0::2] = (s.qweight % 16).double()
        w[:, 1::2] = (s.qweight // 16).double()
        for i in range(groups):
            part = w[:, i * case["group"]:(i + 1) * case["group"]]
            part -= 8.0 if s.zeros is None else s.zeros[i].double()[:, None]
            part *= s.scales[i].double()[:, None]
        y = torch.nn.functional.linear(s.x.double(), w)
        return y if s.bias is None else y + s.bias.double()
    if s.kind == "rope":
        # each pair as a complex number, turned by its angle
        turn = torch.polar(torch.full((1,), s.factor, dtype=torch.float64, device="cuda"),
                           torch.outer(s.positions.double(), s.freq))[:, None]
        out = []
        for x in (s.q, s.k):
            y = x.double().clone()
            rot = y[..., :case["rot"]]
            pairs = rot.unflatten(-1, (-1, 2)) if case["interleaved"] else \
                rot.unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            y[..., :case["rot"]] = (z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2)
            out.append(y)
        return tuple(out)
    group = case["hq"] // case["hkv"]
    parts, start = [], 0
    for i, (r, n) in enumerate(zip(s.rows, s.keys)):
        ids = s.table[i, :-(-n // case["block"])].long()
        k = s.k_cache[ids].double().flatten(0, 1)[:n] * s.k_scale.double()
        v = s.v_cache[ids].double().flatten(0, 1)[:n] * s.v_scale.double()
        q = s.q[start:start + r].double().unflatten(1, (case["hkv"], group))
        start += r
        scores = torch.einsum("rhgd,nhd->hgrn", q, k) * s.scale
        seen = torch.arange(n, device="cuda")[None] <= torch.arange(n - r, n, device="cuda")[:, None]
        w = torch.softmax(scores.masked_fill(~seen, float("-inf")), dim=-1)
        parts.append(torch.einsum("hgrn,nhd->rhgd", w, v).flatten(1, 2))
    return torch.cat(parts)

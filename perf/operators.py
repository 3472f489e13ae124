"""Timed cases of the paged key-value cache: what a service does with it, from one live stream's next token to the
prompts of a full batch.

The cache is pages of ``page`` positions, ``[pages, kv heads, page, head dim]``, found through a table ``[slots, width]``
of page numbers; its elements are bf16, or e4m3 with one power of two for each (position, kv head) vector.  Query head h
reads kv head ``h // (heads // kv)``.  The shapes are the omniASR-LLM decoder's (8 heads x 512), the benchmark stack's
(32 x 128) and generic grouped ones (32 heads over 8, 16 over 2).

Kinds:

* ``write``   the new tokens' q and k rotated, k and v written into their pages; then the same positions read back;
* ``read``    whole cached contexts read back (the keys a continued prompt attends to, a slot moved elsewhere);
* ``decode``  the attention of a step: 1 + drafts queries of each slot over its own pages;
* ``prompt``  the causal attention of packed prompts of different lengths, with cached positions before them or without.
"""

import math

import numpy as np
import torch

own = False

E4M3_MAX = 448.0
POSITIONS = 8192  # rows of the rotation table: the decoder's position cap
SHAPES = ((8, 8, 512), (32, 32, 128), (32, 8, 128), (16, 2, 256))


def listed():
    return [
        # one live stream: the newest token into the cache
        {"name": "write_1_token", "kind": "write", "heads": 8, "kv": 8, "dim": 512, "page": 64, "fp8": True,
         "slots": 1, "lo": 1, "hi": 1, "past": 1433},
        # the drafted step of a full batch: 8 slots, the newest token and 4 drafts each
        {"name": "write_8x5_bf16", "kind": "write", "heads": 32, "kv": 32, "dim": 128, "page": 16, "fp8": False,
         "slots": 8, "lo": 5, "hi": 5, "past": 2000},
        # the prompts of a full batch, from a first segment to two segments and text
        {"name": "write_8_prompts", "kind": "write", "heads": 8, "kv": 8, "dim": 512, "page": 64, "fp8": True,
         "slots": 8, "lo": 750, "hi": 2400, "past": 0},
        # the cached contexts of 8 slots, for prompts that go on behind them
        {"name": "read_8_contexts", "kind": "read", "heads": 8, "kv": 8, "dim": 512, "page": 64, "fp8": True,
         "slots": 8, "lo": 750, "hi": 2400},
        # one short context with odd length over small pages
        {"name": "read_1_context", "kind": "read", "heads": 32, "kv": 8, "dim": 128, "page": 16, "fp8": False,
         "slots": 1, "lo": 333, "hi": 333},
        # one live stream decoded greedily: the next token over a segment's audio and the text before it
        {"name": "decode_1_slot", "kind": "decode", "heads": 8, "kv": 8, "dim": 512, "page": 64, "fp8": True,
         "slots": 1, "tokens": 1, "lo": 1433, "hi": 1433, "idle": 0},
        # the drafted batch of a service on both head layouts, in both element types
        {"name": "decode_8x5", "kind": "decode", "heads": 8, "kv": 8, "dim": 512, "page": 64, "fp8": True,
         "slots": 8, "tokens": 5, "lo": 750, "hi": 2400, "idle": 0},
        {"name": "decode_8x5_32x128_bf16", "kind": "decode", "heads": 32, "kv": 32, "dim": 128, "page": 16,
         "fp8": False, "slots": 8, "tokens": 5, "lo": 750, "hi": 2400, "idle": 1},
        # long generations up to the position cap, grouped heads
        {"name": "decode_16_long_grouped", "kind": "decode", "heads": 32, "kv": 8, "dim": 128, "page": 128, "fp8": True,
         "slots": 16, "tokens": 1, "lo": 4000, "hi": 8188, "idle": 0},
        # continuous batching: a slot fell free and one prompt is filled in
        {"name": "prompt_1", "kind": "prompt", "heads": 32, "kv": 32, "dim": 128, "seqs": 1, "lo": 1433, "hi": 1433,
         "past": 0},
        # the first fill of a batch
        {"name": "prompt_8", "kind": "prompt", "heads": 8, "kv": 8, "dim": 512, "seqs": 8, "lo": 750, "hi": 2400,
         "past": 0},
        # many short prompts behind cached contexts, grouped heads
        {"name": "prompt_16_grouped_past", "kind": "prompt", "heads": 32, "kv": 8, "dim": 128, "seqs": 16, "lo": 1,
         "hi": 500, "past": 900},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["write", "write", "read"] + ["decode"] * 4 + ["prompt"] * 3)
    heads, kv, dim = rng.choice(SHAPES)
    case = {"kind": kind, "heads": heads, "kv": kv, "dim": dim}
    if kind == "prompt":
        seqs, past = _log_int(rng, 1, 8), rng.choice([0, 0, _log_int(rng, 1, 1000)])
        hi = _log_int(rng, 3, 600 if past else 1400 if seqs > 4 else 2000)
        return {**case, "seqs": seqs, "lo": rng.randint(0 if seqs > 3 and hi > 30 else 1, hi), "hi": hi, "past": past}
    case |= {"page": rng.choice([16, 32, 64, 128, 256]), "fp8": rng.random() < 0.6}
    slots = _log_int(rng, 1, 16)
    if kind == "write":
        hi = _log_int(rng, 1, 750)
        return {**case, "slots": slots, "lo": rng.randint(1, hi), "hi": hi, "past": rng.randint(0, 3000)}
    if kind == "read":
        hi = _log_int(rng, 1, 750)
        return {**case, "slots": slots, "lo": rng.randint(1, hi), "hi": hi}
    # the cap keeps a case within the largest listed ones: 8 slots of 750 to 2400 keys x 4096 elements
    hi = _log_int(rng, 1, min(8188, 8 * 1200 * 4096 // (slots * kv * dim)))
    return {**case, "slots": slots, "tokens": rng.choice([1, 1, 2, 5, 5, 9, 16]), "lo": rng.randint(0, hi), "hi": hi,
            "idle": rng.choice([0, 0, 1])}


# ------------------------------------------------------------------------------------------------ inputs

def _lengths(case, count, seed):
    """``count`` lengths of U[lo, hi], fixed by the case (the work is the same for every seed) but dealt to the rows by
    the seed; the ``idle`` last ones are finished slots, which see no cached key."""
    lengths = np.random.default_rng([case["lo"], case["hi"], count]).integers(case["lo"], case["hi"] + 1, count)
    if case.get("idle"):
        lengths[-case["idle"]:] = 0
    return np.random.default_rng(int(seed)).permutation(lengths)


def _normal(shape, g, spread=False):
    """N(0, 1) in bf16; ``spread``: each vector at a size of its own, 2^-3 .. 2^3."""
    x = torch.empty(shape, device="cuda", dtype=torch.float32).normal_(generator=g)
    if spread:
        x *= torch.exp2(torch.rand(*shape[:-1], 1, device="cuda", generator=g) * 6 - 3)
    return x.to(torch.bfloat16)


def _table(reach, page, seed):
    """Pages for ``reach`` positions of each slot, spread over a pool that other slots have shares of too; table
    entries behind a slot's last page are unset."""
    need = [-(-int(n) // page) for n in reach]
    pool = sum(need) + len(need) + 3
    order = np.random.default_rng(int(seed) + 1).permutation(pool)
    table = np.full((len(need), max(max(need), 1)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return torch.tensor(table, device="cuda"), pool


def _pages(case, pool, g):
    shape = (pool, case["kv"], case["page"], case["dim"])
    s = {"k_pages": _normal(shape, g), "v_pages": _normal(shape, g), "k_scale": None, "v_scale": None}
    if case["fp8"]:
        for a in "kv":
            s[a + "_pages"], s[a + "_scale"] = _quantised(s[a + "_pages"].float())
    return s


def _angles(dim):
    inv = 10000.0 ** (-torch.arange(0, dim, 2, device="cuda", dtype=torch.float64) / dim)
    a = torch.arange(POSITIONS, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float()


def _tokens(counts, first):
    """Slots and positions of ``counts[b]`` tokens of each slot b from position ``first[b]`` on."""
    slots = np.repeat(np.arange(len(counts)), counts)
    pos = np.concatenate([np.arange(n) + f for n, f in zip(counts, first)])
    return torch.tensor(slots, device="cuda"), torch.tensor(pos, device="cuda")


def _starts(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    heads, kv, dim, kind = case["heads"], case["kv"], case["dim"], case["kind"]
    if kind == "prompt":
        lengths = _lengths(case, case["seqs"], seed)
        past = np.random.default_rng(int(seed)).integers(0, case["past"] + 1, case["seqs"])
        n, m = int(lengths.sum()), int((lengths + past).sum())
        s = {"q": _normal((n, heads, dim), g), "k": _normal((m, kv, dim), g), "starts": _starts(lengths),
             "k_starts": None, "longest": int(lengths.max()), "longest_k": int((lengths + past).max()),
             "scale": dim ** -0.5}
        if case["past"]:
            s["k_starts"], s["v"] = _starts(lengths + past), _normal((m, kv, dim), g)
        else:  # v as it stands in the projection's output, beside the q and k it was computed with
            s["v"] = _normal((n, heads + 2 * kv, dim), g)[:, heads + kv:]
        return s
    if kind == "decode":
        lengths = _lengths(case, case["slots"], seed)
        reach = lengths + case["tokens"] - 1
        table, pool = _table(reach, case["page"], seed)
        return {**_pages(case, pool, g), "table": table, "lengths": torch.tensor(lengths, device="cuda"),
                "reach": int(reach.max()), "tokens": case["tokens"], "scale": dim ** -0.5,
                "q": _normal((case["slots"] * case["tokens"], heads, dim), g)}
    counts = _lengths(case, case["slots"], seed)
    first = np.random.default_rng(int(seed) + 2).integers(case.get("past", 0) // 2, case.get("past", 0) + 1, len(counts))
    table, pool = _table(counts + first, case["page"], seed)
    s = {**_pages(case, pool, g), "table": table}
    s["slots"], s["pos"] = _tokens(counts, first)
    if kind == "write":
        s["qkv"] = _normal((int(counts.sum()), heads + 2 * kv, dim), g, spread=True).flatten(1)
        s["cs"], s["heads"] = _angles(dim), heads
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _quantised(x):
    """e4m3 codes and exponent bytes (e + 127) of fp32 ``x`` [..., D]: e the least with max |x| <= 448 * 2^e."""
    mantissa, e = torch.frexp(x.abs().amax(-1))
    e = (e - 9 + (mantissa > 0.875)).clamp(-126, 120)  # 448 = 0.875 * 2^9
    e = torch.where(mantissa > 0, e, 0).int()
    down = ((127 - e) << 23).view(torch.float32)  # 2^-e, exact
    return (x * down[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _values(pages, scale):
    """fp32 values of gathered page rows."""
    if scale is None:
        return pages.float()
    return pages.float() * (scale.int() << 23).view(torch.float32)[..., None]


def _cells(s, slots, pos):
    page = s["k_pages"].size(2)
    return s["table"][slots, pos // page].long(), pos % page


def _gather(s, a, slots, pos):
    """k (a = "k") or v of the tokens at (slots, pos), fp32 [..., kv, D]."""
    at, off = _cells(s, slots, pos)
    pages, scale = s[a + "_pages"], s[a + "_scale"]
    if scale is None:
        return pages[at, :, off].float()
    return _values(pages.view(torch.uint8)[at, :, off].view(torch.float8_e4m3fn), scale[at, :, off])


def _write(s):
    heads, kv, dim = s["heads"], s["k_pages"].size(1), s["k_pages"].size(3)
    x = s["qkv"].view(len(s["pos"]), heads + 2 * kv, dim).float()
    c, sn = s["cs"][s["pos"]][:, None].unbind(-1)
    re, im = x[:, : heads + kv, ::2], x[:, : heads + kv, 1::2]
    turned = torch.stack([re * c - im * sn, re * sn + im * c], -1).flatten(-2)
    at, off = _cells(s, s["slots"], s["pos"])
    for a, new in (("k", turned[:, heads:]), ("v", x[:, heads + kv:])):
        if s[a + "_scale"] is None:
            s[a + "_pages"][at, :, off] = new.to(torch.bfloat16)
        else:
            codes, scale = _quantised(new)
            s[a + "_pages"].view(torch.uint8)[at, :, off] = codes.view(torch.uint8)
            s[a + "_scale"][at, :, off] = scale
    return turned[:, :heads].to(torch.bfloat16)


def _softmax_product(scores, seen, v):
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > float("-inf"), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return (p @ v) / torch.where(total > 0, total, 1.0)


def _decode(s):
    t, q = s["tokens"], s["q"].float()
    b, (heads, dim), kv = q.size(0) // t, q.shape[1:], s["k_pages"].size(1)
    pos = torch.arange(max(s["reach"], 1), device=q.device)
    total = s["lengths"][:, None] + torch.arange(t, device=q.device)  # keys that query i of a slot sees
    used = torch.minimum(pos, (total[:, -1:] - 1).clamp(min=0))  # behind a slot's last key: that key again
    rows = torch.arange(b, device=q.device)[:, None]
    k, v = (_gather(s, a, rows, used).transpose(1, 2).contiguous() for a in "kv")  # [b, kv, L, D]
    q = q.view(b, t, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)  # [b, kv, group, t, D]
    scores = (q.flatten(2, 3) @ k.transpose(2, 3).contiguous()) * s["scale"]
    seen = (pos < total[..., None])[:, None, None].expand(b, kv, heads // kv, t, len(pos)).flatten(2, 3)
    o = _softmax_product(scores, seen, v).unflatten(2, (heads // kv, t))
    return o.permute(0, 3, 1, 2, 4).reshape(b * t, heads, dim).to(torch.bfloat16)


def _prompt(s):
    q, k, v, starts = s["q"], s["k"], s["v"], s["starts"]
    k_starts = starts if s["k_starts"] is None else s["k_starts"]
    n, heads, dim = q.shape
    kv, b = k.size(1), starts.numel() - 1
    nq, nk = starts.diff()[:, None], k_starts.diff()[:, None]
    i, j = (torch.arange(x, device=q.device) for x in (s["longest"], s["longest_k"]))
    at_q = (starts[:-1, None] + i).clamp(max=max(n - 1, 0))
    at_k = (k_starts[:-1, None] + j).clamp(max=max(k.size(0) - 1, 0))
    qq = q[at_q].float().view(b, len(i), kv, heads // kv, dim).permute(0, 2, 3, 1, 4).flatten(2, 3)
    kk, vv = (x[at_k].float().transpose(1, 2).contiguous() for x in (k, v))
    scores = (qq @ kk.transpose(2, 3).contiguous()) * s["scale"]
    seen = (j <= (i + nk - nq)[..., None]) & (j < nk[..., None]) & (i < nq)[..., None]
    seen = seen[:, None, None].expand(b, kv, heads // kv, len(i), len(j)).flatten(2, 3)
    o = _softmax_product(scores, seen, vv).unflatten(2, (heads // kv, len(i))).permute(0, 3, 1, 2, 4)
    out = torch.empty(n + 1, heads, dim, device=q.device, dtype=q.dtype)  # the last row takes what is no query's
    out[torch.where(i < nq, at_q, n)] = o.reshape(b, len(i), heads, dim).to(q.dtype)
    return out[:n]


def _own_kernels():
    import importlib

    return importlib.import_module("omniasr-trt_amd").kernels


@torch.inference_mode()
def run(s):
    if own:
        kernels = _own_kernels()
        if "starts" in s:
            return kernels.packed_attention(s["q"], s["k"], s["v"], s["starts"], s["longest"], s["scale"],
                                            k_starts=s["k_starts"])
        scales = {"k_scale": s["k_scale"], "v_scale": s["v_scale"]}
        if "lengths" in s:
            return kernels.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lengths"], s["tokens"],
                                           s["scale"], **scales)
        q = None
        if "qkv" in s:
            q = kernels.rope_kv_paged(s["qkv"], s["cs"], s["pos"], s["k_pages"], s["v_pages"], s["table"], s["heads"],
                                      s["slots"], **scales)
        k, v = kernels.paged_read(s["k_pages"], s["v_pages"], s["table"], s["slots"], s["pos"], **scales)
        return {"q": q, "k": k, "v": v}
    if "starts" in s:
        return _prompt(s)
    if "lengths" in s:
        return _decode(s)
    q = _write(s) if "qkv" in s else None
    k, v = (_gather(s, a, s["slots"], s["pos"]).to(torch.bfloat16) for a in "kv")
    return {"q": q, "k": k, "v": v}


# ------------------------------------------------------------------------------------------------ work

def work(case):
    heads, kv, dim, kind = case["heads"], case["kv"], case["dim"], case["kind"]
    if kind == "prompt":
        nq = _lengths(case, case["seqs"], 0).astype(np.int64)
        past = np.random.default_rng(0).integers(0, case["past"] + 1, case["seqs"])
        return {"bytes": int(2 * dim * (2 * heads * nq.sum() + 2 * kv * (nq + past).sum())) + 16,
                "flops": int(4 * dim * heads * (nq * (nq + 1) // 2 + nq * past).sum())}
    cell = dim + 1 if case["fp8"] else 2 * dim  # bytes of one cached vector
    lengths = _lengths(case, case["slots"], 0).astype(np.int64)
    if kind == "decode":
        t = case["tokens"]
        pairs = int((lengths[:, None] + np.arange(t)).sum())
        return {"bytes": int((lengths + t - 1).sum()) * 2 * kv * cell + 4 * len(lengths) * t * heads * dim,
                "flops": 4 * dim * heads * pairs}
    n = int(lengths.sum())
    read = n * 2 * kv * (cell + 2 * dim)
    if kind == "read":
        return {"bytes": read, "flops": n * 2 * kv * dim}
    return {"bytes": read + n * (2 * dim * (2 * heads + 2 * kv) + 2 * kv * cell + 4 * dim),
            "flops": n * dim * (3 * (heads + kv) + 4 * kv)}


# ------------------------------------------------------------------------------------------------ 64-bit results

def _softmax64(q, k, v, scale, limit):
    """q [T, D], k / v [N, D] in float64; query t sees keys [0, limit[t]), none: zeros."""
    if k.size(0) == 0:
        return torch.zeros_like(q)
    hidden = torch.arange(k.size(0), device=k.device)[None] >= limit[:, None]
    p = torch.softmax(((q @ k.t()) * scale).masked_fill(hidden, float("-inf")), -1)
    return p.masked_fill((limit <= 0)[:, None], 0.0) @ v


def _row64(s, a, slot, n):
    """The first ``n`` cached k or v of a slot in float64 [n, kv, D]."""
    pages, scale = s[a + "_pages"], s[a + "_scale"]
    ids = s["table"][slot, : -(-n // pages.size(2))].long()
    x = pages.view(torch.uint8)[ids].view(pages.dtype).double() if scale is not None else pages[ids].double()
    if scale is not None:
        x = torch.ldexp(x, scale[ids].double()[..., None] - 127)
    return x.transpose(1, 2).flatten(0, 1)[:n]


def _nearest_e4m3(x):
    """The e4m3 values nearest to float64 ``x`` (|x| <= 448), ties to even: spacing 2^(exponent - 3), at least 2^-9."""
    _, e = torch.frexp(x)  # |x| in [2^(e-1), 2^e)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return torch.round(x / step) * step


@torch.inference_mode()
def exact(case, seed):
    s, kind, dim = prepare(case, seed), case["kind"], case["dim"]
    group = case["heads"] // case["kv"]
    if kind == "prompt":
        starts = s["starts"].tolist()
        k_starts = starts if s["k_starts"] is None else s["k_starts"].tolist()
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b in range(len(starts) - 1):
            rows, keys = slice(starts[b], starts[b + 1]), slice(k_starts[b], k_starts[b + 1])
            nq, nk = starts[b + 1] - starts[b], k_starts[b + 1] - k_starts[b]
            limit = torch.arange(nq, device="cuda") + 1 + nk - nq
            for h in range(case["heads"]):
                out[rows, h] = _softmax64(s["q"][rows, h].double(), s["k"][keys, h // group].double(),
                                          s["v"][keys, h // group].double(), s["scale"], limit)
        return out
    if kind == "decode":
        t, out = case["tokens"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lengths"].tolist()):
            k, v = _row64(s, "k", b, n + t - 1), _row64(s, "v", b, n + t - 1)
            rows, limit = slice(b * t, (b + 1) * t), n + torch.arange(t, device="cuda")
            for h in range(case["heads"]):
                out[rows, h] = _softmax64(s["q"][rows, h].double(), k[:, h // group], v[:, h // group], s["scale"],
                                          limit)
        return out
    if kind == "read":
        counts = torch.bincount(s["slots"]).tolist()
        first = [int(s["pos"][s["slots"] == b].min()) for b in range(len(counts))]
        return {"q": None, **{a: torch.cat([_row64(s, a, b, f + n)[f:] for b, (n, f) in enumerate(zip(counts, first))])
                              for a in "kv"}}
    x = s["qkv"].double().view(len(s["pos"]), -1, dim)
    cs = s["cs"].double()[s["pos"]][:, None]
    q, k, v = x.split([case["heads"], case["kv"], case["kv"]], 1)
    turn = torch.view_as_complex(cs)
    q, k = (torch.view_as_real(torch.view_as_complex(a.reshape(*a.shape[:2], -1, 2)) * turn).flatten(2) for a in (q, k))
    if case["fp8"]:
        for a in (k, v):
            unit = torch.exp2(torch.ceil(torch.log2(a.abs().amax(-1, keepdim=True) / E4M3_MAX)))
            a.copy_(_nearest_e4m3(a / unit) * unit)
    return {"q": q, "k": k, "v": v}

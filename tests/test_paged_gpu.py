"""The paged cache's operators on an MI355X against their restatement in float64 (oracle/paged.py).

Bounds: an output is rounded to bf16 once (2^-8 of it) and each weight once before its product with v (2^-8 of the sum of
weights times |v|, ``size``); a score's fp32 sum of D products is off by at most D * 2^-24 * sum |q k| and enters both the
weight and the sum of weights; the rest (exp2, the sums, the merge of splits) is within 2^-16 of ``size``."""

import sys

import pytest
import torch

from oracle import paged as op
from omniasr_trt_amd import _lib, batching, kernels, modeling

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
SHAPES = [(4, 4, 512), (4, 4, 128), (8, 2, 128), (16, 2, 256), (6, 1, 128)]  # heads, kv heads, D


def say(*a):
    print(*a, flush=True, file=sys.stderr)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(shape, g, cuda):
    return torch.randn(shape, generator=g).to(BF).to(cuda)


def close(got, want, size, q, k, scale):
    """``got`` bf16 against ``want`` with the bounds of this file; ``q`` / ``k`` give the largest sum of |q k|."""
    dim = q.size(-1)
    kn = k[k.isfinite().all(-1)] if k.numel() else k
    reach = float(q.double().norm(dim=-1).max() * (kn.double().norm(dim=-1).max() if kn.numel() else 0.0)) * scale
    bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -16 + 2 * dim * 2.0 ** -24 * reach) * size + 1e-30
    off = (got.double() - want).abs()
    worst = float((off / bound).max()) if off.numel() else 0.0
    assert bool((off <= bound).all()), f"{worst:.2f} of the bound"


def make_cache(cuda, g, kv, dim, page, reach, fp8, spare=5, shared=0):
    """Pages of random keys for rows of ``reach`` positions, in random order; the rest of the pool and of the last pages
    holds NaN (e4m3: or, on odd pages, finite codes with exponents that make them infinite or NaN), the table behind a
    row's pages is out of range; the first ``shared`` pages of row 1 are row 0's."""
    need = [-(-n // page) for n in reach]
    pool = sum(need) + spare
    order = torch.randperm(pool, generator=g)
    table = torch.full((len(reach), max(max(need), 1) + 2), 2 ** 30, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    if shared:
        table[1, :shared] = table[0, :shared]
    k, v = (torch.full((pool, kv, page, dim), float("nan")) for _ in "kv")
    for b, n in enumerate(reach):
        for i in range(need[b]):
            rows = min(page, n - i * page)
            for x in (k, v):
                x[int(table[b, i]), :, :rows] = torch.randn(kv, rows, dim, generator=g)
    scales = {}
    out = []
    for name, x in (("k_scale", k), ("v_scale", v)):
        if fp8:
            values, byte = op.quantise(x.to(BF).float())
            codes = (values / torch.exp2(byte.double() - 127)[..., None]).float().to(torch.float8_e4m3fn)
            unused = x[..., 0].isnan()
            unused[::2] = False
            codes.view(torch.uint8)[unused] = 0x7E
            byte[unused] = 254
            byte[1::4] = torch.where(unused[1::4], torch.full_like(byte[1::4], 255), byte[1::4])
            scales[name] = byte.to(cuda)
            out.append(codes.to(cuda))
        else:
            out.append(x.to(BF).to(cuda))
    return out[0], out[1], table.to(cuda), scales


# ---------------------------------------------------------------------------------------------- write and read

def written(qkv, cs, pos, heads, kv, dim, fp8):
    """(q, k, v, rotated k) as they are kept, from the oracle on the CPU: k and v float64."""
    x = qkv.cpu().float().view(len(pos), heads + 2 * kv, dim)
    turned = op.rotate(x[:, : heads + kv], cs.cpu()[pos.cpu()])
    k, v = turned[:, heads:], x[:, heads + kv:]
    kept = [op.quantise(a)[0] for a in (k, v)] if fp8 else [k.to(BF).double(), v.double()]
    return turned[:, :heads].to(BF), *kept, turned[:, heads:].to(BF)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("page", [16, 128])
def test_write_and_read_back(cuda, heads, kv, dim, page, fp8):
    g = gen(heads * dim + page)
    say(f"write heads={heads} kv={kv} dim={dim} page={page} fp8={fp8}")
    lengths = [1, 40, 17]
    k, v, table, scales = make_cache(cuda, g, kv, dim, page, [300, 160, 33], fp8)
    before = [x.clone().view(torch.uint8) for x in (k, v)]
    slots = torch.repeat_interleave(torch.arange(3), torch.tensor(lengths))
    pos = torch.cat([torch.arange(n) + f for n, f in zip(lengths, (299, 100, 0))])
    n = len(pos)
    big = torch.randn(n, heads + 2 * kv, dim + 8, generator=g) * torch.exp2(torch.randint(-30, 30, (n, heads + 2 * kv, 1),
                                                                            generator=g).float())
    wide = big[..., :dim].flatten(1).to(BF).to(cuda)
    qkv = torch.cat([wide, wide], 1)[:, : wide.size(1)]  # a row stride of its own
    cs = modeling.rope_table(modeling.DecoderConfig(model_dim=heads * dim, num_heads=heads, max_seq_len=512)).to(cuda)
    q, rotated = kernels.rope_kv_paged(qkv, cs, pos.to(cuda), k, v, table, heads, slots.to(cuda), rotated=True, **scales)
    kk, vv = kernels.paged_read(k, v, table, slots.to(cuda), pos.to(cuda), **scales)
    torch.cuda.synchronize()
    wq, wk, wv, wr = written(qkv, cs, pos, heads, kv, dim, fp8)
    assert torch.equal(q.cpu(), wq) and torch.equal(rotated.cpu(), wr)
    assert torch.equal(kk.cpu().double(), wk) and torch.equal(vv.cpu().double(), wv)
    # nothing else has changed
    mask = torch.zeros(k.shape[:3], dtype=torch.bool)
    for s, p in zip(slots.tolist(), pos.tolist()):
        page_at, off = op.cell(table, page, k.size(0), s, p)
        mask[page_at, :, off] = True
    for now, was in zip((k, v), before):
        assert torch.equal(now.view(torch.uint8).cpu()[~mask], was.cpu()[~mask])


@pytest.mark.parametrize("fp8", [True, False])
def test_write_outside_the_cache(cuda, fp8):
    """Padding (a negative row), rows and positions past the table and pages past the pool are not written and read as
    zeros; cache positions of their own."""
    g, heads, kv, dim, page = gen(7), 4, 2, 128, 16
    k, v, table, scales = make_cache(cuda, g, kv, dim, page, [40, 20], fp8)
    wide = table.size(1) * page
    slots = torch.tensor([0, -1, 2, 0, 0, 1, 1, 0])
    at = torch.tensor([3, 3, 3, wide, -1, 39, 2 ** 40, 45])  # 39 of row 1 and 45.. of row 0 partly unset in the table
    table[0, 2] = -5
    cells = [op.cell(table, page, k.size(0), s, p) for s, p in zip(slots.tolist(), at.tolist())]
    assert cells[0] is not None and all(c is None for c in cells[1:])
    before = [x.clone().view(torch.uint8) for x in (k, v, *scales.values())]
    qkv = normal((8, (heads + 2 * kv) * dim), g, cuda)
    cs = modeling.rope_table(modeling.DecoderConfig(model_dim=heads * dim, num_heads=heads, max_seq_len=64)).to(cuda)
    pos = torch.arange(8, device=cuda) * 9
    q = kernels.rope_kv_paged(qkv, cs, pos.clamp(max=63), k, v, table, heads, slots.to(cuda), at.to(cuda), **scales)
    kk, vv = kernels.paged_read(k, v, table, slots.to(cuda), at.to(cuda), **scales)
    torch.cuda.synchronize()
    wq, wk, wv, _ = written(qkv, cs, pos.clamp(max=63), heads, kv, dim, fp8)
    assert torch.equal(q.cpu(), wq)
    assert torch.equal(kk[0].cpu().double(), wk[0]) and torch.equal(vv[0].cpu().double(), wv[0])
    assert not kk[1:].any() and not vv[1:].any()
    for now, was in zip((k, v, *scales.values()), before):
        changed = (now.view(torch.uint8) != was).flatten(3).any(-1) if now.dim() == 4 else now != was
        where = changed.nonzero().cpu()
        assert all((r[0].item(), r[2].item()) == cells[0] for r in where)


def test_quantised_vectors_of_zeros_extremes_and_what_is_not_finite(cuda):
    heads, kv, dim, page = 1, 1, 128, 16
    rows = torch.randn(8, dim, generator=gen(3))
    rows[0] = 0
    rows[1, 7] = float("inf")
    rows[2, 9] = float("nan")
    rows[3] = float("-inf")
    rows[4] *= 2.0 ** -133  # bf16 subnormals
    rows[5, 0] = torch.finfo(BF).max
    rows[6] = rows[6].sign() * 448
    rows[7] = (torch.arange(dim) - 64) * 2.0 ** -9  # every subnormal e4m3 code of its scale
    rows[7, 0] = 448 * 2.0
    v = rows.to(BF)
    qkv = torch.cat([torch.zeros(8, 2 * dim, dtype=BF), v], 1).to(cuda)
    k_pages = torch.zeros(1, kv, page, dim, device=cuda).to(torch.float8_e4m3fn)
    v_pages, scale = k_pages.clone(), torch.zeros(1, kv, page, dtype=torch.uint8, device=cuda)
    scales = {"k_scale": scale, "v_scale": scale.clone()}
    table = torch.zeros(1, 1, dtype=torch.int32, device=cuda)
    pos, slots = torch.arange(8, device=cuda), torch.zeros(8, dtype=torch.long, device=cuda)
    cs = modeling.rope_table(modeling.DecoderConfig(model_dim=dim, num_heads=1, max_seq_len=16)).to(cuda)
    kernels.rope_kv_paged(qkv, cs, pos, k_pages, v_pages, table, heads, slots, **scales)
    kk, vv = kernels.paged_read(k_pages, v_pages, table, slots, pos, **scales)
    torch.cuda.synchronize()
    want, byte = op.quantise(v.float())
    assert scales["v_scale"][0, 0, :8].tolist() == byte.tolist() and (scales["k_scale"][0, 0, :8] == 127).all()
    assert not kk.any()
    got = vv[:, 0].cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))


def test_every_code_at_every_exponent_read_back(cuda):
    """code * 2^(byte - 127) in bf16: exact from byte 3 on; at 1 and 2 the least codes lie below bf16's least number, 2^-133,
    and are rounded to a multiple of it."""
    codes = torch.arange(256, dtype=torch.uint8)
    pages = codes.repeat(1, 1, 256, 1).to(cuda).view(torch.float8_e4m3fn)
    byte = torch.arange(256, dtype=torch.uint8)[None, None]
    byte[..., 0], byte[..., 255] = 1, 254  # what is never written
    table, at = torch.zeros(1, 1, dtype=torch.int32, device=cuda), torch.arange(256, device=cuda)
    kk, vv = kernels.paged_read(pages, pages.clone(), table, torch.zeros_like(at), at, k_scale=byte.to(cuda),
                                v_scale=byte.to(cuda))
    torch.cuda.synchronize()
    exact = codes.view(torch.float8_e4m3fn).double() * torch.exp2(byte[0, 0].double() - 127)[:, None]
    want = exact.to(BF)
    fits = exact.abs() < 2.0 ** 128
    assert torch.equal(want[3:].double()[fits[3:]], exact[3:][fits[3:]])
    for got in (kk, vv):
        got = got[:, 0].cpu()
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(0.0, posinf=1.0, neginf=-1.0), want.nan_to_num(0.0, posinf=1.0, neginf=-1.0))
        assert torch.equal(got.isinf(), want.isinf())


def test_read_and_write_nothing(cuda):
    k, v, table, scales = make_cache(cuda, gen(1), 2, 128, 16, [20], True)
    none = torch.zeros(0, dtype=torch.long, device=cuda)
    kk, vv = kernels.paged_read(k, v, table, none, none, **scales)
    assert kk.shape == vv.shape == (0, 2, 128)
    cs = torch.zeros(4, 64, 2, device=cuda)
    q = kernels.rope_kv_paged(torch.zeros(0, 8 * 128, dtype=BF, device=cuda), cs, none, k, v, table, 4, none, **scales)
    assert q.shape == (0, 4, 128)
    out = kernels.paged_attention(torch.zeros(0, 4, 128, dtype=BF, device=cuda), k, v, table, none, 3, 0.1, **scales)
    assert out.shape == (0, 4, 128)


# ---------------------------------------------------------------------------------------------- paged attention

def attention_case(cuda, heads, kv, dim, page, tokens, lengths, fp8, seed, shared=0, scale=None):
    say(f"paged attention heads={heads} kv={kv} dim={dim} page={page} T={tokens} lengths={lengths[:9]} fp8={fp8}")
    g = gen(seed)
    cache = make_cache(cuda, g, kv, dim, page, [n + tokens - 1 for n in lengths], fp8, shared=shared)
    k, v, table, scales = cache
    q = normal((len(lengths) * tokens, heads, dim), g, cuda)
    n = torch.tensor(lengths, device=cuda)
    scale = dim ** -0.5 if scale is None else scale
    out = kernels.paged_attention(q, k, v, table, n, tokens, scale, **scales)
    torch.cuda.synchronize()
    want, size = op.paged_attention(q, k, v, table, lengths, tokens, scale, **scales)
    kf = k.float() * (torch.exp2(scales["k_scale"].float() - 127)[..., None] if fp8 else 1.0)
    close(out, want, size, q, kf, scale)
    return out


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("tokens", [1, 5])
def test_paged_attention(cuda, heads, kv, dim, tokens, fp8):
    attention_case(cuda, heads, kv, dim, 64, tokens, [1, 700, 0, 33, 64], fp8, heads * dim + tokens)
    attention_case(cuda, heads, kv, dim, 16, tokens, [31, 257], fp8, heads * dim + tokens + 1, shared=1)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_paged_attention_lengths_around_tiles_and_pages(cuda, page):
    lengths = [page - 1, page, page + 1, 2 * page + 15, 31, 32, 33, 1]
    attention_case(cuda, 4, 2, 128, page, 1, lengths, True, page)
    attention_case(cuda, 2, 2, 512, page, 3, lengths, False, page + 1)


@pytest.mark.parametrize("tokens", [9, 16])
def test_paged_attention_many_columns(cuda, tokens):
    """More query columns of a kv head than one block of 16."""
    attention_case(cuda, 8, 2, 128, 32, tokens, [40, 0, 300], True, tokens)
    attention_case(cuda, 8, 1, 256, 32, tokens, [77], False, tokens + 1)
    attention_case(cuda, 3, 1, 512, 16, tokens, [130, 2], True, tokens + 2)


def test_paged_attention_of_a_layer_of_a_pool(cuda):
    """Pages that are one layer of a stack, a table that is a part of a wider one, and more rows in it than are asked."""
    g, layers, page, dim = gen(33), 3, 32, 128
    for fp8 in (True, False):
        k, v, table, scales = make_cache(cuda, g, 2, dim, page, [100, 7, 260], fp8)
        stack = [torch.stack([torch.zeros_like(x.view(torch.uint8)), x.view(torch.uint8), torch.zeros_like(x.view(torch.uint8))])
                 .view(x.dtype) for x in (k, v)]
        wide = torch.full((5, table.size(1) + 9), 2 ** 30, dtype=torch.int32, device=cuda)
        wide[:3, 4:4 + table.size(1)] = table
        part = wide[:, 4:4 + table.size(1)]
        q, n = normal((2, 4, dim), g, cuda), torch.tensor([100, 7], device=cuda)
        out = kernels.paged_attention(q, stack[0][1], stack[1][1], part, n, 1, 0.1, **scales)
        same = kernels.paged_attention(q, k, v, table, n, 1, 0.1, **scales)
        at = torch.tensor([99, 0, 6, 259, 300], device=cuda), torch.tensor([0, 0, 1, 2, 2], device=cuda)
        one = kernels.paged_read(stack[0][1], stack[1][1], part, at[1], at[0], **scales)
        two = kernels.paged_read(k, v, table, at[1], at[0], **scales)
        torch.cuda.synchronize()
        assert torch.equal(out, same) and all(torch.equal(a[:4], b[:4]) for a, b in zip(one, two))


@pytest.mark.parametrize("fp8", [True, False])
def test_a_pool_past_32_bits(cuda, fp8):
    """Pages whose elements lie past 2^31: written, read and attended to as in a small pool."""
    g, heads, kv, dim, page, n = gen(34), 4, 2, 512, 256, 300
    pool = 2 ** 31 // (kv * page * dim) + 9
    far = torch.tensor([[pool - 1, pool - 3], [pool - 4, pool - 8]], dtype=torch.int32, device=cuda)
    near = torch.tensor([[0, 2], [3, 1]], dtype=torch.int32, device=cuda)
    slots = torch.arange(2, device=cuda).repeat_interleave(n)
    pos = torch.arange(n, device=cuda).repeat(2)
    qkv = normal((2 * n, (heads + 2 * kv) * dim), g, cuda)
    cs = modeling.rope_table(modeling.DecoderConfig(model_dim=heads * dim, num_heads=heads, max_seq_len=512)).to(cuda)
    got = []
    for table, size in ((far, pool), (near, 4)):
        say("a pool of", size, "pages")
        k, v = (torch.empty(size, kv, page, dim, device=cuda, dtype=torch.float8_e4m3fn if fp8 else BF) for _ in "kv")
        scales = {a: torch.empty(size, kv, page, dtype=torch.uint8, device=cuda) for a in ("k_scale", "v_scale")} if fp8 else {}
        q = kernels.rope_kv_paged(qkv, cs, pos, k, v, table, heads, slots, **scales)
        kk, vv = kernels.paged_read(k, v, table, slots, pos, **scales)
        lengths = torch.tensor([n, 17], device=cuda)
        out = kernels.paged_attention(q[:2], k, v, table, lengths, 1, 0.05, **scales)
        got.append((q, kk, vv, out))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_paged_attention_of_long_rows_and_many_rows(cuda):
    attention_case(cuda, 2, 1, 128, 256, 1, [8188], True, 1)
    attention_case(cuda, 2, 2, 128, 64, 1, [8188, 5, 1433], False, 2)
    attention_case(cuda, 2, 1, 128, 16, 2, [(37 * i) % 91 for i in range(70)], True, 3)


def test_paged_attention_of_very_many_rows(cuda):
    """131072 rows of 0 to 16 keys: right, and in time that grows with the rows (8 times as many: not 64 times)."""
    g, page, dim, heads, took = gen(35), 16, 128, 2, []
    pool = [normal((64, 1, page, dim), g, cuda) for _ in "kv"]
    for rows in (1 << 14, 1 << 17):
        say("paged attention of", rows, "rows")
        at = torch.arange(rows, device=cuda)
        table, lengths = ((at * 7) % 64).int()[:, None], at % 17
        q = normal((4096, heads, dim), g, cuda).repeat(rows // 4096, 1, 1)
        out = kernels.paged_attention(q, *pool, table, lengths, 1, 0.1)
        events = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
        events[0].record()
        for e in events[1:]:
            kernels.paged_attention(q, *pool, table, lengths, 1, 0.1)
            e.record()
        torch.cuda.synchronize()
        took.append(min(a.elapsed_time(b) for a, b in zip(events, events[1:])))
        for some in at.split(1 << 14):
            k, v = (x[table[some, 0].long(), 0].double() for x in pool)
            scores = (q[some].double()[:, :, None] * k[:, None]).sum(-1) * 0.1
            hidden = (torch.arange(page, device=cuda) >= lengths[some, None])[:, None]
            w = torch.softmax(scores.masked_fill(hidden, -torch.inf), -1).masked_fill(hidden, 0.0)
            want, size = ((w[..., None] * x[:, None]).sum(2) for x in (v, v.abs()))
            close(out[some], want, size, q[some], pool[0], 0.1)
    say("ms", took)
    assert took[1] < 24 * took[0]


def test_paged_attention_with_large_scores(cuda):
    """Scores of hundreds: the reference maximum moves, weights underflow."""
    attention_case(cuda, 4, 2, 128, 32, 3, [500, 40], False, 5, scale=1.0)
    attention_case(cuda, 2, 2, 512, 32, 1, [900], True, 6, scale=1.0)


def test_paged_attention_key_counts_are_held_in_the_cache(cuda):
    g = gen(9)
    k, v, table, scales = make_cache(cuda, g, 2, 128, 16, [64, 64], True)
    table = table[:, :4].contiguous()
    q = normal((4, 4, 128), g, cuda)
    out = kernels.paged_attention(q, k, v, table, torch.tensor([2 ** 50, -7], device=cuda), 2, 0.1, **scales)
    same = kernels.paged_attention(q, k, v, table, torch.tensor([64, 0], device=cuda), 2, 0.1, **scales)
    torch.cuda.synchronize()
    assert torch.equal(out, same) and out.isfinite().all()
    want, size = op.paged_attention(q, k, v, table, [64, 0], 2, 0.1, **scales)
    close(out, want, size, q, torch.full((1, 128), 4.0, device=cuda), 0.1)
    assert not out[2].any()


def test_paged_attention_page_numbers_are_held_in_the_pool(cuda):
    """Page numbers out of the pool read some page of it: no fault, and the other rows keep their results."""
    g = gen(10)
    k, v, table, scales = make_cache(cuda, g, 2, 128, 16, [64, 100], True, spare=0)
    k, v = (torch.where(x.float().isnan(), torch.zeros((), device=cuda), x.float()).to(torch.float8_e4m3fn) for x in (k, v))
    q = normal((2, 4, 128), g, cuda)
    n = torch.tensor([64, 100], device=cuda)
    good = kernels.paged_attention(q, k, v, table, n, 1, 0.1, **scales)
    table[0, 0], table[0, 1], table[0, 2] = -1, 2 ** 31 - 1, -2 ** 31
    out = kernels.paged_attention(q, k, v, table, n, 1, 0.1, **scales)
    torch.cuda.synchronize()
    assert torch.equal(out[1], good[1]) and out.isfinite().all()


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("dim", [128, 512])
def test_paged_attention_does_not_see_what_is_masked(cuda, dim, fp8):
    """The newest tokens' keys and values hold NaN (bf16: an infinity too): the earlier queries of the step do not see
    them, the later ones do."""
    g, tokens, n = gen(dim), 4, 45
    k, v, table, scales = make_cache(cuda, g, 2, dim, 16, [n + tokens - 1, 70], fp8)
    q = normal((2 * tokens, 4, dim), g, cuda)
    at = {p: op.cell(table, 16, k.size(0), 0, p) for p in (n, n + 1)}
    flat = [x.view(torch.uint8) if fp8 else x for x in (k, v)]
    nan = 0x7F if fp8 else float("nan")
    flat[1][at[n][0], 1, at[n][1], 5] = nan if fp8 else float("inf")  # seen from query 1 on
    flat[0][at[n + 1][0], 0, at[n + 1][1], 3] = nan  # seen from query 2 on
    flat[1][at[n + 1][0], 1, at[n + 1][1], 77] = nan
    lengths = torch.tensor([n, 67], device=cuda)
    out = kernels.paged_attention(q, k, v, table, lengths, tokens, dim ** -0.5, **scales)
    torch.cuda.synchronize()
    want, size = op.paged_attention(q, k, v, table, lengths.tolist(), tokens, dim ** -0.5, **scales)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isposinf(), want.isposinf())
    assert out[0].isfinite().all() and out[1, :2].isfinite().all() and out[2, :2].isnan().all()
    fine = want.isfinite()
    close(torch.where(fine, out.double(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, size, 0.0), q,
          torch.full((1, dim), 4.0, device=cuda), dim ** -0.5)


def test_paged_attention_of_values_whose_exponent_makes_them_infinite(cuda):
    """A key of the step that an earlier query does not see has v = 448 * 2^127, which is infinite."""
    g, n, tokens = gen(21), 40, 3
    k, v, table, scales = make_cache(cuda, g, 1, 128, 16, [n + tokens - 1], True)
    q = normal((tokens, 2, 128), g, cuda)
    page, off = op.cell(table, 16, k.size(0), 0, n)
    v.view(torch.uint8)[page, 0, off, 9] = 0x7E
    scales["v_scale"][page, 0, off] = 254
    out = kernels.paged_attention(q, k, v, table, torch.tensor([n], device=cuda), tokens, 0.1, **scales)
    torch.cuda.synchronize()
    assert out[0].isfinite().all() and out[1:, :, 9].isposinf().all()
    want, size = op.paged_attention(q[:1], k, v, table, [n], 1, 0.1, **scales)
    close(out[:1], want, size, q, torch.full((1, 128), 4.0, device=cuda), 0.1)


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 512), (16, 2, 256), (32, 8, 128), (8, 8, 128)])
@pytest.mark.parametrize("n", [33, 65, 1433])
def test_paged_attention_of_nan_where_units_are_cut(cuda, heads, kv, dim, n, fp8):
    """A query with a NaN, and one whose newest key, the only one of its tile, has one: NaN wherever the cuts fall."""
    say(f"NaN heads={heads} kv={kv} dim={dim} n={n} fp8={fp8}")
    g = gen(n + dim)
    k, v, table, scales = make_cache(cuda, g, kv, dim, 16, [n, n, n], fp8)
    q, lengths = normal((3, heads, dim), g, cuda), torch.tensor([n, n, n], device=cuda)
    q[0, :, 7] = float("nan")
    page, off = op.cell(table, 16, k.size(0), 1, n - 1)
    if fp8:
        k.view(torch.uint8)[page, :, off, 9] = 0x7F
    else:
        k[page, :, off, 9] = float("nan")
    out = kernels.paged_attention(q, k, v, table, lengths, 1, dim ** -0.5, **scales)
    torch.cuda.synchronize()
    assert out[:2].isnan().all()
    want, size = op.paged_attention(q, k, v, table, [n, n, n], 1, dim ** -0.5, **scales)
    assert want[:2].isnan().all()
    close(out[2], want[2], size[2], q[2:], torch.full((1, dim), 4.0, device=cuda), dim ** -0.5)


# ---------------------------------------------------------------------------------------------- packed attention

def packed_case(cuda, heads, kv, dim, queries, past, seed, longest=None, behind=0, strided=True, scale=None):
    say(f"packed attention heads={heads} kv={kv} dim={dim} queries={queries} past={past}")
    g = gen(seed)
    past = [past] * len(queries) if isinstance(past, int) else past
    keys = [n + p for n, p in zip(queries, past)]
    starts = torch.tensor([0, *queries]).cumsum(0)
    k_starts = torch.tensor([0, *keys]).cumsum(0)
    n, m = int(starts[-1]) + behind, max(int(k_starts[-1]), 0) + behind
    q, k = normal((n, heads, dim), g, cuda), normal((m, kv, dim), g, cuda)
    v = normal((m, heads + 2 * kv, dim), g, cuda)[:, heads + kv:] if strided else normal((m, kv, dim), g, cuda)
    out = torch.full((n, heads, dim), 7.0, dtype=BF, device=cuda)
    scale = dim ** -0.5 if scale is None else scale
    got = kernels.packed_attention(q, k, v, starts.to(cuda), max(queries) if longest is None else longest, scale,
                                   k_starts=None if not any(past) else k_starts.to(cuda), out=out)
    torch.cuda.synchronize()
    assert got is out
    want, size = op.packed_attention(q, k, v, starts.tolist(), k_starts.tolist(), scale)
    used = int(starts[-1])
    close(out[:used], want[:used], size[:used], q, k, scale)
    assert (out[used:] == 7.0).all()
    return out


@pytest.mark.parametrize("heads,kv,dim", SHAPES)
def test_packed_attention(cuda, heads, kv, dim):
    packed_case(cuda, heads, kv, dim, [1, 70, 0, 16, 130, 33], 0, heads * dim, behind=3)
    packed_case(cuda, heads, kv, dim, [5, 129], [300, 31], heads * dim + 1, strided=False)


@pytest.mark.parametrize("dim", [128, 256, 512])
@pytest.mark.parametrize("n", [1, 63, 64, 65, 191, 193, 256, 257, 400])
def test_packed_attention_lengths_around_blocks(cuda, dim, n):
    packed_case(cuda, 2, 1, dim, [n, 3], 0, n + dim)
    packed_case(cuda, 2, 1, dim, [n], [n % 70 + 1], n + dim + 1)


def test_packed_attention_fewer_keys_than_queries(cuda):
    """Queries before the first key see none: zeros."""
    out = packed_case(cuda, 4, 2, 128, [100, 40, 300], [-30, -40, -290], 4)
    assert not out[:30].any() and not out[100:140].any() and not out[140:430].any()
    packed_case(cuda, 2, 2, 512, [100, 70], [-30, -70], 5)
    packed_case(cuda, 2, 2, 256, [100, 70], [-64, -70], 6)


def test_packed_attention_long_prompt_and_many_short_ones(cuda):
    packed_case(cuda, 1, 1, 128, [2100], 0, 1)
    packed_case(cuda, 1, 1, 512, [1500], 600, 2)
    packed_case(cuda, 8, 2, 128, [(13 * i) % 40 for i in range(40)], 0, 3)
    packed_case(cuda, 8, 8, 128, [(13 * i) % 40 for i in range(40)], [(7 * i) % 50 for i in range(40)], 4, longest=1000)


def test_packed_attention_with_large_scores(cuda):
    packed_case(cuda, 2, 2, 128, [300, 90], 0, 8, scale=1.0)
    packed_case(cuda, 2, 1, 512, [200], 50, 9, scale=1.0)


@pytest.mark.parametrize("heads,kv,dim", [(4, 2, 128), (32, 8, 128), (8, 8, 512), (16, 2, 256), (8, 8, 256)])
def test_packed_attention_head_counts(cuda, heads, kv, dim):
    """Two query heads to a block, and the order of blocks for head counts that are multiples of 8."""
    packed_case(cuda, heads, kv, dim, [70, 1, 0, 150], [0, 40, 3, 9], heads + kv)


CHAINED = [(8, 8, 512), (16, 2, 512), (24, 3, 512), (32, 8, 128), (16, 8, 128), (32, 32, 128), (24, 24, 128), (16, 2, 256),
           (8, 8, 256)]


@pytest.mark.parametrize("heads,kv,dim", CHAINED)
def test_packed_attention_in_chains(cuda, heads, kv, dim):
    """Many blocks for each workgroup: one after another, of sequences long, short and empty, behind earlier keys and before
    the first key."""
    packed_case(cuda, heads, kv, dim, [400, 0, 64, 65, 1, 127, 300, 20, 33, 192, 257, 5] * 2, 0, heads, behind=9)
    packed_case(cuda, heads, kv, dim, [400, 0, 64, 65, 1, 127, 300, 20, 33, 192, 257, 5] * 2,
                [30, 7, -64, -65, 500, -100, -290, 64, 0, 1, -10, 2000] * 2, heads + 1, strided=False)
    packed_case(cuda, heads, kv, dim, [(37 * i) % 130 for i in range(64)], [(11 * i) % 90 for i in range(64)], heads + 2,
                longest=300)
    packed_case(cuda, heads, kv, dim, [3, 2], 0, heads + 3, longest=5000, behind=4995)
    packed_case(cuda, heads, kv, dim, [0, 0, 0], 0, heads + 4, longest=5000, behind=4995)
    packed_case(cuda, heads, kv, dim, [700, 900], [-700, -901], heads + 5, longest=4000, behind=2400)


@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 512), (32, 8, 128), (32, 32, 128), (16, 2, 256)])
def test_packed_attention_in_chains_up_to_longest(cuda, heads, kv, dim):
    """Queries past ``longest`` of a sequence are not computed, the others see what they see."""
    g, counts = gen(51), [300, 40, 129, 64, 200, 10, 70, 90, 100, 128, 192, 1, 2, 3, 65, 66]
    starts = torch.tensor([0, *counts]).cumsum(0)
    n = int(starts[-1])
    q, k, v = (normal((n, h, dim), g, cuda) for h in (heads, kv, kv))
    out = torch.full_like(q, 7.0)
    kernels.packed_attention(q, k, v, starts.to(cuda), 256, 0.05, out=out)
    want = kernels.packed_attention(q, k, v, starts.to(cuda), 300, 0.05)
    torch.cuda.synchronize()
    exact, size = op.packed_attention(q, k, v, starts.tolist(), starts.tolist(), 0.05)
    close(want, exact, size, q, k, 0.05)
    kept = torch.ones(n, dtype=torch.bool)
    for s, c in zip(starts.tolist(), counts):
        kept[s + 256:s + c] = False
    assert torch.equal(out[kept], want[kept]) and (out[~kept] == 7.0).all()


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 512), (32, 8, 128), (32, 32, 128), (16, 2, 256)])
def test_packed_attention_in_chains_does_not_see_what_is_masked(cuda, heads, kv, dim):
    g, counts = gen(52), [300, 90, 129, 64, 200, 10, 70, 90, 100, 128, 192, 1, 2, 3, 65, 66]
    starts = torch.tensor([0, *counts]).cumsum(0)
    n = int(starts[-1])
    q, k, v = normal((n, heads, dim), g, cuda), normal((n, kv, dim), g, cuda), normal((n, kv, dim), g, cuda)
    for s, at in ((0, 250), (1, 70), (2, 128), (8, 99), (11, 0), (15, 30)):
        row = int(starts[s]) + at
        v[row, 0, 3], v[row, 1, dim // 2], v[row, 1, dim - 1] = float("inf"), float("nan"), float("-inf")
    k[int(starts[4]) + 150, 1, 9] = float("nan")
    out = [kernels.packed_attention(q, k, v, starts.to(cuda), 300, 0.05) for _ in range(3)]
    torch.cuda.synchronize()
    want, size = op.packed_attention(q, k, v, starts.tolist(), starts.tolist(), 0.05)
    fine = want.isfinite()
    assert not fine.all() and torch.equal(out[0].isnan(), want.isnan()) and torch.equal(out[0].isposinf(), want.isposinf())
    assert all(torch.equal(o.view(torch.int16), out[0].view(torch.int16)) for o in out)
    close(torch.where(fine, out[0].double(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, size, 0.0), q,
          torch.full((1, dim), 4.0, device=cuda), 0.05)


@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 512), (32, 8, 128), (16, 2, 256)])
def test_packed_attention_in_chains_captured(cuda, heads, kv, dim):
    """One captured launch whose chains follow from the lengths of each replay."""
    g = gen(53)
    q, k, v = (normal((1500, h, dim), g, cuda) for h in (heads, kv, kv))
    starts, k_starts = torch.zeros(17, dtype=torch.long, device=cuda), torch.zeros(17, dtype=torch.long, device=cuda)
    out = torch.empty_like(q)
    graphs = batching.GraphCache(cuda, True)
    run = graphs.runner("chains", lambda: kernels.packed_attention(q, k, v, starts, 700, 0.05, k_starts=k_starts, out=out),
                        lambda: [])
    for counts in ([60] * 16, [700, 1] * 2 + [0] * 12, [0] * 15 + [33], [(i * 29) % 90 for i in range(16)]):
        keys = [min(c + 13, 800) for c in counts]
        starts.copy_(torch.tensor([0, *counts]).cumsum(0))
        k_starts.copy_(torch.tensor([0, *keys]).cumsum(0).clamp(max=1500))
        q.copy_(normal(q.shape, g, cuda))
        out.fill_(5.0)
        run()
        torch.cuda.synchronize()
        used = int(starts[-1])
        want, size = op.packed_attention(q, k, v, starts.tolist(), k_starts.tolist(), 0.05)
        close(out[:used], want[:used], size[:used], q, k, 0.05)
        assert (out[used:] == 5.0).all()
        eager = kernels.packed_attention(q, k, v, starts, 700, 0.05, k_starts=k_starts)
        torch.cuda.synchronize()
        assert torch.equal(eager[:used], out[:used])


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (2, 1, 128), (1, 1, 128), (8, 8, 128), (2, 1, 256), (3, 3, 256),
                                          (2, 2, 512), (8, 8, 512)])
def test_packed_attention_of_few_queries_behind_many_keys(cuda, heads, kv, dim):
    """Few blocks, each cut along its keys: one query, a block's worth and one more, keys that end inside a tile."""
    packed_case(cuda, heads, kv, dim, [1], [2999], dim + heads, longest=1)
    packed_case(cuda, heads, kv, dim, [20, 1, 64], [4000, 130, 63], dim + heads + 1)
    packed_case(cuda, heads, kv, dim, [257], [1000], dim + heads + 2)
    packed_case(cuda, heads, kv, dim, [70, 3], [1500, -3], dim + heads + 3, scale=1.0)
    packed_case(cuda, heads, kv, dim, [2000], [-300], dim + heads + 4)


@pytest.mark.parametrize("heads,kv,dim", [(24, 24, 128), (12, 6, 128), (24, 24, 256), (16, 8, 256), (4, 4, 512)])
def test_packed_attention_in_parts_of_smaller_blocks(cuda, heads, kv, dim):
    """Blocks of fewer queries, cut along their keys: around 12 and 24 tiles, and in sequences of unlike lengths."""
    for i, (n, past) in enumerate([(64, 640), (65, 650), (100, 700), (130, 1350), (190, 1410)]):
        packed_case(cuda, heads, kv, dim, [n], [past], dim + heads + i)
    packed_case(cuda, heads, kv, dim, [5, 70], [900, 30], dim + heads + 9)


def test_packed_attention_in_parts_captured(cuda):
    """One captured launch for lengths that are cut and that are not; calls on two streams share nothing."""
    g = gen(41)
    q, k, v = normal((64, 8, 128), g, cuda), normal((4100, 2, 128), g, cuda), normal((4100, 2, 128), g, cuda)
    starts, k_starts = (torch.tensor([0, 64], device=cuda) for _ in range(2))
    out = torch.empty_like(q)
    graphs = batching.GraphCache(cuda, True)
    run = graphs.runner("parts", lambda: kernels.packed_attention(q, k, v, starts, 64, 0.1, k_starts=k_starts, out=out),
                        lambda: [])
    for keys in (4100, 1500, 64, 1601, 0):
        k_starts[1] = keys
        q.copy_(normal(q.shape, g, cuda))
        run()
        torch.cuda.synchronize()
        eager = [torch.empty_like(q) for _ in range(2)]
        for stream, to in zip((torch.cuda.Stream(), torch.cuda.Stream()), eager):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                kernels.packed_attention(q, k, v, starts, 64, 0.1, k_starts=k_starts, out=to)
        torch.cuda.synchronize()
        assert all(torch.equal(out, to) for to in eager)
        want, size = op.packed_attention(q, k, v, [0, 64], [0, keys], 0.1)
        close(out, want, size, q, k, 0.1)


@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (1, 1, 128), (2, 1, 256), (2, 2, 512)])
def test_packed_attention_in_parts_does_not_see_what_is_masked(cuda, heads, kv, dim):
    g, n, past = gen(dim + 5), 90, 700
    q = normal((n, heads, dim), g, cuda)
    k, v = (normal((n + past, kv, dim), g, cuda) for _ in "kv")
    v[past + 40, 0, 7], v[past + 41, 0, 100], v[past + 41, 0, 17] = float("inf"), float("nan"), float("-inf")
    starts, k_starts = torch.tensor([0, n], device=cuda), torch.tensor([0, n + past], device=cuda)
    out = [kernels.packed_attention(q, k, v, starts, n, dim ** -0.5, k_starts=k_starts) for _ in range(3)]
    torch.cuda.synchronize()
    want, size = op.packed_attention(q, k, v, [0, n], [0, n + past], dim ** -0.5)
    fine = want.isfinite()
    assert fine[:40].all() and torch.equal(out[0].isnan(), want.isnan()) and torch.equal(out[0].isposinf(), want.isposinf())
    assert all(torch.equal(o.view(torch.int16), out[0].view(torch.int16)) for o in out)
    close(torch.where(fine, out[0].double(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, size, 0.0), q, k,
          dim ** -0.5)


def litter(cuda):
    """Finite numbers in the memory that the next tensors and workspaces take: what is read unwritten shows."""
    torch.cuda.empty_cache()
    torch.full((512 << 20,), 0x40, dtype=torch.uint8, device=cuda)


@pytest.mark.parametrize("heads,kv,dim,queries,keys,behind", [
    (8, 8, 512, [100], [10], 1990), (8, 8, 512, [600], [200], 1800), (8, 8, 128, [300], [20], 1980),
    (16, 2, 256, [300], [20], 1980), (2, 2, 512, [600] * 8, [200] * 8, 0), (2, 1, 128, [400, 30, 7], [40, 0, 900], 1200),
    (4, 4, 256, [1000, 64], [1, 3], 3000), (1, 1, 512, [900, 900], [800, 30], 700)])
def test_packed_attention_in_parts_of_many_queries_over_few_keys(cuda, heads, kv, dim, queries, keys, behind):
    """A buffer long enough to be cut, sequences of more queries than keys: their first blocks see no key, and no block has
    many tiles."""
    longest, rows = max(queries), sum(keys) + behind
    assert _lib.load().omni_packed_attention_workspace(len(queries), rows, longest, heads, kv, dim) > 0
    for _ in range(2):
        litter(cuda)
        packed_case(cuda, heads, kv, dim, queries, [k - n for n, k in zip(queries, keys)], dim + heads, behind=behind)


@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 128), (8, 8, 128), (2, 1, 256), (2, 1, 512)])
def test_packed_attention_more_sequences_than_are_ranked(cuda, heads, kv, dim):
    packed_case(cuda, heads, kv, dim, [(13 * i) % 70 for i in range(67)], [(7 * i) % 11 for i in range(67)], dim + heads)


def test_packed_attention_strides_and_layers(cuda):
    """K and V as slices of wide rows, and of a stack of layers."""
    g, heads, kv, n = gen(31), 4, 2, 150
    starts = torch.tensor([0, 90, n], device=cuda)
    for dim in (128, 256, 512):
        say("packed attention of slices", dim)
        q = normal((n, heads, dim), g, cuda)
        wide = normal((n, 3 * kv, 2 * dim + 8), g, cuda)
        stack = normal((3, kv, n, dim), g, cuda)
        for k, v in ((wide[:, ::3, :dim], wide[:, 1::3, dim + 8:]), (stack[1].transpose(0, 1), stack[2].transpose(0, 1))):
            out = kernels.packed_attention(q, k, v, starts, 90, dim ** -0.5)
            torch.cuda.synchronize()
            want, size = op.packed_attention(q, k, v, starts.tolist(), starts.tolist(), dim ** -0.5)
            close(out, want, size, q, k, dim ** -0.5)


@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (4, 2, 256), (2, 2, 512)])
def test_packed_attention_captured(cuda, heads, kv, dim):
    """A captured call reads the starts of the replay; lengths and contents change between replays."""
    g = gen(dim + 3)
    q, k, v = (normal((300, h, dim), g, cuda) for h in (heads, kv, kv))
    starts, k_starts = torch.zeros(4, dtype=torch.long, device=cuda), torch.zeros(4, dtype=torch.long, device=cuda)
    out = torch.empty_like(q)
    graphs = batching.GraphCache(cuda, True)
    run = graphs.runner("packed", lambda: kernels.packed_attention(q, k, v, starts, 200, 0.1, k_starts=k_starts, out=out),
                        lambda: [])
    for counts, past in (([100, 0, 200], [0, 0, 0]), ([1, 60, 30], [20, 100, 0]), ([200, 3, 7], [-50, 9, 30])):
        starts.copy_(torch.tensor([0, *counts]).cumsum(0))
        k_starts.copy_(torch.tensor([0, *(a + b for a, b in zip(counts, past))]).cumsum(0))
        q.copy_(normal(q.shape, g, cuda))
        out.fill_(5.0)
        run()
        torch.cuda.synchronize()
        used = int(starts[-1])
        eager = kernels.packed_attention(q, k, v, starts, 200, 0.1, k_starts=k_starts)
        torch.cuda.synchronize()
        assert torch.equal(out[:used], eager[:used]) and (out[used:] == 5.0).all()
        want, size = op.packed_attention(q, k, v, starts.tolist(), k_starts.tolist(), 0.1)
        close(out[:used], want[:used], size[:used], q, k, 0.1)


@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 128), (4, 4, 256), (2, 2, 512)])
def test_packed_attention_past_32_bits(cuda, heads, kv, dim):
    """Sequences whose rows of q, k, v and out lie past 2^31 elements."""
    g, used = gen(dim + 4), 200
    n = 2 ** 31 // (heads * dim) + used
    q, k, v = (torch.empty(n, heads, dim, dtype=BF, device=cuda) for _ in "qkv")
    for x in (q, k, v):
        x[-used:] = normal((used, heads, dim), g, cuda)
    out = torch.empty_like(q)
    starts = torch.tensor([0, 150, used], device=cuda)
    kernels.packed_attention(q, k, v, starts + (n - used), 150, 0.1, out=out)
    near = kernels.packed_attention(q[-used:], k[-used:], v[-used:], starts, 150, 0.1)
    torch.cuda.synchronize()
    assert torch.equal(out[-used:], near)


def test_packed_attention_into_its_inputs_is_refused(cuda):
    x = normal((40, 4, 128), gen(1), cuda)
    starts = torch.tensor([0, 20], device=cuda)
    for out in (x[:20], x[20:]):
        with pytest.raises(ValueError, match="memory of its own"):
            kernels.packed_attention(x[:20], x[20:], x[20:], starts, 20, 0.1, out=out)


def test_packed_attention_nothing(cuda):
    q = torch.zeros(4, 2, 128, dtype=BF, device=cuda)
    k = torch.zeros(0, 2, 128, dtype=BF, device=cuda)
    starts, none = torch.tensor([0, 4], device=cuda), torch.tensor([0, 0], device=cuda)
    out = kernels.packed_attention(q, k, k, starts, 4, 0.1, k_starts=none)
    assert not out.any()
    full = torch.full_like(q, 3.0)
    assert (kernels.packed_attention(q, q, q, none[:1], 4, 0.1, out=full) == 3).all()
    assert (kernels.packed_attention(q, q, q, none, 0, 0.1, out=full) == 3).all()


@pytest.mark.parametrize("heads,kv,dim", [(2, 1, 128), (4, 1, 128), (1, 1, 128), (2, 1, 256), (1, 1, 256), (2, 1, 512)])
def test_packed_attention_does_not_see_what_is_masked(cuda, heads, kv, dim):
    """NaN and infinities in later positions of a prompt, and in its neighbours, do not reach the queries before them."""
    g = gen(dim + 1)
    q, k, v = (normal((230, h, dim), g, cuda) for h in (heads, kv, kv))
    starts = torch.tensor([0, 100, 230], device=cuda)
    k[90, 0, 3], v[95, 0, 7], v[96, 0, 100], v[100] = float("nan"), float("inf"), float("nan"), float("nan")
    out = kernels.packed_attention(q, k, v, starts, 130, dim ** -0.5)
    torch.cuda.synchronize()
    want, size = op.packed_attention(q, k, v, starts.tolist(), starts.tolist(), dim ** -0.5)
    fine = want.isfinite()
    assert fine[:90].all() and not fine[90:].all()
    assert torch.equal(out.isfinite(), fine)
    close(torch.where(fine, out.double(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, size, 0.0), q,
          torch.full((1, dim), 4.0, device=cuda), dim ** -0.5)


@pytest.mark.parametrize("heads,kv,dim", [(8, 8, 512), (32, 8, 128), (8, 8, 128), (16, 2, 256), (3, 1, 512), (3, 1, 128)])
@pytest.mark.parametrize("queries,past", [([130, 70], [0, 0]), ([20, 65], [1500, 63]), ([150] * 30, [64] * 30)])
def test_packed_attention_of_nan_alone_in_a_tile(cuda, heads, kv, dim, queries, past):
    """Queries with a NaN, and a NaN in a key that starts a tile of 64 (the only one that some query sees of it): one block by
    one, in parts and in chains."""
    say(f"packed NaN heads={heads} kv={kv} dim={dim} queries={queries[:2]} past={past[:2]}")
    g = gen(dim + heads)
    starts = torch.tensor([0, *queries]).cumsum(0)
    k_starts = torch.tensor([0, *(a + b for a, b in zip(queries, past))]).cumsum(0)
    q, k, v = (normal((int(n), h, dim), g, cuda) for n, h in ((starts[-1], heads), (k_starts[-1], kv), (k_starts[-1], kv)))
    q[3, :, 7], q[-1, 0, dim - 1] = float("nan"), float("nan")
    k[int(k_starts[1]) + 64, :, 9] = float("nan")  # of the second sequence
    out = kernels.packed_attention(q, k, v, starts.to(cuda), max(queries), dim ** -0.5, k_starts=k_starts.to(cuda))
    torch.cuda.synchronize()
    want, size = op.packed_attention(q, k, v, starts.tolist(), k_starts.tolist(), dim ** -0.5)
    fine = want.isfinite()
    assert want[3].isnan().all() and want[-1, 0].isnan().all() and torch.equal(out.isnan(), want.isnan())
    close(torch.where(fine, out.double(), 0.0), torch.where(fine, want, 0.0), torch.where(fine, size, 0.0),
          torch.full((1, dim), 4.0, device=cuda), torch.full((1, dim), 4.0, device=cuda), dim ** -0.5)


# ---------------------------------------------------------------------------------------------- together

@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 512), (8, 2, 128)])
def test_prompts_then_steps_then_a_continued_prompt(cuda, heads, kv, dim, fp8):
    """As a decoder uses them: packed prompts into the cache and through the attention, drafted steps over it (captured
    and replayed), then prompts that go on behind what is cached -- each result against the oracle over the keys and
    values kept so far."""
    g, page, tokens, prompts = gen(dim), 32, 3, [50, 1, 90]
    scale, vecs = dim ** -0.5, heads + 2 * kv
    cs = modeling.rope_table(modeling.DecoderConfig(model_dim=heads * dim, num_heads=heads, max_seq_len=512)).to(cuda)
    pool = 3 * 8
    k, v = (torch.zeros(pool, kv, page, dim, device=cuda).to(torch.float8_e4m3fn if fp8 else BF) for _ in "kv")
    scales = {a: torch.zeros(pool, kv, page, dtype=torch.uint8, device=cuda) for a in ("k_scale", "v_scale")} if fp8 else {}
    table = torch.randperm(pool, generator=g).int().view(3, 8).to(cuda)

    def fill(counts, first):
        slots = torch.repeat_interleave(torch.arange(3), torch.tensor(counts)).to(cuda)
        pos = torch.cat([torch.arange(n) + f for n, f in zip(counts, first)]).to(cuda)
        return slots, pos, torch.tensor([0, *counts]).cumsum(0).to(cuda)

    slots, pos, starts = fill(prompts, [0, 0, 0])
    qkv = normal((len(pos), vecs * dim), g, cuda)
    q, kr = kernels.rope_kv_paged(qkv, cs, pos, k, v, table, heads, slots, rotated=True, **scales)
    vr = qkv.view(len(pos), vecs, dim)[:, heads + kv:]
    out = kernels.packed_attention(q, kr, vr, starts, max(prompts), scale)
    want, size = op.packed_attention(q, kr, vr, starts.tolist(), starts.tolist(), scale)
    close(out, want, size, q, kr, scale)

    # two drafted steps through one captured graph
    step_qkv = torch.zeros(3 * tokens, vecs * dim, dtype=BF, device=cuda)
    lengths = torch.tensor(prompts, device=cuda) + 1
    held = {}

    def step():
        at = (lengths[:, None] - 1 + torch.arange(tokens, device=cuda)).flatten()
        rows = torch.arange(3, device=cuda).repeat_interleave(tokens)
        held["q"] = kernels.rope_kv_paged(step_qkv, cs, at, k, v, table, heads, rows, **scales)
        held["out"] = kernels.paged_attention(held["q"], k, v, table, lengths, tokens, scale, **scales)

    graphs = batching.GraphCache(cuda, True)
    run = graphs.runner("step", step, lambda: [])
    captured = dict(held)  # the graph's own outputs
    for _ in range(3):
        step_qkv.copy_(normal(step_qkv.shape, g, cuda))
        run()
        torch.cuda.synchronize()
        n = lengths.tolist()
        want, size = op.paged_attention(captured["q"], k, v, table, n, tokens, scale, **scales)
        kf = torch.cat([op.cached(k, scales.get("k_scale"), table[b], n[b], 0) for b in range(3)])
        close(captured["out"], want, size, captured["q"], kf * 1.5, scale)
        step()
        assert torch.equal(captured["out"], held["out"])
        lengths += 2

    # prompts that go on behind the cached positions
    past = (lengths - 1).tolist()
    more = [20, 70, 3]
    slots, pos, starts = fill(more, past)
    qkv = normal((len(pos), vecs * dim), g, cuda)
    q = kernels.rope_kv_paged(qkv, cs, pos, k, v, table, heads, slots, **scales)
    total = [a + b for a, b in zip(past, more)]
    all_slots, all_pos, k_starts = fill(total, [0, 0, 0])
    kk, vv = kernels.paged_read(k, v, table, all_slots, all_pos, **scales)
    out = kernels.packed_attention(q, kk, vv, starts, max(more), scale, k_starts=k_starts)
    torch.cuda.synchronize()
    for b in range(3):
        kept = op.cached(k, scales.get("k_scale"), table[b], total[b], 1)
        assert torch.equal(kk[k_starts[b]:k_starts[b + 1], 1].double(), kept)
    want, size = op.packed_attention(q, kk, vv, starts.tolist(), k_starts.tolist(), scale)
    close(out, want, size, q, kk, scale)


def test_as_the_full_length_caches(cuda):
    """The same step over a full-length cache and over pages of it: the two kernels agree to their roundings."""
    g, b, t, h, d, cap, page = gen(11), 3, 5, 4, 128, 256, 64
    kc, vc, q = normal((b, h, cap, d), g, cuda), normal((b, h, cap, d), g, cuda), normal((b * t, h, d), g, cuda)
    lengths = torch.tensor([200, 0, 77], device=cuda)
    pages = [x.view(b, h, cap // page, page, d).transpose(1, 2).flatten(0, 1).contiguous() for x in (kc, vc)]
    table = torch.arange(b * (cap // page), dtype=torch.int32, device=cuda).view(b, -1)
    one = kernels.draft_attention(q, kc, vc, lengths, t, cap, d ** -0.5)
    two = kernels.paged_attention(q, *pages, table, lengths, t, d ** -0.5)
    _, size = op.paged_attention(q, *pages, table, lengths.tolist(), t, d ** -0.5)
    assert bool(((one.double() - two.double()).abs() <= 2 * (2.0 ** -8 * two.double().abs()
                                                             + (2.0 ** -8 + 2.0 ** -12) * size)).all())


def test_two_streams_at_once(cuda):
    """Calls on two streams share nothing: each equals the call alone."""
    g = gen(12)
    cases = []
    for lengths in ([700, 33], [90, 1200]):
        k, v, table, scales = make_cache(cuda, g, 2, 128, 32, lengths, True)
        cases.append((normal((2, 8, 128), g, cuda), k, v, table, torch.tensor(lengths, device=cuda), scales))
    alone = [kernels.paged_attention(q, k, v, t, n, 1, 0.1, **s) for q, k, v, t, n, s in cases]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i, (q, k, v, t, n, s) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(kernels.paged_attention(q, k, v, t, n, 1, 0.1, **s))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, alone[i]) for x in got[i])

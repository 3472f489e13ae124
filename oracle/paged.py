"""Plain restatement of the paged cache's operators in float64 (test infrastructure): torch on any device, loops where
they are plain.  Tensors as the operators take them; results float64 with, for attention, the sum of weights times |v|
that error bounds are stated in."""

from __future__ import annotations

import torch

E4M3_MAX = 448.0


def e4m3_values() -> torch.Tensor:
    """The 127 finite e4m3 values >= 0 in order, float64: 3 bits of mantissa, exponents -6..8, subnormals of 2^-9."""
    out = [m * 2.0 ** -9 for m in range(8)]
    for e in range(-6, 9):
        out += [(8 + m) * 2.0 ** (e - 3) for m in range(8)]
    return torch.tensor(out[:-1], dtype=torch.float64)  # the last code is NaN


def rotate(x: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    """fp32 ``x`` [N, heads, D] by ``cs`` [N, D/2, 2]: products and sums rounded on their own."""
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    re, im = x[..., ::2], x[..., 1::2]
    return torch.stack([re * c - im * s, re * s + im * c], -1).flatten(-2)


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(values, exponent bytes) of fp32 vectors ``x`` [..., D]: the nearest of e4m3 * 2^e, ties to the even code, in
    float64, of those that bf16 has (at e = 120 not 256 and more); infinities and NaN as NaN."""
    d = x.double()
    top = torch.where(d.isfinite(), d.abs(), 0.0).amax(-1, keepdim=True)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 121):  # the least e with top <= 448 * 2^e
        e = torch.where(top > E4M3_MAX * 2.0 ** k, float(k + 1), e)
    e = torch.where(top == 0, 0.0, e)
    grid = e4m3_values().to(x.device)
    y = d.abs() / torch.exp2(e)
    finite = torch.where(y.isfinite(), y, 0.0)
    hi = torch.searchsorted(grid, finite).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = grid[hi] - finite, finite - grid[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    code = torch.where(e == 120, code.clamp(max=int((grid == 240).nonzero())), code)
    out = torch.where(y.isfinite(), grid[code] * torch.exp2(e) * torch.sign(d), float("nan"))
    return out, (e[..., 0] + 127).to(torch.uint8)


def cell(table: torch.Tensor, page: int, pages: int, slot: int, pos: int):
    """(page, offset) of a position, None outside the cache."""
    if not (0 <= slot < table.size(0) and 0 <= pos < table.size(1) * page):
        return None
    at = int(table[slot, pos // page])
    return (at, pos % page) if 0 <= at < pages else None


def softmax_product(q, k, v, scale: float, limit):
    """q [T, D], k / v [N, D]; query t sees keys [0, limit[t]).  (out, sum of weights |v|), float64; none: zeros.  Keys and
    values that a query does not see take no part, whatever they hold."""
    q, k, v = q.double(), k.double(), v.double()
    limit = torch.tensor([int(x) for x in limit], device=q.device)
    seen = torch.arange(k.size(0), device=q.device) < limit[:, None]
    w = torch.softmax(((q @ k.T) * scale).masked_fill(~seen, -torch.inf), 1).masked_fill(~seen, 0.0)
    fine = v.isfinite()
    kept = v.masked_fill(~fine, 0.0)
    out, size = w @ kept, w @ kept.abs()
    for n in (~fine).any(1).nonzero().flatten().tolist():  # an infinity or NaN, to the queries that see it
        out[seen[:, n]] += v[n].masked_fill(fine[n], 0.0)
        size[seen[:, n]] += v[n].masked_fill(fine[n], 0.0).abs()
    return out, size


def cached(pages: torch.Tensor, scale, table_row: torch.Tensor, n: int, head: int) -> torch.Tensor:
    """The first ``n`` positions of a row for one kv head, float64 [n, D]."""
    page = pages.size(2)
    ids = table_row[: -(-n // page)].long()
    if scale is None:
        x = pages[ids, head].double()
    else:
        x = pages.view(torch.uint8)[ids, head].view(torch.float8_e4m3fn).double()
        x = x * torch.exp2(scale[ids, head].double() - 127)[..., None]
    return x.flatten(0, 1)[:n]


def paged_attention(q, k_pages, v_pages, table, lengths, tokens: int, scale: float, k_scale=None, v_scale=None):
    """(out, size) [B*T, H, D] float64."""
    heads, kv = q.size(1), k_pages.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    room = table.size(1) * k_pages.size(2)
    for b in range(q.size(0) // tokens):
        n = min(max(int(lengths[b]), 0), room)
        last = min(n + tokens - 1, room)
        rows = slice(b * tokens, (b + 1) * tokens)
        for h in range(heads):
            k = cached(k_pages, k_scale, table[b], last, h // (heads // kv))
            v = cached(v_pages, v_scale, table[b], last, h // (heads // kv))
            out[rows, h], size[rows, h] = softmax_product(q[rows, h], k, v, scale,
                                                          [min(n + i, last) for i in range(tokens)])
    return out, size


def packed_attention(q, k, v, starts, k_starts, scale: float):
    """(out, size) [N, H, D] float64, zeros in rows of no sequence."""
    heads, kv = q.size(1), k.size(1)
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(out)
    for s in range(len(starts) - 1):
        rows, keys = slice(starts[s], starts[s + 1]), slice(k_starts[s], k_starts[s + 1])
        nq, nk = starts[s + 1] - starts[s], k_starts[s + 1] - k_starts[s]
        for h in range(heads):
            out[rows, h], size[rows, h] = softmax_product(q[rows, h], k[keys, h // (heads // kv)],
                                                          v[keys, h // (heads // kv)], scale,
                                                          [i + 1 + nk - nq for i in range(nq)])
    return out, size

"""The paged cache's operators without a GPU: the oracle's own facts, and what the entry points refuse."""

import ctypes

import pytest
import torch

from oracle import paged as op
from omniasr_trt_amd import _lib, kernels

FAKE = ctypes.c_void_p(0x10000)  # never dereferenced: every call below fails its checks before any launch


def test_e4m3_values_are_torch_s():
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(op.e4m3_values(), codes)


def test_quantise_against_torch_s_rounding():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(64, 128, generator=g) * torch.exp2(torch.randint(-40, 40, (64, 1), generator=g).float())
    x[0] = 0.0
    x[1, 5] = 448.0 * 2 ** 60
    values, byte = op.quantise(x)
    scale = torch.exp2(byte.double() - 127)[:, None]
    assert torch.equal(values, (x.double() / scale).float().to(torch.float8_e4m3fn).double() * scale)
    assert byte[0] == 127 and (values[0] == 0).all()
    assert byte[1] == 187 and values[1, 5] == 448.0 * 2 ** 60
    top = x.double().abs().amax(1)
    assert (top <= 448 * scale[:, 0]).all() and (top[1:] > 224 * scale[1:, 0]).all()  # the least such power of two
    # the kept values are bf16 numbers, and half a step of e4m3 away at most
    assert torch.equal(values.to(torch.bfloat16).double(), values)
    assert ((values - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, scale * 2.0 ** -10)).all()


def test_quantise_keeps_what_is_not_finite_apart():
    x = torch.ones(3, 128)
    x[0, 3], x[1, 4], x[2, 5] = float("inf"), float("nan"), -float("inf")
    values, byte = op.quantise(x)
    assert byte.tolist() == [119] * 3  # 1 <= 448 * 2^-8
    assert values.isnan().sum().item() == 3 and (values[~values.isnan()] == 1).all()


def _cache(kv=2, page=16, dim=128, rows=3, width=4, fp8=True):
    pages = torch.zeros(8, kv, page, dim).to(torch.float8_e4m3fn if fp8 else torch.bfloat16)
    scale = torch.full((8, kv, page), 127, dtype=torch.uint8) if fp8 else None
    return pages, pages.clone(), torch.zeros(rows, width, dtype=torch.int32), scale


def _refused(call, what, *args, **kw):
    with pytest.raises((ValueError, RuntimeError), match=what):
        call(*args, **kw)


@pytest.mark.parametrize("change,what", [
    (dict(k=torch.zeros(8, 2, 16, 64).to(torch.float8_e4m3fn)), "one dtype"),
    (dict(k=torch.zeros(8, 2, 16, 128)), "one dtype"),
    (dict(scale=None), "k_scale"),
    (dict(scale=torch.zeros(8, 2, 16, dtype=torch.int8)), "k_scale"),
    (dict(scale=torch.zeros(8, 2, 8, dtype=torch.uint8)), "k_scale"),
    (dict(table=torch.zeros(3, 4, dtype=torch.long)), "table"),
    (dict(table=torch.zeros(4, 3, dtype=torch.int32).t()), "table"),
    ({}, "on the GPU"),
])
def test_cache_refusals(change, what):
    k, v, table, scale = _cache()
    k, scale, table = change.get("k", k), change.get("scale", scale), change.get("table", table)
    at = torch.zeros(3, dtype=torch.long)
    _refused(kernels.paged_read, what, k, v, table, at, at, k_scale=scale, v_scale=scale)
    qkv = torch.zeros(3, (4 + 2 * 2) * 128, dtype=torch.bfloat16)
    _refused(kernels.rope_kv_paged, what, qkv, torch.zeros(64, 64, 2), at, k, v, table, 4, at, k_scale=scale,
             v_scale=scale)
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    _refused(kernels.paged_attention, what, q, k, v, table, at, 1, 0.1, k_scale=scale, v_scale=scale)


def test_page_and_head_dim_refusals():
    for shape in ((8, 2, 24, 128), (8, 2, 8, 128), (8, 2, 512, 128), (8, 2, 16, 64), (8, 2, 16, 96)):
        pages = torch.zeros(shape, dtype=torch.bfloat16)
        _refused(kernels.paged_read, "pages of 16", pages, pages, torch.zeros(3, 4, dtype=torch.int32),
                 torch.zeros(1, dtype=torch.long), torch.zeros(1, dtype=torch.long))
    k, v, table, _ = _cache(fp8=False)
    at = torch.zeros(3, dtype=torch.long)
    _refused(kernels.paged_read, "e4m3 pages only", k, v, table, at, at, k_scale=torch.zeros(8, 2, 16, dtype=torch.uint8))


def test_call_refusals():
    k, v, table, scale = _cache()
    kw = {"k_scale": scale, "v_scale": scale}
    at, cs = torch.zeros(3, dtype=torch.long), torch.zeros(64, 64, 2)
    _refused(kernels.rope_kv_paged, "qkv", torch.zeros(3, 8 * 128, dtype=torch.bfloat16), cs, at, k, v, table, 5, **kw)
    _refused(kernels.rope_kv_paged, "bfloat16", torch.zeros(3, 8 * 128), cs, at, k, v, table, 4, **kw)
    q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    _refused(kernels.paged_attention, "tokens", q, k, v, table, at, 17, 0.1, **kw)
    _refused(kernels.paged_attention, "tokens", q, k, v, table, at, 2, 0.1, **kw)
    _refused(kernels.paged_attention, "tokens", q, k, v, table, at, 0, 0.1, **kw)
    _refused(kernels.paged_attention, "multiple", torch.zeros(3, 5, 128, dtype=torch.bfloat16), k, v, table, at, 1, 0.1,
             **kw)
    _refused(kernels.paged_attention, "B rows", torch.zeros(4, 4, 128, dtype=torch.bfloat16), k, v, table, at, 1, 0.1,
             **kw)
    kk = torch.zeros(7, 2, 128, dtype=torch.bfloat16)
    starts = torch.tensor([0, 3])
    _refused(kernels.packed_attention, "D = 128", torch.zeros(3, 4, 64, dtype=torch.bfloat16), kk, kk, starts, 3, 0.1)
    _refused(kernels.packed_attention, "k / v", q, kk, kk[:6], starts, 3, 0.1)
    _refused(kernels.packed_attention, "multiple", q, kk[:, :1].repeat(1, 3, 1), kk[:, :1].repeat(1, 3, 1), starts, 3, 0.1)
    _refused(kernels.packed_attention, "unit stride", q, kk.transpose(1, 2).contiguous().transpose(1, 2), kk, starts, 3, 0.1)
    _refused(kernels.packed_attention, "on the GPU", q, kk, kk, starts, 3, 0.1)


def test_shared_memory_of_tensors():
    x = torch.zeros(6, 4, 8)
    assert kernels._share_memory(x, x) and kernels._share_memory(x[2:4], x[3:]) and kernels._share_memory(x[3:], x[:, :1])
    assert not kernels._share_memory(x[:3], x[3:]) and not kernels._share_memory(x[3:], x[:3])
    assert not kernels._share_memory(x[0, :2], x[0, 2:]) and not kernels._share_memory(x, x[:0])
    assert not kernels._share_memory(x, torch.zeros_like(x))


def test_c_abi_refusals_before_launch():
    lib = _lib.load()
    other = [ctypes.c_void_p(0x10000 * i) for i in (2, 3, 4)]
    pages = [FAKE, *other, 64, 16, FAKE, 8]  # k, v, scales, pages, page, table, its row stride
    rope = [FAKE, 1024, FAKE, 8192, FAKE, None, None, FAKE, None, *pages, 3, 8, 5, 4, 2, 128, _lib.E4M3, _lib.BF16, None]

    def changed(args, at, value):
        return [*args[:at], value, *args[at + 1:]]

    assert lib.omni_rope_kv_paged(*changed(rope, 24, _lib.F32)) == -2
    assert lib.omni_rope_kv_paged(*changed(rope, 23, _lib.F32)) == -2
    assert lib.omni_rope_kv_paged(*changed(rope, 22, 64)) == -3
    assert lib.omni_rope_kv_paged(*changed(rope, 14, 24)) == -3  # a page that is no power of two
    assert lib.omni_rope_kv_paged(*changed(rope, 11, None)) == -1  # e4m3 without scales
    assert lib.omni_rope_kv_paged(*changed(rope, 1, 1016)) == -1  # a row shorter than its vectors
    assert lib.omni_rope_kv_paged(*changed(rope, 16, 7)) == -1  # table rows shorter than their width
    assert lib.omni_rope_kv_paged(*changed(rope, 19, 0)) == 0
    assert lib.omni_rope_kv_paged(*changed(rope, 10, FAKE)) == -1  # K and V in the same pages
    assert lib.omni_rope_kv_paged(*changed(rope, 12, rope[11])) == -1
    assert lib.omni_rope_kv_paged(*changed(rope, 19, 2 ** 24)) == -3
    read = [*pages, 3, 8, FAKE, FAKE, 5, 2, 128, _lib.E4M3, FAKE, FAKE, None]
    assert lib.omni_paged_read(*changed(read, 5, 512)) == -3
    assert lib.omni_paged_read(*changed(read, 10, None)) == -1
    assert lib.omni_paged_read(*changed(read, 12, 0)) == 0
    assert lib.omni_paged_read(*changed(read, 12, 2 ** 24)) == -3
    ws = lib.omni_paged_attention_workspace(3, 2, 4, 2, 128, 16, 8)
    assert ws > 0
    attn = [FAKE, *pages, 8, FAKE, 3, 2, 4, 2, 128, 0.1, FAKE, FAKE, ws, _lib.E4M3, _lib.BF16, None]
    assert lib.omni_paged_attention(*changed(attn, 12, 17)) == -3
    assert lib.omni_paged_attention(*changed(attn, 14, 3)) == -1
    assert lib.omni_paged_attention(*changed(attn, 16, 0.0)) == -1
    assert lib.omni_paged_attention(*changed(attn, 16, float("nan"))) == -1
    assert lib.omni_paged_attention(*changed(attn, 19, ws - 1)) == -4
    assert lib.omni_paged_attention(*changed(attn, 18, ctypes.c_void_p(0x10010))) == -4
    assert lib.omni_paged_attention(*changed(attn, 11, 0)) == 0
    assert lib.omni_paged_attention(*changed(attn, 11, 2 ** 23)) == -3
    packed = [FAKE, FAKE, FAKE, 256, 128, 256, 128, FAKE, other[0], 2, 9, 9, 5, 4, 2, 128, 0.1, FAKE]
    packed[11] = 4000
    ws = lib.omni_packed_attention_workspace(2, 4000, 5, 4, 2, 128)
    assert ws > 0 and lib.omni_packed_attention_workspace(65, 4000, 5, 4, 2, 128) == 0
    packed += [FAKE, ws, _lib.BF16, None]
    assert lib.omni_packed_attention(*changed(packed, 19, ws - 1)) == -4
    assert lib.omni_packed_attention(*changed(packed, 18, None)) == -4
    assert lib.omni_packed_attention(*changed(packed, 20, _lib.F32)) == -2
    assert lib.omni_packed_attention(*changed(packed, 15, 64)) == -3
    assert lib.omni_packed_attention(*changed(packed, 3, 252)) == -1
    assert lib.omni_packed_attention(*changed(packed, 16, -1.0)) == -1
    assert lib.omni_packed_attention(*changed(packed, 1, ctypes.c_void_p(0x10008))) == -1
    assert lib.omni_packed_attention(*changed(packed, 9, 0)) == 0
    assert lib.omni_packed_attention(*changed(packed, 9, 65536)) == -3
    big = [*packed[:9], 65535, 2 ** 30, 2 ** 30, 2 ** 24, 4, 4, 512, *packed[16:]]  # 65535 x 2^18 x 4 blocks
    assert lib.omni_packed_attention(*big) == -3
    assert lib.omni_packed_attention(*big[:9], 1, 2 ** 30, 2 ** 30, 2 ** 30, 4, 1, 128, *big[16:]) == -3  # 2^25 along x


def test_packed_attention_workspace_of_every_size():
    lib = _lib.load()
    most = max(lib.omni_packed_attention_workspace(sequences, keys, longest, kv * group, kv, dim)
               for sequences in (1, 2, 3, 9, 40, 64) for keys in (500, 704, 1472, 1473, 9000, 200000)
               for longest in (1, 64, 65, 128, 257, 1000, 5000) for kv in (1, 3, 8, 25) for group in (1, 2, 4, 7)
               for dim in (128, 256, 512))
    assert 32 << 20 < most <= 66 << 20

"""CPU: calls of the 8-bit cache's and the norms' C entry points that are right but for one argument are refused, and for that argument: the same call with
it put right gets as far as the device.  The addresses are made up, so none of this meets a device."""
import ctypes

import pytest
import torch

EINVAL, EUNSUPPORTED, EWORKSPACE = 1, 2, 5
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no kernel can start")


@pytest.fixture(scope="module")
def lib():
    from minfer.kernels.torch_ext import _lib
    return _lib


def filled(p, args):
    for name, v in args.items():
        if isinstance(v, tuple):
            for i, x in enumerate(v):
                getattr(p, name)[i] = x
        else:
            setattr(p, name, v)
    return p


def check(struct, entry, right, bad, code):
    call = lambda args: entry(ctypes.byref(filled(struct(), args)), None)  # noqa: E731
    assert call(right) not in (EINVAL, EUNSUPPORTED, EWORKSPACE), "the call without the bad argument is refused as well"
    assert call({**right, **bad}) == code


# q [2, 3, 8, 128] and k, v [2, 3, 2, 128]; caches [2, 2, 64, 128] with a scale for each block of 64 rows, or three pages of 64 rows
NORM = dict(q=0x10000, k=0x20000, v=0x30000, start=0x38000, batch=2, seq=3, n_heads=8, n_kv_heads=2, head_dim=128, rotary_dim=128, freq_base=10000.0, eps=1e-6,
            max_len=64, q_stride=(4096, 1024, 128), kv_stride=(768, 256, 128))
WEIGHTED = dict(NORM, q_weight=0x40000, k_weight=0x41000)
C16 = dict(NORM, k_cache=0x50000, v_cache=0x60000, cache_stride=(2 * 64 * 128, 64 * 128, 128))
C8 = dict(C16, k_scale=0x70000, v_scale=0x71000, scale_stride=(2, 1), cache_format=2, block_size=64)
P16 = dict(C16, block_table=0x72000, page_size=64, table_stride=1, n_pages=3)
P8 = dict(C8, block_table=0x72000, page_size=64, table_stride=1, n_pages=3)
HOST = dict(C16, start=None, start_pos=10)          # the position comes from the host


@pytest.mark.parametrize("right,bad,code", [
    (NORM, dict(batch=0), EINVAL), (NORM, dict(seq=0), EINVAL), (NORM, dict(seq=-1), EINVAL), (NORM, dict(head_dim=120), EINVAL), (NORM, dict(head_dim=0), EINVAL),
    (NORM, dict(head_dim=272), EUNSUPPORTED), (NORM, dict(seq=1 << 30), EINVAL), (NORM, dict(dtype=2), EINVAL), (NORM, dict(dtype=-1), EINVAL),
    (NORM, dict(style=2), EINVAL), (NORM, dict(style=-1), EINVAL), (NORM, dict(rotary_dim=144), EINVAL), (NORM, dict(rotary_dim=12), EINVAL),
    (dict(NORM, style=1, rotary_dim=32), dict(rotary_dim=24), EINVAL), (NORM, dict(rotary_dim=-8), EINVAL), (NORM, dict(freq_base=0.0), EINVAL),
    (NORM, dict(freq_base=-1.0), EINVAL), (NORM, dict(freq_base=float("nan")), EINVAL), (NORM, dict(freq_base=float("inf")), EINVAL),
    (NORM, dict(q=0x10008), EINVAL), (NORM, dict(k=0x20008), EINVAL), (C16, dict(v=0x30008), EINVAL), (NORM, dict(n_heads=0), EINVAL),
    (NORM, dict(n_kv_heads=0), EINVAL), (NORM, dict(n_heads=65536), EUNSUPPORTED), (NORM, dict(n_kv_heads=65536), EUNSUPPORTED),
    *[(NORM, {s: tuple(x + (4 if i == j else 0) for j, x in enumerate(NORM[s]))}, EINVAL) for s in ("q_stride", "kv_stride") for i in range(3)],
    *[(NORM, {s: tuple(-x if i == j else x for j, x in enumerate(NORM[s]))}, EINVAL) for s in ("q_stride", "kv_stride") for i in range(3)],
    (WEIGHTED, dict(q_weight=None), EINVAL), (WEIGHTED, dict(k_weight=None), EINVAL), (WEIGHTED, dict(q_weight=0x40008), EINVAL),
    (WEIGHTED, dict(k_weight=0x41008), EINVAL), (WEIGHTED, dict(weight_dtype=3), EINVAL), (WEIGHTED, dict(weight_dtype=-1), EINVAL),
    (WEIGHTED, dict(weight_stride=(4, 0)), EINVAL), (WEIGHTED, dict(weight_stride=(0, 4)), EINVAL), (WEIGHTED, dict(weight_stride=(-8, 0)), EINVAL),
    (dict(WEIGHTED, weight_dtype=2, weight_stride=(132, 4)), dict(weight_stride=(132, 2)), EINVAL),
    (WEIGHTED, dict(eps=-1.0), EINVAL), (WEIGHTED, dict(eps=float("nan")), EINVAL),
    (HOST, dict(start_pos=-1), EINVAL), (HOST, dict(start_pos=62), EINVAL), (dict(NORM, start=None, start_pos=0x7FFFFFFC), dict(start_pos=0x7FFFFFFD), EINVAL),
    (NORM, dict(start=0x38002), EINVAL), (NORM, dict(flags=1), EUNSUPPORTED), (NORM, dict(status=0x1002), EINVAL),
    (NORM, dict(cache_format=1), EINVAL), (NORM, dict(cache_format=2), EINVAL), (NORM, dict(block_table=0x72000), EINVAL), (NORM, dict(k_cache=0x50000), EINVAL),
    (C16, dict(v_cache=None), EINVAL), (C16, dict(k_cache=None), EINVAL), (C16, dict(v=None), EINVAL), (C16, dict(k=None), EINVAL), (C16, dict(max_len=0), EINVAL),
    (C16, dict(k_cache=0x50008), EINVAL), (C16, dict(v_cache=0x60008), EINVAL), (C16, dict(cache_format=1), EINVAL),
    *[(C16, dict(cache_stride=tuple(x + (4 if i == j else 0) for j, x in enumerate(C16["cache_stride"]))), EINVAL) for i in range(3)],
    *[(C8, dict(cache_stride=tuple(x + (8 if i == j else 0) for j, x in enumerate(C16["cache_stride"]))), EINVAL) for i in range(3)],
    *[(C8, dict(cache_stride=tuple(-x if i == j else x for j, x in enumerate(C16["cache_stride"]))), EINVAL) for i in range(3)],
    (dict(C8, head_dim=64, rotary_dim=64), dict(head_dim=96), EUNSUPPORTED), (C8, dict(head_dim=256), EUNSUPPORTED),
    (C8, dict(block_size=48), EINVAL), (C8, dict(block_size=0), EINVAL), (C8, dict(block_size=256), EINVAL), (C8, dict(block_size=8), EINVAL),
    (C8, dict(k_scale=None), EINVAL), (C8, dict(v_scale=None), EINVAL), (C8, dict(k_scale=0x70002), EINVAL), (C8, dict(v_scale=0x71002), EINVAL),
    (C8, dict(scale_stride=(-2, 1)), EINVAL), (C8, dict(scale_stride=(2, -1)), EINVAL),
    (dict(P8, page_size=128, block_size=128), dict(page_size=64), EINVAL),                      # a page holds no whole block
    (P16, dict(page_size=0), EINVAL), (P16, dict(table_stride=0), EINVAL), (P16, dict(n_pages=0), EINVAL), (P16, dict(block_table=0x72002), EINVAL),
    (P16, dict(max_len=65), EINVAL), (P8, dict(page_size=0), EINVAL), (P8, dict(table_stride=0), EINVAL), (P8, dict(n_pages=0), EINVAL),
    (P8, dict(block_table=0x72002), EINVAL), (P8, dict(max_len=65), EINVAL)])
def test_norm_rope(lib, right, bad, code):
    check(lib.NormRopeParams, lib.lib.minfer_attn_norm_rope_append, right, bad, code)


DEC = dict(q=0x10000, k_cache=0x20000, v_cache=0x30000, k_scale=0x40000, v_scale=0x41000, lens=0x42000, out=0x50000, batch=2, n_heads=8, n_kv_heads=2, max_len=100,
           head_dim=128, cache_format=2, block_size=16, q_stride=(1024, 128), out_stride=(1024, 128), kv_stride=(2 * 100 * 128, 100 * 128, 128), scale_stride=(14, 7))
DEC_P = dict(DEC, block_table=0x60000, page_size=48, table_stride=3, n_pages=9, max_len=144)
LONG = dict(DEC, batch=1, n_heads=8, n_kv_heads=1, max_len=1 << 18, workspace=0x100000, workspace_bytes=1 << 30)


@pytest.mark.parametrize("right,bad,code", [
    *[(DEC, {name: None}, EINVAL) for name in ("q", "k_cache", "v_cache", "k_scale", "v_scale", "lens", "out")],
    *[(DEC, {name: DEC[name] + 8}, EINVAL) for name in ("q", "k_cache", "v_cache", "out")], *[(DEC, {name: DEC[name] + 2}, EINVAL) for name in ("k_scale", "v_scale", "lens")],
    (DEC, dict(batch=0), EINVAL), (DEC, dict(n_heads=0), EINVAL), (DEC, dict(n_kv_heads=0), EINVAL), (DEC, dict(max_len=0), EINVAL), (DEC, dict(n_heads=9), EINVAL),
    (DEC, dict(n_heads=34), EUNSUPPORTED), (DEC, dict(batch=65536), EUNSUPPORTED), (dict(DEC, n_heads=65535, n_kv_heads=65535), dict(n_heads=65536, n_kv_heads=65536), EUNSUPPORTED),
    (DEC, dict(head_dim=96), EUNSUPPORTED), (DEC, dict(dtype=2), EINVAL), (DEC, dict(cache_format=0), EINVAL), (DEC, dict(cache_format=1), EINVAL),
    (DEC, dict(block_size=8), EINVAL), (DEC, dict(q_stride=(4, 128)), EINVAL), (DEC, dict(q_stride=(1024, -8)), EINVAL), (DEC, dict(out_stride=(1024, 132)), EINVAL),
    (DEC, dict(out_stride=(-1024, 128)), EINVAL), *[(DEC, dict(kv_stride=tuple(x + (8 if i == j else 0) for j, x in enumerate(DEC["kv_stride"]))), EINVAL) for i in range(3)],
    (DEC, dict(scale_stride=(14, -7)), EINVAL), (DEC, dict(scale_stride=(-14, 7)), EINVAL), (DEC, dict(softmax_scale=-1.0), EINVAL), (DEC, dict(softmax_scale=float("nan")), EINVAL),
    (DEC, dict(flags=1), EUNSUPPORTED), (DEC, dict(status=0x1002), EINVAL),
    (DEC_P, dict(page_size=56), EINVAL), (DEC_P, dict(page_size=32), EINVAL), (DEC_P, dict(table_stride=2), EINVAL), (DEC_P, dict(n_pages=0), EINVAL),
    (DEC_P, dict(block_table=0x60002), EINVAL), (DEC_P, dict(max_len=145), EINVAL), (dict(DEC_P, block_size=16), dict(block_size=32), EINVAL),
    (LONG, dict(workspace_bytes=4096), EWORKSPACE), (LONG, dict(workspace=0x100004), EWORKSPACE)])
def test_decode(lib, right, bad, code):
    check(lib.DecodeB8Params, lib.lib.minfer_attn_decode_b8, right, bad, code)


READ = dict(k_cache=0x10000, v_cache=0x20000, k_scale=0x30000, v_scale=0x31000, lens=0x32000, k_out=0x40000, v_out=0x50000, batch=2, n_kv_heads=2, max_len=100, out_rows=50,
            head_dim=64, cache_format=3, block_size=32, cache_stride=(2 * 100 * 64, 100 * 64, 64), scale_stride=(8, 4), out_stride=(2 * 50 * 64, 50 * 64, 64))
READ_P = dict(READ, block_table=0x60000, page_size=32, table_stride=4, n_pages=9, max_len=128)


@pytest.mark.parametrize("right,bad,code", [
    *[(READ, {name: None}, EINVAL) for name in ("k_cache", "v_cache", "k_scale", "v_scale", "lens", "k_out", "v_out")],
    *[(READ, {name: READ[name] + 8}, EINVAL) for name in ("k_cache", "v_cache", "k_out", "v_out")], *[(READ, {name: READ[name] + 2}, EINVAL) for name in ("k_scale", "v_scale", "lens")],
    (READ, dict(batch=0), EINVAL), (READ, dict(n_kv_heads=0), EINVAL), (READ, dict(max_len=0), EINVAL), (READ, dict(out_rows=0), EINVAL), (READ, dict(dtype=2), EINVAL),
    (READ, dict(cache_format=0), EINVAL), (READ, dict(cache_format=1), EINVAL), (READ, dict(block_size=33), EINVAL), (READ, dict(head_dim=72), EUNSUPPORTED),
    *[(READ, dict(out_stride=tuple(x + (4 if i == j else 0) for j, x in enumerate(READ["out_stride"]))), EINVAL) for i in range(3)],
    *[(READ, dict(cache_stride=tuple(x + (8 if i == j else 0) for j, x in enumerate(READ["cache_stride"]))), EINVAL) for i in range(3)],
    (READ, dict(scale_stride=(-8, 4)), EINVAL), (READ, dict(scale_stride=(8, -4)), EINVAL), (READ, dict(flags=2), EUNSUPPORTED), (READ, dict(status=0x1002), EINVAL),
    (READ, dict(batch=1 << 29), EINVAL), (dict(READ, batch=1, n_kv_heads=1, max_len=0x7FFFFFFF, out_rows=0x7FFFFFFF - 128), dict(out_rows=0x7FFFFFFF), EINVAL),
    (READ_P, dict(page_size=16), EINVAL), (READ_P, dict(page_size=48), EINVAL), (READ_P, dict(table_stride=3), EINVAL), (READ_P, dict(n_pages=0), EINVAL),
    (READ_P, dict(block_table=0x60002), EINVAL), (READ_P, dict(max_len=129), EINVAL)])
def test_read(lib, right, bad, code):
    check(lib.KvReadB8Params, lib.lib.minfer_attn_kv_read_b8, right, bad, code)

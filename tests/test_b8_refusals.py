"""CPU: the C entry points of the 8-bit cache and of the norms refuse bad arguments before touching a device; the ops have no CPU path."""
import ctypes

import pytest
import torch

EINVAL, EUNSUPPORTED, EWORKSPACE = 1, 2, 5


@pytest.fixture(scope="module")
def lib():
    from minfer.kernels.torch_ext import _lib
    return _lib


def norm(lib, **kw):
    p = lib.NormRopeParams()
    p.q = p.k = p.v = 0x1000
    p.batch, p.seq, p.n_heads, p.n_kv_heads, p.head_dim, p.rotary_dim = 2, 3, 8, 2, 128, 128
    p.freq_base, p.eps, p.max_len = 10000.0, 1e-6, 64
    p.start = 0x1000
    for k, v in kw.items():
        if isinstance(v, tuple):
            for i, x in enumerate(v):
                getattr(p, k)[i] = x
        else:
            setattr(p, k, v)
    return lib.lib.minfer_attn_norm_rope_append(ctypes.byref(p), None)


B8 = dict(k_cache=0x1000, v_cache=0x1000, k_scale=0x1000, v_scale=0x1000, cache_format=2, block_size=64)


@pytest.mark.parametrize("bad,code", [
    (dict(q=None, k=None), EINVAL), (dict(batch=0), EINVAL), (dict(seq=0), EINVAL), (dict(head_dim=120), EINVAL), (dict(head_dim=272), EUNSUPPORTED),
    (dict(batch=1 << 16, seq=1 << 15), EINVAL), (dict(dtype=2), EINVAL), (dict(style=2), EINVAL), (dict(rotary_dim=144), EINVAL),
    (dict(rotary_dim=12), EINVAL), (dict(style=1, rotary_dim=24), EINVAL), (dict(rotary_dim=-8), EINVAL), (dict(freq_base=0.0), EINVAL),
    (dict(freq_base=float("nan")), EINVAL), (dict(freq_base=float("inf")), EINVAL), (dict(q=0x1008), EINVAL), (dict(q_stride=(4, 0, 0)), EINVAL),
    (dict(kv_stride=(0, -8, 0)), EINVAL), (dict(q_weight=0x1000), EINVAL), (dict(k_weight=0x1000), EINVAL),
    (dict(q_weight=0x1000, k_weight=0x1008), EINVAL), (dict(q_weight=0x1000, k_weight=0x1000, weight_dtype=3), EINVAL),
    (dict(q_weight=0x1000, k_weight=0x1000, weight_stride=(4, 8)), EINVAL), (dict(q_weight=0x1000, k_weight=0x1000, eps=-1.0), EINVAL),
    (dict(q_weight=0x1000, k_weight=0x1000, eps=float("nan")), EINVAL), (dict(start=None, start_pos=-1), EINVAL),
    (dict(start=None, start_pos=0x7FFFFFFF), EINVAL), (dict(start=0x1002), EINVAL), (dict(flags=1), EUNSUPPORTED), (dict(status=0x1001), EINVAL),
    (dict(k_cache=0x1000), EINVAL), (dict(cache_format=1), EINVAL), (dict(cache_format=2), EINVAL), (dict(block_table=0x1000), EINVAL),
    (dict(k_cache=0x1000, v_cache=0x1000, v=None), EINVAL), (dict(k_cache=0x1000, v_cache=0x1000, cache_stride=(4, 8, 8)), EINVAL),
    (dict(k_cache=0x1000, v_cache=0x1000, start=None, start_pos=62), EINVAL), (dict(k_cache=0x1000, v_cache=0x1000, max_len=0), EINVAL),
    ({**B8, "head_dim": 96, "rotary_dim": 96}, EUNSUPPORTED), ({**B8, "block_size": 48}, EINVAL), ({**B8, "block_size": 0}, EINVAL),
    ({**B8, "block_size": 256}, EINVAL), ({**B8, "k_scale": None}, EINVAL), ({**B8, "v_scale": 0x1002}, EINVAL),
    ({**B8, "cache_stride": (8, 16, 16)}, EINVAL), ({**B8, "scale_stride": (-1, 0)}, EINVAL),
    ({**B8, "block_table": 0x1000, "page_size": 32, "table_stride": 2, "n_pages": 4}, EINVAL),     # a page holds no whole block
    ({**B8, "block_table": 0x1000, "page_size": 64, "table_stride": 0, "n_pages": 4}, EINVAL),
    ({**B8, "block_table": 0x1000, "page_size": 64, "table_stride": 1, "n_pages": 0}, EINVAL),
    ({**B8, "block_table": 0x1002, "page_size": 64, "table_stride": 1, "n_pages": 4}, EINVAL),
    ({**B8, "block_table": 0x1000, "page_size": 64, "table_stride": 1, "n_pages": 4, "max_len": 65}, EINVAL)])
def test_norm_rope_refusals(lib, bad, code):
    assert norm(lib, **bad) == code


def fill(p, base, changes):
    for k, v in {**base, **changes}.items():
        if isinstance(v, tuple):
            for i, x in enumerate(v):
                getattr(p, k)[i] = x
        else:
            setattr(p, k, v)
    return p


DEC = dict(q=0x1000, k_cache=0x1000, v_cache=0x1000, k_scale=0x1000, v_scale=0x1000, lens=0x1000, out=0x1000, batch=2, n_heads=8, n_kv_heads=2,
           max_len=100, head_dim=128, cache_format=2, block_size=16)


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), EINVAL), (dict(k_scale=None), EINVAL), (dict(lens=None), EINVAL), (dict(batch=0), EINVAL), (dict(max_len=0), EINVAL),
    (dict(n_heads=9), EINVAL), (dict(n_heads=34), EUNSUPPORTED), (dict(head_dim=96), EUNSUPPORTED), (dict(dtype=2), EINVAL), (dict(cache_format=0), EINVAL),
    (dict(cache_format=1), EINVAL), (dict(block_size=8), EINVAL), (dict(q=0x1004), EINVAL), (dict(k_cache=0x1008), EINVAL), (dict(v_scale=0x1001), EINVAL),
    (dict(kv_stride=(16, 8, 16)), EINVAL), (dict(q_stride=(4, 8)), EINVAL), (dict(scale_stride=(0, -1)), EINVAL), (dict(softmax_scale=-1.0), EINVAL),
    (dict(softmax_scale=float("nan")), EINVAL), (dict(batch=70000), EUNSUPPORTED), (dict(flags=1), EUNSUPPORTED), (dict(status=0x1002), EINVAL),
    (dict(block_table=0x1000, page_size=24, table_stride=9, n_pages=9), EINVAL), (dict(block_table=0x1000, page_size=32, table_stride=3, n_pages=9), EINVAL)])
def test_decode_refusals(lib, bad, code):
    assert lib.lib.minfer_attn_decode_b8(ctypes.byref(fill(lib.DecodeB8Params(), DEC, bad)), None) == code


READ = dict(k_cache=0x1000, v_cache=0x1000, k_scale=0x1000, v_scale=0x1000, lens=0x1000, k_out=0x1000, v_out=0x1000, batch=2, n_kv_heads=2, max_len=100,
            out_rows=50, head_dim=64, cache_format=3, block_size=32)


@pytest.mark.parametrize("bad,code", [
    (dict(k_out=None), EINVAL), (dict(out_rows=0), EINVAL), (dict(n_kv_heads=0), EINVAL), (dict(dtype=2), EINVAL), (dict(cache_format=0), EINVAL),
    (dict(block_size=33), EINVAL), (dict(head_dim=72), EUNSUPPORTED), (dict(k_out=0x1008), EINVAL), (dict(lens=0x1001), EINVAL),
    (dict(out_stride=(8, 8, 4)), EINVAL), (dict(cache_stride=(16, 16, 8)), EINVAL), (dict(flags=2), EUNSUPPORTED),
    (dict(batch=1 << 20, n_kv_heads=1 << 11), EINVAL), (dict(block_table=0x1000, page_size=16, table_stride=9, n_pages=9), EINVAL)])
def test_read_refusals(lib, bad, code):
    assert lib.lib.minfer_attn_kv_read_b8(ctypes.byref(fill(lib.KvReadB8Params(), READ, bad)), None) == code


def test_null_parameter_blocks(lib):
    for name in ("minfer_attn_norm_rope_append", "minfer_attn_decode_b8", "minfer_attn_kv_read_b8"):
        assert getattr(lib.lib, name)(None, None) == EINVAL


def test_workspace_too_small(lib):
    """Where a shape uses a workspace, one that is too small or unaligned is refused."""
    need = lib.lib.minfer_attn_decode_b8_workspace_bytes(1, 8, 1, 1 << 18, 128)
    assert lib.lib.minfer_attn_decode_b8_workspace_bytes(0, 8, 1, 64, 128) == 0 and lib.lib.minfer_attn_decode_b8_workspace_bytes(1, 8, 1, 64, 96) == 0
    if need:
        shape = dict(batch=1, n_heads=8, n_kv_heads=1, max_len=1 << 18)
        for bad in (dict(workspace=0x1000, workspace_bytes=need - 1), dict(workspace=0x1004, workspace_bytes=need)):
            assert lib.lib.minfer_attn_decode_b8(ctypes.byref(fill(lib.DecodeB8Params(), DEC, {**shape, **bad})), None) == EWORKSPACE


def test_struct_layouts_match_the_header(lib, tmp_path):
    """Sizes and the last fields' offsets of the ctypes structures, against the C compiler's."""
    import os
    import shutil
    import subprocess
    from conftest import ROOT
    cc = shutil.which("gcc") or shutil.which("cc")
    names = {"MinferNormRopeParams": lib.NormRopeParams, "MinferAttnDecodeB8Params": lib.DecodeB8Params, "MinferKvReadB8Params": lib.KvReadB8Params}
    src = tmp_path / "layout.c"
    lines = "".join(f'printf("{n} %zu", sizeof({n}));' + "".join(f'printf(" %zu", offsetof({n}, {f[0]}));' for f in c._fields_) + 'printf("\\n");'
                    for n, c in names.items())
    src.write_text(f'#include <stdio.h>\n#include <stddef.h>\n#include "{os.path.join(ROOT, "include", "minfer_attn.h")}"\nint main(void) {{ {lines} return 0; }}\n')
    subprocess.run([cc, str(src), "-o", str(tmp_path / "layout")], check=True)
    for line in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True, check=True).stdout.splitlines():
        n, *sizes = line.split()
        assert [int(x) for x in sizes] == [ctypes.sizeof(names[n])] + [getattr(names[n], f[0]).offset for f in names[n]._fields_], n


def test_no_cpu_path():
    from minfer.kernels import KernelBackend
    k = KernelBackend("torch_ext")
    q, kv = torch.zeros(1, 1, 4, 64, dtype=torch.float16), torch.zeros(1, 1, 2, 64, dtype=torch.float16)
    c, s, n, w = torch.zeros(1, 2, 64, 64, dtype=torch.int8), torch.zeros(1, 2, 4), torch.zeros(1, dtype=torch.int32), torch.ones(64)
    out16 = torch.zeros(1, 2, 64, 64, dtype=torch.float16)
    for call in (lambda: k.qk_norm_rope(64, 1e4, 0, 1e-6, q, kv, w, w, n), lambda: k.rope_kv_append_b8(64, 1e4, 0, q, kv, kv, c, c, s, s, 16, n),
                 lambda: k.flash_attn_decode_b8(q.transpose(1, 2), c, c, s, s, 16, n, q.transpose(1, 2).clone()),
                 lambda: k.kv_read_b8(c, c, s, s, 16, n, out16, out16.clone())):
        with pytest.raises(NotImplementedError):
            call()


# These calls are right but for one argument, or altogether, and their addresses are made up: they must never meet a device.
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no kernel can start")

STRIDES = dict(q=0x10000, k=0x20000, v=0x30000, q_stride=(4096, 1024, 128), kv_stride=(768, 256, 128))
CACHES = dict(k_cache=0x40000, v_cache=0x50000, cache_stride=(2 * 64 * 128, 64 * 128, 128))
CACHES_B8 = dict(CACHES, k_scale=0x60000, v_scale=0x61000, scale_stride=(2, 1), cache_format=2, block_size=64)
PAGES_B8 = dict(CACHES_B8, block_table=0x70000, page_size=64, table_stride=1, n_pages=3)


@no_device
@pytest.mark.parametrize("base,bad", [
    ({}, dict(k=0x10000)), ({}, dict(q_stride=(0, 1024, 128))), ({}, dict(q_stride=(4096, 0, 128))), ({}, dict(q_stride=(4096, 1024, 0))),
    ({}, dict(kv_stride=(0, 256, 128))), ({}, dict(kv_stride=(768, 0, 128))), ({}, dict(kv_stride=(768, 256, 0))),
    (CACHES, dict(k=0x10000)), (CACHES, dict(v=0x10000)), (CACHES, dict(v_cache=0x40000)), (CACHES, dict(q_stride=(0, 1024, 128))),
    (CACHES, dict(cache_stride=(0, 64 * 128, 128))), (CACHES, dict(cache_stride=(2 * 64 * 128, 0, 128))), (CACHES, dict(cache_stride=(2 * 64 * 128, 64 * 128, 0))),
    (CACHES_B8, dict(v_cache=0x40000)), (CACHES_B8, dict(v_scale=0x60000)), (CACHES_B8, dict(scale_stride=(0, 1))), (CACHES_B8, dict(scale_stride=(2, 0))),
    (PAGES_B8, dict(cache_stride=(0, 64 * 128, 128))), (PAGES_B8, dict(scale_stride=(0, 1)))])
def test_what_is_written_lies_apart(lib, base, bad):
    """Expanded tensors that are written, and one tensor given twice, are refused; the same call without them gets as far as the device."""
    assert norm(lib, **STRIDES, **base) not in (EINVAL, EUNSUPPORTED)
    assert norm(lib, **{**STRIDES, **base, **bad}) == EINVAL


@no_device
def test_expanded_inputs_are_read(lib):
    """k and v that are only read, and dimensions of one entry, may have any stride."""
    assert norm(lib, **{**STRIDES, **CACHES, "kv_stride": (0, 0, 0)}) not in (EINVAL, EUNSUPPORTED)
    one = dict(batch=1, seq=1, n_heads=1, n_kv_heads=1, q_stride=(0, 0, 0), kv_stride=(0, 0, 0), cache_stride=(0, 0, 128))
    assert norm(lib, **{**STRIDES, **CACHES, **one}) not in (EINVAL, EUNSUPPORTED)


@no_device
def test_outputs_lie_apart(lib):
    dec = dict(q_stride=(1024, 128), out_stride=(1024, 128), out=0x20000)
    call = lambda **kw: lib.lib.minfer_attn_decode_b8(ctypes.byref(fill(lib.DecodeB8Params(), DEC, {**dec, **kw})), None)  # noqa: E731
    assert call() not in (EINVAL, EUNSUPPORTED)
    assert call(out_stride=(0, 128)) == EINVAL and call(out_stride=(1024, 0)) == EINVAL and call(q_stride=(0, 0)) not in (EINVAL, EUNSUPPORTED)
    read = dict(k_out=0x20000, v_out=0x30000, out_stride=(2 * 50 * 64, 50 * 64, 64))
    call = lambda **kw: lib.lib.minfer_attn_kv_read_b8(ctypes.byref(fill(lib.KvReadB8Params(), READ, {**read, **kw})), None)  # noqa: E731
    assert call() not in (EINVAL, EUNSUPPORTED)
    assert call(v_out=0x20000) == EINVAL
    for i in range(3):
        assert call(out_stride=tuple(0 if j == i else x for j, x in enumerate(read["out_stride"]))) == EINVAL
    assert call(batch=1, n_kv_heads=1, max_len=0x7FFFFFFF, out_rows=0x7FFFFFFF) == EINVAL      # row numbers are rounded up in 32 bits
    assert call(batch=1, n_kv_heads=1, max_len=0x7FFFFFFF) not in (EINVAL, EUNSUPPORTED)        # the outputs have few

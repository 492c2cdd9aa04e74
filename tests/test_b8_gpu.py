"""GPU parity of the block-scaled 8-bit KV cache: append, read-back, decode, and a run of them together.

Appended values: v, and k that is neither rotated nor normed, have exact inputs, so codes and scales have to be the definition's, bit for
bit.  Rotated or normed k is known to the kernel to 2^-18 of its row's largest value (the arithmetic of test_norm_rope_gpu.py): a
code may differ from the nearest one only if it is as near as that, and a scale follows a largest value that is off by as much."""
import pytest
import torch

from _b8 import Cache, raw
from oracle import oracle as O

pytestmark = pytest.mark.gpu
BASE = 500000.0


def inputs(seed, dtype, B, L, Hq, Hkv, D):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, L, (Hq + 2 * Hkv) * D, generator=g)
    qkv *= torch.exp(torch.randn(B, L, 1, generator=g))               # tokens of different magnitude: scales grow
    qkv = qkv.to(dtype)
    split = lambda t: (t[..., :Hq * D].view(B, L, Hq, D), t[..., Hq * D:(Hq + Hkv) * D].view(B, L, Hkv, D),  # noqa: E731
                       t[..., (Hq + Hkv) * D:].view(B, L, Hkv, D))
    return split(qkv), split(qkv.cuda()), (1 + 0.2 * torch.randn(D, generator=g)).to(dtype), (1 + 0.2 * torch.randn(D, generator=g)).to(dtype)


def append(kerns, c, tensors, rot, style, q, k, v, start, qw=None, kw=None):
    w = (None, None) if qw is None else (qw.cuda(), kw.cuda())
    if c.page:
        kerns.rope_kv_append_b8_paged(rot, BASE, style, q, k, v, *tensors, c.block, c.table.cuda(), start.cuda(), *w, 1e-6)
    else:
        kerns.rope_kv_append_b8(rot, BASE, style, q, k, v, *tensors, c.block, start.cuda(), *w, 1e-6)


def check_append(c, tensors, y, start, i, exact, what):
    """y [B, L, Hkv, D] float64: what was appended to tensor i (0 k, 1 v) of cache c, whose state before is in c; updates c to the
    state that the kernel left."""
    got_c, got_s = c.back(tensors[i], tensors[2 + i])
    B, L, H, _ = y.shape
    for b in range(B):
        for h in range(H):
            want_c, want_s = O.b8_append(c.codes[i][b, h], c.scale[i][b, h], y[b, :, h], int(start[b]), c.block, c.int8)
            if exact:
                assert torch.equal(got_s[b, h], want_s), f"{what}: scales of sequence {b}, head {h}"
                assert torch.equal(got_c[b, h], want_c), f"{what}: codes of sequence {b}, head {h}"
                continue
            p0, p1 = int(start[b]), int(start[b]) + L
            j0, j1 = p0 // c.block, -(-p1 // c.block)
            err = y[b, :, h].abs().amax() * 2.0 ** -18
            s = got_s[b, h]
            assert torch.equal(s[:j0], want_s[:j0]) and torch.equal(s[j1:], want_s[j1:]), what
            if c.int8:
                assert ((s - want_s).abs() <= want_s * 2.0 ** -24 + err / 127).all(), what
            else:   # a power of two: another one only where the largest value is that near to the border
                for j in range(j0, j1):
                    if s[j] != want_s[j]:
                        rows = y[b, max(0, j * c.block - p0):(j + 1) * c.block - p0, h]
                        assert (rows.abs().amax() / (448 * torch.minimum(s[j], want_s[j])) - 1).abs() < 2.0 ** -17, what
            per_row = s.repeat_interleave(c.block)[p0:p1, None]
            near = (y[b, :, h] - O.b8_codes(y[b, :, h], per_row, c.int8) * per_row).abs()
            assert ((y[b, :, h] - got_c[b, h, p0:p1] * per_row).abs() <= near + 2 * err).all(), f"{what}: codes of sequence {b}, head {h}"
            # the rows before, under the scale that the block has now
            lo = j0 * c.block
            old = c.codes[i][b, h, lo:p0]
            if p0 > lo:
                want_old = old if s[j0] == c.scale[i][b, h, j0] else O.b8_codes((old * c.scale[i][b, h, j0]).float().double(), s[j0], c.int8)
                assert torch.equal(got_c[b, h, lo:p0], want_old), f"{what}: earlier rows of sequence {b}, head {h}"
            assert torch.equal(got_c[b, h, :lo], c.codes[i][b, h, :lo]) and torch.equal(got_c[b, h, p1:], c.codes[i][b, h, p1:]), what
    c.codes[i], c.scale[i] = got_c, got_s


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("page", [0, 128])
@pytest.mark.parametrize("dtype,D,block,Hq,Hkv", [(torch.float16, 128, 64, 8, 2), (torch.bfloat16, 64, 16, 3, 3), (torch.float16, 64, 128, 10, 5),
                                                  (torch.bfloat16, 128, 128, 4, 1), (torch.float16, 128, 16, 6, 3), (torch.bfloat16, 64, 32, 2, 2),
                                                  (torch.float16, 128, 32, 4, 4), (torch.float16, 64, 64, 4, 2)])
def test_append_without_rotation_is_exact(kerns, fmt, page, dtype, D, block, Hq, Hkv):
    """A history of calls on one cache: prompts, single tokens, short runs; blocks begun, crossed, filled and grown."""
    B = 3
    c = Cache(fmt, B, Hkv, 640, D, block, page, seed=block + D)
    t = c.to_gpu()
    start = torch.tensor([0, 37, 200], dtype=torch.int32)
    for step, L in enumerate((50, 1, 1, 1, 3, 130, 1, 2, block, 1, 17)):
        (q, k, v), (qd, kd, vd), _, _ = inputs(100 + step, dtype, B, L, Hq, Hkv, D)
        append(kerns, c, t, 0, step & 1, qd, kd, vd, start)
        torch.cuda.synchronize()
        what = f"call {step} of {L} tokens"
        assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v), what
        check_append(c, t, k.double(), start, 0, True, what + ", k")
        check_append(c, t, v.double(), start, 1, True, what + ", v")
        start += L


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("dtype,D,rot,block,page,norm", [(torch.float16, 128, 128, 64, 0, True), (torch.bfloat16, 128, 64, 32, 64, False),
                                                         (torch.float16, 64, 64, 16, 48, True), (torch.bfloat16, 64, 32, 128, 0, True)])
def test_append_rotated_and_normed(kerns, fmt, style, dtype, D, rot, block, page, norm):
    B, Hq, Hkv = 2, 6, 3
    c = Cache(fmt, B, Hkv, 480, D, block, page, seed=5)
    t = c.to_gpu()
    start = torch.tensor([11, 160], dtype=torch.int32)
    for step, L in enumerate((70, 1, 1, 4, 1, 129)):
        (q, k, v), (qd, kd, vd), qw, kw = inputs(200 + step, dtype, B, L, Hq, Hkv, D)
        append(kerns, c, t, rot, style, qd, kd, vd, start, *((qw, kw) if norm else ()))
        torch.cuda.synchronize()
        want_q = O.norm_rope(q, qw if norm else None, rot, BASE, style, start, 1e-6)
        tol = want_q.abs() * torch.finfo(dtype).eps / 2 + want_q.abs().amax(-1, keepdim=True) * 2.0 ** -18 + 2.0 ** -25
        assert ((qd.cpu().double() - want_q).abs() <= tol).all()
        check_append(c, t, O.norm_rope(k, kw if norm else None, rot, BASE, style, start, 1e-6), start, 0, False, f"call {step}, k")
        check_append(c, t, v.double(), start, 1, True, f"call {step}, v")
        start += L


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("L", [1, 3])
def test_values_at_the_edges(kerns, fmt, L):
    """Zeros (scale 0, also in a block that held anything), infinities (saturated), NaN, the smallest and largest finite values,
    and values half way between two codes."""
    B, H, D, block = 1, 8, 64, 16
    c = Cache(fmt, B, H, 64, D, block, seed=3)
    dtype = torch.bfloat16
    x = torch.zeros(B, L, H, D, dtype=dtype)
    x[0, :, 1, 0] = 1.0
    x[0, :, 2] = torch.arange(D).to(dtype) * 0.5 - 16                       # ties of both codes
    x[0, :, 2, 0] = 127.0
    x[0, :, 3, 0], x[0, :, 3, 1], x[0, :, 3, 2] = float("inf"), -float("inf"), 3e38
    x[0, :, 4, 0], x[0, :, 4, 1] = 1e-38, 9e-39
    x[0, :, 5, 0], x[0, :, 5, 1] = 448.0, 449.0
    x[0, :, 6, 0], x[0, :, 6, 1] = float("nan"), 2.0
    x[0, :, 7, 0], x[0, :, 7, 1] = 1.0, 0.5                                  # int8: 63.5 steps of 1 / 127
    for start in (16, 21):                                                   # a block that begins here, and one that was begun
        t = c.to_gpu()
        xd = x.cuda()
        append(kerns, c, t, 0, 0, xd.clone(), xd, xd, torch.tensor([start], dtype=torch.int32))
        torch.cuda.synchronize()
        for i in range(2):
            got_c, got_s = c.back(t[i], t[2 + i])
            for h in range(H):
                want_c, want_s = O.b8_append(c.codes[i][0, h], c.scale[i][0, h], x[0, :, h].double(), start, block, c.int8)
                assert torch.equal(got_s[0, h], want_s), (start, i, h)
                assert torch.equal(torch.nan_to_num(got_c[0, h], nan=777.0), torch.nan_to_num(want_c, nan=777.0)), (start, i, h)


@pytest.mark.parametrize("L", [1, 40])
def test_rows_outside_the_cache_are_dropped_and_reported(kerns, L):
    from minfer.kernels.torch_ext.ops import check_status
    B, H, D, block = 3, 2, 128, 16
    c = Cache("e4m3", B, H, 60, D, block, seed=8)
    t = c.to_gpu()
    (q, k, v), (qd, kd, vd), _, _ = inputs(1, torch.float16, B, L, 2, H, D)
    start = torch.tensor([60 if L == 1 else 30, -1 if L == 1 else -8, 20], dtype=torch.int32)
    check_status()
    append(kerns, c, t, 0, 0, qd, kd, vd, start)
    with pytest.raises(RuntimeError, match="cache position out of range"):
        check_status()
    for i, x in ((0, k), (1, v)):
        got_c, got_s = c.back(t[i], t[2 + i])
        for b in range(B):
            first, n = max(0, -int(start[b])), min(L, 60 - int(start[b]))
            for h in range(H):
                want = (c.codes[i][b, h], c.scale[i][b, h])
                if n > first:
                    want = O.b8_append(*want, x[b, first:n, h].double(), int(start[b]) + first, block, False)
                assert torch.equal(got_c[b, h], want[0]) and torch.equal(got_s[b, h], want[1]), (b, h)
    p = Cache("int8", 2, H, 64, D, 32, 32, seed=9)
    t = p.to_gpu()
    before = [x.clone() for x in t]
    p.table = torch.tensor([[int(p.table[0, 0]), 99], [-1, int(p.table[1, 1])]], dtype=torch.int32)
    (q, k, v), (qd, kd, vd), _, _ = inputs(2, torch.float16, 2, L, 2, H, D)
    append(kerns, p, t, 0, 0, qd, kd, vd, torch.tensor([31, 0], dtype=torch.int32))
    # (31 + 40 tokens also pass the end of the cache: the word holds whichever was seen first)
    with pytest.raises(RuntimeError, match="block-table entry outside the page pool" if L == 1 else "block-table entry|cache position out of range"):
        check_status()
    changed = torch.tensor([not torch.equal(raw(t[0])[i], raw(before[0])[i]) for i in range(p.n_pages)])
    wanted = {int(p.table[0, 0])} | ({int(p.table[1, 1])} if L > 1 else set())
    assert set(torch.nonzero(changed).flatten().tolist()) == wanted


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,block,page,rows", [(128, 64, 0, 700), (64, 16, 48, 333), (128, 128, 256, 1000), (64, 128, 0, 129)])
def test_read_back(kerns, fmt, dtype, D, block, page, rows):
    B, H = 4, 3
    c = Cache(fmt, B, H, rows, D, block, page, seed=rows)
    lens = torch.tensor([0, 1, rows - 1, rows], dtype=torch.int32)
    t = c.to_gpu(lens)
    for out_rows in (rows, rows // 2, rows + 5):
        store = torch.full((2, B, out_rows, H, D), 7.0, dtype=dtype, device="cuda")
        ko, vo = store[0].transpose(1, 2), store[1].transpose(1, 2)
        args = (*t, block) + ((c.table.cuda(),) if page else ()) + (lens.cuda(), ko, vo)
        (kerns.kv_read_b8_paged if page else kerns.kv_read_b8)(*args)
        torch.cuda.synchronize()
        for i, got in ((0, ko), (1, vo)):
            want = torch.full((B, H, out_rows, D), 7.0, dtype=dtype)
            # code * scale in fp32 (exact to 2^-24), then the type: the product of a few bits and a float32 rounds once, to the same value
            val = c.values(i).float().to(dtype)
            for b in range(B):
                n = min(int(lens[b]), out_rows)
                want[b, :, :n] = val[b, :, :n]
            assert torch.equal(got.cpu(), want), (out_rows, i)


def decode(kerns, c, t, q, lens, out):
    if c.page:
        kerns.flash_attn_decode_b8_paged(q, *t, c.block, c.table.cuda(), lens.cuda(), out)
    else:
        kerns.flash_attn_decode_b8(q, *t, c.block, lens.cuda(), out)


def check_decode(kerns, c, q, lens, dtype, what="", qd=None, out=None):
    t = c.to_gpu(lens)
    out = torch.full(q.shape, float("nan"), dtype=dtype, device="cuda") if out is None else out
    decode(kerns, c, t, q.cuda() if qd is None else qd, lens, out)
    torch.cuda.synchronize()
    want, tol = O.b8_decode(q, c.values(0), c.values(1), lens, dtype)
    err = (out.cpu().double() - want).abs()
    assert torch.isfinite(out).all(), what
    assert (err <= tol).all(), f"{what}: worst {(err / tol.clamp_min(1e-30)).max():.2f} of the tolerance"
    return out


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,H,Hkv,block,page", [(128, 32, 8, 64, 0), (64, 8, 2, 16, 0), (128, 12, 2, 32, 64), (64, 16, 1, 128, 128), (128, 5, 5, 16, 48),
                                                (128, 22, 2, 128, 0), (64, 9, 1, 64, 192)])
def test_decode(kerns, fmt, dtype, D, H, Hkv, block, page):
    B, rows = 8, 1100
    c = Cache(fmt, B, Hkv, rows, D, block, page, seed=D + H)
    lens = torch.tensor([0, 1, 15, 16, 17, 513, 1025, 1100], dtype=torch.int32)
    q = torch.randn(B, H, 1, D, generator=torch.Generator().manual_seed(H)).to(dtype)
    out = check_decode(kerns, c, q, lens, dtype)
    assert (out[0] == 0).all()


@pytest.mark.parametrize("B,Hkv,rows", [(1, 1, 1), (1, 1, 17), (1, 2, 5000), (2, 8, 300), (40, 4, 250), (1, 1, 20000), (130, 1, 70), (300, 1, 33)])
def test_decode_shapes_of_the_split(kerns, B, Hkv, rows):
    c = Cache("e4m3", B, Hkv, rows, 64, 16, seed=rows)
    lens = torch.randint(0, rows + 1, (B,), generator=torch.Generator().manual_seed(B), dtype=torch.int32)
    lens[0] = rows
    check_decode(kerns, c, torch.randn(B, 4 * Hkv, 1, 64, generator=torch.Generator().manual_seed(1)).half(), lens, torch.float16)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_decode_scales_over_many_orders(kerns, fmt):
    """Blocks whose values differ by 10^12, blocks of zeros, weights that sit on blocks of small values: the fp16 weights follow
    weight times scale, so none of it is lost."""
    B, Hkv, D, block, rows = 2, 2, 128, 16, 640
    c = Cache(fmt, B, Hkv, rows, D, block, seed=4, spread=0.3)
    g = torch.Generator().manual_seed(6)
    c.scale[1] = (c.scale[1] * 10 ** (12 * torch.rand(c.scale[1].shape, generator=g, dtype=torch.float64) - 8)).float().double()
    c.scale[1][:, :, 3] = 0
    c.codes[1][:, :, 48:64] = 0
    c.scale[0][:, :, 7] = 0                                   # keys of zeros: score 0
    c.codes[0][:, :, 112:128] = 0
    q = torch.randn(B, 8, 1, D, generator=g).bfloat16()
    check_decode(kerns, c, q, torch.tensor([640, 601], dtype=torch.int32), torch.bfloat16, "spread scales")
    for j in range(c.blocks):                                 # sharp attention to a block of the smallest scale
        if j != 5:
            c.scale[0][:, :, j] *= 0.01
    c.scale[0] = c.scale[0].float().double()
    c.scale[1][:, :, 5] = 2.0 ** -30
    check_decode(kerns, c, 20 * q, torch.tensor([640, 601], dtype=torch.int32), torch.bfloat16, "weight on the smallest block")


def test_decode_query_magnitudes(kerns):
    """bfloat16 queries far outside fp16's range, heads of zeros, and heads that differ by 10^20."""
    c = Cache("e4m3", 1, 2, 100, 64, 32, seed=14)
    q = torch.randn(1, 8, 1, 64, generator=torch.Generator().manual_seed(3))
    q *= torch.tensor([1e-20, 1e-6, 1.0, 0.0, 3e4, 1e-30, 10.0, 1e-3]).view(1, 8, 1, 1)
    check_decode(kerns, c, q.bfloat16(), torch.tensor([100], dtype=torch.int32), torch.bfloat16)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_decode_strided_queries_streams_and_graphs(kerns, fmt):
    B, H, Hkv, D, rows = 3, 8, 2, 128, 400
    c = Cache(fmt, B, Hkv, rows, D, 32, seed=2)
    lens = torch.tensor([400, 3, 77], dtype=torch.int32)
    big = torch.randn(B, 1, H + 4, D + 8, generator=torch.Generator().manual_seed(5)).half()
    view = lambda x: x[:, :, 2:2 + H, :D].transpose(1, 2)  # noqa: E731
    store = torch.full(big.shape, 7.0, dtype=torch.float16, device="cuda")
    check_decode(kerns, c, view(big), lens, torch.float16, qd=view(big.cuda()), out=view(store))
    kept = store.clone()
    view(kept).fill_(7.0)
    assert (kept == 7.0).all()
    t, qd, ld, out = c.to_gpu(), view(big).contiguous().cuda(), lens.cuda(), torch.zeros(B, H, 1, D, dtype=torch.float16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        decode(kerns, c, t, qd, lens, out)
    side.synchronize()
    eager = out.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kerns.flash_attn_decode_b8(qd, *t, c.block, ld, out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, eager)
    ld.copy_(torch.tensor([1, 399, 0], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    want, tol = O.b8_decode(view(big), c.values(0), c.values(1), ld.cpu(), torch.float16)
    assert ((out.cpu().double() - want).abs() <= tol).all()


def test_decode_nan_reaches_its_sequence_only(kerns):
    c = Cache("e4m3", 2, 1, 64, 64, 16, seed=31)
    lens = torch.tensor([40, 40], dtype=torch.int32)
    t = c.to_gpu(lens)
    raw(t[1])[0, 0, 5, 3] = 0x7F                                # a NaN among the visible values of sequence 0, dimension 3
    q = torch.randn(2, 2, 1, 64, generator=torch.Generator().manual_seed(8)).half()
    out = torch.zeros(2, 2, 1, 64, dtype=torch.float16, device="cuda")
    decode(kerns, c, t, q.cuda(), lens, out)
    nan = torch.isnan(out.cpu())
    assert nan[0, :, 0, 3].all() and int(nan.sum()) == 2


def test_decode_bad_page_is_reported_not_followed(kerns):
    from minfer.kernels.torch_ext.ops import check_status
    c = Cache("int8", 2, 1, 64, 64, 16, 16, seed=32)
    t = c.to_gpu()
    q = torch.randn(2, 2, 1, 64, generator=torch.Generator().manual_seed(8)).half()
    out = torch.zeros(2, 2, 1, 64, dtype=torch.float16, device="cuda")
    lens = torch.tensor([20, 64], dtype=torch.int32)
    c.table[0, 2:] = 1 << 30                                    # behind the sequence: never read
    check_status()
    decode(kerns, c, t, q.cuda(), lens, out)
    check_status()
    c.table[1, 1] = c.n_pages
    decode(kerns, c, t, q.cuda(), lens, out)
    with pytest.raises(RuntimeError, match="block-table entry outside the page pool"):
        check_status()
    ko = torch.zeros(2, 1, 64, 64, dtype=torch.float16, device="cuda")
    kerns.kv_read_b8_paged(*t, c.block, c.table.cuda(), lens.cuda(), ko, torch.zeros_like(ko))
    with pytest.raises(RuntimeError, match="block-table entry outside the page pool"):
        check_status()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("page", [0, 64])
def test_prompt_chunk_and_tokens_together(kerns, fmt, page):
    """As a model uses them: a prompt (append, read back, causal attention), a second chunk behind it, then tokens (append, decode)."""
    B, Hq, Hkv, D, block, style = 2, 8, 2, 128, 32, 1
    c = Cache(fmt, B, Hkv, 384, D, block, page, seed=77)
    for s in c.scale:
        s.zero_()
    for x in c.codes:
        x.zero_()
    t = c.to_gpu()
    table = (c.table.cuda(),) if page else ()
    dec = kerns.flash_attn_decode_b8_paged if page else kerns.flash_attn_decode_b8
    read = kerns.kv_read_b8_paged if page else kerns.kv_read_b8
    n = 0
    for step, L in enumerate((150, 45, 1, 1, 1, 1)):
        (q, k, v), (qd, kd, vd), qw, kw = inputs(300 + step, torch.bfloat16, B, L, Hq, Hkv, D)
        start = torch.full((B,), n, dtype=torch.int32)
        append(kerns, c, t, D, style, qd, kd, vd, start, qw, kw)
        n += L
        lens = torch.full((B,), n, dtype=torch.int32, device="cuda")
        out = torch.zeros(B, Hq, L, D, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        check_append(c, t, O.norm_rope(k, kw, D, BASE, style, start, 1e-6), start, 0, False, f"step {step}, k")
        check_append(c, t, v.double(), start, 1, True, f"step {step}, v")
        qt = qd.transpose(1, 2)
        if L > 1:
            ko, vo = (torch.zeros(B, Hkv, n, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            read(*t, block, *table, lens, ko, vo)
            kerns.flash_attn_causal(qt, ko, vo, out)
            want = O.prefill_oracle(qt.cpu(), ko.cpu(), vo.cpu(), causal=True) if L == n else None
            if want is None:
                mask = torch.ones(L, n, dtype=torch.bool).tril(n - L)
                want = torch.softmax((qt.cpu().double() @ ko.cpu().double().repeat_interleave(Hq // Hkv, 1).transpose(2, 3) / D ** 0.5)
                                     .masked_fill(~mask, float("-inf")), -1) @ vo.cpu().double().repeat_interleave(Hq // Hkv, 1)
            scale = vo.cpu().double().abs().amax()
            assert ((out.cpu().double() - want.double()).abs() <= scale * 2.0 ** -7).all()      # bf16 weights and outputs, 2^-8 each
        else:
            dec(qt, *t, block, *table, lens, out)
            want, tol = O.b8_decode(qt.cpu(), c.values(0), c.values(1), lens.cpu(), torch.bfloat16)
            assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("fmt,dtype,B,H,Hkv,D,block,page,rows,lens", [
    ("e4m3", torch.float16, 1, 32, 8, 128, 64, 0, 16400, [16400]), ("int8", torch.bfloat16, 3, 6, 1, 64, 16, 96, 87456, [87456, 0, 33]),
    ("e4m3", torch.bfloat16, 1, 20, 2, 64, 128, 0, 131100, [131075]), ("int8", torch.float16, 2, 22, 2, 128, 32, 0, 33000, [17, 32999]),
    ("e4m3", torch.float16, 24, 1, 1, 128, 128, 0, 5500, None)])
def test_decode_split_over_all_sms(kerns, fmt, dtype, B, H, Hkv, D, block, page, rows, lens):
    """Few pairs of a long padded cache: partial outputs through the workspace; long, short, empty and padded sequences alike."""
    from minfer.kernels.torch_ext import _lib
    assert _lib.lib.minfer_attn_decode_b8_workspace_bytes(B, H, Hkv, rows, D) > 0, "this shape is to take the split form"
    c = Cache(fmt, B, Hkv, rows, D, block, page, seed=rows)
    g = torch.Generator().manual_seed(B)
    lens = torch.tensor(lens, dtype=torch.int32) if lens else torch.randint(0, rows + 1, (B,), generator=g, dtype=torch.int32)
    check_decode(kerns, c, torch.randn(B, H, 1, D, generator=g).to(dtype), lens, dtype)


def test_split_decode_in_two_graphs_and_on_two_streams(kerns):
    """Calls that use a workspace at the same time: each has its own."""
    D, H, Hkv, rows = 128, 8, 2, 66000
    caches = [Cache("e4m3", 1, Hkv, rows, D, 128, seed=50 + i) for i in range(2)]
    lens = torch.tensor([rows], dtype=torch.int32)
    ts, ld = [c.to_gpu() for c in caches], lens.cuda()
    qs = [torch.randn(1, H, 1, D, generator=torch.Generator().manual_seed(i)).half() for i in range(2)]
    qd, outs = [q.cuda() for q in qs], [torch.zeros(1, H, 1, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    call = lambda i: kerns.flash_attn_decode_b8(qd[i], *ts[i], 128, ld, outs[i])  # noqa: E731
    for i in range(2):
        call(i)
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    for i, c in enumerate(caches):
        ref, tol = O.b8_decode(qs[i], c.values(0), c.values(1), lens, torch.float16)
        assert ((want[i].cpu().double() - ref).abs() <= tol).all()
    graphs = []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            call(i)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for run in (lambda i: graphs[i].replay(), call):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    run(i)
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


def test_codes_of_other_writers(kerns):
    """Scales that are no power of two, the int8 code -128, negative zero and every finite e4m3 code: what another program wrote is read as
    code * scale, and an append behind it codes the rows again from those values."""
    D, block = 64, 16
    for fmt in ("e4m3", "int8"):
        c = Cache(fmt, 1, 1, 48, D, block, seed=6)
        every = torch.arange(256, dtype=torch.uint8)
        if fmt == "e4m3":
            every = every[(every & 0x7F) != 0x7F]
        vals = every.view(torch.float8_e4m3fn if fmt == "e4m3" else torch.int8).float().double()
        for i in range(2):
            c.codes[i][0, 0, :32] = vals.repeat(9)[:32 * D].view(32, D)
            c.scale[i][0, 0] = torch.tensor([0.0123, 0.7, 1.9]).double()
        check_decode(kerns, c, torch.randn(1, 2, 1, D, generator=torch.Generator().manual_seed(1)).half(), torch.tensor([32], dtype=torch.int32), torch.float16)
        t = c.to_gpu()
        ko, vo = (torch.zeros(1, 1, 32, D, dtype=torch.float16, device="cuda") for _ in range(2))
        kerns.kv_read_b8(*t, block, torch.tensor([32], dtype=torch.int32, device="cuda"), ko, vo)
        assert torch.equal(ko.cpu(), c.values(0)[:, :, :32].float().half()) and torch.equal(vo.cpu(), c.values(1)[:, :, :32].float().half())
        for L in (1, 5):                                           # grows the block that holds rows 16 .. 26
            t = c.to_gpu()
            x = torch.full((1, L, 1, D), 3000.0, dtype=torch.float16)
            append(kerns, c, t, 0, 0, x.cuda(), x.cuda(), x.cuda(), torch.tensor([27], dtype=torch.int32))
            torch.cuda.synchronize()
            got_c, got_s = c.back(t[0], t[2])
            want_c, want_s = O.b8_append(c.codes[0][0, 0], c.scale[0][0, 0], x[0, :, 0].double(), 27, block, c.int8)
            assert torch.equal(got_c[0, 0], want_c) and torch.equal(got_s[0, 0], want_s), (fmt, L)


@pytest.mark.parametrize("block", [16, 64, 128])
@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("start", [0, 100_000])
def test_angles_are_exact_to_fp32(kerns, block, style, start):
    """An int8 block with one value in it has that value's magnitude / 127 as its scale, in 32 bits: with 1 in one half of a pair, the
    larger of |cos| and |sin| of that pair's angle."""
    d, n = 64, 8 * block
    first = start // block * block
    k = torch.zeros(1, n, 1, d, dtype=torch.float16, device="cuda")
    rows = torch.arange(8) * block + (torch.arange(8) * 37 + 5) % block
    pair = torch.arange(8) * 5 % (d // 2)
    k[0, rows, 0, pair * 2 if style == 0 else pair] = 1.0
    q = torch.zeros(1, n, 1, d, dtype=torch.float16, device="cuda")
    lmax = first + n
    kc, vc = (torch.zeros(1, 1, lmax, d, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(1, 1, (lmax + block - 1) // block, device="cuda") for _ in range(2))
    kerns.rope_kv_append_b8(d, 10000.0, style, q, k, torch.zeros_like(k), kc, vc, ks, vs, block,
                            torch.tensor([first], dtype=torch.int32, device="cuda"))
    got = ks[0, 0, first // block:].double().cpu() * 127
    angle = (first + rows).double() * 10000.0 ** (-2.0 * pair.double() / d)
    want = torch.maximum(angle.cos().abs(), angle.sin().abs())
    # In units of 2^-24: sincospif is within 1 of values below 1, its argument (an eighth of a turn) is rounded by pi / 8; a row's angle
    # is the sum of two such, (1 + pi / 8) * 2 * sqrt 2 = 3.94, and the sum's two roundings make it 4.94; relative to sqrt 1/2 or more 6.99,
    # and the scale's own rounding is 1.
    assert ((got - want).abs() / want).max() <= 8 * 2.0 ** -24


def test_decode_shares_of_a_sequence_that_pass_32_bits(kerns):
    """301 million keys, nearly all of them the same page: keys of zeros weigh the same, so the output is the share of each page's values.
    The last fifth of the table names the second page: shares that went wrong leave it out."""
    page, n0, n1, d, block = 65536, 3700, 900, 64, 128
    kc = torch.zeros(2, 1, page, d, device="cuda").to(torch.float8_e4m3fn)
    vc = torch.ones(2, 1, page, d, device="cuda")
    vc[1] = -1.0
    s = torch.ones(2, 1, page // block, device="cuda")
    table = torch.tensor([[0] * n0 + [1] * n1], dtype=torch.int32, device="cuda")
    q = torch.ones(1, 1, 1, d, dtype=torch.float16, device="cuda")
    out = torch.full_like(q, float("nan"))
    kerns.flash_attn_decode_b8_paged(q, kc, vc.to(torch.float8_e4m3fn), s, s.clone(), block, table, torch.tensor([page * (n0 + n1)], dtype=torch.int32, device="cuda"), out)
    want = (n0 - n1) / (n0 + n1)
    # A warp's sums are of equal powers of two, fewer than 2^24: exact.  Adding up 296 blocks' (of 4 warps) parts rounds 300 times at most,
    # in numerator and denominator; then one rounding to fp16.
    assert (out.double() - want).abs().max() <= want * (2.0 ** -11 + 2 * 300 * 2.0 ** -24)


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "16"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("seq", [1, 150])
def test_offsets_that_pass_32_bits(kerns, fmt, paged, seq):
    """The last sequence (the last page) of a cache lies beyond 2^32 bytes: append, read-back and decode give the same bits as in a small one."""
    page, D, block = 1024, 64, 64
    size = 2 if fmt == "16" else 1
    far = (1 << 32) // (page * D * size) + 3                          # pages before the far one
    dt = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8, "16": torch.float16}[fmt]
    g = torch.Generator(device="cuda").manual_seed(seq)
    q = torch.randn(2, seq, 4, D, generator=g, device="cuda", dtype=torch.float16)
    k, v = (torch.randn(2, seq, 1, D, generator=g, device="cuda", dtype=torch.float16) for _ in range(2))
    w = torch.rand(D, generator=g, device="cuda") + 0.5
    start = torch.zeros(2, dtype=torch.int32, device="cuda")

    def run(last):
        def laid(*shape, dtype):  # sequences (pages) 0 and `last`, with nothing else touched in between
            step = shape[1] * shape[2] * (shape[3] if len(shape) == 4 else 1)
            flat = torch.empty((last + 1) * step, dtype=dtype, device="cuda")
            if paged:
                t = flat.view(last + 1, *shape[1:])
                ends = t.view(torch.int8) if dtype.itemsize == 1 else t
            else:
                strides = (last * step, step, *((shape[3], 1) if len(shape) == 4 else (1,)))
                t = flat.as_strided(shape, strides)
                ends = flat.view(torch.int8).as_strided(shape, strides) if dtype.itemsize == 1 else t
            ends[0].zero_()
            ends[-1].zero_()
            return t
        kc, vc = (laid(2, 1, page, D, dtype=dt) for _ in range(2))
        table = torch.tensor([[0], [last]], dtype=torch.int32, device="cuda")
        turn = (D, 10000.0, 0)
        qq = q.clone()
        pages = (table,) if paged else ()
        if fmt == "16":
            name = "qk_norm_rope_kv_append" + ("_paged" if paged else "")
            getattr(kerns, name)(*turn, 1e-6, qq, k, v, w, w, kc, vc, *pages, start)
            return [qq.cpu(), kc[0].cpu(), kc[-1].cpu(), vc[0].cpu(), vc[-1].cpu()]
        ks, vs = (laid(2, 1, page // block, dtype=torch.float32) for _ in range(2))
        tail = "_paged" if paged else ""
        getattr(kerns, "rope_kv_append_b8" + tail)(*turn, qq, k, v, kc, vc, ks, vs, block, *pages, start, w, w, 1e-6)
        lens = start + seq
        ko, vo = (torch.zeros(2, 1, seq, D, dtype=torch.float16, device="cuda") for _ in range(2))
        getattr(kerns, "kv_read_b8" + tail)(kc, vc, ks, vs, block, *pages, lens, ko, vo)
        q1 = qq[:, -1:].transpose(1, 2).contiguous()
        out = torch.empty_like(q1)
        getattr(kerns, "flash_attn_decode_b8" + tail)(q1, kc, vc, ks, vs, block, *pages, lens, out)
        return [qq.cpu(), *(raw(c[i].contiguous()).cpu() for c in (kc, vc) for i in (0, -1)), *(s[i].cpu() for s in (ks, vs) for i in (0, -1)), ko.cpu(), vo.cpu(), out.cpu()]

    near, there = run(1), run(far)
    assert all(torch.equal(a, b) for a, b in zip(near, there))
    assert near[2].any() and near[4].any()                             # (something was written there)

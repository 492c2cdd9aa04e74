"""GPU: calls at the edges of the 8-bit cache's operators that test_b8_gpu.py does not make."""
import pytest
import torch

from _b8 import Cache
from oracle import oracle as O
from test_b8_gpu import append, check_append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [0, 48])
def test_read_back_of_negative_lengths_touches_nothing(kerns, page):
    """A negative length is a length of none, down to the smallest int32, from which no row number may be taken away in 32 bits.  129 rows: the last
    warp's 16 pass the end of the cache."""
    B, H, D, rows = 4, 2, 64, 129
    c = Cache("e4m3", B, H, rows, D, 16, page, seed=1)
    t = c.to_gpu()
    lens = torch.tensor([-1, -2 ** 31, -2 ** 31 + 40, 5], dtype=torch.int32)
    store = torch.full((2, B, H, c.rows + 64, D), 7.0, dtype=torch.float16, device="cuda")
    ko, vo = store[0, :, :, :c.rows], store[1, :, :, :c.rows]
    args = (*t, 16) + ((c.table.cuda(),) if page else ()) + (lens.cuda(), ko, vo)
    (kerns.kv_read_b8_paged if page else kerns.kv_read_b8)(*args)
    got = store.cpu()
    for i in range(2):
        want = torch.full((B, H, c.rows + 64, D), 7.0, dtype=torch.float16)
        want[3, :, :5] = c.values(i)[3, :, :5].half()
        assert torch.equal(got[i], want), i


def values_near_borders(dtype, scale, n):
    """The n finite values of the type, of those that a block with this e4m3 scale takes without growing, whose quotient lies nearest to a border between two codes
    (ties among them), half of them negative; shuffled."""
    x = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dtype).double()
    m, e = torch.frexp(torch.tensor(float(scale), dtype=torch.float64))
    x = x[torch.isfinite(x) & (x > scale * 2.0 ** -11) & (x <= 448 * torch.ldexp(torch.ones((), dtype=torch.float64), e - 1))]
    y = x / scale
    step = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)
    order = ((y / step - torch.floor(y / step) - 0.5).abs() * step / y).argsort()
    x = x[order[:n]].repeat(-(-n // min(n, len(x))))[:n]
    g = torch.Generator().manual_seed(n)
    return (x * (1 - 2 * torch.randint(0, 2, (n,), generator=g)))[torch.randperm(n, generator=g)].to(dtype)


@pytest.mark.parametrize("dtype,scale", [(t, s) for t in (torch.float16, torch.bfloat16) for s in (7.0, 49 / 448, 0.3, 1.9, 3 * 2.0 ** -10)] +
                                        [(torch.bfloat16, 1.25 * 2.0 ** -66)])
@pytest.mark.parametrize("L,D,block,page", [(1, 128, 16, 0), (1, 64, 64, 64), (5, 64, 16, 48), (100, 128, 128, 0), (40, 128, 64, 128), (60, 64, 128, 0)])
def test_e4m3_codes_under_scales_of_other_writers(kerns, dtype, scale, L, D, block, page):
    """A block that another program began keeps its scale while the new rows need no larger one, whatever number it is: their codes are the nearest
    ones, ties to even, of the exact quotient, as under a power of two."""
    B, H = 2, 4
    c = Cache("e4m3", B, H, 256, D, block, page, seed=12)
    scale = float(torch.tensor(scale, dtype=torch.float32))
    for i in range(2):
        c.scale[i][:] = scale
    start = torch.tensor([1, block - 2], dtype=torch.int32)            # the second sequence's call goes on into blocks of its own
    x = values_near_borders(dtype, scale, 2 * B * L * H * D).view(2, B, L, H, D)
    k, v = x[0], x[1]
    t = c.to_gpu()
    append(kerns, c, t, 0, 0, k.cuda(), k.cuda(), v.cuda(), start)
    torch.cuda.synchronize()
    kept = c.scale[0].clone()
    check_append(c, t, k.double(), start, 0, True, "k")
    check_append(c, t, v.double(), start, 1, True, "v")
    assert torch.equal(c.scale[0][0, :, 0], kept[0, :, 0]) and torch.equal(c.scale[0][1, :, 0], kept[1, :, 0]), "the scale was to stay"


def test_append_of_nearly_two_to_the_31_tokens(kerns):
    """Positions behind the cache are dropped and reported, so the C entry takes a call of 2^31 - 100 tokens whose k and v are one row, expanded; the number of
    blocks that such a call touches passes 32 bits on the way."""
    import ctypes

    from minfer.kernels.torch_ext import _lib
    D, H, rows, block = 64, 2, 64, 128
    c = Cache("e4m3", 1, H, rows, D, block, seed=4)
    t = c.to_gpu()
    x = torch.randn(2, H, D, generator=torch.Generator().manual_seed(2)).half()
    xd, start, status = x.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    p = _lib.NormRopeParams()
    p.k, p.v, p.start, p.status = xd[0].data_ptr(), xd[1].data_ptr(), start.data_ptr(), status.data_ptr()
    p.k_cache, p.v_cache, p.k_scale, p.v_scale = (y.data_ptr() for y in t)
    p.kv_stride[2] = D
    for i in range(3):
        p.cache_stride[i] = t[0].stride(i)
    p.scale_stride[0], p.scale_stride[1] = t[2].stride(0), t[2].stride(1)
    p.batch, p.seq, p.n_kv_heads, p.head_dim, p.max_len = 1, 2 ** 31 - 100, H, D, rows
    p.freq_base, p.dtype, p.cache_format, p.block_size = 10000.0, _lib.F16, _lib.KV_E4M3, block
    rc = _lib.lib.minfer_attn_norm_rope_append(ctypes.byref(p), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    torch.cuda.synchronize()
    assert status.tolist() == [102, 0, rows, rows]
    for i in range(2):
        check_append(c, t, x[i].double().expand(1, rows, H, D), torch.zeros(1, dtype=torch.int32), i, True, str(i))


@pytest.mark.parametrize("dtype,style", [(torch.bfloat16, 1), (torch.float16, 0)])
@pytest.mark.parametrize("D,block", [(64, 16), (128, 32), (128, 64), (64, 128), (128, 128)])
def test_tokens_in_one_call_or_one_by_one(kerns, dtype, style, D, block):
    """e4m3: the same scales, and v's codes differ only where a value lies below the smallest normal code of the final scale.  So do k's where a thread
    works on one row of a block (blocks of 4096 values and fewer); else a row's angle may be the sum of two, which moves k by 2^-18 of its row's
    largest value at most in either form, and codes and scales where a border is as near as twice that."""
    B, L, Hq, Hkv, rot = 2, 150, 4, 2, D
    g = torch.Generator().manual_seed(D + block)
    q, k, v = ((torch.randn(B, L, h, D, generator=g) * torch.exp(torch.randn(B, L, 1, 1, generator=g))).to(dtype) for h in (Hq, Hkv, Hkv))
    qw, kw = (1 + 0.2 * torch.randn(D, generator=g), 1 + 0.2 * torch.randn(D, generator=g))
    caches, tensors, qs = [], [], []
    for whole in (True, False):
        c = Cache("e4m3", B, Hkv, 256, D, block, seed=1)
        t = c.to_gpu()
        qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
        for p in ([(0, L)] if whole else [(i, i + 1) for i in range(L)]):
            append(kerns, c, t, rot, style, qd[:, p[0]:p[1]], kd[:, p[0]:p[1]], vd[:, p[0]:p[1]], torch.full((B,), p[0], dtype=torch.int32), qw, kw)
        torch.cuda.synchronize()
        caches.append(c)
        tensors.append(t)
        qs.append(qd.cpu())
    assert torch.equal(*qs)                                            # q's angles are formed in one way
    y = O.norm_rope(k, kw, rot, 500000.0, style, [0] * B, 1e-6).transpose(1, 2), v.double().transpose(1, 2)
    for i in range(2):
        (ca, sa), (cb, sb) = (c.back(t[i], t[2 + i]) for c, t in zip(caches, tensors))
        near = y[i].abs().amax(-1, keepdim=True) * (2.0 ** -17 if i == 0 and block * D > 4096 else 0.0)
        blocks = -(-L // block)
        for j in range(blocks):
            top = y[i][:, :, j * block:(j + 1) * block].abs().amax((-1, -2))
            low = torch.minimum(sa[:, :, j], sb[:, :, j])
            assert ((sa[:, :, j] == sb[:, :, j]) | ((top - 448 * low).abs() <= near.amax())).all(), (i, j)
        s = torch.maximum(sa, sb).repeat_interleave(block, -1)[:, :, :L, None]
        a, b = (c[:, :, :L] * w.repeat_interleave(block, -1)[:, :, :L, None] for c, w in ((ca, sa), (cb, sb)))
        z = y[i] / s
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp_min(2.0 ** -6))) - 3)
        border = ((z / step - torch.floor(z / step) - 0.5).abs() * step * s)
        fine = (a == b) | (z.abs() < 2.0 ** -6) | (border <= near)
        assert fine.all(), (i, int((~fine).sum()))
        assert (z.abs() < 2.0 ** -6).double().mean() < 0.2             # (the rule above is about a few)
        assert torch.equal(ca[:, :, L:], cb[:, :, L:])


def test_decode_of_the_largest_queries(kerns):
    """bfloat16 queries up to the type's last binade, 2^127 and more: finite scores, so a result as for any other query.  Scores differ by 2^119 and more from key
    to key: the output is the value of the key with the largest."""
    D, H, rows = 64, 4, 40
    c = Cache("e4m3", 1, 1, rows, D, 16, seed=21)
    c.codes[0].zero_()
    c.scale[0][:] = 2.0 ** -10
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(4))
    ladder = torch.tensor([m * 2.0 ** e for e in range(3, 8) for m in (1, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875)], dtype=torch.float64)
    c.codes[0][0, 0, order, 5] = ladder[:rows]
    q = torch.zeros(1, H, 1, D)
    q[0, :, 0, 5] = torch.tensor([2.0 ** 125, 2.0 ** 126, -(2.0 ** 127), 2.0 ** 127 * 1.9921875])
    q = q.bfloat16()
    out = torch.zeros(1, H, 1, D, dtype=torch.bfloat16, device="cuda")
    kerns.flash_attn_decode_b8(q.cuda(), *c.to_gpu(), 16, torch.tensor([rows], dtype=torch.int32, device="cuda"), out)
    score = q[0, :, 0, 5, None].double() * c.values(0)[0, 0, :, 5] / 8
    assert score.abs().max() < torch.finfo(torch.float32).max
    assert torch.equal(out.cpu()[0, :, 0], c.values(1)[0, 0, score.argmax(1)].bfloat16())


@pytest.mark.parametrize("L", [1, 30])
@pytest.mark.parametrize("page", [0, 64])
def test_the_int8_code_of_minus_128_saturates_under_a_scale_that_grew_little(kerns, L, page):
    """Another program's -128 is read as what it is; coded again under a scale up to 128 / 127 of the old one it lies beyond -127 steps, the last code there is."""
    B, H, D, block = 1, 4, 64, 64
    c = Cache("int8", B, H, 128, D, block, page, seed=9)
    for i in range(2):
        c.codes[i][:, :, :20] = torch.where(torch.arange(D) % 3 == 0, -128.0, c.codes[i][:, :, :20])
        c.scale[i][:, :, 0] = 1.0
    t = c.to_gpu()
    x = torch.ones(B, L, H, D)
    x[0, 0, :, 7] = torch.tensor([127.0625, 127.5, 128.0, 129.0])     # scales of 1.0005, 1.004, 1.0079 and 1.0157
    x = x.half()
    start = torch.tensor([20], dtype=torch.int32)
    append(kerns, c, t, 0, 0, x.cuda(), x.cuda(), x.cuda(), start)
    torch.cuda.synchronize()
    for i in range(2):
        check_append(c, t, x.double(), start, i, True, str(i))
        assert c.codes[i].min() == -127.0

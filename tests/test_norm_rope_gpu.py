"""GPU parity of qk_norm_rope and its appending forms against the definition in 64 bits.

Tolerance, derived: one rounding to the output type (half a step, eps / 2 relative), and the fp32 arithmetic in front of it.
That is at most: 2^-24 * 16 for the sum of squares, the reciprocal root and the two products (relative to x), and for
the rotated pair (a, b) the error of cos and sin - the angle is good to 2^-24 * pi, sincospi to two ulp - times |a| + |b|.
Together below 2^-19 of |a| + |b|, hence of sqrt(2) * the row's largest value: 2^-18 * max|y| absolute covers it.  Subnormal fp16
results add half their step, 2^-25."""
import pytest
import torch

from oracle import oracle as O

pytestmark = pytest.mark.gpu


def close(got, want, dtype, what=""):
    got, want = got.detach().cpu().double(), want.double()
    assert torch.isfinite(got).all(), what
    tol = want.abs() * (torch.finfo(dtype).eps / 2) + want.abs().amax(-1, keepdim=True) * 2.0 ** -18 + 2.0 ** -25
    bad = (got - want).abs() > tol * 1.0001
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / tol).max():.2f} of the tolerance"


def draw(seed, dtype, B, L, Hq, Hkv, D, wdt=None, per_head=False):
    g = torch.Generator().manual_seed(seed)
    qkv = torch.randn(B, L, (Hq + 2 * Hkv) * D, generator=g).to(dtype)
    split = lambda t: (t[..., :Hq * D].view(B, L, Hq, D), t[..., Hq * D:(Hq + Hkv) * D].view(B, L, Hkv, D),  # noqa: E731
                       t[..., (Hq + Hkv) * D:].view(B, L, Hkv, D))
    qw = (1 + 0.2 * torch.randn(*((Hq, D) if per_head else (D,)), generator=g)).to(wdt or dtype)
    kw = (1 + 0.2 * torch.randn(*((Hkv, D) if per_head else (D,)), generator=g)).to(wdt or dtype)
    return split(qkv), split(qkv.cuda()), qw, kw


@pytest.mark.parametrize("style", [0, 1])
@pytest.mark.parametrize("dtype,wdt,per_head", [(torch.float16, None, False), (torch.bfloat16, torch.float32, True),
                                                (torch.float16, torch.bfloat16, True), (torch.bfloat16, None, False)])
@pytest.mark.parametrize("B,L,Hq,Hkv,D,rot", [(1, 1, 32, 8, 128, 128), (3, 37, 6, 2, 64, 32), (2, 130, 10, 2, 128, 64), (1, 5, 3, 3, 16, 16),
                                              (2, 9, 4, 1, 80, 48), (1, 33, 2, 2, 256, 256), (2, 3, 5, 1, 192, 96), (300, 1, 4, 2, 64, 64),
                                              (2, 700, 12, 4, 128, 128), (1, 3000, 4, 4, 64, 0)])
def test_in_place(kerns, style, dtype, wdt, per_head, B, L, Hq, Hkv, D, rot):
    (q, k, v), (qd, kd, vd), qw, kw = draw(B + L + D, dtype, B, L, Hq, Hkv, D, wdt, per_head)
    start = torch.randint(0, 100000, (B,), generator=torch.Generator().manual_seed(L), dtype=torch.int32)
    kerns.qk_norm_rope(rot, 500000.0, style, 1e-5, qd, kd, qw.cuda(), kw.cuda(), start.cuda())
    torch.cuda.synchronize()
    close(qd, O.norm_rope(q, qw, rot, 500000.0, style, start, 1e-5), dtype, "q")
    close(kd, O.norm_rope(k, kw, rot, 500000.0, style, start, 1e-5), dtype, "k")
    assert torch.equal(vd.cpu(), v)


@pytest.mark.parametrize("pos", [0, 1, 65536, 16777217, 2000000000])
def test_angles_of_far_positions(kerns, pos):
    """fp32 products of position and frequency would be off by 2^-24 of the angle: 0.06 at 10^6, anything at 2 * 10^9."""
    x = torch.ones(1, 2, 1, 128, dtype=torch.float16)
    q, k = x.cuda(), x.cuda()
    w = torch.ones(128)
    start = torch.tensor([pos], dtype=torch.int32)
    kerns.qk_norm_rope(128, 10000.0, 1, 0.0, q, k, w.cuda(), w.cuda(), start.cuda())
    torch.cuda.synchronize()
    # the oracle's own angle: 2 * 10^9 in 64 bits is off by 2^-22, below the tolerance
    close(q, O.norm_rope(x, w, 128, 10000.0, 1, start, 0.0), torch.float16, f"position {pos}")


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("style,dtype,B,L,D", [(0, torch.float16, 3, 21, 128), (1, torch.bfloat16, 4, 1, 128), (1, torch.float16, 2, 300, 64),
                                               (0, torch.bfloat16, 2, 7, 96)])
def test_append(kerns, paged, style, dtype, B, L, D):
    Hq, Hkv, rot, base, Lmax, page = 6, 2, D, 500000.0, 480, 24
    (q, k, v), (qd, kd, vd), qw, kw = draw(7 + L, dtype, B, L, Hq, Hkv, D)
    start = torch.tensor([0, 100, 163, 31][:B], dtype=torch.int32)
    if paged:
        table = torch.randperm(B * Lmax // page, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(B, -1)
        kc, vc = (torch.full((B * Lmax // page, Hkv, page, D), 7.0, dtype=dtype) for _ in range(2))
    else:
        kc, vc = (torch.full((B, Hkv, Lmax, D), 7.0, dtype=dtype) for _ in range(2))
    kcd, vcd = kc.cuda(), vc.cuda()
    args = (rot, base, style, 1e-6, qd, kd, vd, qw.cuda(), kw.cuda(), kcd, vcd)
    if paged:
        kerns.qk_norm_rope_kv_append_paged(*args, table.cuda(), start.cuda())
    else:
        kerns.qk_norm_rope_kv_append(*args, start.cuda())
    torch.cuda.synchronize()
    close(qd, O.norm_rope(q, qw, rot, base, style, start, 1e-6), dtype, "q")
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v)          # written to the caches only
    want_k, want_v = kc.double(), vc.clone()
    ky = O.norm_rope(k, kw, rot, base, style, start, 1e-6)
    for b in range(B):
        for t in range(L):
            p = int(start[b]) + t
            o, r = (int(table[b, p // page]), p % page) if paged else (b, p)
            want_k[o, :, r], want_v[o, :, r] = ky[b, t], v[b, t]
    close(kcd, want_k, dtype, "k cache")
    assert torch.equal(vcd.cpu(), want_v)
    # (the cache's other rows: want_k holds their fill, which close() compares)


def test_rows_outside_the_cache_are_dropped_and_reported(kerns):
    from minfer.kernels.torch_ext.ops import check_status
    B, L, H, D, Lmax = 3, 2, 2, 64, 32
    (q, k, v), (qd, kd, vd), qw, kw = draw(3, torch.float16, B, L, H, H, D)
    kc, vc = (torch.full((B, H, Lmax, D), 7.0, dtype=torch.float16, device="cuda") for _ in range(2))
    start = torch.tensor([3, Lmax - 1, -1], dtype=torch.int32)
    check_status()
    kerns.qk_norm_rope_kv_append(D, 1e4, 0, 1e-6, qd, kd, vd, qw.cuda(), kw.cuda(), kc, vc, start.cuda())
    with pytest.raises(RuntimeError, match="cache position out of range"):
        check_status()
    wrote = torch.zeros(B, Lmax, dtype=torch.bool)
    wrote[0, 3:5] = wrote[1, Lmax - 1] = wrote[2, 0] = True
    assert torch.equal((kc != 7.0).any(-1).any(1).cpu(), wrote) and torch.equal((vc != 7.0).any(-1).any(1).cpu(), wrote)
    close(qd, O.norm_rope(q, qw, D, 1e4, 0, start, 1e-6), torch.float16, "q of every token")
    pool = torch.full((4, H, 16, D), 7.0, dtype=torch.float16, device="cuda")
    table = torch.tensor([[0, 1], [9, 2], [3, -5]], dtype=torch.int32, device="cuda")
    pool_v = pool.clone()
    kerns.qk_norm_rope_kv_append_paged(D, 1e4, 0, 1e-6, qd, kd, vd, qw.cuda(), kw.cuda(), pool, pool_v, table,
                                       torch.tensor([0, 0, 15], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="block-table entry outside the page pool"):
        check_status()
    wrote = torch.zeros(4, 16, dtype=torch.bool)
    wrote[0, :2] = wrote[3, 15] = True
    assert torch.equal((pool != 7.0).any(-1).any(1).cpu(), wrote)


def test_strided_views_other_streams_and_graphs(kerns):
    """Storage with gaps, a call on another stream, and a captured call replayed on new inputs."""
    B, L, Hq, Hkv, D = 2, 19, 4, 2, 128
    g = torch.Generator().manual_seed(9)
    big = torch.randn(B, Hq + 3, L + 2, D + 16, generator=g).half()
    qw, kw = torch.randn(D, generator=g), torch.randn(D, generator=g)
    start = torch.tensor([5, 900], dtype=torch.int32)
    view = lambda t, h: t[:, 1:1 + h, 1:1 + L, 8:8 + D].transpose(1, 2)  # noqa: E731
    qd, kd = big.cuda(), big.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kerns.qk_norm_rope(D, 1e4, 0, 1e-6, view(qd, Hq), view(kd, Hkv), qw.cuda(), kw.cuda(), start.cuda())
    side.synchronize()
    for got, h, w in ((qd, Hq, qw), (kd, Hkv, kw)):
        close(view(got, h), O.norm_rope(view(big, h), w, D, 1e4, 0, start, 1e-6), torch.float16)
        kept = got.cpu()
        view(kept, h).copy_(view(big, h))
        assert torch.equal(kept, big)                                     # nothing beside the views
    sq, sk, st = view(big, Hq).contiguous().cuda(), view(big, Hkv).contiguous().cuda(), start.cuda()
    qwd, kwd = qw.cuda(), kw.cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kerns.qk_norm_rope(D, 1e4, 1, 1e-6, sq, sk, qwd, kwd, st)
    x, y = torch.randn(B, L, Hq, D, generator=g).half(), torch.randn(B, L, Hkv, D, generator=g).half()
    sq.copy_(x)
    sk.copy_(y)
    st += 1
    graph.replay()
    torch.cuda.synchronize()
    close(sq, O.norm_rope(x, qw, D, 1e4, 1, start + 1, 1e-6), torch.float16)
    close(sk, O.norm_rope(y, kw, D, 1e4, 1, start + 1, 1e-6), torch.float16)


def test_zero_rows_and_non_finite_values_stay_in_their_row(kerns):
    B, L, H, D = 1, 4, 2, 128
    (q, k, v), (qd, kd, vd), qw, kw = draw(21, torch.float16, B, L, H, H, D)
    qd[0, 1] = 0
    qd[0, 2, 0, 5] = float("inf")
    qd[0, 3, 1, 7] = float("nan")
    q = qd.cpu().clone()
    kerns.qk_norm_rope(D, 1e4, 0, 1e-6, qd, kd, qw.cuda(), kw.cuda(), torch.zeros(1, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    want = O.norm_rope(q, qw, D, 1e4, 0, [0], 1e-6)
    rows = torch.ones(L, H, dtype=torch.bool)
    rows[2, 0] = rows[3, 1] = False
    close(qd[0][rows.cuda()], want[0][rows], torch.float16)
    assert (qd[0, 1] == 0).all() and torch.isnan(qd[0, 3, 1]).all() and torch.isnan(qd[0, 2, 0, 5])

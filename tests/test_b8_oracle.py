"""CPU: the 64-bit definitions of the 8-bit cache against torch's own conversions, and their invariants."""
import pytest
import torch

from oracle import oracle as O


def test_e4m3_codes_are_torchs():
    g = torch.Generator().manual_seed(1)
    x = torch.cat([torch.randn(20000, generator=g) * 10 ** (6 * torch.rand(20000, generator=g) - 4), torch.tensor([0.0, 448.0, -448.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10])])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).float().double()
    assert torch.equal(O.b8_codes(x, torch.ones(()), False), want)


def test_scales():
    a = torch.tensor([0.0, 448.0, 449.0, 447.0, 224.0, 224.5, 1.75, 1.7500001, 1e-45, 3e38, float("inf")])
    s = O.b8_scale(a, False)
    assert s.tolist()[:8] == [0, 1, 2, 1, 0.5, 1, 2.0 ** -8, 2.0 ** -7]
    fin = a.double().clamp_max(torch.finfo(torch.float32).max)
    ok = (fin <= 448 * s) & ((fin > 224 * s) | (s == 2.0 ** -126))
    assert ok[1:].all()
    s8 = O.b8_scale(a, True)
    assert s8[0] == 0 and float(s8[1]) == float(torch.tensor(448.0) / 127) and s8[8] == 2.0 ** -126


@pytest.mark.parametrize("int8", [False, True])
def test_append_in_pieces_keeps_earlier_rows_within_a_step(int8):
    """Rows that are coded again under a grown scale stay within one more half step of the grown block."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(100, 64, generator=g, dtype=torch.float64) * torch.exp(torch.randn(100, 1, generator=g, dtype=torch.float64))
    codes, scale = torch.full((112, 64), 99.0, dtype=torch.float64), torch.full((7,), 99.0, dtype=torch.float64)
    p = 0
    for n in (1, 1, 5, 1, 30, 2, 1, 59):
        codes, scale = O.b8_append(codes, scale, x[p:p + n], p, 16, int8)
        p += n
    assert p == 100 and (codes[100:] == 99).all()
    y = O.b8_dequantize(codes, scale, 16)[:100]
    top = scale.repeat_interleave(16)[:100, None]
    # half a step: int8 0.5 of the scale; e4m3 2^-4 of the value, 2^-10 of the scale below the normal codes
    half = top * 0.5 if int8 else torch.maximum(x.abs() * 2.0 ** -4, top * 2.0 ** -10)
    assert ((y - x).abs() <= (4 if int8 else 1.1) * half).all()      # int8: a growth adds half a (smaller) step each
    whole, s1 = O.b8_append(torch.zeros(112, 64, dtype=torch.float64), torch.zeros(7, dtype=torch.float64), x, 0, 16, int8)
    assert torch.equal(s1[:6], scale[:6]) or not int8
    if not int8:                                                      # powers of two: growth loses nothing above the smallest normal code
        a, b = O.b8_dequantize(whole, s1, 16)[:100], y
        assert torch.equal(s1[:7], scale[:7]) and ((a == b) | (a.abs() < 2.0 ** -5 * top)).all()

"""Caches held in 8 bits for the tests: made, poisoned and read on the CPU."""
import torch

from oracle import oracle as O

TORCH = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
POISON = {"e4m3": 0x7F, "int8": 0x80}       # NaN; the one int8 that no code takes


def raw(t):
    return t.view(torch.int8)


class Cache:
    """k and v codes (float64 values), scales and, paged, a block table; `to_gpu` gives the tensors of a call."""

    def __init__(self, fmt, B, Hkv, rows, D, block, page=0, seed=0, spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.fmt, self.int8, self.block, self.page, self.B = fmt, fmt == "int8", block, page, B
        unit = page or block
        self.rows = rows if not page else -(-rows // unit) * unit
        self.blocks = -(-self.rows // block)
        self.codes, self.scale = [], []
        for _ in range(2):
            x = torch.randn(B, Hkv, self.rows, D, generator=g, dtype=torch.float64)
            x *= torch.exp(spread * torch.randn(B, Hkv, self.rows, 1, generator=g, dtype=torch.float64))
            pad = torch.zeros(B, Hkv, self.blocks * block, D, dtype=torch.float64)
            pad[:, :, :self.rows] = x
            amax = pad.view(B, Hkv, self.blocks, block, D).abs().amax((-1, -2))
            s = O.b8_scale(amax, self.int8)
            self.scale.append(s)
            self.codes.append(O.b8_codes(x, s.repeat_interleave(block, -1)[:, :, :self.rows, None], self.int8))
        self.table = None
        if page:
            n = B * self.rows // page
            self.table = torch.randperm(n + 3, generator=g)[:n].to(torch.int32).view(B, -1)
            self.n_pages = n + 3

    def values(self, i):
        return O.b8_dequantize(self.codes[i], self.scale[i], self.block)

    def _lay_out(self, t, per, fill):
        """[B, Hkv, n, ...] -> itself, or pages of `per` entries."""
        if not self.page:
            return t.contiguous()
        B, H, n = t.shape[:3]
        pool = torch.full((self.n_pages, H, per, *t.shape[3:]), fill, dtype=t.dtype)
        pool[self.table.long().view(-1)] = t.view(B, H, n // per, per, *t.shape[3:]).transpose(1, 2).reshape(-1, H, per, *t.shape[3:])
        return pool

    def to_gpu(self, lens=None):
        """k codes, v codes, k scales, v scales.  With `lens` everything behind them is poison: codes that are no values, NaN scales."""
        out = []
        for i in range(2):
            c = raw(self.codes[i].float().to(TORCH[self.fmt]).contiguous()).clone()
            s = self.scale[i].float()
            if lens is not None:
                s = s.clone()
                for b in range(self.B):
                    n = int(lens[b])
                    c[b, :, n:] = POISON[self.fmt] - (256 if POISON[self.fmt] > 127 else 0)
                    s[b, :, -(-n // self.block):] = float("nan")
            out.append((self._lay_out(c, self.page, 0).cuda().view(TORCH[self.fmt]), self._lay_out(s, (self.page or 1) // self.block or 1, 1.0).cuda()))
        return out[0][0], out[1][0], out[0][1], out[1][1]

    def back(self, codes, scale):
        """Tensors of a call -> [B, Hkv, rows, D] float64 code values and [B, Hkv, blocks] float64."""
        c, s = codes.cpu().float().double(), scale.cpu().double()
        if self.page:
            def gather(t):
                x = t[self.table.long()]                                  # [B, pages, H, per, ...]
                return x.transpose(1, 2).reshape(self.B, t.size(1), -1, *t.shape[3:])
            return gather(c), gather(s)
        return c, s

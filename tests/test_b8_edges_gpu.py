"""GPU: calls at the edges of the 8-bit cache's operators that test_b8_gpu.py does not make."""
import pytest
import torch

from _b8 import Cache

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

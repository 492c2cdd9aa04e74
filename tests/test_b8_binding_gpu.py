"""The Python side of the 8-bit cache and the norms: argument checks, both bindings and the direct entry points, opcheck."""
import os
import subprocess
import sys

import pytest
import torch

from conftest import PKG_ROOT

pytestmark = pytest.mark.gpu


def tensors(D=64, L=1):
    g = torch.Generator().manual_seed(4)
    r = lambda *s: torch.randn(*s, generator=g).half().cuda()  # noqa: E731
    d = dict(q=r(2, L, 4, D), k=r(2, L, 2, D), v=r(2, L, 2, D), w=r(D), n=torch.tensor([3, 20], dtype=torch.int32, device="cuda"))
    d["c"] = torch.randint(-127, 128, (2, 2, 64, D), generator=g, dtype=torch.int8).cuda()
    d["d"] = d["c"].clone()
    d["s"] = torch.rand(2, 2, 4, generator=g).cuda()
    d["u"] = d["s"].clone()
    d["o"] = torch.zeros(2, 4, 1, D, dtype=torch.float16, device="cuda")
    d["x"], d["y"] = (torch.zeros(2, 2, 64, D, dtype=torch.float16, device="cuda") for _ in range(2))
    d["t"] = torch.arange(2, dtype=torch.int32, device="cuda").view(2, 1)
    return d


def calls(kerns, **over):
    d = {**tensors(), **over}
    g = lambda *names: [d[n] for n in names]  # noqa: E731
    rot = over.get("rot", 64)
    blk = over.get("blk", 16)
    return {
        "norm": lambda: kerns.qk_norm_rope(rot, 1e4, 0, 1e-6, *g("q", "k", "w", "w", "n")),
        "append": lambda: kerns.rope_kv_append_b8(rot, 1e4, 0, *g("q", "k", "v", "c", "d", "s", "u"), blk, d["n"]),
        "append_norm": lambda: kerns.rope_kv_append_b8(rot, 1e4, 0, *g("q", "k", "v", "c", "d", "s", "u"), blk, *g("n", "w", "w"), 1e-5),
        "append_paged": lambda: kerns.rope_kv_append_b8_paged(rot, 1e4, 0, *g("q", "k", "v", "c", "d", "s", "u"), blk, *g("t", "n")),
        "decode": lambda: kerns.flash_attn_decode_b8(d["q"].transpose(1, 2), *g("c", "d", "s", "u"), blk, *g("n", "o")),
        "decode_paged": lambda: kerns.flash_attn_decode_b8_paged(d["q"].transpose(1, 2), *g("c", "d", "s", "u"), blk, *g("t", "n", "o")),
        "read": lambda: kerns.kv_read_b8(*g("c", "d", "s", "u"), blk, *g("n", "x", "y")),
        "read_paged": lambda: kerns.kv_read_b8_paged(*g("c", "d", "s", "u"), blk, *g("t", "n", "x", "y")),
    }


def test_the_calls_themselves_pass(kerns):
    for name, call in calls(kerns).items():
        assert call() is None, name
    torch.cuda.synchronize()


@pytest.mark.parametrize("which,change", [
    ("norm", lambda d: dict(k=d["k"].bfloat16())), ("norm", lambda d: dict(w=d["w"][:32])), ("norm", lambda d: dict(w=d["w"].double())),
    ("norm", lambda d: dict(n=d["n"].long())), ("norm", lambda d: dict(n=d["n"][:1])), ("norm", lambda d: dict(n=d["n"].cpu())),
    ("norm", lambda d: dict(rot=72)), ("norm", lambda d: dict(q=d["q"].float(), k=d["k"].float())), ("norm", lambda d: dict(w=d["w"].expand(3, 64))),
    ("append", lambda d: dict(c=d["c"].half())), ("append", lambda d: dict(d=d["d"].view(torch.float8_e4m3fn))), ("append", lambda d: dict(blk=48)),
    ("append", lambda d: dict(blk=32)), ("append", lambda d: dict(s=d["s"].half(), u=d["u"].half())), ("append", lambda d: dict(s=d["s"][:, :, :3])),
    ("append", lambda d: dict(v=d["v"].transpose(0, 1))), ("append", lambda d: dict(s=d["s"].cpu())), ("append", lambda d: dict(c=d["c"][:, :1], d=d["d"][:, :1])),
    ("append", lambda d: dict(c=d["c"].view(torch.uint8), d=d["d"].view(torch.uint8))),
    ("append_paged", lambda d: dict(t=d["t"].long())), ("append_paged", lambda d: dict(t=d["t"][:1])), ("append_paged", lambda d: dict(t=d["t"].cpu())),
    ("decode", lambda d: dict(q=torch.cat([d["q"]] * 2, 1))), ("decode", lambda d: dict(o=d["o"].bfloat16())), ("decode", lambda d: dict(blk=128)),
    ("decode", lambda d: dict(c=d["c"][..., :32], d=d["d"][..., :32])), ("decode", lambda d: dict(c=d["c"][:1], d=d["d"][:1])),
    ("decode", lambda d: dict(s=d["s"].transpose(1, 2).contiguous().transpose(1, 2), u=d["u"].transpose(1, 2).contiguous().transpose(1, 2))),
    ("read", lambda d: dict(y=d["y"].bfloat16())), ("read", lambda d: dict(x=d["x"].float(), y=d["y"].float())),
    ("read", lambda d: dict(x=d["x"][:, :1], y=d["y"][:, :1])), ("read_paged", lambda d: dict(t=d["t"].float()))])
def test_refusals(kerns, which, change):
    with pytest.raises(RuntimeError):
        calls(kerns, **change(tensors()))[which]()


def test_one_weight_without_the_other_is_refused(kerns):
    d = tensors()
    for w in ((d["w"], None), (None, d["w"])):
        with pytest.raises(RuntimeError):
            kerns.rope_kv_append_b8(64, 1e4, 0, d["q"], d["k"], d["v"], d["c"], d["d"], d["s"], d["u"], 16, d["n"], *w)


def test_opcheck():
    import minfer.kernels.torch_ext  # noqa: F401
    d = tensors()
    ops, only = torch.ops.minfer, ("test_schema", "test_faketensor")
    g = lambda *names: [d[n] for n in names]  # noqa: E731
    w2 = d["w"].clone()
    torch.library.opcheck(ops.qk_norm_rope.default, (64, 1e4, 0, 1e-6, *g("q", "k", "w"), w2, d["n"]), test_utils=only)
    kc, vc = torch.zeros(2, 2, 64, 64, dtype=torch.float16, device="cuda"), torch.zeros(2, 2, 64, 64, dtype=torch.float16, device="cuda")
    torch.library.opcheck(ops.qk_norm_rope_kv_append.default, (64, 1e4, 0, 1e-6, *g("q", "k", "v", "w"), w2, kc, vc, d["n"]), test_utils=only)
    torch.library.opcheck(ops.qk_norm_rope_kv_append_paged.default, (64, 1e4, 0, 1e-6, *g("q", "k", "v", "w"), w2, kc, vc, *g("t", "n")), test_utils=only)
    torch.library.opcheck(ops.rope_kv_append_b8.default, (64, 1e4, 0, *g("q", "k", "v", "c", "d", "s", "u"), 16, d["n"], d["w"], w2, 1e-6), test_utils=only)
    torch.library.opcheck(ops.rope_kv_append_b8_paged.default, (64, 1e4, 0, *g("q", "k", "v", "c", "d", "s", "u"), 16, *g("t", "n")), test_utils=only)
    q1 = d["q"].transpose(1, 2).contiguous()
    torch.library.opcheck(ops.flash_attn_decode_b8.default, (q1, *g("c", "d", "s", "u"), 16, *g("n", "o")), test_utils=only)
    torch.library.opcheck(ops.flash_attn_decode_b8_paged.default, (q1, *g("c", "d", "s", "u"), 16, *g("t", "n", "o")), test_utils=only)
    torch.library.opcheck(ops.kv_read_b8.default, (*g("c", "d", "s", "u"), 16, *g("n", "x", "y")), test_utils=only)
    torch.library.opcheck(ops.kv_read_b8_paged.default, (*g("c", "d", "s", "u"), 16, *g("t", "n", "x", "y")), test_utils=only)


_RUN = """
import sys, torch
sys.path[:0] = [{pkg!r}, {tests!r}]
import test_b8_binding_gpu as T
from minfer.kernels import KernelBackend
from minfer.kernels.torch_ext import ops
assert ops.BINDING == {binding!r}, ops.BINDING
d = T.tensors(128, 5)
for call in T.calls(KernelBackend("torch_ext"), **{{**d, "q": d["q"][:, :1], "k": d["k"], "rot": 128}}).items():
    if call[0] in ("decode", "decode_paged", "read", "read_paged"):
        call[1]()
kerns = KernelBackend("torch_ext")
kerns.rope_kv_append_b8(128, 1e4, 1, d["q"], d["k"], d["v"], d["c"], d["d"], d["s"], d["u"], 16, d["n"], d["w"], d["w"], 1e-6)
kerns.rope_kv_append_b8_paged(128, 1e4, 1, d["q"], d["k"], d["v"], d["c"], d["d"], d["s"], d["u"], 16, d["t"], d["n"])
kerns.qk_norm_rope(128, 1e4, 0, 1e-6, d["q"], d["k"], d["w"], d["w"], d["n"])
h, i = d["x"].clone(), d["y"].clone()
kerns.qk_norm_rope_kv_append(128, 1e4, 0, 1e-6, d["q"], d["k"], d["v"], d["w"], d["w"], h, i, d["n"])
kerns.qk_norm_rope_kv_append_paged(128, 1e4, 0, 1e-6, d["q"], d["k"], d["v"], d["w"], d["w"], h, i, d["t"], d["n"])
torch.cuda.synchronize()
torch.save([x.cpu() for x in (*d.values(), h, i)], {out!r})
"""


@pytest.mark.parametrize("binding", ["ctypes", "stable"])
def test_both_bindings_give_the_bits_of_the_direct_entry_points(tmp_path, binding):
    got = {}
    for choice, name in (("auto", "stable"), (binding, binding)):
        out = str(tmp_path / f"{choice}.pt")
        code = _RUN.format(pkg=PKG_ROOT, tests=os.path.dirname(os.path.abspath(__file__)), binding=name, out=out)
        env = dict(os.environ, MINFER_ATTN_BINDING=choice)
        r = subprocess.run([sys.executable, "-c", code], env=env, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        got[choice] = torch.load(out)
    a, b = got.values()
    assert all(torch.equal(x, y) for x, y in zip(a, b))

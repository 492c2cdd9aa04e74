"""Performance cases of the block-scaled 8-bit KV cache and of the query/key norms in front of it.

The operators, as `KernelBackend("torch_ext")` offers them:

  qk_norm_rope                        RMS norm of every query and key head, then the position rotation, in place
  qk_norm_rope_kv_append[_paged]      the same with keys and values written to a 16-bit cache
  rope_kv_append_b8[_paged]           rotation (with or without norms) and append to a cache held in 8 bits, one fp32
                                      scale for each block of tokens and head
  kv_read_b8[_paged]                  cached rows back as 16-bit values, for a prompt's attention behind a cached prefix
  flash_attn_decode_b8[_paged]        one query token per sequence over that cache

With `own` false `run` computes the same in elementary torch operations.  Run from the repository's root.
"""
import math
import os
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_BASE = 500000.0
_EPS = 1e-6
_E4M3_MAX = 448.0


def _case(name, kind, batch, heads, kv_heads, head_dim, dtype, seq, len_lo, len_hi, fmt="16", block=0, page=0, style=0,
          rot=None, norm=True, weights="row"):
    return {"name": name, "kind": kind, "batch": batch, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "dtype": dtype, "seq": seq, "len_lo": len_lo, "len_hi": len_hi, "fmt": fmt, "block": block, "page": page,
            "style": style, "rot": head_dim if rot is None else rot, "norm": norm, "weights": weights}


def listed():
    return [
        # one token of one conversation: the step before attention, where latency counts
        _case("norm_token", "norm", 1, 32, 8, 128, "bf16", 1, 778, 778, style=1),
        # three prompts of a length that fills no tile, a weight for each head, half of the dimensions rotated
        _case("norm_prompts_997", "norm", 3, 24, 8, 64, "fp16", 997, 997, 2000, rot=32, weights="head_fp32"),
        # a serving step of 64 conversations on a paged 16-bit cache
        _case("norm_append_paged_step", "norm_append", 64, 32, 8, 128, "bf16", 1, 512, 8192, page=64, style=1),
        # the prefill benchmark's prompts into the contiguous cache
        _case("norm_append_l4096", "norm_append", 4, 32, 8, 128, "fp16", 4096, 4096, 4096),
        # a serving step on the 8-bit paged cache: one token into blocks that are partly filled
        _case("append_b8_step", "append", 64, 32, 8, 128, "bf16", 1, 512, 8192, "e4m3", 64, 64, 1),
        # prompts into the 8-bit cache, no norms
        _case("append_b8_l4096", "append", 4, 32, 8, 128, "fp16", 4096, 4096, 4096, "e4m3", 128, norm=False),
        # chunked prefill: 1000 tokens behind 15 k cached ones, appended, and all rows read back for their attention
        _case("chunk_b8_int8_16k", "chunk", 1, 32, 8, 128, "bf16", 1000, 16000, 16000, "int8", 64, 256, 1),
        # the end-to-end configuration's prompts, small blocks
        _case("chunk_b8_batch8_d64", "chunk", 8, 32, 8, 64, "fp16", 512, 512, 512, "e4m3", 16, norm=False),
        # one conversation's next token
        _case("decode_b8_777", "decode", 1, 32, 8, 128, "bf16", 1, 777, 777, "e4m3", 64, norm=False),
        # the decode benchmark's batch
        _case("decode_b8_batch64", "decode", 64, 32, 8, 128, "fp16", 1, 512, 8192, "e4m3", 64, norm=False),
        # ragged conversations on int8 pages, six query heads to a key head
        _case("decode_b8_int8_paged", "decode", 24, 48, 8, 128, "bf16", 1, 700, 10001, "int8", 32, 64, norm=False),
        # one very long document
        _case("decode_b8_long", "decode", 1, 64, 8, 128, "fp16", 1, 131072, 131072, "e4m3", 128, norm=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


_HEADS = ((32, 8), (32, 8), (64, 8), (48, 8), (24, 8), (16, 16), (8, 1), (10, 2))
_MOST_BYTES = 500 << 20


def draw(rng):
    kind = rng.choice(("norm", "norm_append", "append", "append", "chunk", "decode", "decode", "decode"))
    heads, kv_heads = rng.choice(_HEADS)
    head_dim = rng.choice((64, 128, 128))
    dtype = rng.choice(("fp16", "bf16"))
    style = rng.randrange(2)
    rot = rng.choice((head_dim, head_dim, head_dim // 2))
    norm = kind in ("norm", "norm_append") or rng.random() < 0.5
    weights = rng.choice(("row", "row_fp32", "head", "head_fp32"))
    fmt = "16" if kind in ("norm", "norm_append") else rng.choice(("e4m3", "e4m3", "int8"))
    if kind == "append":
        fmt = "e4m3"
    block = 0 if fmt == "16" else rng.choice((16, 32, 64, 128))
    page = rng.choice((0, 16, 64, 256)) if kind != "norm" else 0
    if page:
        page = max(page, block)
    batch = _log_int(rng, 1, 96)
    if kind == "decode":
        seq = 1
        most = _MOST_BYTES // (batch * kv_heads * head_dim * 2)
        len_hi = max(1, min(_log_int(rng, 1, 131072), most))
        len_lo = max(1, round(len_hi * rng.choice((0.05, 0.3, 1.0))))
    else:
        seq = 1 if rng.random() < 0.4 else _log_int(rng, 2, 8192)
        row = head_dim * (4 * heads + 8 * kv_heads)
        seq = max(1, min(seq, (_MOST_BYTES // 2) // (batch * row)))
        behind = 0 if rng.random() < 0.4 else _log_int(rng, 1, 16384)
        behind = min(behind, (_MOST_BYTES // 2) // (batch * kv_heads * head_dim * 4))
        len_lo = seq + (behind if rng.random() < 0.5 else behind // 3)
        len_hi = seq + behind
    case = _case("", kind, batch, heads, kv_heads, head_dim, dtype, seq, len_lo, len_hi, fmt, block, page, style, rot, norm,
                 weights)
    del case["name"]
    return case


def _lengths(case):
    """Lengths after this call, evenly spread, so that a case's work does not hang on the seed."""
    n, lo, hi = case["batch"], case["len_lo"], case["len_hi"]
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def work(case):
    h, g, d, b, n = case["heads"], case["kv_heads"], case["head_dim"], case["batch"], case["seq"]
    total = sum(_lengths(case))
    tokens = b * n
    if case["kind"] == "decode":
        return {"bytes": total * g * 2 * (d + 4 / case["block"]) + 4 * b * h * d, "flops": 4 * h * d * total}
    flops = tokens * d * (6 * h + 6 * g)                                     # squares, scales and rotation
    moved = 4 * tokens * h * d                                               # q there and back
    if case["kind"] == "norm":
        return {"bytes": moved + 4 * tokens * g * d, "flops": flops}
    moved += 4 * tokens * g * d                                              # the new keys and values
    if case["fmt"] == "16":
        return {"bytes": moved + 4 * tokens * g * d, "flops": flops}
    moved += 2 * tokens * g * (d + 4 / case["block"])
    if case["kind"] == "chunk":
        moved += 2 * (total - tokens) * g * (d + 4 / case["block"]) + 4 * total * g * d   # cached rows; all of them as 16-bit
        flops += 2 * total * g * d
    return {"bytes": moved, "flops": flops}


# ---- inputs ----

class _Draws:
    def __init__(self, case, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)
        self.dtype = _DTYPES[case["dtype"]]

    def normal(self, *dims, dtype=None):
        return torch.randn(*dims, generator=self.gen, device="cuda", dtype=dtype or self.dtype)

    def permutation(self, n):
        return torch.randperm(n, generator=self.gen, device="cuda")


def _filled_cache(draws, case, outer, rows):
    """Cached rows [outer, kv heads, rows, D] whose tokens differ in magnitude, with the scale of each block."""
    g, d, blk = case["kv_heads"], case["head_dim"], case["block"]
    codes = torch.empty(outer, g, rows, d, dtype=torch.float8_e4m3fn if case["fmt"] == "e4m3" else torch.int8, device="cuda")
    scale = torch.empty(outer, g, rows // blk, dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (g * rows * d))
    for i in range(0, outer, step):
        n = min(step, outer - i)
        x = draws.normal(n, g, rows // blk, blk, d, dtype=torch.float32)
        x *= torch.exp(0.5 * draws.normal(n, g, rows // blk, blk, 1, dtype=torch.float32))
        s = _scale_of(x.abs().amax((-1, -2)), case["fmt"])
        scale[i:i + n] = s
        x /= s[..., None, None]
        codes[i:i + n] = (x if case["fmt"] == "e4m3" else x.round()).to(codes.dtype).view(n, g, rows, d)
    return codes, scale


def prepare(case, seed):
    draws = _Draws(case, seed)
    b, h, g, d, n = case["batch"], case["heads"], case["kv_heads"], case["head_dim"], case["seq"]
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")[draws.permutation(b)].contiguous()
    state = {"case": case, "lens": lens, "start": (lens - n).contiguous(), "table": None}
    blk = case["block"] or 1
    unit = case["page"] or case["block"] or 8
    # rows behind the longest sequence: a padded cache has them, and the plain form looks at whole blocks
    max_len = -(-(case["len_hi"] + 2 * blk) // unit) * unit
    outer, rows = b, max_len
    if case["page"]:
        per_seq = max_len // case["page"]
        outer, rows = b * per_seq, case["page"]
        state["table"] = draws.permutation(outer).to(torch.int32).view(b, per_seq)
    if case["kind"] == "decode":
        state["q"] = draws.normal(b, h, 1, d)
        state["out"] = torch.zeros_like(state["q"])
    else:
        # the fused projection's output, as views
        qkv = draws.normal(b, n, (h + 2 * g) * d)
        state["q"] = qkv[..., :h * d].view(b, n, h, d)
        state["k"] = qkv[..., h * d:(h + g) * d].view(b, n, g, d)
        state["v"] = qkv[..., (h + g) * d:].view(b, n, g, d)
        wt = torch.float32 if case["weights"].endswith("fp32") else draws.dtype
        per_head = case["weights"].startswith("head")
        state["qw"] = (1 + 0.1 * draws.normal(*((h, d) if per_head else (d,)), dtype=torch.float32)).to(wt)
        state["kw"] = (1 + 0.1 * draws.normal(*((g, d) if per_head else (d,)), dtype=torch.float32)).to(wt)
    if case["fmt"] == "16":
        if case["kind"] != "norm":
            state["k_cache"], state["v_cache"] = draws.normal(outer, g, rows, d), draws.normal(outer, g, rows, d)
    else:
        state["k_cache"], state["k_scale"] = _filled_cache(draws, case, outer, rows)
        state["v_cache"], state["v_scale"] = _filled_cache(draws, case, outer, rows)
    if case["kind"] == "chunk":
        state["k_out"] = torch.zeros(b, g, case["len_hi"], d, dtype=draws.dtype, device="cuda")
        state["v_out"] = torch.zeros_like(state["k_out"])
    return state


# ---- the plain form ----

def _scale_of(amax, fmt):
    if fmt == "int8":
        return amax / 127
    # the smallest power of two that brings the largest magnitude to 448 or less
    mant, ex = torch.frexp(amax)
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), ex - 9 + (mant > 0.875)), torch.zeros_like(amax))


def _coded(x, scale, fmt):
    """Values and the scale of each (broadcast) as codes."""
    if fmt == "int8":
        y = torch.where(scale > 0, x.double() / scale.double(), torch.zeros((), dtype=torch.float64, device=x.device))
        return y.round().clamp(-127, 127).to(torch.int8)
    y = torch.where(scale > 0, x / scale, torch.zeros((), dtype=x.dtype, device=x.device))
    return y.clamp(-_E4M3_MAX, _E4M3_MAX).to(torch.float8_e4m3fn)


def _angles(case, start):
    """cos and sin [B, L, 1, rot / 2]; the angles of far positions want 64 bits."""
    i = torch.arange(case["rot"] // 2, dtype=torch.float64, device=start.device)
    pos = start.double()[:, None] + torch.arange(case["seq"], device=start.device)
    ang = pos[:, :, None, None] * _BASE ** (-2 * i / case["rot"])
    return ang.cos().float(), ang.sin().float()


def _rotated(x, case, cos, sin):
    rot, half = case["rot"], case["rot"] // 2
    if case["style"] == 0:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:rot]
        y = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _normed(x, weight):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS) * weight.float()


def _turned(s, name):
    """Queries or keys of the call in fp32: normed (where the case says so) and rotated."""
    case = s["case"]
    x = s[name].float()
    if case["norm"]:
        x = _normed(x, s[name + "w"])
    return _rotated(x, case, *_angles(case, s["start"]))


def _places(s, pos):
    """Positions [B, n] of the sequences as (outer index, row) of the cache."""
    case = s["case"]
    if case["page"]:
        return s["table"].long().gather(1, pos // case["page"]), pos % case["page"]
    return torch.arange(case["batch"], device=pos.device)[:, None].expand_as(pos), pos


def _gathered(t, o, r):
    """t[o, :, r]: [B, n, Hkv, ...]"""
    return t.view(torch.int8)[o, :, r].view(t.dtype) if t.element_size() == 1 else t[o, :, r]


def _append_16(s, k):
    pos = s["start"].long()[:, None] + torch.arange(s["case"]["seq"], device=k.device)
    o, r = _places(s, pos)
    s["k_cache"][o, :, r] = k.to(s["k_cache"].dtype)
    s["v_cache"][o, :, r] = s["v"]


def _append_8(s, x, cache, scale):
    """The new rows x [B, L, Hkv, D] (fp32) into the blocks they fall into; a block that was begun keeps its rows, under a larger
    scale where the new ones need it."""
    case = s["case"]
    blk, n, fmt = case["block"], case["seq"], case["fmt"]
    b, _, g, d = x.shape
    start = s["start"].long()
    first = start // blk
    nb = (n + blk - 2) // blk + 1
    pos = first[:, None] * blk + torch.arange(nb * blk, device=x.device)                  # all rows of those blocks
    at = pos - start[:, None]                                                             # which new row
    new = (at >= 0) & (at < n)
    o, r = _places(s, pos)
    held = _gathered(cache, o, r).view(torch.int8)                                             # [B, rows, Hkv, D], their bytes
    old = held.view(cache.dtype).float()
    so, sr = _places(s, (first[:, None] + torch.arange(nb, device=x.device)) * blk)
    s_old = scale[so, :, sr // blk]                                                       # [B, nb, Hkv]
    begun = ((start % blk != 0)[:, None] & (torch.arange(nb, device=x.device) == 0))[..., None]
    s0 = torch.where(begun, s_old, torch.zeros_like(s_old))
    fresh = x.gather(1, at.clamp(0, n - 1)[:, :, None, None].expand(b, nb * blk, g, d))
    amax = torch.where(new[:, :, None, None], fresh.abs(), torch.zeros_like(fresh)).view(b, nb, blk, g, d).amax((2, 4))
    s1 = torch.maximum(s0, _scale_of(amax, fmt))
    rows = lambda t: t.repeat_interleave(blk, 1)[..., None]  # noqa: E731
    value = torch.where(new[:, :, None, None], fresh, old * rows(s0))
    keep = (at >= n)[:, :, None, None]                                                    # rows behind the call's last token
    codes = torch.where(keep, held, _coded(value, rows(s1), fmt).view(torch.int8))
    cache.view(torch.int8)[o, :, r] = codes
    scale[so, :, sr // blk] = torch.where(new.view(b, nb, blk).any(-1)[..., None], s1, s_old)


def _read_8(s, cache, scale, out):
    case = s["case"]
    n = out.size(2)
    pos = torch.arange(n, device=out.device).expand(case["batch"], n)
    o, r = _places(s, pos)
    x = _gathered(cache, o, r).float() * scale[o, :, r // case["block"]][..., None]               # [B, n, Hkv, D]
    live = (pos < s["lens"][:, None])[:, None, :, None]
    out.copy_(torch.where(live, x.transpose(1, 2).to(out.dtype), out))


def _decode_plain(s):
    case = s["case"]
    b, h, g, d = case["batch"], case["heads"], case["kv_heads"], case["head_dim"]
    pos = torch.arange(case["len_hi"], device=s["q"].device).expand(b, -1)
    if case["page"]:
        o, r = _places(s, pos)
        k, v = (_gathered(s[c], o, r).transpose(1, 2) for c in ("k_cache", "v_cache"))
        ks, vs = (s[c][o, :, r // case["block"]].transpose(1, 2) for c in ("k_scale", "v_scale"))
    else:
        k, v = (s[c][:, :, :case["len_hi"]] for c in ("k_cache", "v_cache"))
        ks, vs = (s[c].repeat_interleave(case["block"], 2)[:, :, :case["len_hi"]] for c in ("k_scale", "v_scale"))
    q = s["q"].float().view(b, g, h // g, d)
    t = q @ k.float().transpose(2, 3) * (ks[:, :, None] / math.sqrt(d))
    t = t.masked_fill((pos >= s["lens"][:, None])[:, None, None], float("-inf"))
    p = torch.exp(t - t.amax(-1, keepdim=True))
    o = (p * vs[:, :, None]) @ v.float() / p.sum(-1, keepdim=True)
    s["out"].copy_(o.view(b, h, 1, d))


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "decode":
        return _decode_plain(s)
    k = _turned(s, "k")
    s["q"].copy_(_turned(s, "q"))
    if case["kind"] == "norm":
        s["k"].copy_(k)
    elif case["kind"] == "norm_append":
        _append_16(s, k)
    else:
        _append_8(s, k, s["k_cache"], s["k_scale"])
        _append_8(s, s["v"].float(), s["v_cache"], s["v_scale"])
        if case["kind"] == "chunk":
            _read_8(s, s["k_cache"], s["k_scale"], s["k_out"])
            _read_8(s, s["v_cache"], s["v_scale"], s["v_out"])


# ---- the framework's calls ----

def _kernels():
    global _KERNS
    if _KERNS is None:
        pkg = os.path.abspath("minfer-python_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from minfer.kernels import KernelBackend
        _KERNS = KernelBackend("torch_ext")
    return _KERNS


_KERNS = None


def _run_own(s):
    kern, case, table = _kernels(), s["case"], s["table"]
    turn = (case["rot"], _BASE, case["style"])
    if case["kind"] == "norm":
        kern.qk_norm_rope(*turn, _EPS, s["q"], s["k"], s["qw"], s["kw"], s["start"])
        return
    if case["kind"] == "norm_append":
        if table is None:
            kern.qk_norm_rope_kv_append(*turn, _EPS, s["q"], s["k"], s["v"], s["qw"], s["kw"], s["k_cache"], s["v_cache"], s["start"])
        else:
            kern.qk_norm_rope_kv_append_paged(*turn, _EPS, s["q"], s["k"], s["v"], s["qw"], s["kw"], s["k_cache"], s["v_cache"], table,
                                              s["start"])
        return
    cache = (s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], case["block"])
    if case["kind"] == "decode":
        if table is None:
            kern.flash_attn_decode_b8(s["q"], *cache, s["lens"], s["out"])
        else:
            kern.flash_attn_decode_b8_paged(s["q"], *cache, table, s["lens"], s["out"])
        return
    qw, kw = (s["qw"], s["kw"]) if case["norm"] else (None, None)
    if table is None:
        kern.rope_kv_append_b8(*turn, s["q"], s["k"], s["v"], *cache, s["start"], qw, kw, _EPS)
    else:
        kern.rope_kv_append_b8_paged(*turn, s["q"], s["k"], s["v"], *cache, table, s["start"], qw, kw, _EPS)
    if case["kind"] == "chunk":
        if table is None:
            kern.kv_read_b8(*cache, s["lens"], s["k_out"], s["v_out"])
        else:
            kern.kv_read_b8_paged(*cache, table, s["lens"], s["k_out"], s["v_out"])


def run(state):
    if own:
        _run_own(state)
    else:
        _run_plain(state)
    kind = state["case"]["kind"]
    if kind == "decode":
        return state["out"]
    if kind == "norm":
        return state["q"], state["k"]
    if kind == "norm_append":
        return state["q"], state["k_cache"], state["v_cache"]
    if kind == "append":
        # e4m3 codes are values as they are; the scales beside them
        return state["q"], state["k_cache"], state["v_cache"], state["k_scale"], state["v_scale"]
    return state["q"], state["k_out"], state["v_out"], state["k_scale"], state["v_scale"]


# ---- the definition in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    b, n, g, d, blk = case["batch"], case["seq"], case["kv_heads"], case["head_dim"], case["block"]
    group = case["heads"] // g
    starts, lens = s["start"].tolist(), s["lens"].tolist()

    def rows_of(cache, i, lo, hi, per=1):
        """Rows lo .. hi (or their blocks) of sequence i: [Hkv, hi - lo, ...], gathered from its pages one index at a time."""
        p = torch.arange(lo, hi, device="cuda")
        raw = cache.view(torch.int8) if cache.element_size() == 1 else cache               # (indexing knows no 8-bit floats)
        if case["page"]:
            got = raw[s["table"][i].long()[p // case["page"]], :, (p % case["page"]) // per].transpose(0, 1)
        else:
            got = raw[i][:, p // per]
        return got.contiguous().view(cache.dtype)

    if case["kind"] == "decode":
        out = torch.zeros(b, case["heads"], 1, d, dtype=torch.float64, device="cuda")
        for i in range(b):
            k, v = (rows_of(s[c], i, 0, lens[i]).double() for c in ("k_cache", "v_cache"))
            k *= rows_of(s["k_scale"], i, 0, lens[i], blk).double()[..., None]
            v *= rows_of(s["v_scale"], i, 0, lens[i], blk).double()[..., None]
            q = s["q"][i].double().view(g, group, d)
            p = torch.softmax(torch.einsum("ghd,gld->ghl", q, k) / math.sqrt(d), -1)
            out[i] = torch.einsum("ghl,gld->ghd", p, v).reshape(case["heads"], 1, d)
        return out

    def turn(x, w, first):
        x = x.double()
        if case["norm"]:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + _EPS) * w.double()
        half = case["rot"] // 2
        freq = torch.tensor([_BASE ** (-2.0 * i / case["rot"]) for i in range(half)], dtype=torch.float64, device="cuda")
        z = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), (first + torch.arange(n, device="cuda"))[:, None] * freq)[:, None]
        y = x.clone()
        if case["style"] == 0:
            y[..., :2 * half] = torch.view_as_real(torch.view_as_complex(x[..., :2 * half].reshape(*x.shape[:-1], half, 2).contiguous()) * z).flatten(-2)
        else:
            c = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * z
            y[..., :half], y[..., half:2 * half] = c.real, c.imag
        return y

    q = torch.stack([turn(s["q"][i], s["qw"], starts[i]) for i in range(b)])
    k = torch.stack([turn(s["k"][i], s["kw"], starts[i]) for i in range(b)])
    if case["kind"] == "norm":
        return q, k
    v = s["v"].double()

    def where(i, p):
        return (int(s["table"][i, p // case["page"]]), p % case["page"]) if case["page"] else (i, p)

    if case["kind"] == "norm_append":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for i in range(b):
            p = torch.arange(starts[i], starts[i] + n, device="cuda")
            o = s["table"][i].long()[p // case["page"]] if case["page"] else torch.full_like(p, i)
            r = p % case["page"] if case["page"] else p
            kc[o, :, r], vc[o, :, r] = k[i], v[i]
        return q, kc, vc

    def scale_for(top):
        if case["fmt"] == "int8":
            return (top / 127).float().double()
        e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448))
        e = torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, e)
        return torch.where(top > 0, torch.exp2(e), torch.zeros_like(top))

    def nearest(x, sc):
        y = torch.where(sc > 0, x / sc.clamp_min(1e-300), torch.zeros_like(x))
        if case["fmt"] == "int8":
            return torch.clamp(torch.round(y), -127, 127)
        step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.clamp(torch.round(y / step) * step, -448, 448)

    if b * (n // blk + 2) > 6000:
        return None
    got = {}
    for name, x in (("k", k), ("v", v)):
        codes, scale = s[name + "_cache"].double(), s[name + "_scale"].double()
        for i in range(b):
            p = starts[i]
            while p < starts[i] + n:
                lo, hi = p // blk * blk, min(p // blk * blk + blk, starts[i] + n)
                o, r = where(i, lo)
                new = x[i, p - starts[i]:hi - starts[i]].transpose(0, 1)                   # [Hkv, rows, D]
                s0 = scale[o, :, r // blk] if p > lo else torch.zeros(g, dtype=torch.float64, device="cuda")
                s1 = torch.maximum(s0, scale_for(new.abs().amax((1, 2))))
                if p > lo:
                    codes[o, :, r:r + p - lo] = nearest(codes[o, :, r:r + p - lo] * s0[:, None, None], s1[:, None, None])
                codes[o, :, r + p - lo:r + hi - lo] = nearest(new, s1[:, None, None])
                scale[o, :, r // blk] = s1
                p = hi
        got[name] = codes, scale
    if case["kind"] == "append":
        return q, got["k"][0], got["v"][0], got["k"][1], got["v"][1]
    read = {}
    for name in "kv":
        out = torch.zeros(b, g, case["len_hi"], d, dtype=torch.float64, device="cuda")
        for i in range(b):
            out[i, :, :lens[i]] = rows_of(got[name][0], i, 0, lens[i]) * rows_of(got[name][1], i, 0, lens[i], blk)[..., None]
        read[name] = out
    return q, read["k"], read["v"], got["k"][1], got["v"][1]

"""Dispatch facade with the reference's shape (src/minfer/kernels/__init__.py:2-18).

Only the attention path's attributes exist: `flash_attn`, `il_rope` and `neox_rope`
keep the reference's signatures; `flash_attn_causal`, `flash_attn_decode` (also over a
Q8_0, a paged or a block-scaled 8-bit cache, "b8"), `rope_kv_append` (likewise),
`qk_norm_rope` and `kv_read_b8` are additions.
"""


class KernelBackend:
    def __init__(self, backend: str):
        if backend == "torch_ext":
            from .torch_ext import flash_attn, flash_attn_causal, flash_attn_decode
            from .torch_ext import il_rope, neox_rope, rope_kv_append
            from .torch_ext import flash_attn_decode_q8, rope_kv_append_q8
            from .torch_ext import flash_attn_decode_paged, rope_kv_append_paged
            from .torch_ext import qk_norm_rope, qk_norm_rope_kv_append, qk_norm_rope_kv_append_paged
            from .torch_ext import rope_kv_append_b8, flash_attn_decode_b8, kv_read_b8
            from .torch_ext import rope_kv_append_b8_paged, flash_attn_decode_b8_paged, kv_read_b8_paged
            self.qk_norm_rope = qk_norm_rope
            self.qk_norm_rope_kv_append = qk_norm_rope_kv_append
            self.qk_norm_rope_kv_append_paged = qk_norm_rope_kv_append_paged
            self.rope_kv_append_b8 = rope_kv_append_b8
            self.flash_attn_decode_b8 = flash_attn_decode_b8
            self.kv_read_b8 = kv_read_b8
            self.rope_kv_append_b8_paged = rope_kv_append_b8_paged
            self.flash_attn_decode_b8_paged = flash_attn_decode_b8_paged
            self.kv_read_b8_paged = kv_read_b8_paged
            self.flash_attn_decode_paged = flash_attn_decode_paged
            self.rope_kv_append_paged = rope_kv_append_paged
            self.flash_attn_decode_q8 = flash_attn_decode_q8
            self.rope_kv_append_q8 = rope_kv_append_q8
            self.il_rope = il_rope
            self.neox_rope = neox_rope
            self.rope_kv_append = rope_kv_append
            self.flash_attn = flash_attn
            self.flash_attn_causal = flash_attn_causal
            self.flash_attn_decode = flash_attn_decode
        else:
            raise ValueError(f"KernelBackend init: unsupported backend {backend}")

"""GPU: the generate app with q/k norms and 8-bit caches against an fp32 CPU twin that recomputes every step, its keys and values
coded as the 64-bit definition codes them.  Tolerance: that of the 16-bit app's test (fp16 matrix products)."""
import pytest
import torch
import torch.nn.functional as F

from oracle import oracle as O
from test_generate_gpu import load_generate_app

pytestmark = pytest.mark.gpu


def coded(x, pieces, block, int8):
    """x [B, T, H, D], appended in `pieces` -> the values that the cache stands for."""
    B, T, H, D = x.shape
    out = torch.empty(B, T, H, D, dtype=torch.float64)
    blocks = -(-T // block)
    for b in range(B):
        for h in range(H):
            codes, scale, p = torch.zeros(T, D, dtype=torch.float64), torch.zeros(blocks, dtype=torch.float64), 0
            for n in pieces:
                codes, scale = O.b8_append(codes, scale, x[b, p:p + n, h].double(), p, block, int8)
                p += n
            out[b, :, h] = O.b8_dequantize(codes, scale, block)
    return out.float()


def twin_logits(model, tokens, pieces):
    s = model.s
    x = model.embed.float().cpu()[tokens.cpu()]
    B, T, _ = x.shape
    nq, nkv = s.heads * s.head_dim, s.kv_heads * s.head_dim
    for lay in model.layers:
        h = F.rms_norm(x, (s.hidden,), lay["attn_norm"].float().cpu(), s.eps)
        qkv = F.linear(h, lay["wqkv"].float().cpu())
        turn = lambda t, w: O.norm_rope(t, lay[w].cpu() if s.qk_norm else None, s.head_dim, s.rope_theta, s.rope_style, [0] * B, s.eps).float()  # noqa: E731
        q = turn(qkv[..., :nq].reshape(B, T, s.heads, s.head_dim), "q_norm")
        k = turn(qkv[..., nq:nq + nkv].reshape(B, T, s.kv_heads, s.head_dim), "k_norm")
        v = qkv[..., nq + nkv:].reshape(B, T, s.kv_heads, s.head_dim)
        if s.kv_cache != "16bit":
            k, v = (coded(t, pieces, s.kv_block, s.kv_cache == "int8") for t in (k, v))
        a = O.attention_f64(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), causal=True)
        x = x + F.linear(a.transpose(1, 2).reshape(B, T, nq), lay["wo"].float().cpu())
        h = F.rms_norm(x, (s.hidden,), lay["ffn_norm"].float().cpu(), s.eps)
        gu = F.linear(h, lay["w_gate_up"].float().cpu())
        x = x + F.linear(F.silu(gu[..., :s.ffn]) * gu[..., s.ffn:], lay["w_down"].float().cpu())
    x = F.rms_norm(x[:, -1], (s.hidden,), model.final_norm.float().cpu(), s.eps)
    return F.linear(x, model.lm_head.float().cpu())


@pytest.mark.parametrize("qk_norm,kv_cache,kv_block,rope_style,head_dim", [(True, "16bit", 64, 1, 128), (True, "e4m3", 16, 1, 64), (False, "int8", 64, 0, 128)])
def test_prefill_then_decode_matches_twin(qk_norm, kv_cache, kv_block, rope_style, head_dim):
    G = load_generate_app()
    shape = G.Shape(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=head_dim, ffn=512, vocab=500, rope_theta=500000.0, rope_style=rope_style,
                    qk_norm=qk_norm, kv_cache=kv_cache, kv_block=kv_block)
    B, L, steps = 2, 150, 3
    model = G.Decoder(shape, B, L + steps)
    tokens = torch.randint(0, shape.vocab, (B, L), generator=torch.Generator().manual_seed(5))
    pieces = [L]
    with torch.no_grad():
        got, want = model.forward(tokens.cuda()), twin_logits(model, tokens, pieces)
        assert torch.allclose(got.float().cpu(), want, atol=2e-2, rtol=2e-2), (got.float().cpu() - want).abs().max()
        for _ in range(steps):
            nxt = want.argmax(dim=-1)                      # teacher forcing with the twin's choice
            tokens = torch.cat([tokens, nxt[:, None]], dim=1)
            pieces.append(1)
            got, want = model.forward(nxt[:, None].cuda()), twin_logits(model, tokens, pieces)
            assert torch.allclose(got.float().cpu(), want, atol=2e-2, rtol=2e-2), (got.float().cpu() - want).abs().max()


@pytest.mark.parametrize("kv_cache", ["e4m3", "int8"])
def test_graph_replay_gives_the_eager_tokens(kv_cache):
    G = load_generate_app()
    shape = G.Shape(layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, ffn=512, vocab=300, qk_norm=True, kv_cache=kv_cache, kv_block=32)
    model = G.Decoder(shape, 3, 64 + 6)
    prompts = torch.randint(0, 300, (3, 64), generator=torch.Generator().manual_seed(1)).cuda()
    with torch.no_grad():
        ids, _ = G.generate(model, prompts, 6)
        model.lens.zero_()
        ids_g, _ = G.generate(model, prompts, 6, False, use_graph=True)
    assert torch.equal(ids, ids_g)

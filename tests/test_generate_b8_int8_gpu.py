"""GPU: the generate app on an int8 cache, in a model whose logits show what the cache holds."""
import pytest
import torch

import test_generate_b8_gpu as T

pytestmark = pytest.mark.gpu


def logits_with(monkeypatch, change, *args):
    """The twin's logits with what its cache stands for changed: change(values, coded values, is_k)."""
    real, calls = T.coded, [0]

    def other(t, *a):
        calls[0] += 1
        return change(t.float(), real(t, *a), calls[0] % 2 == 1)      # (k and v of each layer in turn)
    with monkeypatch.context() as m:
        m.setattr(T, "coded", other)
        return T.twin_logits(*args)


def test_the_logits_depend_on_the_codes(monkeypatch):
    """A pair of k's dimensions carries eight times the rest (and q's an eighth), as keys of real models do, so that int8 keys are coarse.  The
    app's matrix products in fp16, emulated on the CPU, move the logits by up to 0.0085; leaving out the coding moves them by 0.042, keys 5 % too large by 0.059.
    0.02 lies between the two by a factor of 2."""
    G = T.load_generate_app()
    shape = G.Shape(layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, ffn=512, vocab=500, rope_theta=500000.0, rope_style=0, qk_norm=True, kv_cache="int8",
                    kv_block=64)
    B, L, steps = 2, 150, 3
    model = G.Decoder(shape, B, L + steps)
    for lay in model.layers:
        lay["k_norm"][:2] *= 8.0
        lay["q_norm"][:2] /= 8.0
    tokens = torch.randint(0, shape.vocab, (B, L), generator=torch.Generator().manual_seed(5))
    pieces = [L]
    with torch.no_grad():
        got = model.forward(tokens.cuda()).float().cpu()
        for step in range(steps + 1):
            want = T.twin_logits(model, tokens, pieces)
            assert (got - want).abs().max() <= 0.02, step
            for change in (lambda t, c, is_k: t, lambda t, c, is_k: c * 1.05 if is_k else c):
                assert (logits_with(monkeypatch, change, model, tokens, pieces) - want).abs().max() > 0.03, "the twin does not depend on the codes"
            if step < steps:
                nxt = want.argmax(dim=-1)                              # teacher forcing with the twin's choice
                tokens = torch.cat([tokens, nxt[:, None]], dim=1)
                pieces.append(1)
                got = model.forward(nxt[:, None].cuda()).float().cpu()

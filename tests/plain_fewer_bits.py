"""The plain Qwen3 decoder with its matrices and the rows they meet in 8 bits, and its keys and values in 4: every value is
replaced by the one that its code stands for, and the arithmetic stays in 64 bits.

A value next to the border of two codes takes either one, whichever way a rounding before it went: with values that differ by a
share e, about e / step of the codes move, by a whole step each, so that results differ by about sqrt(e step), far more than by e, and
the next layer's by the root of that again.  ``noise`` shows how much: every value is multiplied by 1 + noise * N(0, 1) before it
is brought to a code."""
import torch

import plain_qwen3 as plain


# (a quotient is rounded to 32 bits before it is rounded to a code, as the definition has it: half of a row's largest magnitude is 63.5
# steps, which bfloat16 weights meet often)
def int8_rows(x):
    scale = (x.abs().amax(-1, keepdim=True) / 127).float().to(x.dtype)
    return torch.where(scale > 0, (x / scale).float().round().clamp(-127, 127).to(x.dtype) * scale, torch.zeros_like(x))


def int4_heads(x):
    zero = x.amin(-1, keepdim=True).bfloat16().to(x.dtype)
    scale = ((x.amax(-1, keepdim=True) - zero) / 15).bfloat16().to(x.dtype)
    return torch.where(scale > 0, zero + ((x - zero) / scale).float().round().clamp(0, 15).to(x.dtype) * scale, zero)


def logits(cfg, w, ids, weights8, cache4, noise=0.0, seed=0):
    g = torch.Generator().manual_seed(seed)
    shaken = lambda x: x * (1 + noise * torch.randn(x.shape, generator=g, dtype=x.dtype)) if noise else x

    def product(h, name):
        m, h = w[name + ".weight"], shaken(h)
        y = int8_rows(h) @ int8_rows(m).T if weights8 else h @ m.T
        return y + w[name + ".bias"] if name + ".bias" in w else y

    H, Hkv, D, eps = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"], cfg["rms_norm_eps"]
    T = len(ids)
    cos, sin = plain.rope_tables(D, cfg["rope_theta"], T, torch.float64)
    r = w["model.embed_tokens.weight"][torch.as_tensor(ids)]
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        h = plain.rms_norm(r, w[p + "input_layernorm.weight"], eps)
        q, k, v = (product(h, p + f"self_attn.{n}_proj").view(T, -1, D) for n in "qkv")
        q, k = (plain.apply_rope(plain.rms_norm(x, w[p + f"self_attn.{n}_norm.weight"], eps), cos, sin) for n, x in (("q", q), ("k", k)))
        if cache4:
            k, v = int4_heads(shaken(k)), int4_heads(shaken(v))
        r = r + product(plain.causal_attention(q, k, v, D ** -0.5, plain.layer_window(cfg, i)).reshape(T, H * D), p + "self_attn.o_proj")
        h = plain.rms_norm(r, w[p + "post_attention_layernorm.weight"], eps)
        act = torch.nn.functional.silu(product(h, p + "mlp.gate_proj")) * product(h, p + "mlp.up_proj")
        r = r + product(act, p + "mlp.down_proj")
    hidden = plain.rms_norm(r, w["model.norm.weight"], eps)
    return hidden @ (w["model.embed_tokens.weight"] if cfg["tie_word_embeddings"] else w["lm_head.weight"]).T

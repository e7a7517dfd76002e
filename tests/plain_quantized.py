"""Quantised Llama layers in plain torch, float64: the oracle of ``linear_type`` "int4" and "fp8".

int4: the layers' matrices stand for (q - z) s, a group's 15 steps spanning its values and zero.
fp8: the layers' matrices and the rows that meet them stand for e4m3 values times a float32 scale a row.  Rounding rows to 4 bits
magnifies what came before, so the oracle rounds to bfloat16 where the engine hands a tensor on in bfloat16."""
import re

import torch

import plain_llama as pl

MATRICES = re.compile(r"model\.layers\.\d+\.(self_attn|mlp)\.\w+_proj\.weight")


def int4_of(w, group):
    """What a matrix rounded to 4 bits stands for: the scale in bfloat16, everything to the nearest."""
    out, dim = w.shape
    group = min(group, (dim + 31) // 32 * 32)
    wide = torch.zeros(out, -(-dim // group) * group)
    wide[:, :dim] = w.float()
    wide = wide.view(out, -1, group)
    low, high = wide.amin(2, keepdim=True).clamp(max=0), wide.amax(2, keepdim=True).clamp(min=0)
    scale = ((high - low) / 15).bfloat16().float()
    step = torch.where(scale > 0, scale, torch.ones_like(scale))
    zero = (-low / step).round().clamp(0, 15)
    return ((((wide / step).round() + zero).clamp(0, 15) - zero).double() * scale.double()).view(out, -1)[:, :dim]


def nearest_e4m3(v):
    """The nearest e4m3 value of each, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def e4m3_rows(x):
    most = x.abs().amax(1, keepdim=True)
    safe = torch.where(most > 0, most, torch.ones_like(most))
    return nearest_e4m3(x * 448 / safe) * (most / 448).float().double()


def bf16(x):
    return x.float().bfloat16().double()


class Int4Llama(pl.PlainLlama):
    def __init__(self, path, group):
        super().__init__(path)
        self.w = {k: int4_of(t, group) if MATRICES.fullmatch(k) else t for k, t in self.w.items()}


class Fp8Llama(pl.PlainLlama):
    def __init__(self, path):
        super().__init__(path)
        self.w = {k: e4m3_rows(t) if MATRICES.fullmatch(k) else t for k, t in self.w.items()}

    def block(self, i, x, positions, window=0):
        c, w, p, s = self.c, self.w, f"model.layers.{i}.", x.shape[0]

        def product(h, name):
            return h @ w[p + name + ".weight"].T + w.get(p + name + ".bias", 0.0)

        h = e4m3_rows(pl.plain_rmsnorm(x, w[p + "input_layernorm.weight"], c["eps"]))
        q, k, v = (bf16(product(h, f"self_attn.{n}_proj")).view(s, -1, c["head_dim"]) for n in "qkv")
        q, k = (bf16(pl.plain_rope(t, positions, self.inv_freq)) for t in (q, k))
        a = bf16(pl.plain_attention(q, k, v, window=window).reshape(s, -1))
        x = x + bf16(product(e4m3_rows(a), "self_attn.o_proj"))
        h = e4m3_rows(pl.plain_rmsnorm(x, w[p + "post_attention_layernorm.weight"], c["eps"]))
        f = bf16(torch.nn.functional.silu(product(h, "mlp.gate_proj")) * product(h, "mlp.up_proj"))
        return x + bf16(product(e4m3_rows(f), "mlp.down_proj"))

"""Test infrastructure of the generation tests: the attention of a layer by hand in 64 bits with the spread that its roundings
cause, and a small language model on the CPU oracle, both on weights whose scores spread by several units - on freshly initialised
ones softmax is nearly flat, and neither the rotation nor the scale shows.  What a mistake in the wiring (positions, rotation,
scale) does to them is planted here, in the oracle."""
import contextlib
import math

import numpy as np
import torch

import golden_params
from oracle import neox_layer_oracle as O

U = 2.0 ** -8  # largest relative error of a rounding to bf16
ATTENTION = [(256, 4, 0.25), (256, 2, 1.0), (512, 8, 0.25)]  # hidden size, heads, rotated part
_rotary_tables = O.rotary_tables
MISTAKES = ["no rotation", "positions halved", "positions of new tokens from 0", "positions one behind", "scale halved"]


def sharpened(w, heads, by=3.2):
    """The query and key rows of a fused QKV weight scaled: queries and keys of standard deviation 2 instead of 0.63 from inputs of
    1, so that scores have one of 4."""
    w = w.clone()
    w.view(heads, 3, w.size(0) // (3 * heads), w.size(1))[:, :2] *= by
    return w


def layer_params(h, heads, seed=4):
    """Master parameters of a layer whose attention returns the context itself: the output projection is the identity."""
    p = golden_params.master_params(np.random.default_rng(seed), h)
    p["attention.query_key_value.weight"] = sharpened(p["attention.query_key_value.weight"], heads)
    p["attention.dense.weight"] = torch.eye(h)
    return p


def tables(positions, d):
    """The bf16 module's tables at these positions (any order), exact in 64 bits."""
    cos, sin = _rotary_tables(int(max(positions)) + 1, d, dtype=torch.bfloat16)
    at = torch.as_tensor(positions, dtype=torch.long)
    return cos.double()[at], sin.double()[at]


def wrong(mistake, s, new):
    """(positions of the rows, factor of the scale) of a sequence of s rows whose last `new` came one at a time."""
    pos, scale = list(range(s)), 1.0
    if mistake == "positions halved":
        pos = [p // 2 for p in pos]
    elif mistake == "positions of new tokens from 0":
        pos = [p if p < s - new else p - (s - new) for p in pos]
    elif mistake == "positions one behind":  # of the new tokens
        pos = [p if p < s - new else p - 1 for p in pos]
    elif mistake == "scale halved":
        scale = 0.5
    return pos, scale


def attention_by_hand(p, heads, d, x, mistake=None, new=0):
    """(out, spread) [s, h] in 64 bits of a sequence's rows x [s, h] through QKV, rotation, causal attention, on the bf16 weights.

    spread is a bound of an element's standard deviation under the path's roundings, a rounding being uniform within U of its value
    (deviation U / sqrt(3)): q and k are rounded behind the projection, and behind the rotation where rotated; a score then
    deviates by sigma_j.  Deviations of different keys may go together (they share the query), so they are added up:
    sum_j w_j sigma_j |v_j - out|.  Values and probabilities are rounded once each, the context once."""
    s, h = x.shape
    hn = h // heads
    w, b = (p["attention.query_key_value." + n].bfloat16().double() for n in ("weight", "bias"))
    mixed = (x.double() @ w.t() + b).view(s, heads, 3, hn)
    q, k, v = mixed.unbind(2)
    pos, factor = wrong(mistake, s, new)
    cos, sin = (t[:, None] for t in tables(pos, d))
    one = U * U / 3.0

    def rotated(t):
        var = one * t ** 2
        if mistake == "no rotation":
            return t, var
        r = t[..., :d]
        y = r * cos + O.rotate_half(r) * sin
        vy = one * ((r * cos) ** 2 + (O.rotate_half(r) * sin) ** 2 + y ** 2)
        return torch.cat((y, t[..., d:]), -1), torch.cat((vy, var[..., d:]), -1)

    (q, vq), (k, vk) = rotated(q), rotated(k)
    scale = factor / math.sqrt(hn)
    out, spread = torch.zeros(s, heads, hn, dtype=torch.float64), torch.zeros(s, heads, hn, dtype=torch.float64)
    hidden = torch.triu(torch.ones(s, s, dtype=torch.bool), 1)
    for i in range(heads):
        sc = (q[:, i] @ k[:, i].t()) * scale
        prob = torch.softmax(sc.masked_fill(hidden, -math.inf), -1)
        sigma = scale * (vq[:, i] @ (k[:, i] ** 2).t() + (q[:, i] ** 2) @ vk[:, i].t()).sqrt()
        o = prob @ v[:, i]
        out[:, i] = o
        far = (v[None, :, i] - o[:, None]).abs()  # [row, key, dim]
        spread[:, i] = ((prob * sigma)[:, :, None] * far).sum(1) + one ** 0.5 * (2 ** 0.5 * prob @ v[:, i].abs() + o.abs())
    return out.view(s, h), spread.view(s, h)


# ------------------------------------------------------------------------------------------------- a small language model
MODEL = dict(V=1024, h=256, n=4, L=2, rotary_pct=0.25)  # harness.CONFIGS["tiny"]


def model_params(seed=12):
    p = golden_params.stack_init(np.random.default_rng(seed), MODEL["V"], MODEL["h"], MODEL["L"])
    for i in range(MODEL["L"]):
        key = f"l{i}.attention.query_key_value.weight"
        p[key] = sharpened(p[key], MODEL["n"])
    return p


@contextlib.contextmanager
def planted(mistake, new):
    """The oracle's layers with a mistake (None: with the bf16 module's tables, whatever the oracle computes in)."""
    rotary, rotate, attend = O.rotary_tables, O.apply_rotary, O.self_attention

    def bf16_tables(s, d, base=10000, dtype=None):
        cos, sin = tables(wrong(mistake, s, new)[0], d)
        return cos.to(dtype), sin.to(dtype)

    def scaled(cfg, p, x, mask, prefix="attention."):
        w = p[prefix + "query_key_value.weight"].clone()
        b = p[prefix + "query_key_value.bias"].clone()
        factor = wrong(mistake, x.size(0), new)[1]  # of the scores: of the queries
        w.view(cfg.num_attention_heads, 3, -1, w.size(1))[:, 0] *= factor
        b.view(cfg.num_attention_heads, 3, -1)[:, 0] *= factor
        return attend(cfg, {**p, prefix + "query_key_value.weight": w, prefix + "query_key_value.bias": b}, x, mask, prefix)

    O.rotary_tables, O.self_attention = bf16_tables, scaled
    if mistake == "no rotation":
        O.apply_rotary = lambda q, k, cos, sin, offset=0: (q, k)
    try:
        yield
    finally:
        O.rotary_tables, O.apply_rotary, O.self_attention = rotary, rotate, attend


@torch.no_grad()
def model_logits(p, tokens, dtype, mistake=None, new=0):
    """Logits [s, V] of one sequence on the oracle, weights rounded to bf16, computed in dtype."""
    q = {k: v.bfloat16().to(dtype) for k, v in p.items()}
    cfg = O.LayerConfig(MODEL["h"], MODEL["n"], rotary_pct=MODEL["rotary_pct"], gpt_j_residual=True, bias_gelu_fusion=True)
    x = q["emb"][tokens][:, None]
    with planted(mistake, new):
        for i in range(MODEL["L"]):
            x = O.layer_forward(cfg, [{k: q[f"l{i}.{k}"] for k in golden_params.PARAM_ORDER}], x, O.causal_mask(x.size(0)))
    return torch.nn.functional.linear(O.layer_norm(x[:, 0], q["fln.w"], q["fln.b"]), q["head"]).float()


def off(a, b):
    """Relative difference of two sets of rows."""
    return float((a - b).norm() / b.norm())

"""Microscaled numbers written plainly, in 64 bits: blocks of 32 with a power of two each, elements e4m3 or e2m1."""
import torch

BLOCK = 32
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
E4M3 = [(m / 8) * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127]   # the 128th is NaN
GRID = {"mxfp4": E2M1, "mxfp8": E4M3}


def element_values(codes: torch.Tensor, form: str) -> torch.Tensor:
    half = len(GRID[form])
    table = GRID[form] + ([float("nan")] if form == "mxfp8" else [])
    table = torch.tensor(table + [-v for v in table], dtype=torch.float64)
    assert table.numel() in (16, 256) and half in (8, 127)
    return table[codes.long()]


def scale_values(codes: torch.Tensor) -> torch.Tensor:
    return torch.where(codes == 255, torch.nan, torch.exp2(codes.double() - 127))


def dequantize(elements: torch.Tensor, scales: torch.Tensor, form: str) -> torch.Tensor:
    """codes a byte each [T, W], scale codes [T, ceil(W / 32)] -> float64 [T, W]"""
    return element_values(elements, form) * scale_values(scales).repeat_interleave(BLOCK, 1)[:, :elements.shape[1]]


def quantize(x: torch.Tensor, form: str):
    """(element codes [T, W], scale codes [T, ceil(W / 32)]) of float64 rows, block by block: the smallest power of two from 2^-127 up with
    which no number is past the largest, the nearest element, of two equally near the one with the even code."""
    grid = torch.tensor(GRID[form], dtype=torch.float64)
    sign = 8 if form == "mxfp4" else 128
    T, W = x.shape
    elements, scales = torch.zeros(T, W, dtype=torch.uint8), torch.zeros(T, -(-W // BLOCK), dtype=torch.uint8)
    powers = torch.exp2(torch.arange(255, dtype=torch.float64) - 127)
    for b in range(scales.shape[1]):
        v = x[:, b * BLOCK:(b + 1) * BLOCK]
        bad = ~torch.isfinite(v).all(1)
        v = torch.where(bad[:, None], torch.zeros_like(v), v)
        code = (v.abs().amax(1)[:, None] > grid[-1] * powers[None]).sum(1)
        a = v.abs() / powers[code][:, None]
        apart = (a[..., None] - grid).abs()
        nearest = apart.amin(-1, keepdim=True)
        near = apart == nearest
        even = near & (torch.arange(len(grid)) % 2 == 0)
        at = torch.where(even.any(-1), even.int().argmax(-1), near.int().argmax(-1))
        e = at + sign * torch.signbit(v).int()
        elements[:, b * BLOCK:(b + 1) * BLOCK] = torch.where(bad[:, None], torch.zeros_like(e), e).to(torch.uint8)
        scales[:, b] = torch.where(bad, torch.full_like(code, 255), code).to(torch.uint8)
    return elements, scales


def unpack(rows) -> tuple:
    """(element codes a byte each, scale codes) of arle_amd's MXRows, on the CPU, padding included."""
    e, s = rows.elements.view(torch.uint8).cpu(), rows.scales.view(torch.uint8).cpu()
    if rows.form == "mxfp4":
        e = torch.stack([e & 15, e >> 4], dim=-1).flatten(1)
    return e, s


def norm(residual, delta, weight, eps):
    """(residual + delta, its root-mean-square norm) in 64 bits; delta None, [T, H] or a stack."""
    h = residual.double()
    if delta is not None:
        h = h + (delta.double().sum(0) if delta.dim() == 3 else delta.double())
    return h, h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * weight.double()


def gated(x, w):
    """silu(x . gate^T) * (x . up^T), w the gate's rows and then the up's"""
    y = x @ w.T
    gate, up = y.chunk(2, dim=1)
    return gate * torch.sigmoid(gate) * up


def round_rows(x, form):
    """The numbers that rows in blocks stand for."""
    return dequantize(*quantize(x, form), form)


def qwen3_logits(weights, cfg, tokens, weight_form, row_form):
    """Logits of the plain Qwen3 decoder in 64 bits whose projections hold their weights as `weight_form` and meet rows as `row_form` (None: as
    they are): the norms' rows, the attention's output and the activation's products."""
    import plain_qwen3 as q

    w = {n: t.double() for n, t in weights.items()}
    held = {n: round_rows(t, weight_form) if weight_form and ("_proj.weight" in n) else t for n, t in w.items()}
    rows = (lambda x: round_rows(x, row_form)) if row_form else (lambda x: x)
    T, eps = len(tokens), cfg["rms_norm_eps"]
    nq, nkv, D = cfg["num_attention_heads"], cfg["num_key_value_heads"], cfg["head_dim"]
    cos, sin = q.rope_cos_sin(range(T), D, cfg["rope_theta"], dtype=torch.float64)
    h = q.embedding(w["model.embed_tokens.weight"], tokens)
    for i in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{i}."
        x = rows(q.rms_norm(h, w[p + "input_layernorm.weight"], eps))
        of = lambda name, heads: (x @ held[f"{p}self_attn.{name}_proj.weight"].T).view(T, heads, D)
        qs = q.prepare_heads(of("q", nq), w[p + "self_attn.q_norm.weight"], eps, cos, sin)
        ks = q.prepare_heads(of("k", nkv), w[p + "self_attn.k_norm.weight"], eps, cos, sin)
        a = q.causal_attention(qs, ks, of("v", nkv), nkv).reshape(T, nq * D)
        h = h + rows(a) @ held[p + "self_attn.o_proj.weight"].T
        x = rows(q.rms_norm(h, w[p + "post_attention_layernorm.weight"], eps))
        act = q.silu(x @ held[p + "mlp.gate_proj.weight"].T) * (x @ held[p + "mlp.up_proj.weight"].T)
        h = h + rows(act) @ held[p + "mlp.down_proj.weight"].T
    f = q.rms_norm(h, w["model.norm.weight"], eps)
    return f @ (w["model.embed_tokens.weight"] if cfg["tie_word_embeddings"] else w["lm_head.weight"]).T

"""Plain 64-bit forms of the long-sequence operators on the CPU, with bounds on what rounding may do to a kernel that
computes them: u = 2^-24 for each 32-bit operation, r = 2^-8 (bf16) or 0 (fp32) for each value that is rounded to the
tensors' type."""
import math

import torch

U = 2.0 ** -24


def visible(n_q, n, window, sinks, causal, length):
    i, j = torch.arange(n_q)[:, None], torch.arange(n)[None, :]
    if causal:
        seen = (j <= i) & ((i - j < window) | (j < sinks))
    else:
        seen = ((i - j).abs() < window) | (j < sinks) | (i < sinks)
    return seen & (i < length) & (j < length)


def attention(q, k, v, seen, scale, r, d_o=None):
    """One head: q [n, dh], k, v [m, dh], seen [n, m] in 64 bits.  {name: (value, bound)} for o and, with d_o, dq, dk, dv.

    A score is off by dh u sum|q k| scale, which is its probability's relative error, twice for the normaliser, and a few u
    for the exponential; probabilities and score gradients are rounded (r) as operands of the next product; a sum of
    m terms adds m u of their absolute sum; results are rounded (r)."""
    dh, m = q.shape[1], k.shape[0]
    s = (q @ k.t() * scale).masked_fill(~seen, -math.inf)
    top = s.amax(1, keepdim=True) if m else s.new_zeros(q.shape[0], 1)
    top = torch.where(top.isinf(), torch.zeros_like(top), top)
    e = torch.exp(s - top)
    p = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    size = ((q.abs() @ k.abs().t()) * scale).masked_fill(~seen, 0.0)
    size = size.amax(1, keepdim=True) if m else s.new_zeros(q.shape[0], 1)
    rel = 2 * dh * U * size + (48 + m) * U
    e_p = rel * p
    o = p @ v
    e_o = (e_p + (r + m * U) * p) @ v.abs()
    out = {"o": (o, e_o + (r + U) * o.abs())}
    if d_o is not None:
        dp = d_o @ v.t()
        delta = (p * dp).sum(1, keepdim=True)
        ds = p * (dp - delta)
        e_dp = dh * U * (d_o.abs() @ v.abs().t())
        # the output that delta reads holds 7 bits behind a rounded one's
        e_delta = (d_o.abs() * e_o).sum(1, keepdim=True) + (r * 2.0 ** -7 + (dh + 4) * U) * (d_o.abs() * o.abs()).sum(1, keepdim=True)
        e_ds = e_p * (dp.abs() + delta.abs()) + p * (e_dp + e_delta) + (r + 4 * U) * ds.abs()
        for name, val, err in (("dq", ds @ k * scale, (e_ds + m * U * ds.abs()) @ k.abs() * scale),
                               ("dk", ds.t() @ q * scale, (e_ds + q.shape[0] * U * ds.abs()).t() @ q.abs() * scale),
                               ("dv", p.t() @ d_o, (e_p + (r + q.shape[0] * U) * p).t() @ d_o.abs())):
            out[name] = (val, err + (r + U) * val.abs())
    return out


def sliding_attention(q, k, v, window, sinks, causal, lengths, scale, r, d_o=None):
    """[B, N, H, dh] tensors; {name: (value, bound)} laid out like them."""
    q, k, v = (t.detach().double().cpu() for t in (q, k, v))
    d_o = None if d_o is None else d_o.detach().double().cpu()
    B, N, Hq, dh = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    out = {"o": [torch.zeros_like(q) for _ in range(2)]}
    if d_o is not None:
        out.update(dq=[torch.zeros_like(q) for _ in range(2)], dk=[torch.zeros_like(k) for _ in range(2)],
                   dv=[torch.zeros_like(v) for _ in range(2)])
    for b in range(B):
        n = N if lengths is None else min(max(int(lengths[b]), 0), N)
        seen = visible(n, n, window, sinks, causal, n)
        for h in range(Hq):
            got = attention(q[b, :n, h], k[b, :n, h // G], v[b, :n, h // G], seen, scale, r,
                            None if d_o is None else d_o[b, :n, h])
            for name, pair in got.items():
                for dst, src in zip(out[name], pair):
                    if name in ("dk", "dv"):
                        dst[b, :n, h // G] += src
                    else:
                        dst[b, :n, h] = src
    return {name: tuple(x) for name, x in out.items()}


def rope(x, pos, pairs, base, interleaved, inverse=False):
    """(value, bound without the final rounding) of x [B, N, H, dh]."""
    x = x.detach().double().cpu()
    pos = pos.detach().cpu().double()
    pos = pos if pos.dim() == 3 else pos[None]
    angle = torch.cat([pos[..., a:a + 1] * base ** (-torch.arange(n, dtype=torch.float64) / n) for a, n in enumerate(pairs)], -1)
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None] * (-1 if inverse else 1)
    P = sum(pairs)
    first, second = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    y, e = x.clone(), torch.zeros_like(x)
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    # cosine and sine: an angle of at most half a turn, rounded, then two units of the function; a product and a sum
    e[..., first] = e[..., second] = 10 * U * (x[..., first].abs() + x[..., second].abs())
    return y, e


def adamw(p, g, m, v, t, coef, lr, betas, eps, wd):
    """One step in 64 bits: (p, m, v), each with its bound."""
    b1, b2 = betas
    g = g * coef
    m1, v1 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    e_m = 5 * U * (b1 * m.abs() + (1 - b1) * g.abs())
    e_v = 7 * U * v1
    up = lr / (1 - b1 ** t) * m1 / ((v1 / (1 - b2 ** t)).sqrt() + eps)
    e_up = lr / (1 - b1 ** t) * e_m / ((v1 / (1 - b2 ** t)).sqrt() + eps) + 12 * U * up.abs()
    p1 = p * (1 - lr * wd) - up
    return (p1, 3 * U * p.abs() + e_up + U * p1.abs()), (m1, e_m), (v1, e_v)


# ----------------------------------------------------------------------------- 8-bit states, bit for bit
TOP, BLOCK = 448.0, 256


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def adamw8(p, g, mc, ms, vc, vs, t, coef, lr, betas, eps, wd, seed=0,
           sqrt=torch.sqrt):
    """One step of one flat fp32 tensor with e4m3 states, in single 32-bit roundings on the CPU; updated values of all five.
    ``sqrt``: the device's, whose last bit is not always the CPU's.  The neighbours of a value are looked up in a table of the codes."""
    n = p.numel()
    b1, b2 = betas

    def widen(scale):
        return scale.repeat_interleave(BLOCK)[:n]

    m = mc.float() * widen(ms)
    v = vc.float() * widen(vs)
    v = v * v
    g = g * torch.tensor(coef, dtype=torch.float32)
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    root = sqrt(v)
    den = root * (1.0 / math.sqrt(1.0 - b2 ** t)) + eps
    p = p * (1.0 - lr * wd) - (m / den) * (lr / (1.0 - b1 ** t))
    table = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    word = _mix(torch.arange(n) ^ int(_mix(torch.tensor((seed + t * 0x9E3779B1) & 0xFFFFFFFF))))
    pad = -n % BLOCK
    out = []
    for x, second in ((m, False), (root, True)):
        top = torch.nn.functional.pad(x.abs(), (0, pad)).view(-1, BLOCK).amax(1)
        some = top >= 2.0 ** -112
        inv = torch.where(some, torch.tensor(TOP) / top, torch.zeros_like(top))
        scale = torch.where(some, top * torch.tensor(1.0 / TOP), torch.zeros_like(top))
        y = x * widen(inv)
        a = y.abs().clamp(max=TOP)
        at = (torch.searchsorted(table, a, right=True) - 1).clamp(0, 125)
        lo, hi = table[at], table[at + 1]
        if second:
            u = ((word >> 16).float() + 0.5) * 2.0 ** -16
            code = torch.where(u * (hi * hi - lo * lo) < y * y - lo * lo, hi, lo)
            code = torch.where(y > 0, code.clamp_min(2.0 ** -9), code)
        else:
            # the 20 bits below the code's last one, plus a word of 20 bits, carry into it
            step = (hi - lo).double()
            frac = torch.where(a < 2.0 ** -6, (a + 2.0 ** -6).double() - 2.0 ** -6 - lo, a.double() - lo) / step * 2 ** 20
            code = torch.where(frac + ((word & 0xFFFF) * 16 + 8) >= 2 ** 20, hi, lo)
            code = torch.where(y < 0, -code, code)
        out += [code.to(torch.float8_e4m3fn), scale]
    return [p] + out


# ----------------------------------------------------------------------------- a ViT with rotary positions and a window
def vit_logits(params, images, patch, layers, heads, grid, window, sinks, pairs, base):
    """Logits of a pre-LN ViT (class token first) in the type of ``params`` (a state dict by the model's names)."""
    P = {k.replace("transformer.", "", 1) if k.startswith("transformer.") else k: v for k, v in params.items()}
    F = torch.nn.functional

    def norm(x, name):
        return F.layer_norm(x, x.shape[-1:], P[name + ".weight"], P[name + ".bias"], 1e-6)

    def linear(x, name):
        return F.linear(x, P[name + ".weight"], P[name + ".bias"])

    x = F.conv2d(images, P["embeddings.patch_embeddings.weight"], P["embeddings.patch_embeddings.bias"], stride=patch)
    B, D = x.shape[:2]
    x = torch.cat([P["embeddings.cls_token"].expand(B, -1, -1), x.flatten(2).transpose(1, 2)], 1) + P["embeddings.position_embeddings"]
    N, dh = x.shape[1], D // heads
    at = torch.tensor([[0, 0]] + [[r, c] for r in range(grid[0]) for c in range(grid[1])], dtype=x.dtype)
    angle = torch.cat([at[:, a:a + 1] * base ** (-torch.arange(n, dtype=x.dtype) / n) for a, n in enumerate(pairs)], 1)[:, None]
    cos, sin, S = angle.cos(), angle.sin(), sum(pairs)

    def turned(t):
        a, b = t[..., :S], t[..., S:2 * S]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, t[..., 2 * S:]], -1)

    seen = visible(N, N, window, sinks, False, N)
    for i in range(layers):
        L = f"encoder.layer.{i}."
        h = norm(x, L + "attention_norm")
        q, k, v = (linear(h, L + "attn." + n).view(B, N, heads, dh) for n in ("query", "key", "value"))
        q, k, v = (t.transpose(1, 2) for t in (turned(q), turned(k), v))
        p = torch.softmax((q @ k.transpose(-1, -2) / math.sqrt(dh)).masked_fill(~seen, -math.inf), -1)
        x = x + linear((p @ v).transpose(1, 2).reshape(B, N, D), L + "attn.out")
        x = x + linear(F.gelu(linear(norm(x, L + "ffn_norm"), L + "ffn.fc1")), L + "ffn.fc2")
    return linear(norm(x, "encoder.encoder_norm")[:, 0], "head")

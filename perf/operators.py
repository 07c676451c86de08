"""What the long-sequence operators of this framework are measured on.

Four operators: rotary positions with several axes (`vitk.ops.axial_rope`), attention with a sliding window and first
tokens that stay visible (`vitk.ops.sliding_attention`), its single-token form over a cache
(`vitk.ops.sliding_attention_decode`), and the AdamW step over many tensors with states in 32 or 8 bits
(`utils.optim.FusedAdamW`).

    run(prepare(case, seed))     one pass: the plain form in elementary torch operations, or, with `own`, the framework's calls
    exact(case, seed)            the same outputs from the definition in 64 bits
"""
import math
import os
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 256                    # elements that share a scale in an 8-bit optimizer state
TOP = 448.0                    # largest e4m3 value
SMALLEST = 2.0 ** -112         # a block whose largest value is below this is held as zeros


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token for each of eight streams, time | height | width positions far into the stream: latency
        dict(name="rope_token", op="rope", B=8, T=1, Y=1, X=1, lead=0, heads=16, dh=64, axes="8,12,12", dtype="bf16",
             interleaved=False, real=False, each=True, offset=1_000_000, train=False),
        # query | key of a 384 x 384 image at patch 16 (577 tokens, class token first), 12 + 12 heads, patch centres
        dict(name="rope_image_train", op="rope", B=64, T=1, Y=24, X=24, lead=1, heads=24, dh=64, axes="16,16", dtype="bf16",
             interleaved=False, real=True, each=False, offset=0, train=True),
        # a clip of 32 frames of 14 x 14 patches in fp32, interleaved pairs, part of the head left as it is
        dict(name="rope_clip_train_fp32", op="rope", B=4, T=32, Y=14, X=14, lead=1, heads=32, dh=64, axes="8,10,10",
             dtype="fp32", interleaved=True, real=False, each=False, offset=4096, train=True),
        # a handful of tokens (a 96 x 96 image at patch 16 with its class token): latency
        dict(name="attn_few_tokens", op="attn", B=1, N=37, Hq=3, Hkv=3, dh=64, dtype="bf16", causal=False, window=9, sinks=1,
             ragged=False, train=False),
        # a 768 x 768 image at patch 16 (2304 patches and the class token), 12 heads, training
        dict(name="attn_image_train", op="attn", B=8, N=2305, Hq=12, Hkv=12, dh=64, dtype="bf16", causal=False, window=145,
             sinks=1, ragged=False, train=True),
        # a long stream of frames, causal, shared key heads of 128, training
        dict(name="attn_stream_train", op="attn", B=1, N=16384, Hq=8, Hkv=2, dh=128, dtype="bf16", causal=True, window=1024,
             sinks=4, ragged=False, train=True),
        # the same kind of stream read in without gradients, padded sequences
        dict(name="attn_stream_read", op="attn", B=4, N=4099, Hq=16, Hkv=8, dh=64, dtype="bf16", causal=True, window=512,
             sinks=16, ragged=True, train=False),
        # fp32 instance on padded odd lengths, training
        dict(name="attn_ragged_train_fp32", op="attn", B=6, N=577, Hq=8, Hkv=4, dh=32, dtype="fp32", causal=False, window=97,
             sinks=5, ragged=True, train=True),
        # one stream, one token: latency of a serving step
        dict(name="decode_one", op="decode", B=1, cap=4096, Hq=12, Hkv=12, dh=64, dtype="bf16", window=1024, sinks=4),
        # many streams, one token each, long caches
        dict(name="decode_many", op="decode", B=32, cap=16387, Hq=32, Hkv=8, dh=128, dtype="bf16", window=8192, sinks=64),
        # the tensors of ViT-B/16 at 224 x 224, states in 32 bits
        dict(name="adamw32_b16", op="adamw", tensors="vit", hidden=768, layers=12, tokens=197, classes=1000, bits=32, t=1000),
        # the tensors of ViT-L/16 at 384 x 384, states in 8 bits
        dict(name="adamw8_l16", op="adamw", tensors="vit", hidden=1024, layers=24, tokens=577, classes=100, bits=8, t=20),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "attn", "attn", "decode", "adamw"))
    if op == "rope":
        dh = rng.choice((32, 64, 128))
        A = rng.choice((1, 2, 3))
        axes, left = [], dh // 2
        for _ in range(A):
            n = rng.randint(1, max(1, left - (A - 1 - len(axes)))) if len(axes) < A - 1 else left
            n = min(n, dh // 4 + dh // (4 * A))
            axes.append(n)
            left -= n
        axes = [n for n in axes if n > 0]
        heads = rng.randint(1, 32)
        T, Y, X = (1 if A < 3 else _log(rng, 1, 16)), (1 if A < 2 else _log(rng, 1, 24)), _log(rng, 1, 24 if A > 1 else 4096)
        each = T * Y * X
        B = _log(rng, 1, max(1, min(256, 1_600_000 // (each * heads * dh // 32 + 1) + 1)))
        return dict(op=op, B=B, T=T, Y=Y, X=X, lead=rng.randint(0, 2), heads=heads, dh=dh, axes=",".join(map(str, axes)),
                    dtype=rng.choice(("bf16", "fp32")), interleaved=rng.random() < 0.5, real=rng.random() < 0.3,
                    each=rng.random() < 0.3, offset=rng.choice((0, _log(rng, 10, 10_000_000))), train=rng.random() < 0.6)
    if op == "attn":
        Hkv = rng.choice((1, 2, 3, 4, 6, 8))
        Hq = Hkv * rng.choice((1, 1, 2, 3, 4))
        N = _log(rng, 1, 8192)
        B = _log(rng, 1, max(1, min(64, 500_000_000 // (N * N * Hq))))
        case = dict(op=op, B=B, N=N, Hq=Hq, Hkv=Hkv, dh=rng.choice((32, 64, 64, 128)), dtype=rng.choice(("bf16", "bf16", "fp32")),
                    causal=rng.random() < 0.5, window=_log(rng, 1, max(2, min(N, 2048))), sinks=rng.choice((0, 1, 4, _log(rng, 1, 70))),
                    ragged=rng.random() < 0.5, train=rng.random() < 0.7)
        while work(case)["flops"] > 2e11 and case["window"] > 1:
            case["window"] = (case["window"] + 1) // 2
        return case
    if op == "decode":
        Hkv = rng.choice((1, 2, 3, 4, 8))
        Hq = Hkv * rng.choice((1, 2, 4, 5, 8))
        cap = _log(rng, 1, 16384)
        dh = rng.choice((32, 64, 64, 128))
        B = _log(rng, 1, max(1, min(64, 400_000_000 // (cap * Hkv * dh))))
        return dict(op=op, B=B, cap=cap, Hq=Hq, Hkv=Hkv, dh=dh, dtype=rng.choice(("bf16", "bf16", "fp32")),
                    window=_log(rng, 1, max(2, cap)), sinks=rng.choice((0, 1, 4, _log(rng, 1, 70))))
    bits, t = rng.choice((8, 32)), _log(rng, 1, 20000)
    if rng.random() < 0.5:       # the per-task factors of the task-conditioned models: many small tensors
        return dict(op=op, tensors="factors", hidden=64 * rng.randint(1, 16), layers=rng.randint(1, 24), tokens=0,
                    classes=rng.randint(2, 1000), bits=bits, t=t)
    return dict(op=op, tensors="vit", hidden=64 * rng.randint(2, 12), layers=rng.randint(1, 12), tokens=rng.randint(2, 600),
                classes=rng.randint(2, 1000), bits=bits, t=t)


# ------------------------------------------------------------------------------------------------ inputs
def _framework():
    pkg = os.path.join(os.getcwd(), "vit-pytorch_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _axes(case):
    return tuple(int(n) for n in case["axes"].split(","))


def _lengths(case):
    """Tokens of each sequence: a padded batch from the full length down to half of it."""
    N, B = case["N"], case["B"]
    return [N - (N * b) // (2 * B) for b in range(B)] if case["ragged"] else [N] * B


def _cached(case):
    """Tokens that each stream of a decode batch holds: from the whole cache down to half of it."""
    cap, B = case["cap"], case["B"]
    return [cap - (cap * b) // (2 * B) for b in range(B)]


def _shapes(case):
    """The tensors of a model with `hidden` columns, or of the factors its layers have for each task."""
    D, F = case["hidden"], 4 * case["hidden"]
    out = []
    if case["tensors"] == "vit":
        out += [(D, 3, 16, 16), (D,), (1, case["tokens"], D), (1, 1, D)]
        for _ in range(case["layers"]):
            out += [(D,), (D,), (D,), (D,)] + [(D, D), (D,)] * 4 + [(F, D), (F,), (D, F), (D,)]
        out += [(D,), (D,)]
    else:
        for _ in range(case["layers"]):
            for i, o in ((D, D),) * 4 + ((D, F), (F, D)):
                out += [(i, 2), (2, o), (o,)]
    return out + [(case["classes"], D), (case["classes"],)]


def _adamw_settings():
    return dict(lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if own:
        _framework()

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV).to(dtype)

    if op == "rope":
        B, N = case["B"], case["lead"] + case["T"] * case["Y"] * case["X"]
        A = len(_axes(case))
        ax = [torch.arange(n, device=DEV) for n in (case["T"], case["Y"], case["X"])]
        grid = torch.stack(torch.meshgrid(*ax, indexing="ij"), -1).reshape(-1, 3)[:, 3 - A:]
        grid = grid + torch.tensor([case["offset"]] + [0] * (A - 1), device=DEV)     # the first axis is far along
        pos = torch.cat([torch.zeros(case["lead"], A, dtype=torch.int64, device=DEV), grid])
        if case["each"]:
            pos = pos[None] + torch.randint(0, 100, (B, 1, 1), generator=g, device=DEV)
        if case["real"]:
            pos = (pos + 0.5).float()
        dt = DTYPES[case["dtype"]]
        packed = randn(B, N, case["heads"] * case["dh"] * 3 // 2 if case["heads"] % 2 == 0 else case["heads"] * case["dh"], dtype=dt)
        s.update(pos=pos, axes=_axes(case), x=packed[:, :, :case["heads"] * case["dh"]].view(B, N, case["heads"], case["dh"]))
        if case["train"]:
            s["dy"] = randn(B, N, case["heads"], case["dh"], dtype=dt)
            s["x"].requires_grad_(own)
    elif op == "attn":
        B, N, Hq, Hkv, dh, dt = (case[k] for k in ("B", "N", "Hq", "Hkv", "dh", "dtype"))
        qkv = randn(B, N, Hq + 2 * Hkv, dh, dtype=DTYPES[dt])
        q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
        s.update(q=q, k=k, v=v, lengths=torch.tensor(_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] else None)
        if case["train"]:
            s["do"] = randn(B, N, Hq, dh, dtype=DTYPES[dt])
            for t in (q, k, v):
                t.requires_grad_(own)
    elif op == "decode":
        B, cap, Hkv, dh, dt = case["B"], case["cap"], case["Hkv"], case["dh"], DTYPES[case["dtype"]]
        s.update(q=randn(B, case["Hq"], dh, dtype=dt), k=randn(B, cap, Hkv, dh, dtype=dt), v=randn(B, cap, Hkv, dh, dtype=dt),
                 lengths=torch.tensor(_cached(case), dtype=torch.int32, device=DEV))
    else:
        shapes = _shapes(case)
        sizes = [math.prod(x) for x in shapes]
        room = [-(-n // BLOCK) * BLOCK for n in sizes]       # every tensor starts at a block of its own
        starts = np.concatenate([[0], np.cumsum(room)]).tolist()
        total = starts[-1]
        p, grad = 0.02 * randn(total), 0.003 * randn(total)
        m, r = 0.001 * randn(total), 0.003 * randn(total).abs()
        spread = torch.exp(randn(total // BLOCK, 1)).expand(-1, BLOCK).reshape(-1)      # layers differ in size
        grad, m, r = grad * spread, m * spread, r * spread
        real = torch.cat([torch.arange(w, device=DEV) < n for n, w in zip(sizes, room)])
        index = torch.cat([torch.arange(w, device=DEV, dtype=torch.int32) for w in room])
        for x in (p, grad, m, r):
            x.mul_(real)
        s.update(p=p, g=grad, index=index, t=case["t"])
        if case["bits"] == 8:
            for name, x in (("m", m), ("v", r)):
                top = x.view(-1, BLOCK).abs().amax(1)
                s[name + "_scale"] = top / TOP
                s[name] = (x.view(-1, BLOCK) / s[name + "_scale"].clamp_min(1e-30)[:, None]).view(-1).to(torch.float8_e4m3fn)
        else:
            s.update(m=m, v=r * r)
        if own:
            from utils.optim import FusedAdamW
            params = []
            for shape, n, o in zip(shapes, sizes, starts):
                x = torch.nn.Parameter(p[o:o + n].view(shape))
                x.grad = grad[o:o + n].view(shape)
                params.append(x)
            opt = FusedAdamW(params, state_bits=case["bits"], **_adamw_settings())
            for x, shape, n, o in zip(params, shapes, sizes, starts):
                st = dict(step=case["t"], exp_avg=s["m"][o:o + n].view(shape), exp_avg_sq=s["v"][o:o + n].view(shape))
                if case["bits"] == 8:
                    b0, b1 = o // BLOCK, (o + n + BLOCK - 1) // BLOCK
                    st.update(exp_avg_scale=s["m_scale"][b0:b1], exp_avg_sq_scale=s["v_scale"][b0:b1])
                opt.state[x] = st
            s["opt"] = opt
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    return {"rope": _rope, "attn": _attn, "decode": _decode, "adamw": _adamw}[case["op"]](s, case)


def _rotate(x, cos, sin, P, interleaved):
    """The first 2 P elements of each head in pairs, (2 i, 2 i + 1) or (i, i + P), turned by their angles."""
    a, b = (x[..., 0:2 * P:2], x[..., 1:2 * P:2]) if interleaved else (x[..., :P], x[..., P:2 * P])
    u, w = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((y, x[..., 2 * P:]), -1)


def _rope(s, case):
    if own:
        from vitk import ops
        y = ops.axial_rope(s["x"], s["pos"], s["axes"], interleaved=case["interleaved"])
        if not case["train"]:
            return {"y": y}
        return {"y": y.detach(), "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    # angles of far positions lose their fraction of a turn in 32 bits
    freq = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float64, device=DEV) / n) for n in s["axes"]])
    axis = torch.repeat_interleave(torch.arange(len(s["axes"]), device=DEV), torch.tensor(s["axes"], device=DEV), output_size=sum(s["axes"]))
    angle = s["pos"].double()[..., axis] * freq
    cos, sin = angle.cos().float().unsqueeze(-2), angle.sin().float().unsqueeze(-2)
    P = sum(s["axes"])
    dt = s["x"].dtype
    out = {"y": _rotate(s["x"].float(), cos, sin, P, case["interleaved"]).to(dt)}
    if case["train"]:
        out["dx"] = _rotate(s["dy"].float(), cos, -sin, P, case["interleaved"]).to(dt)
    return out


def _attn(s, case):
    q, k, v, lengths = s["q"], s["k"], s["v"], s["lengths"]
    if own:
        from vitk import ops
        o = ops.sliding_attention(q, k, v, case["window"], sinks=case["sinks"], causal=case["causal"], lengths=lengths)
        if not case["train"]:
            return {"o": o}
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    B, N, Hq, dh = q.shape
    Hkv, dt, scale = k.shape[2], q.dtype, dh ** -0.5
    G = Hq // Hkv
    qf = q.float().view(B, N, Hkv, G, dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, dh)
    kf, vf = (x.float().permute(0, 2, 1, 3).contiguous() for x in (k, v))
    i, j = torch.arange(N, device=DEV)[:, None], torch.arange(N, device=DEV)[None, :]
    if case["causal"]:
        seen = (j <= i) & ((i - j < case["window"]) | (j < case["sinks"]))
    else:
        seen = ((i - j).abs() < case["window"]) | (j < case["sinks"]) | (i < case["sinks"])
    if lengths is not None:
        n = lengths.view(B, 1, 1)
        seen = (seen & (i < n) & (j < n)).view(B, 1, 1, N, N)
    sc = torch.matmul(qf, kf.transpose(-1, -2)).view(B, Hkv, G, N, N).mul_(scale)
    sc.masked_fill_(~seen, -math.inf)
    top = sc.amax(-1, keepdim=True)
    top.masked_fill_(top == -math.inf, 0.0)
    p = sc.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30)).view(B, Hkv, G * N, N)

    def back(x, H):        # [B, Hkv, rows, dh] -> [B, N, H, dh]
        return x.view(B, Hkv, H // Hkv, N, dh).permute(0, 3, 1, 2, 4).reshape(B, N, H, dh).to(dt)

    out = {"o": back(torch.matmul(p, vf), Hq)}
    if case["train"]:
        do = s["do"].float().view(B, N, Hkv, G, dh).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * N, dh)
        out["dv"] = back(torch.matmul(p.transpose(-1, -2), do), Hkv)
        ds = torch.matmul(do, vf.transpose(-1, -2))
        ds = ds.sub_((p * ds).sum(-1, keepdim=True)).mul_(p).mul_(scale)
        out["dq"] = back(torch.matmul(ds, kf), Hq)
        out["dk"] = back(torch.matmul(ds.transpose(-1, -2), qf), Hkv)
    return out


def _decode(s, case):
    q, k, v, lengths = s["q"], s["k"], s["v"], s["lengths"]
    if own:
        from vitk import ops
        return {"o": ops.sliding_attention_decode(q, k, v, lengths, case["window"], sinks=case["sinks"])}
    B, Hq, dh = q.shape
    Hkv, w, first = k.shape[2], min(case["window"], case["cap"]), min(case["sinks"], case["cap"])
    # only what can be seen is read: the first tokens, then the last ones behind them
    n = lengths.long().view(B, 1)
    last = n - w + torch.arange(w, device=DEV)
    at = torch.cat((torch.arange(first, device=DEV).expand(B, -1), last), 1)
    seen = torch.cat((at[:, :first] < n, (last >= first) & (last >= 0)), 1)
    rows = (at.clamp(0, case["cap"] - 1) + torch.arange(B, device=DEV)[:, None] * case["cap"]).view(-1)
    kf = k.view(-1, Hkv, dh)[rows].view(B, -1, Hkv, dh).float().permute(0, 2, 3, 1)
    vf = v.view(-1, Hkv, dh)[rows].view(B, -1, Hkv, dh).float().permute(0, 2, 1, 3)
    sc = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, dh), kf).mul_(dh ** -0.5)
    sc.masked_fill_(~seen[:, None, None, :], -math.inf)
    p = (sc - sc.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    return {"o": torch.matmul(p, vf).view(B, Hq, dh).to(q.dtype)}


def _mix(x):
    """32-bit mixing of non-negative int64 values."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _floor_e4m3(a):
    """(largest e4m3 value <= a, the next one) for 0 <= a <= 448."""
    tiny = a < 2.0 ** -6
    b = torch.where(tiny, a + 2.0 ** -6, a).view(torch.int32) & ~0xFFFFF
    less = tiny.float() * 2.0 ** -6
    return b.view(torch.float32) - less, (b + 0x100000).view(torch.float32) - less


def _to_blocks(x):
    """x in units of its block's largest value / 448, and those units (zeros where there is nothing to hold)."""
    x = x.view(-1, BLOCK)
    top = x.abs().amax(1, keepdim=True)
    some = top >= SMALLEST
    inv = torch.where(some, torch.full_like(top, TOP) / top, torch.zeros_like(top))
    return (x * inv).view(-1), torch.where(some, top * (1.0 / TOP), torch.zeros_like(top)).view(-1)


def _adamw(s, case):
    names = ("p", "m", "v") + (("m_scale", "v_scale") if case["bits"] == 8 else ())
    if own:
        norm = s["opt"].step(max_grad_norm=1.0)
        return dict({x: s[x] for x in names}, norm=norm)
    c = _adamw_settings()
    lr, (b1, b2), eps, wd = c["lr"], c["betas"], c["eps"], c["weight_decay"]
    s["t"] += 1
    norm = torch.sum(s["g"].double().square_()).sqrt()                  # a long sum
    g = s["g"] * (1.0 / (norm + 1e-6)).clamp_max(1.0).float()
    m, v = s["m"], s["v"]
    if case["bits"] == 8:
        m = (m.float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        v = (v.float().view(-1, BLOCK) * s["v_scale"][:, None]).view(-1).square()
    m = (m * b1).add_(g * (1.0 - b1))
    v = (v * b2).add_((g * g).mul_(1.0 - b2))
    root = v.sqrt()
    s["p"].mul_(1.0 - lr * wd)
    step = lr / (1.0 - b1 ** s["t"])
    s["p"].sub_((m / (root * (1.0 / math.sqrt(1.0 - b2 ** s["t"]))).add_(eps)).mul_(step))
    if case["bits"] == 8:
        # rounded at random: the word of (seed 0, step, element) decides between the two neighbours, for the first
        # moment in proportion to the value, for the second in proportion to its square
        key = int(_mix(torch.tensor((s["t"] * 0x9E3779B1) & 0xFFFFFFFF)))
        word = _mix(s["index"].long() ^ key)
        y, s["m_scale"] = _to_blocks(m)
        a = y.abs()
        tiny = a < 2.0 ** -6
        b = torch.where(tiny, a + 2.0 ** -6, a).view(torch.int32) + (((word & 0xFFFF) << 4) + 8).int()
        a = ((b & ~0xFFFFF).view(torch.float32) - tiny.float() * 2.0 ** -6).clamp_max_(TOP)
        s["m"] = torch.where(y < 0, -a, a).to(torch.float8_e4m3fn)
        y, s["v_scale"] = _to_blocks(root)
        lo, hi = _floor_e4m3(y.clamp_max(TOP))
        hi.clamp_max_(TOP)
        u = ((word >> 16).float() + 0.5) * 2.0 ** -16
        up = u * (hi * hi - lo * lo) < y * y - lo * lo
        a = torch.where(up, hi, lo)
        s["v"] = torch.where(y > 0, a.clamp_min(2.0 ** -9), a).to(torch.float8_e4m3fn)
    else:
        s["m"], s["v"] = m, v
    return dict({x: s[x] for x in names}, norm=norm.float())


# ------------------------------------------------------------------------------------------------ the least there is to do
def _pairs(case, n):
    """(query, key) pairs that a sequence of n tokens has to look at."""
    w, f = case["window"], case["sinks"]
    i = np.arange(n, dtype=np.int64)
    if case["causal"]:
        band = np.minimum(i + 1, w)                                    # i - w < j <= i
        extra = np.clip(np.minimum(f, i - w + 1), 0, None)             # first tokens before the band
        return int((band + extra).sum())
    lo, hi = np.maximum(0, i - w + 1), np.minimum(n, i + w)
    width = hi - lo if w > 0 else np.zeros_like(i)
    extra = np.clip(np.minimum(f, lo), 0, None) if w > 0 else np.full_like(i, min(f, n))
    return int(np.where(i < f, n, width + extra).sum())


def work(case):
    op = case["op"]
    e = 2 if case.get("dtype") == "bf16" else 4
    if op == "rope":
        n = case["B"] * (case["lead"] + case["T"] * case["Y"] * case["X"]) * case["heads"] * case["dh"]
        passes = 2 if case["train"] else 1
        return {"bytes": passes * 2 * n * e, "flops": passes * 3 * n}
    if op == "attn":
        per, Hq, Hkv, dh = sum(_lengths(case)), case["Hq"], case["Hkv"], case["dh"]
        pairs = sum(_pairs(case, n) for n in _lengths(case)) * Hq
        q, kv, full = per * Hq * dh * e, per * Hkv * dh * e, case["B"] * case["N"] * dh * e
        if not case["train"]:
            return {"bytes": q + 2 * kv + full * Hq, "flops": 4 * pairs * dh}
        return {"bytes": 2 * q + 2 * kv + full * (2 * Hq + 2 * Hkv), "flops": 14 * pairs * dh}
    if op == "decode":
        rows = sum(min(n, case["window"] + min(case["sinks"], max(0, n - case["window"]))) for n in _cached(case))
        return {"bytes": e * case["dh"] * (2 * rows * case["Hkv"] + 2 * case["B"] * case["Hq"]), "flops": 4 * rows * case["Hq"] * case["dh"]}
    n = sum(math.prod(x) for x in _shapes(case))
    state = 4.0 if case["bits"] == 32 else 1.0 + 4.0 / BLOCK
    return {"bytes": n * (4 + 8 + 4 * state), "flops": 16 * n}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    return {"rope": _exact_rope, "attn": _exact_attn, "decode": _exact_decode, "adamw": _exact_adamw}[case["op"]](s, case)


def _exact_rope(s, case):
    P = sum(s["axes"])
    turns = []
    for a, n in enumerate(s["axes"]):
        for i in range(n):
            turns.append(s["pos"][..., a].double() / 10000.0 ** (i / n))
    unit = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), torch.stack(turns, -1))[..., None, :]

    def turned(x, unit):
        y = x.double().clone()
        re, im = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if case["interleaved"] else (slice(0, P), slice(P, 2 * P))
        z = torch.complex(y[..., re], y[..., im]) * unit
        y[..., re], y[..., im] = z.real, z.imag
        return y

    out = {"y": turned(s["x"], unit)}
    if case["train"]:
        out["dx"] = turned(s["dy"], unit.conj())
    return out


def _exact_attn(s, case):
    """One sequence and key head after the other, gradients by automatic differentiation."""
    B, N, Hq, dh = s["q"].shape
    Hkv, w, f = case["Hkv"], case["window"], case["sinks"]
    G = Hq // Hkv
    names = ("q", "k", "v")
    out = {"o": torch.zeros(B, N, Hq, dh, dtype=torch.float64, device=DEV)}
    if case["train"]:
        out.update({"d" + x: torch.zeros(s[x].shape, dtype=torch.float64, device=DEV) for x in names})
    for b, n in enumerate(_lengths(case)):
        at = torch.arange(n, device=DEV)
        far = at[:, None] - at[None, :]
        hidden = far >= w
        if case["causal"]:
            hidden = (hidden & (at[None, :] >= f)) | (far < 0)
        else:
            hidden = (hidden | (far <= -w)) & (at[None, :] >= f) & (at[:, None] >= f)
        for h in range(Hkv):
            heads = slice(h * G, (h + 1) * G)
            q = s["q"][b, :n, heads].detach().double().transpose(0, 1).contiguous().requires_grad_(case["train"])
            k = s["k"][b, :n, h].detach().double().contiguous().requires_grad_(case["train"])
            v = s["v"][b, :n, h].detach().double().contiguous().requires_grad_(case["train"])
            p = torch.softmax((q @ k.t() / math.sqrt(dh)).masked_fill(hidden, -math.inf), -1)
            o = p @ v
            out["o"][b, :n, heads] = o.detach().transpose(0, 1)
            if case["train"]:
                dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"][b, :n, heads].double().transpose(0, 1))
                out["dq"][b, :n, heads], out["dk"][b, :n, h], out["dv"][b, :n, h] = dq.transpose(0, 1), dk, dv
    return out


def _exact_decode(s, case):
    B, Hq, dh = s["q"].shape
    G = Hq // case["Hkv"]
    out = torch.zeros(B, Hq, dh, dtype=torch.float64, device=DEV)
    for b, n in enumerate(_cached(case)):
        back = max(0, n - case["window"])
        at = torch.cat((torch.arange(min(case["sinks"], back), device=DEV), torch.arange(back, n, device=DEV)))
        for h in range(case["Hkv"]):
            sc = s["q"][b, h * G:(h + 1) * G].double() @ s["k"][b, at, h].double().t() / math.sqrt(dh)
            out[b, h * G:(h + 1) * G] = torch.softmax(sc, -1) @ s["v"][b, at, h].double()
    return {"o": out}


def _exact_adamw(s, case):
    c = _adamw_settings()
    (b1, b2), t = c["betas"], case["t"] + 1
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    g = g / torch.clamp(norm + 1e-6, min=1.0)
    m, v = s["m"].double(), s["v"].double()
    if case["bits"] == 8:
        m = m * s["m_scale"].double().repeat_interleave(BLOCK)
        v = (v * s["v_scale"].double().repeat_interleave(BLOCK)) ** 2
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = s["p"].double()
    p = p - c["lr"] * c["weight_decay"] * p - c["lr"] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + c["eps"])
    out = {"p": p, "norm": norm}
    if case["bits"] == 32:
        return dict(out, m=m, v=v)
    del g, p
    # the word of every element, in numpy's 32-bit arithmetic
    with np.errstate(over="ignore"):
        def mixed(x):
            x ^= x >> np.uint32(16)
            x *= np.uint32(0x7FEB352D)
            x ^= x >> np.uint32(15)
            x *= np.uint32(0x846CA68B)
            x ^= x >> np.uint32(16)
            return x
        key = mixed(np.array([(t * 0x9E3779B1) % 2 ** 32], dtype=np.uint32))
        word = mixed(s["index"].cpu().numpy().view(np.uint32) ^ key)
    low = torch.from_numpy((word & np.uint32(0xFFFF)).astype(np.int32)).to(DEV)
    high = torch.from_numpy((word >> np.uint32(16)).astype(np.int32)).to(DEV)
    table = torch.arange(127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).double()       # 0 ... 448

    def held(x, chance):
        top = x.view(-1, BLOCK).abs().amax(1).repeat_interleave(BLOCK)
        a = torch.where(top >= SMALLEST, x.abs() / top * TOP, torch.zeros_like(x)).clamp(max=TOP)
        at = torch.searchsorted(table, a, right=True).sub_(1).clamp_(0, 125)
        lo, hi = table[at], table[at + 1]
        return torch.where(chance(a, lo, hi), hi, lo), a, top[::BLOCK] / TOP

    a, _, out["m_scale"] = held(m, lambda a, lo, hi: (low + 0.5) / 65536 + (a - lo) / (hi - lo) >= 1)
    out["m"] = torch.where(m < 0, -a, a)
    a, y, out["v_scale"] = held(v.sqrt(), lambda a, lo, hi: (high + 0.5) / 65536 * (hi ** 2 - lo ** 2) < a ** 2 - lo ** 2)
    out["v"] = torch.where(y > 0, a.clamp(min=2.0 ** -9), a)
    return out

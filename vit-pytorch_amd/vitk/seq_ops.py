"""Operators of long token sequences (large images, clips, streams of frames): rotary positions with several axes,
attention with a sliding window and first tokens that stay visible, and its single-token form over a cache.

All of them take ``[batch, tokens, heads, head size]`` tensors in bf16 or fp32 with any strides, run on the current
stream of the tensors' device (whichever device is current) and raise ``VitkError`` for what they do not take, forward-mode
derivatives among it.
They are offered through ``vitk.ops``.
"""
import ctypes
import math

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import Rope, SlideAttn, SlideCache, VitkError, check, dtype_code, lib
from .ops import convert


class _On:
    """The device of the tensors as the current one for the length of a call; `.stream` is its current stream."""
    __slots__ = ("device", "before", "stream")

    def __init__(self, device):
        self.device = device.index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.device:
            torch.cuda.set_device(self.device)
        self.stream = torch._C._cuda_getCurrentRawStream(self.device)
        return self

    def __exit__(self, *_):
        if self.before != self.device:
            torch.cuda.set_device(self.before)


def _one_device(what, first, *ts):
    if not first.is_cuda:
        raise VitkError(f"{what}: vitk kernels run on the GPU only: got a tensor on {first.device}")
    device = first.device
    for t in ts:
        if t is not None and t.device != device:
            raise VitkError(f"{what}: tensors on {device} and {t.device}")


def _no_tangents(what, *ts):
    """Forward-mode derivatives are refused: a call that records nothing for backward would drop them without a word."""
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise VitkError(f"{what}: no forward-mode derivatives")


def _rows(t, apart=1 << 23):
    """`t` as the kernels address it: consecutive elements inside a head, pointer and strides multiples of 16 bytes, tokens
    less than `apart` elements from one to the next (attention's tiles count bytes in 32 bits, a decoded cache is addressed in 64)."""
    st, unit = t.stride(), 16 // t.element_size()
    if t.data_ptr() % 16 == 0 and st[-1] == 1 and st[1] < apart and not any(s % unit for s in st[:-1]):
        return t
    return t.clone(memory_format=torch.contiguous_format)


# ----------------------------------------------------------------------------- rotary positions
_POS_KIND = {torch.int64: 0, torch.int32: 1, torch.float32: 2, torch.float64: 3}


def grid_positions(sizes, lead=0, device="cuda"):
    """Positions of the cells of a grid, row-major, behind ``lead`` tokens at the origin: int64 [lead + cells, axes]."""
    ax = [torch.arange(int(n)) for n in sizes]
    grid = torch.stack(torch.meshgrid(*ax, indexing="ij"), -1).reshape(-1, len(ax))
    return torch.cat([torch.zeros(lead, len(ax), dtype=torch.int64), grid]).to(device)


def _rope_call(x, y, pos, pairs, base, interleaved, inverse, on):
    B, N, H, dh = x.shape
    xs, ys = x.stride(), y.stride()
    a = Rope(x.data_ptr(), y.data_ptr(), pos.data_ptr(), xs[0], xs[1], xs[2], ys[0], ys[1], ys[2],
             pos.shape[1] * pos.shape[2] if pos.dim() == 3 else 0, B, N, H, dh, len(pairs), _POS_KIND[pos.dtype],
             int(interleaved), int(inverse), (ctypes.c_int * 8)(*pairs), base)
    check(lib.vitk_axial_rope(ctypes.byref(a), dtype_code(x.dtype), on.stream), "vitk_axial_rope")


def _rope_args(x, positions, pairs, base):
    """Checks; (positions contiguous, pairs as ints, base)."""
    if x.dim() != 4:
        raise VitkError(f"axial_rope: x is [batch, tokens, heads, head size], got {tuple(x.shape)}")
    dtype_code(x.dtype)
    pairs = tuple(int(n) for n in pairs)
    B, N, H, dh = x.shape
    if dh % 2 or dh > 256 or dh == 0:
        raise VitkError(f"axial_rope: even head sizes up to 256, got {dh}")
    if B * N >= 1 << 31 or H * dh >= 1 << 28:
        raise VitkError(f"axial_rope: fewer than 2^31 tokens of fewer than 2^28 elements, got {tuple(x.shape)}")
    if not 1 <= len(pairs) <= 8 or min(pairs) < 1 or sum(pairs) > dh // 2:
        raise VitkError(f"axial_rope: 1 to 8 axes of at least one pair, {dh // 2} pairs in all: got {pairs}")
    if positions.dtype not in _POS_KIND:
        raise VitkError(f"axial_rope: positions are int64, int32, float32 or float64, got {positions.dtype}")
    if positions.requires_grad:
        raise VitkError("axial_rope: positions have no gradient")
    if tuple(positions.shape) not in ((N, len(pairs)), (B, N, len(pairs))):
        raise VitkError(f"axial_rope: positions are [{N}, {len(pairs)}] or [{B}, {N}, {len(pairs)}], got {tuple(positions.shape)}")
    if not (base > 0 and math.isfinite(base)):
        raise VitkError(f"axial_rope: base must be positive, got {base}")
    _no_tangents("axial_rope", x, positions)
    _one_device("axial_rope", x, positions)
    return positions.contiguous(), pairs, float(base)


def _odd(t):
    """Whether a head of `t` may begin at an odd element: the kernel moves interleaved pairs as wholes."""
    st = t.stride()
    return (t.data_ptr() // t.element_size() | st[0] | st[1] | st[2]) & 1


def _rope_rows(x, interleaved):
    return x if x.stride(-1) == 1 and not (interleaved and _odd(x)) else x.clone(memory_format=torch.contiguous_format)


def _meets(x, out):
    """Whether a write to `out` may land on elements of `x` other than the one it comes from, which another workgroup may not have
    read yet.  Both have the same shape; a layout too tangled to tell counts as one that meets."""
    B, N, H, dh = x.shape
    (a, b, c, d), (e, f, g, h) = x.stride(), out.stride()
    at = (out.data_ptr() - x.data_ptr()) // x.element_size()
    if (at > (B - 1) * a + (N - 1) * b + (H - 1) * c + (dh - 1) * d or -at > (B - 1) * e + (N - 1) * f + (H - 1) * g + (dh - 1) * h
            or x.numel() == 0):
        return False
    st = [0 if n == 1 else s for s, n in zip(x.stride(), x.shape)]
    to = [0 if n == 1 else s for s, n in zip(out.stride(), x.shape)]
    if st != to:
        return True
    dims = sorted(((s, n) for s, n in zip(st, x.shape) if n > 1), reverse=True)
    if any(s <= sum((m - 1) * t for t, m in dims[i + 1:]) for i, (s, _) in enumerate(dims)):
        return True

    def hits(at, dims):                # whether a difference of two elements' indices is `at` apart
        if not dims:
            return at == 0
        (s, n), c = dims[0], at // dims[0][0]
        return any(abs(k) < n and hits(at - k * s, dims[1:]) for k in (c, c + 1))

    return at != 0 and hits(at, dims)


def _rope_new(x, pos, pairs, base, interleaved, inverse):
    x = _rope_rows(x, interleaved)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if y.numel():
        with _On(x.device) as on:
            _rope_call(x, y, pos, pairs, base, interleaved, inverse, on)
    return y


class AxialRopeFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, pos, pairs, base, interleaved):
        ctx.save_for_backward(pos)
        ctx.meta = (pairs, base, interleaved)
        return _rope_new(x, pos, pairs, base, interleaved, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        (pos,) = ctx.saved_tensors
        return _rope_new(dy, pos, *ctx.meta, True), None, None, None, None


def axial_rope(x, positions, pairs, base=10000.0, interleaved=False, out=None):
    """Rotary positions with one or several axes (time, height, width, ...).

    x [B, N, H, dh]; positions [N, axes] or [B, N, axes] (int64, int32, float32 or float64; on x's device); ``pairs``: how many
    element pairs of a head turn with each axis, ``sum(pairs) <= dh / 2``; the rest of the head is copied.  Pair i of
    axis a turns by ``positions[..., a] * base ** (-i / pairs[a])``.  With P = sum(pairs), pairs are elements (i, i + P), or
    (2 i, 2 i + 1) when ``interleaved``.  Angles are reduced to one turn in 64 bits, so positions may be far.
    Returns a new contiguous tensor, or writes ``out`` (same shape and type, consecutive elements inside a head; it may be
    x itself, in a part of a cache, overlap x, ...; not differentiable; for autograd it counts as modified in place)."""
    if out is not None:
        _no_tangents("axial_rope", out)
    pos, pairs, base = _rope_args(x, positions, pairs, base)
    interleaved = bool(interleaved)
    if out is None:
        if torch.is_grad_enabled() and x.requires_grad:
            return AxialRopeFn.apply(x, pos, pairs, base, interleaved)
        return _rope_new(x, pos, pairs, base, interleaved, False)
    if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
        raise VitkError("axial_rope: out= is not differentiable")
    if out.shape != x.shape or out.dtype != x.dtype or out.stride(-1) != 1:
        raise VitkError("axial_rope: out has x's shape and type and consecutive elements inside a head")
    if any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise VitkError("axial_rope: out holds an element in more than one place")
    _one_device("axial_rope", x, out)
    if (interleaved and _odd(out)) or _meets(x, out):
        return out.copy_(_rope_new(x, pos, pairs, base, interleaved, False))
    x = _rope_rows(x, interleaved)
    if out.numel():
        with _On(x.device) as on:
            _rope_call(x, out, pos, pairs, base, interleaved, False, on)
        if not out.is_inference():             # written through a raw pointer: a graph that keeps `out` has to know
            torch.autograd.graph.increment_version(out)
    return out


# ----------------------------------------------------------------------------- attention with a window and sinks
def _heads(what, q, k, v):
    B, Hq, dh = q.shape[0], q.shape[-2], q.shape[-1]
    if k.dim() != 4 or v.shape != k.shape or k.shape[0] != B or k.shape[3] != dh:
        raise VitkError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not go together")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise VitkError(f"{what}: q, k and v have one type, got {q.dtype}, {k.dtype}, {v.dtype}")
    dtype_code(q.dtype)
    if dh not in (32, 64, 128):
        raise VitkError(f"{what}: head sizes 32, 64 and 128, got {dh}")
    if k.shape[2] == 0 or Hq % k.shape[2]:
        raise VitkError(f"{what}: {Hq} query heads do not share {k.shape[2]} key heads evenly")


def _reach(what, window, sinks, scale, tokens, dh):
    window = tokens if window is None else int(window)
    sinks = int(sinks)
    if window < 0 or sinks < 0:
        raise VitkError(f"{what}: window and sinks count tokens, got {window} and {sinks}")
    scale = 1.0 / math.sqrt(dh) if scale is None else float(scale)
    if not 2.0 ** -126 <= scale < 2.0 ** 127:           # in 32 bits, times the 1.44 of the base-2 exponential too
        raise VitkError(f"{what}: scale must be positive and a number in 32 bits, got {scale}")
    return min(window, tokens), min(sinks, tokens), scale


def _lengths(what, lengths, B):
    if lengths.dtype != torch.int32 or lengths.shape != (B,):
        raise VitkError(f"{what}: lengths is int32 [{B}], got {lengths.dtype} {tuple(lengths.shape)}")
    return lengths.contiguous()


def _p(t):
    return None if t is None else t.data_ptr()


def _slide_args(q, k, v, o, rest, lse, lengths, meta, d_o=None, delta=None, dq=None, dk=None, dv=None):
    window, sinks, causal, scale = meta
    st = []
    for t in (q, k, v, d_o, dq, dk, dv):
        st += t.stride()[:3] if t is not None else (0, 0, 0)
    return SlideAttn(_p(q), _p(k), _p(v), _p(o), _p(rest), _p(lse), _p(lengths), _p(d_o), _p(delta), _p(dq), _p(dk), _p(dv),
                     None, *st, q.shape[0], q.shape[1], q.shape[2], k.shape[2], q.shape[3], window, sinks, int(causal), scale)


def _slide_workspace(a, code, backward, device):
    """The records of the first tokens (16-byte aligned memory of this call and stream)."""
    n = lib.vitk_slide_attn_workspace(ctypes.byref(a), code, int(backward))
    if not n:
        return None
    ws = torch.empty(n // 4, dtype=torch.float32, device=device)
    a.workspace = ws.data_ptr()
    return ws


def _slide_forward(q, k, v, lengths, meta, keep):
    """(o, what its rounding left or None, lse or None): the last two are what a backward pass needs besides o (`keep`)."""
    B, N, Hq, dh = q.shape
    o = torch.empty((B, N, Hq, dh), dtype=q.dtype, device=q.device)
    rest = torch.empty((B, N, Hq, dh), dtype=torch.int8, device=q.device) if keep and q.dtype != torch.float32 else None
    lse = torch.empty((B, Hq, N), dtype=torch.float32, device=q.device) if keep else None
    if o.numel():
        with _On(q.device) as on:
            a = _slide_args(q, k, v, o, rest, lse, lengths, meta)
            code = dtype_code(q.dtype)
            ws = _slide_workspace(a, code, False, q.device)  # noqa: F841  (lives until the launch is enqueued)
            check(lib.vitk_slide_attn_fwd(ctypes.byref(a), code, on.stream), "vitk_slide_attn_fwd")
    return o, rest, lse


def _slide_backward(q, k, v, o, rest, lse, lengths, meta, d_o, dq, dk, dv):
    if d_o.dtype != q.dtype:
        d_o = convert(d_o, q.dtype)
    d_o = _rows(d_o)
    delta = torch.empty_like(lse)
    with _On(q.device) as on:
        a = _slide_args(q, k, v, o, rest, lse, lengths, meta, d_o, delta, dq, dk, dv)
        code = dtype_code(q.dtype)
        ws = _slide_workspace(a, code, True, q.device)  # noqa: F841
        check(lib.vitk_slide_attn_bwd(ctypes.byref(a), code, on.stream), "vitk_slide_attn_bwd")


class SlidingAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, meta):
        keep = any(ctx.needs_input_grad[:3])
        q, k, v = _rows(q), _rows(k), _rows(v)
        o, rest, lse = _slide_forward(q, k, v, lengths, meta, keep)
        if keep:
            ctx.save_for_backward(q, k, v, o, rest, lse, lengths)
            ctx.meta = meta
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o):
        q, k, v, o, rest, lse, lengths = ctx.saved_tensors
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        new = torch.empty if q.numel() else torch.zeros              # keys without queries: gradients of 0
        dq = new(q.shape, dtype=q.dtype, device=q.device) if need_q else None
        dk, dv = (new(k.shape, dtype=k.dtype, device=k.device) for _ in range(2)) if need_k or need_v else (None, None)
        if q.numel():
            _slide_backward(q, k, v, o, rest, lse, lengths, ctx.meta, d_o, dq, dk, dv)
        return dq, (dk if need_k else None), (dv if need_v else None), None, None


def sliding_attention(q, k, v, window, sinks=0, causal=False, lengths=None, scale=None):
    """Attention in which a token sees the tokens nearer than ``window`` and the first ``sinks`` tokens of its sequence.

    q [B, N, Hq, dh], k, v [B, N, Hkv, dh] (Hq a multiple of Hkv; dh 32, 64 or 128; any strides).  ``causal``: query i sees key
    j <= i when i - j < window or j < sinks; otherwise when |i - j| < window or j < sinks or i < sinks (first tokens
    such as a class token see everything).  ``window`` None: no limit.  ``lengths`` int32 [B] on the same device: how many tokens
    of each sequence there are; tokens behind it may hold anything, their outputs and gradients are 0, as are those of
    a query that sees nothing.  A query that looks at a NaN, or at an infinity whose score is no number or plus infinity, gives NaN, and
    so does its gradient (one in v, or in a gradient, may also reach those up to 62 tokens beyond, and of the same 32 as a first token).
    Returns [B, N, Hq, dh]."""
    what = "sliding_attention"
    if q.dim() != 4:
        raise VitkError(f"{what}: q is [batch, tokens, heads, head size], got {tuple(q.shape)}")
    _heads(what, q, k, v)
    if k.shape[1] != q.shape[1]:
        raise VitkError(f"{what}: {q.shape[1]} queries, {k.shape[1]} keys")
    window, sinks, scale = _reach(what, window, sinks, scale, q.shape[1], q.shape[3])
    if lengths is not None:
        lengths = _lengths(what, lengths, q.shape[0])
    _no_tangents(what, q, k, v)
    _one_device(what, q, k, v, lengths)
    meta = (window, sinks, bool(causal), scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return SlidingAttentionFn.apply(q, k, v, lengths, meta)
    return _slide_forward(_rows(q), _rows(k), _rows(v), lengths, meta, False)[0]


class SlidingAttentionQkvFn(torch.autograd.Function):
    """The same on a packed projection [B*N, 3 H dh], with the rotation of queries and keys in between: rotated
    queries and keys are kept for backward, which writes one packed gradient and turns its query and key part back."""

    @staticmethod
    def forward(ctx, qkv, shape, meta, rope):
        B, N, H = shape
        x = qkv.view(B, N, 3 * H, -1)
        if rope is None:
            qk, pos = x, None
        else:
            pos, pairs, base, interleaved = rope
            qk = torch.empty((B, N, 2 * H, x.shape[3]), dtype=x.dtype, device=x.device)
            with _On(x.device) as on:
                _rope_call(x[:, :, :2 * H], qk, pos, pairs, base, interleaved, False, on)
        q, k, v = qk[:, :, :H], qk[:, :, H:2 * H], x[:, :, 2 * H:]
        o, rest, lse = _slide_forward(q, k, v, None, meta, ctx.needs_input_grad[0])
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(qkv, qk if rope is not None else None, o, rest, lse, pos)
            ctx.meta = (shape, meta, rope[1:] if rope is not None else None)
        return o.view(B * N, -1)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_o):
        qkv, qk, o, rest, lse, pos = ctx.saved_tensors
        (B, N, H), meta, rope = ctx.meta
        x = qkv.view(B, N, 3 * H, -1)
        qk = x if qk is None else qk
        dqkv = torch.empty_like(qkv)
        g = dqkv.view(B, N, 3 * H, -1)
        _slide_backward(qk[:, :, :H], qk[:, :, H:2 * H], x[:, :, 2 * H:], o, rest, lse, None, meta,
                        d_o.reshape(B, N, H, -1), g[:, :, :H], g[:, :, H:2 * H], g[:, :, 2 * H:])
        if rope is not None:
            pairs, base, interleaved = rope
            with _On(qkv.device) as on:
                _rope_call(g[:, :, :2 * H], g[:, :, :2 * H], pos, pairs, base, interleaved, True, on)
        return dqkv, None, None, None


def sliding_attention_qkv(qkv, B, N, H, window, sinks=0, causal=False, scale=None, positions=None, pairs=None,
                          base=10000.0, interleaved=False):
    """`sliding_attention` on a fused projection qkv [B*N, 3*H*dh] (query | key | value, as `attention` takes it), after
    `axial_rope` of its queries and keys when ``positions`` and ``pairs`` are given.  Returns the context [B*N, H*dh]."""
    what = "sliding_attention_qkv"
    if qkv.dim() != 2 or B < 1 or N < 1 or H < 1 or qkv.shape[0] != B * N or qkv.shape[1] % (3 * H):
        raise VitkError(f"{what}: qkv {tuple(qkv.shape)} is not [{B} * {N}, 3 * {H} heads]")
    if (positions is None) != (pairs is None):
        raise VitkError(f"{what}: positions and pairs go together")
    _no_tangents(what, qkv)
    _one_device(what, qkv)
    qkv = qkv if qkv.is_contiguous() and qkv.data_ptr() % 16 == 0 else qkv.clone(memory_format=torch.contiguous_format)
    x = qkv.detach().view(B, N, 3 * H, -1)
    _heads(what, x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:])
    window, sinks, scale = _reach(what, window, sinks, scale, N, x.shape[3])
    rope = None
    if positions is not None:
        rope = _rope_args(x[:, :, :2 * H], positions, pairs, base) + (bool(interleaved),)
    return SlidingAttentionQkvFn.apply(qkv, (B, N, H), (window, sinks, bool(causal), scale), rope)


_CUS = {}         # compute units of each device


def _splits(B, Hkv, G, window, sinks, dh, esz, device):
    """Workgroups that share the keys of one (sequence, key head): as many as give each CU one in all, none with fewer than 32
    keys a wave.  One stream of 65536 tokens, 8 key heads of 4 x 128: 575 us unsplit, 50 us with 32 each; 12 heads of 64, 16384
    tokens: 111 us unsplit, 18.5 us with 21 each, 21.8 with 22, which is more than there are CUs.
    One workgroup alone while its waves have no more than 24 KB of keys each: shared, the kernels are faster, but a second launch
    costs an eager call 4 us of host time.  Microseconds alone and shared, eager | replayed from a graph, by KB a wave:
      12 heads of 64, bf16    8: 12.7 16.8 | 5.1 6.6    20: 12.7 17.0 | 8.9 6.8    24: 12.6 16.9 | 11.4 6.8   32: 14.5 17.0 | 14.3 7.1
      8 of 4 x 128, bf16     16: 12.7 16.9 | 6.7 8.0    24: 12.7 16.9 | 10.4 8.2   40: 13.3 17.0 | 12.9 8.3   48: 17.7 16.9 | 17.3 8.4
      4 of 2 x 32, bf16      12: 12.7 16.7 | 7.9 6.0    16: 12.7 16.8 | 9.8 6.1    24: 13.6 16.8 | 13.2 7.0   32: 17.0 16.8 | 16.7 7.2
      12 heads of 64, fp32   16: 12.8 16.9 | 9.4 8.6    24: 12.8 16.9 | 11.9 8.7   40: 18.2 17.0 | 17.8 8.7   48: 21.0 16.9 | 20.6 8.8
      4 of 4 x 128, fp32     32: 16.2 17.1 | 16.0 12.5  48: 20.9 17.0 | 20.5 12.4
    Up to about 24 KB an eager call gains what a replay loses, and beyond it does not.  The rule does not ask whether a
    graph is being captured, so that a replay gives the bits of the eager call."""
    cus = _CUS.get(device.index)
    if cus is None:
        cus = _CUS[device.index] = torch.cuda.get_device_properties(device).multi_processor_count
    groups = B * Hkv * ((G + 31) // 32)
    tiles = -(-window // 32) + -(-sinks // 32)
    turns = -(-tiles // (8 if esz == 2 else 4))
    if turns * 32 * dh * esz <= 24 * 1024:
        return 1
    return max(1, min(turns, cus // groups, 64))


def sliding_attention_decode(q, k_cache, v_cache, lengths, window, sinks=0, scale=None):
    """One new token per sequence against a cache: the query at position lengths[b] - 1 sees the first ``sinks`` and the
    last ``window`` of the lengths[b] cached tokens (its own key and value among them).

    q [B, Hq, dh]; k_cache, v_cache [B, capacity, Hkv, dh] (any strides); lengths int32 [B] on the same device, at most the
    capacity; 0 gives a row of zeros, a NaN among what is seen a row of NaN.  ``window`` None: no limit.  Not differentiable.
    Returns [B, Hq, dh]."""
    what = "sliding_attention_decode"
    if q.dim() != 3:
        raise VitkError(f"{what}: q is [batch, heads, head size], got {tuple(q.shape)}")
    if torch.is_grad_enabled() and (q.requires_grad or k_cache.requires_grad or v_cache.requires_grad):
        raise VitkError(f"{what}: not differentiable; call it under torch.no_grad()")
    _no_tangents(what, q, k_cache, v_cache)
    _heads(what, q, k_cache, v_cache)
    B, Hq, dh = q.shape
    cap, Hkv = k_cache.shape[1:3]
    window, sinks, scale = _reach(what, window, sinks, scale, cap, dh)
    lengths = _lengths(what, lengths, B)
    _one_device(what, q, k_cache, v_cache, lengths)
    if B == 0 or Hq == 0 or cap == 0:
        return torch.zeros(q.shape, dtype=q.dtype, device=q.device)
    q, k, v = (_rows(t, 1 << 62) for t in (q, k_cache, v_cache))
    with _On(q.device) as on:
        o = torch.empty((B, Hq, dh), dtype=q.dtype, device=q.device)
        splits = _splits(B, Hkv, Hq // Hkv, window, sinks, dh, q.element_size(), q.device)
        ws = torch.empty(B * Hq * splits * (dh + 2), dtype=torch.float32, device=q.device) if splits > 1 else None
        a = SlideCache(_p(q), _p(k), _p(v), _p(o), _p(lengths), _p(ws), *q.stride()[:2], *k.stride()[:3], *v.stride()[:3],
                       B, cap, Hq, Hkv, dh, window, sinks, splits, scale)
        check(lib.vitk_slide_decode(ctypes.byref(a), dtype_code(q.dtype), on.stream), "vitk_slide_decode")
    return o

"""Long-sequence operators against their plain 64-bit forms.  Every bound is the rounding bound that the oracle derives
beside the value (oracle/seq_oracle.py); nothing here is measured first."""
import math

import pytest
import torch

from oracle import seq_oracle as SO

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, FP = torch.bfloat16, torch.float32
R = {BF: 2.0 ** -8, FP: 0.0}


def _rand(*shape, dtype=FP, seed=0):
    g = torch.Generator().manual_seed(seed + 7919 * len(shape) + sum(shape))
    return torch.randn(*shape, generator=g).to(dtype)


def _hold(name, got, value, bound, tiny=1e-30):
    got = got.detach().double().cpu()
    assert got.shape == value.shape, name
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = ((got - value).abs() / (bound + tiny)).max() if got.numel() else torch.tensor(0.0)
    assert worst <= 1.0, f"{name}: {float(worst):.2f} of the bound"


# ----------------------------------------------------------------------------- rotary positions
ROPE = [  # (B, N, H, dh, pairs, interleaved, dtype, kind, each)
    (1, 1, 1, 2, (1,), False, FP, torch.int64, False), (2, 7, 3, 64, (16, 16), False, BF, torch.int64, False),
    (2, 7, 3, 64, (16, 16), True, BF, torch.float32, True), (3, 5, 2, 64, (8, 12, 12), False, FP, torch.int32, True),
    (1, 33, 5, 128, (64,), True, FP, torch.float64, False), (2, 9, 1, 32, (3, 4), False, BF, torch.int64, False),
    (2, 9, 1, 32, (3, 4), True, BF, torch.int64, True), (1, 3, 2, 6, (1, 1, 1), False, BF, torch.float32, False),
    (4, 1, 16, 256, (100, 28), False, BF, torch.int64, True), (1, 2, 3, 96, (5, 10), False, FP, torch.int64, False),
    (1, 17, 2, 64, (4,) * 8, True, FP, torch.int32, False), (2, 1025, 1, 64, (15, 15), False, BF, torch.int64, False)]


@pytest.mark.parametrize("B,N,H,dh,pairs,inter,dt,kind,each", ROPE)
def test_axial_rope_and_its_gradient(B, N, H, dh, pairs, inter, dt, kind, each):
    from vitk import ops
    x, dy = _rand(B, N, H, dh, dtype=dt, seed=1), _rand(B, N, H, dh, dtype=dt, seed=2)
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(-5, 3000, (B, N, len(pairs)) if each else (N, len(pairs)), generator=g).to(kind)
    if kind.is_floating_point:
        pos = pos + 0.25
    xd = x.to(DEV).requires_grad_(True)
    y = ops.axial_rope(xd, pos.to(DEV), pairs, base=1000.0, interleaved=inter)
    y.backward(dy.to(DEV))
    for name, got, src, inv in (("y", y, x, False), ("dx", xd.grad, dy, True)):
        val, e = SO.rope(src, pos, pairs, 1000.0, inter, inv)
        _hold(name, got, val, e + (R[dt] + SO.U) * val.abs())


def test_axial_rope_far_positions_strides_and_places():
    from vitk import ops
    B, N, H, dh, pairs = 2, 6, 4, 64, (8, 24)
    packed = _rand(B, N, 3 * H * dh, dtype=BF).to(DEV)
    pos = torch.tensor([[2 ** 31 + 5 * i, 10_000_019 * i] for i in range(N)])
    x = packed.view(B, N, 3 * H, dh)[:, :, :H]
    val, e = SO.rope(x, pos, pairs, 10000.0, False)
    # 2^31 turns less by 2^53-rounded products: 2^31 * 2^-52 of a radian at most, below one unit of the sine
    bound = e + R[BF] * val.abs()
    _hold("view", ops.axial_rope(x, pos.to(DEV), pairs), val, bound)
    turned = x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)              # heads outside tokens
    _hold("heads first", ops.axial_rope(turned, pos.to(DEV), pairs), val, bound)
    last = x.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2)                # elements not consecutive
    _hold("transposed", ops.axial_rope(last, pos.to(DEV), pairs), val, bound)
    odd = torch.empty(B * N * H * dh + 3, dtype=BF, device=DEV)[3:].view(B, N, H, dh).copy_(x)      # 2-byte aligned
    _hold("odd pointer", ops.axial_rope(odd, pos.to(DEV), pairs), val, bound)
    one = x[:, :, :1].expand(B, N, H, dh)                                        # one head broadcast
    _hold("broadcast", ops.axial_rope(one, pos.to(DEV), pairs)[:, :, 2:3], val[:, :, :1], bound[:, :, :1])
    cache = torch.full((B, 20, H, dh), 7.0, dtype=BF, device=DEV)                # into a part of a cache
    assert ops.axial_rope(x, pos.to(DEV), pairs, out=cache[:, 3:3 + N]) .data_ptr() == cache[:, 3:].data_ptr()
    _hold("cache", cache[:, 3:3 + N], val, bound)
    assert (cache[:, :3] == 7).all() and (cache[:, 3 + N:] == 7).all()
    for inter in (False, True):                                                  # in place
        want = ops.axial_rope(x, pos.to(DEV), pairs, interleaved=inter)
        same = x.clone()
        ops.axial_rope(same, pos.to(DEV), pairs, interleaved=inter, out=same)
        assert torch.equal(same, want)
    assert ops.axial_rope(x[:, :0], pos[:0].to(DEV), pairs).shape == (B, 0, H, dh)
    # broadcast leaf: its gradient is the sum over the copies
    leaf = x[:, :, :1].detach().float().requires_grad_(True)
    ops.axial_rope(leaf.expand(B, N, H, dh), pos.to(DEV), pairs).sum().backward()
    val, e = SO.rope(torch.full((B, N, 1, dh), float(H)), pos, pairs, 10000.0, False, True)
    _hold("sum", leaf.grad, val, H * e + 8 * SO.U * val.abs())


# ----------------------------------------------------------------------------- sliding-window attention
ATTN = [  # (B, N, Hq, Hkv, dh, causal, window, sinks, lengths)
    (1, 1, 1, 1, 64, True, 1, 0, None), (1, 1, 1, 1, 64, False, 1, 1, None), (2, 2, 2, 1, 32, False, 1, 0, (1, 2)),
    (1, 31, 2, 2, 64, True, 4, 0, None), (1, 33, 2, 1, 64, False, 4, 1, None), (2, 64, 2, 2, 64, True, 64, 0, None),
    (1, 65, 1, 1, 128, True, 17, 3, None), (1, 129, 2, 1, 64, False, 33, 2, None), (3, 197, 4, 2, 64, False, 40, 1, (197, 100, 1)),
    (4, 200, 2, 2, 32, True, 64, 5, (200, 0, 1, 130)), (1, 300, 6, 2, 64, False, 20, 70, None), (1, 300, 3, 3, 128, True, 50, 140, None),
    (2, 257, 4, 1, 64, True, 1000, 0, (257, 250)), (1, 257, 4, 4, 64, False, None, 0, None), (2, 160, 2, 2, 64, True, 0, 2, (160, 9)),
    (1, 96, 2, 2, 64, False, 0, 0, None), (1, 96, 2, 2, 64, False, 0, 3, None), (1, 513, 2, 2, 128, False, 128, 0, None),
    (1, 700, 5, 1, 64, True, 128, 4, None), (1, 1025, 1, 1, 64, False, 65, 33, (999,)),
    # few key heads, many queries a key: several workgroups to a band of keys
    (2, 700, 8, 1, 64, False, 150, 3, (700, 90)), (1, 150, 8, 1, 32, False, 100, 4, None), (2, 390, 12, 2, 128, True, None, 0, (390, 0)),
    (1, 520, 16, 1, 128, True, 100, 40, (333,)), (1, 4100, 4, 1, 32, True, 1, 2, None), (1, 1500, 2, 1, 64, True, None, 0, None), (1, 260, 20, 1, 128, False, 70, 2, None)]


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,N,Hq,Hkv,dh,causal,window,sinks,lengths", ATTN)
def test_sliding_attention_and_its_gradients(B, N, Hq, Hkv, dh, causal, window, sinks, lengths, dt):
    from vitk import ops
    q, k, v = (_rand(B, N, h, dh, dtype=dt, seed=s) for s, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    d_o = _rand(B, N, Hq, dh, dtype=dt, seed=4)
    want = SO.sliding_attention(q, k, v, N if window is None else window, sinks, causal, lengths, dh ** -0.5, R[dt], d_o)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o = ops.sliding_attention(*leaves, window, sinks=sinks, causal=causal, lengths=n)
    o.backward(d_o.to(DEV))
    for name, got in (("o", o), ("dq", leaves[0].grad), ("dk", leaves[1].grad), ("dv", leaves[2].grad)):
        _hold(name, got, *want[name])
    with torch.no_grad():
        again = ops.sliding_attention(*leaves, window, sinks=sinks, causal=causal, lengths=n)
    assert torch.equal(again, o)


def _case(dt, B=2, N=150, Hq=4, Hkv=2, dh=64):
    return tuple(_rand(B, N, h, dh, dtype=dt, seed=s).to(DEV) for s, h in ((1, Hq), (2, Hkv), (3, Hkv), (4, Hq)))


def _grads(q, k, v, d_o, **kw):
    from vitk import ops
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = ops.sliding_attention(*leaves, **kw)
    return [o.detach()] + list(torch.autograd.grad(o, leaves, d_o))


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_what_lies_behind_a_sequence_is_not_looked_at(dt, causal):
    q, k, v, d_o = _case(dt)
    lengths = torch.tensor([150, 71], dtype=torch.int32, device=DEV)
    kw = dict(window=20, sinks=3, causal=causal, lengths=lengths)
    clean = _grads(q, k, v, d_o, **kw)
    for bad in (float("nan"), float("inf"), torch.finfo(dt).min):
        dirty = [t.clone() for t in (q, k, v, d_o)]
        for t in dirty:
            t[1, 71:] = bad
        for a, b in zip(_grads(*dirty, **kw), clean):
            assert torch.equal(a, b)
            assert (a[1, 71:] == 0).all()


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,window,sinks,causal,lengths", [(1, 1, 0, True, None), (1, 9, 2, False, None), (150, 1, 0, True, None),
                                                           (150, 1, 0, False, (150, 33)), (3000, 0, 1, True, None), (90, 20, 3, False, (1, 1))])
def test_scores_of_queries_that_see_one_key_have_no_gradient(dt, N, window, sinks, causal, lengths):
    q, k, v, d_o = _case(dt, N=N)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o, dq, dk, dv = _grads(q, k, v, d_o, window=window, sinks=sinks, causal=causal, lengths=n)
    assert not dq.any() and not dk.any() and dv.any()


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("level", [-900.0, 900.0])
def test_scores_far_from_zero(dt, causal, level):
    """Every score near -900 or 900: the sums' logarithms lie far outside the range of an exponential."""
    from vitk import ops
    B, N, H, dh = 1, 333, 2, 64
    q, k, v, d_o = (_rand(B, N, H, dh, dtype=dt, seed=s) for s in range(4))
    q, k = q * 0.25, k * 0.25
    q[..., 0], k[..., 0] = 85.0, level * 8 / 85.0
    kw = dict(window=20, sinks=3, causal=causal)
    want = SO.sliding_attention(q, k, v, 20, 3, causal, None, dh ** -0.5, R[dt], d_o)
    for name, got in zip(("o", "dq", "dk", "dv"), _grads(*(t.to(DEV) for t in (q, k, v, d_o)), **kw)):
        _hold(name, got, *want[name])


def test_strides_orders_and_repeats_give_the_same_bits():
    q, k, v, d_o = _case(BF)
    kw = dict(window=33, sinks=2, causal=True)
    want = _grads(q, k, v, d_o, **kw)

    def same(got, what):
        for a, b in zip(got, want):
            assert torch.equal(a, b), what

    same(_grads(q, k, v, d_o, **kw), "again")
    heads = [t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for t in (q, k, v, d_o)]
    same(_grads(*heads, **kw), "heads first")
    last = [t.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2) for t in (q, k, v, d_o)]
    same(_grads(*last, **kw), "elements apart")
    packed = torch.cat([q, k, v], 2)
    same(_grads(packed[:, :, :4], packed[:, :, 4:6], packed[:, :, 6:], d_o, **kw), "packed")
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k, v, d_o)]
    same(_grads(*odd, **kw), "2-byte aligned")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _grads(q, k, v, d_o, **kw)
    torch.cuda.current_stream().wait_stream(side)
    same(got, "another stream")
    one = [t[:1].contiguous() for t in (q, k, v, d_o)]
    want = _grads(*one, **kw)
    same(_grads(*[t.as_strided(t.shape, (7, *t.stride()[1:])) for t in one], **kw), "a batch of one, any stride")


def test_two_captured_passes_replayed_at_once():
    """Each graph holds the records of its first tokens in memory of its own: replayed side by side on two streams, with
    other work of the same kind in between, both give what they give alone."""
    from vitk import ops
    first = _case(BF, B=1, N=3000)
    cases = [first, tuple(t.flip(1) for t in first)]
    kw = dict(window=40, sinks=3)
    graphs, outs, want = [], [], []
    with torch.no_grad():
        for q, k, v, _ in cases:
            want.append(ops.sliding_attention(q, k, v, **kw))
        torch.cuda.synchronize()
        for q, k, v, _ in cases:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(ops.sliding_attention(q, k, v, **kw))
            graphs.append(g)
        streams = [torch.cuda.Stream() for _ in graphs]
        for turn in range(4):
            for o in outs:
                o.zero_()
            torch.cuda.synchronize()
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
            ops.sliding_attention(*cases[0][:3], **kw)
            torch.cuda.synchronize()
            for o, w in zip(outs, want):
                assert torch.equal(o, w), turn


def test_some_gradients_only_and_shared_inputs():
    from vitk import ops
    q, k, v, d_o = _case(FP, Hq=2, Hkv=2)
    kw = dict(window=30, sinks=1)
    _, dq, dk, dv = _grads(q, k, v, d_o, **kw)
    for wanted in (0, 1, 2):
        leaves = [t.detach().requires_grad_(i == wanted) for i, t in enumerate((q, k, v))]
        got = torch.autograd.grad(ops.sliding_attention(*leaves, **kw), leaves[wanted], d_o)[0]
        assert torch.equal(got, (dq, dk, dv)[wanted])
    x = q.detach().requires_grad_(True)              # one tensor in all three places
    o = ops.sliding_attention(x, x, x, **kw)
    got = torch.autograd.grad(o, x, d_o)[0]
    _, a, b, c = _grads(q, q, q, d_o, **kw)
    val = (a.double() + b.double() + c.double()).cpu()
    _hold("sum", got, val, 3 * SO.U * (a.abs() + b.abs() + c.abs()).double().cpu())
    one = k[:, :, :1].detach().requires_grad_(True)  # one key head broadcast to two: the gradient of a shared head
    o = ops.sliding_attention(q, one.expand(-1, -1, 2, -1), v, **kw)
    shared = torch.autograd.grad(o, one, d_o)[0]
    _, _, both, _ = _grads(q, k[:, :, :1].expand(-1, -1, 2, -1), v, d_o, **kw)
    _hold("shared", shared, both.double().sum(2, keepdim=True).cpu(), 3 * SO.U * both.abs().double().sum(2, keepdim=True).cpu())
    for n in (0, 3):
        e = torch.zeros(2 if n else 0, 0 if n else 5, 2, 64, device=DEV, requires_grad=True)
        o = ops.sliding_attention(e, e, e, 3)
        assert o.shape == e.shape
        o.sum().backward()
        assert e.grad.shape == e.shape


def test_gradients_against_differences():
    """fp32, random directions: (f(x + h d) - f(x - h d)) / 2h = <grad, d> up to h^2 and rounding / h."""
    from vitk import ops
    q, k, v, d_o = (t * 0.5 for t in _case(FP, B=1, N=70, Hq=2, Hkv=1, dh=32))
    for causal in (True, False):
        kw = dict(window=11, sinks=2, causal=causal)
        _, *grads = _grads(q, k, v, d_o, **kw)
        for at, g in enumerate(grads):
            d = _rand(*g.shape, seed=20 + at).to(DEV)
            d = d / d.norm()
            h = 0.05

            def f(step):
                x = [q, k, v]
                x[at] = x[at] + step * d
                return float((ops.sliding_attention(*x, **kw).double() * d_o.double()).sum())

            # Richardson: the h^2 term cancels, what is left is of order h^4; sums of 4480 terms of size < 1, u each
            diff = (4 * (f(h / 2) - f(-h / 2)) / h - (f(h) - f(-h)) / (2 * h)) / 3
            want = float((g.double() * d.double()).sum())
            scale = float(g.double().norm())
            assert abs(diff - want) <= 1e-3 * scale, (causal, at, diff, want)


@pytest.mark.parametrize("Hkv,dh", [(2, 64), (1, 128)])
@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
def test_captured_training_pass_replays(dt, Hkv, dh):
    from vitk import ops
    q, k, v, d_o = _case(dt, B=1, N=190, Hkv=Hkv, dh=dh)
    static = [t.clone().requires_grad_(True) for t in (q, k, v)]
    sd = d_o.clone()
    kw = dict(window=25, sinks=2, causal=False)

    def once():
        o = ops.sliding_attention(*static, **kw)
        return [o] + list(torch.autograd.grad(o, static, sd))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        once()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = once()
    for turn in range(3):
        fresh = [_rand(*t.shape, dtype=dt, seed=50 + turn + i).to(DEV) for i, t in enumerate((q, k, v, d_o))]
        with torch.no_grad():
            for s, t in zip(static + [sd], fresh):
                s.copy_(t)
        want = _grads(*fresh, **kw)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b), turn


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_form_is_rotation_then_attention(dt, causal):
    from vitk import ops
    B, N, H, dh, pairs = 2, 50, 3, 64, (16, 16)
    qkv = _rand(B * N, 3 * H * dh, dtype=dt).to(DEV).requires_grad_(True)
    d_o = _rand(B * N, H * dh, dtype=dt, seed=9).to(DEV)
    pos = ops.grid_positions((7, 7), lead=1)
    kw = dict(window=9, sinks=1, causal=causal)
    o = ops.sliding_attention_qkv(qkv, B, N, H, positions=pos, pairs=pairs, **kw)
    (got,) = torch.autograd.grad(o, qkv, d_o)
    x = qkv.detach().view(B, N, 3 * H, dh)
    q, k = (ops.axial_rope(x[:, :, a:a + H], pos, pairs) for a in (0, H))
    want, dq, dk, dv = _grads(q, k, x[:, :, 2 * H:], d_o.view(B, N, H, dh), **kw)
    assert torch.equal(o, want.view(B * N, -1))
    dq, dk = (ops.axial_rope(g, -pos, pairs) for g in (dq, dk))       # turned back
    parts = got.view(B, N, 3 * H, dh)
    for name, a, b in (("dq", parts[:, :, :H], dq), ("dk", parts[:, :, H:2 * H], dk), ("dv", parts[:, :, 2 * H:], dv)):
        assert torch.equal(a, b), name
    plain = ops.sliding_attention_qkv(qkv, B, N, H, **kw)
    assert torch.equal(plain.view(B, N, H, dh), ops.sliding_attention(x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:], **kw))


def test_whole_window_is_plain_attention():
    """No limit and no sinks: the framework's full attention, each side within its own rounding of the other."""
    from vitk import ops
    B, N, H, dh = 2, 77, 2, 64
    qkv = _rand(B * N, 3 * H * dh, dtype=FP).to(DEV)
    a = ops.sliding_attention_qkv(qkv, B, N, H, None)
    b, _ = ops.attention(qkv, B, N, H)
    x = qkv.view(B, N, 3 * H, dh)
    want = SO.sliding_attention(x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:], N, 0, False, None, dh ** -0.5, 0.0)["o"]
    _hold("o", a.view(B, N, H, dh), *want)
    _hold("full", b.view(B, N, H, dh), want[0], 2 * want[1])


# ----------------------------------------------------------------------------- one token over a cache
DECODE = [  # (B, cap, Hq, Hkv, dh, window, sinks, lengths)
    (1, 1, 1, 1, 64, 1, 0, (1,)), (3, 40, 4, 2, 64, 8, 3, (0, 1, 40)), (2, 33, 2, 2, 32, 100, 0, (33, 32)),
    (2, 300, 6, 1, 128, 65, 40, (299, 50)), (1, 1000, 40, 1, 64, 512, 4, (1000,)), (2, 1000, 8, 8, 64, None, 0, (1000, 31)),
    (2, 129, 3, 3, 64, 0, 5, (129, 2)), (2, 64, 2, 2, 64, 0, 0, (64, 64)), (1, 2050, 2, 2, 128, 1500, 700, (2050,)),
    (5, 97, 35, 5, 32, 31, 31, (97, 96, 62, 61, 33)), (1, 9000, 2, 1, 64, 8000, 33, (8999,)),
    (1, 5000, 3, 1, 32, None, 2, (4990,)), (3, 3000, 40, 1, 64, 2500, 4, (3000, 17, 0))]


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,cap,Hq,Hkv,dh,window,sinks,lengths", DECODE)
def test_sliding_attention_decode(B, cap, Hq, Hkv, dh, window, sinks, lengths, dt):
    from vitk import ops
    q, k, v = _rand(B, Hq, dh, dtype=dt, seed=1), _rand(B, cap, Hkv, dh, dtype=dt, seed=2), _rand(B, cap, Hkv, dh, dtype=dt, seed=3)
    n = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    value, bound = torch.zeros(B, Hq, dh, dtype=torch.float64), torch.zeros(B, Hq, dh, dtype=torch.float64)
    for b, L in enumerate(lengths):
        seen = torch.zeros(1, L, dtype=torch.bool)
        seen[:, max(0, L - (cap if window is None else window)):] = True
        seen[:, :sinks] = True
        for h in range(Hq if L else 0):
            kk, vv = (t[b, :L, h // (Hq // Hkv)].double() for t in (k, v))
            value[b, h], bound[b, h] = (t[0] for t in SO.attention(q[b, h:h + 1].double(), kk, vv, seen, dh ** -0.5, R[dt])["o"])
    dirty = [t.to(DEV) for t in (k, v)]
    for b, L in enumerate(lengths):                  # rows behind a sequence hold anything
        for t in dirty:
            t[b, L:] = float("nan")
    o = ops.sliding_attention_decode(q.to(DEV), *dirty, n, window, sinks=sinks)
    _hold("o", o, value, bound)
    assert torch.equal(o, ops.sliding_attention_decode(q.to(DEV), *dirty, n, window, sinks=sinks))


def test_decode_layouts_graph_and_growing_cache():
    """A serving loop: the cache grows by one token per replay of a captured step; each step is the last row of the
    training form on the tokens so far."""
    from vitk import ops
    B, cap, Hq, Hkv, dh, pairs = 2, 70, 4, 2, 64, (10, 22)
    kw = dict(window=13, sinks=2)
    xs = _rand(B, cap, Hq + 2 * Hkv, dh, dtype=BF).to(DEV)
    pos = torch.stack([torch.arange(cap), 3 * torch.arange(cap)], 1).to(DEV)
    cache = torch.full((2, B, Hkv, cap, dh), float("nan"), dtype=BF, device=DEV).permute(0, 1, 3, 2, 4)    # heads outside tokens
    step = torch.zeros(B, 1, Hq + 2 * Hkv, dh, dtype=BF, device=DEV)
    at = torch.zeros(1, 2, dtype=torch.int64, device=DEV)
    n = torch.zeros(B, dtype=torch.int32, device=DEV)

    def once():
        q = ops.axial_rope(step[:, :, :Hq], at, pairs)
        return ops.sliding_attention_decode(q[:, 0], cache[0], cache[1], n, **kw)

    with torch.no_grad():
        once()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o = once()
        full_q = ops.axial_rope(xs[:, :, :Hq], pos, pairs)
        full_k = ops.axial_rope(xs[:, :, Hq:Hq + Hkv], pos, pairs)
        want = SO.sliding_attention(full_q, full_k, xs[:, :, Hq + Hkv:], 13, 2, True, None, dh ** -0.5, R[BF])["o"]
        for t in range(cap):
            step.copy_(xs[:, t:t + 1])
            at.copy_(pos[t:t + 1])
            n.fill_(t + 1)
            ops.axial_rope(step[:, :, Hq:Hq + Hkv], at, pairs, out=cache[0][:, t:t + 1])
            cache[1][:, t].copy_(step[:, 0, Hq + Hkv:])
            graph.replay()
            _hold(f"token {t}", o, want[0][:, t], want[1][:, t])


def test_decode_in_a_cache_beyond_32_bit_offsets():
    from vitk import ops
    cap, Hkv, dh = (1 << 18) + 77, 64, 128              # 2^31 elements and more in each cache
    q = _rand(1, Hkv, dh, dtype=BF).to(DEV)
    k = torch.zeros(1, cap, Hkv, dh, dtype=BF, device=DEV)
    v = torch.zeros(1, cap, Hkv, dh, dtype=BF, device=DEV)
    tail = 40
    rows = torch.cat([torch.arange(3), torch.arange(cap - tail, cap)])
    kk, vv = _rand(len(rows), Hkv, dh, dtype=BF, seed=2), _rand(len(rows), Hkv, dh, dtype=BF, seed=3)
    k[0, rows.to(DEV)], v[0, rows.to(DEV)] = kk.to(DEV), vv.to(DEV)
    o = ops.sliding_attention_decode(q, k, v, torch.tensor([cap], dtype=torch.int32, device=DEV), tail, sinks=3)
    seen = torch.ones(1, len(rows), dtype=torch.bool)
    for h in (0, 1, 31, 63):
        val, e = SO.attention(q[0, h:h + 1].double().cpu(), kk[:, h].double(), vv[:, h].double(), seen, dh ** -0.5, R[BF])["o"]
        _hold(f"head {h}", o[0, h:h + 1], val, e)


# ----------------------------------------------------------------------------- AdamW
SHAPES = [(64, 48), (257,), (1,), (3, 5, 7), (8193,), (4, 2049), (2, 8192), (31, 1025)]


def _optim(shapes, bits, seed=0, **kw):
    from utils.optim import FusedAdamW
    init = [_rand(*s, seed=seed + i) for i, s in enumerate(shapes)]
    params = [torch.nn.Parameter(p.clone().to(DEV)) for p in init]
    return init, params, FusedAdamW(params, state_bits=bits, **kw)


@pytest.mark.parametrize("clip", [None, 1.0])
@pytest.mark.parametrize("betas,wd", [((0.9, 0.999), 0.05), ((0.0, 0.5), 0.0)])
def test_adamw_32_bit_step(clip, betas, wd):
    kw = dict(lr=3e-3, betas=betas, eps=1e-7, weight_decay=wd)
    init, params, opt = _optim(SHAPES, 32, **kw)
    ref = [(p.double(), torch.zeros_like(p).double(), torch.zeros_like(p).double()) for p in init]
    for t in range(1, 5):
        grads = [_rand(*s, seed=100 * t + i) * (3.0 if t == 2 else 0.01) for i, s in enumerate(SHAPES)]
        for p, g in zip(params, grads):
            p.grad = g.to(DEV)
        norm = opt.step(max_grad_norm=clip)
        true = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        coef = 1.0
        if clip is not None:
            assert abs(float(norm) - true) <= 2 * SO.U * true
            coef = float(torch.tensor(min(1.0, clip / (true + 1e-6)), dtype=FP))
        else:
            assert norm is None
        for i, p in enumerate(params):
            st = opt.state[p]
            assert st["step"] == t
            new = SO.adamw(ref[i][0], grads[i].double(), ref[i][1], ref[i][2], t, coef, **{"wd" if k == "weight_decay" else k: v for k, v in kw.items()})
            for name, got, (val, e) in zip(("p", "m", "v"), (p, st["exp_avg"], st["exp_avg_sq"]), new):
                _hold(f"{name} {i} step {t}", got, val, e, tiny=1e-38)
            # the next step starts from what the kernel holds: bounds of one step each
            ref[i] = tuple(x.detach().double().cpu() for x in (p, st["exp_avg"], st["exp_avg_sq"]))


def test_adamw_32_bit_follows_torch():
    init, params, opt = _optim(SHAPES, 32, lr=1e-3, weight_decay=0.1)
    other = [torch.nn.Parameter(p.clone().double()) for p in init]
    ref = torch.optim.AdamW(other, lr=1e-3, weight_decay=0.1)
    sched = [torch.optim.lr_scheduler.LambdaLR(o, lambda k: 1.0 / (1 + k)) for o in (opt, ref)]
    for t in range(3):
        for i, (p, q) in enumerate(zip(params, other)):
            g = _rand(*p.shape, seed=300 + 10 * t + i)
            p.grad, q.grad = g.to(DEV), g.double()
        opt.step()
        ref.step()
        for s in sched:
            s.step()
    for p, q in zip(params, other):
        # three steps of at most 1e-3 each; a gradient near zero makes its own relative error in m / sqrt(v)
        _hold("p", p, q.detach(), 16 * SO.U * (q.detach().abs() + 1.0))


@pytest.mark.parametrize("clip", [None, 0.5])
def test_adamw_8_bit_step_bit_for_bit(clip):
    kw = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.05)
    init, params, opt = _optim(SHAPES, 8, seed=40, **{**kw, "lr": 3e-3})
    opt.seed = 12345
    held = [[p.clone().view(-1)] + [torch.zeros(p.numel()).to(torch.float8_e4m3fn), torch.zeros(-(-p.numel() // 256))] * 2 for p in init]
    for t in range(1, 6):
        grads = [_rand(*s, seed=100 * t + i) * 10.0 ** (i - 4) for i, s in enumerate(SHAPES)]
        if t == 3:
            grads[0].zero_()
            grads[1][:5] = 1e-20
        for p, g in zip(params, grads):
            p.grad = g.to(DEV)
        opt.step(max_grad_norm=clip)
        true = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        coef = 1.0 if clip is None else min(1.0, clip / (true + 1e-6))
        for i, p in enumerate(params):
            st = opt.state[p]
            held[i] = SO.adamw8(held[i][0], grads[i].view(-1), *held[i][1:], t, coef, kw["lr"], kw["betas"], kw["eps"], kw["weight_decay"], seed=12345,
                               sqrt=lambda x: x.to(DEV).sqrt().cpu())
            got = [p.detach().view(-1), st["exp_avg"].view(-1).view(torch.uint8), st["exp_avg_scale"],
                   st["exp_avg_sq"].view(-1).view(torch.uint8), st["exp_avg_sq_scale"]]
            for name, a, b in zip(("p", "m", "m scale", "v", "v scale"), got, held[i]):
                b = b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b
                a = a.cpu()
                if name == "p":
                    # three steps of at most lr / (1 - b1) each by a reciprocal of 2^-23, and a rounding of p each
                    assert ((a - b).abs() <= t * (2.0 ** -22 * kw["lr"] * 10 + 2 * SO.U * b.abs())).all(), (i, t)
                    continue
                if a.dtype == torch.uint8:                              # -0 and 0 are one value
                    a, b = torch.where(a == 128, 0, a), torch.where(b == 128, 0, b)
                assert torch.equal(a, b), (name, i, t)


def test_adamw_8_bit_moments_are_held_without_bias():
    """65536 elements, gradients of unit size: 400 steps of rounding leave the mean of the second moment where it is.
    One element's held value wanders by about a third of itself (a code's neighbours are 1/16 to 1/8 apart, of which a
    step of 1/1000 takes one at a time); the mean of 65536 of them by 0.3 / 256, and 2 % is 17 times that."""
    n = 65536
    _, params, opt = _optim([(n,)], 8, lr=0.0, weight_decay=0.0)
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    for _ in range(400):
        x = torch.randn(n, generator=g, device=DEV) + 0.5
        params[0].grad = x
        opt.step()
        m = 0.9 * m + 0.1 * x
        v = 0.999 * v + 0.001 * x * x
    st = opt.state[params[0]]
    hm = st["exp_avg"].float() * st["exp_avg_scale"].repeat_interleave(256)
    hv = (st["exp_avg_sq"].float() * st["exp_avg_sq_scale"].repeat_interleave(256)).square()
    assert abs(float(hv.mean() / v.mean()) - 1) < 0.02
    assert abs(float(hm.mean() / m.mean()) - 1) < 0.02
    assert float((hm - m).square().mean().sqrt()) < 0.15 * float(m.square().mean().sqrt())


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_groups_missing_gradients_alignment_and_state_dict(bits):
    from utils.optim import FusedAdamW
    shapes = [(300,), (40, 30), (5,), (0, 4), (9000,)]
    store = torch.cat([_rand(n, seed=n).view(-1) for n in (301, 1201, 6, 1, 9001)]).to(DEV)

    def build(odd):
        params, at = [], 1 if odd else 0
        for s in shapes:                                    # views of one buffer, at odd addresses or in tensors of their own
            n = math.prod(s)
            x = store[at:at + n] if odd else store[at + 1:at + 1 + n].clone()
            params.append(torch.nn.Parameter(x.view(s)))
            at += n
        opt = FusedAdamW([dict(params=params[:2], lr=1e-2), dict(params=params[2:], weight_decay=0.0, betas=(0.8, 0.9))], lr=1e-3,
                         weight_decay=0.1, state_bits=bits)
        return params, opt

    plain, opt_a = build(False)
    odd, opt_b = build(True)
    for t in range(4):
        for i, (p, q) in enumerate(zip(plain, odd)):
            if t == 1 and i in (1, 4):                       # no gradient: left alone, one step behind from here
                p.grad = q.grad = None
                continue
            g = _rand(*p.shape, seed=70 + 10 * t + i).to(DEV)
            p.grad = g
            q.grad = torch.empty(g.numel() + 1, device=DEV)[1:].view(g.shape).copy_(g)
        before = [p.detach().clone() for p in plain]
        na, nb = opt_a.step(max_grad_norm=5.0), opt_b.step(max_grad_norm=5.0)
        assert abs(float(na) - float(nb)) <= 2 * SO.U * float(na)        # other pieces, another order of 64-bit sums
        if t == 1:
            assert torch.equal(plain[1], before[1]) and torch.equal(plain[4], before[4])
        for p, q in zip(plain, odd):
            assert torch.equal(p, q)
        if t == 2:                                           # saved, restored into a new optimizer, and on
            sd = opt_a.state_dict()
            opt_a = build(False)[1]
            for grp, new in zip(opt_a.param_groups, (plain[:2], plain[2:])):
                grp["params"] = new
            opt_a.load_state_dict(sd)
    assert [opt_a.state[p]["step"] for p in plain if p.numel()] == [4, 3, 4, 3]
    with pytest.raises(ValueError):
        build(False)[1].__class__([torch.nn.Parameter(torch.zeros(3, device=DEV))], state_bits=40 - bits).load_state_dict(
            dict(sd, param_groups=sd["param_groups"][:1]))


def test_adamw_loads_torch_state_and_refuses():
    from utils.optim import FusedAdamW
    p, q = (torch.nn.Parameter(_rand(100).to(DEV)) for _ in range(2))
    ref, opt = torch.optim.AdamW([p], lr=1e-2), FusedAdamW([q], lr=1e-2)
    p.grad = _rand(100, seed=5).to(DEV)
    ref.step()
    with torch.no_grad():
        q.copy_(p)
    opt.load_state_dict(ref.state_dict())
    q.grad = p.grad.clone()
    ref.step()
    opt.step()
    _hold("p", q, p.detach().double().cpu(), 16 * SO.U * (p.detach().double().cpu().abs() + 1e-2))
    with pytest.raises(ValueError, match="moments"):          # another tensor behind the same parameter
        q.data = torch.zeros(101, device=DEV)
        q.grad = torch.zeros(101, device=DEV)
        opt.step()
    for bad in (torch.zeros(4, device=DEV, dtype=BF), torch.zeros(4, 6, device=DEV).t()):
        x = torch.nn.Parameter(bad)
        x.grad = torch.zeros_like(x)
        with pytest.raises(ValueError):
            FusedAdamW([x]).step()
    y = torch.nn.Parameter(torch.zeros(4, device=DEV))
    y.grad = torch.zeros(4, device=DEV)
    opt = FusedAdamW([y])
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    held = torch.zeros(4, device=DEV)
    with torch.cuda.graph(graph):
        held += 1
        with pytest.raises(RuntimeError, match="captured"):
            opt.step()


# ----------------------------------------------------------------------------- together
@pytest.mark.parametrize("bits", [32, 8])
def test_vit_with_rotary_positions_and_a_window_trains_with_adamw(bits):
    """Positions, attention and update in one model, fp32 compute: loss and every gradient within 1e-5 of their scale
    (the framework's fp32 bar), every updated parameter within the step's own rounding of the gradients it was given."""
    import vitk
    from models.config import get_tiny_config
    from models.ViT.modeling import VisionTransformer
    from utils.optim import FusedAdamW
    torch.manual_seed(3)
    cfg = get_tiny_config()
    cfg.transformer.update(attention_window=4, attention_sinks=1, rope_pairs=(12, 20), rope_base=100.0)
    kw = dict(lr=1e-3, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.05)
    with vitk.compute_dtype(FP):
        model = VisionTransformer(cfg, (48, 80), num_classes=7).to(DEV).train()
        assert not any("positions" in k and "embeddings" not in k for k in model.state_dict())
        with torch.no_grad():
            for p in model.parameters():
                p.add_(0.05 * torch.randn_like(p))
        opt = FusedAdamW(model.parameters(), state_bits=bits, **kw)
        for step in (1, 2):
            images, labels = _rand(3, 3, 48, 80, seed=step), torch.tensor([1, 5, 2])
            loss = model(images.to(DEV), labels.to(DEV))
            loss.backward()
            ref = {k: v.detach().double().cpu().requires_grad_(True) for k, v in model.named_parameters()}
            logits = SO.vit_logits(ref, images.double(), 16, 2, 2, (3, 5), 4, 1, (12, 20), 100.0)
            want = torch.nn.functional.cross_entropy(logits, labels)
            want.backward()
            assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(want))
            for name, p in model.named_parameters():
                g, r = p.grad.double().cpu(), ref[name].grad
                scale = r.abs().max()
                if name.endswith("attn.key.bias"):     # zero but for rounding: judged by the query bias's
                    scale = torch.maximum(scale, ref[name.replace("key", "query")].grad.abs().max())
                assert (g - r).abs().max() <= 1e-5 * scale + 1e-7, name
            before = {k: (p.detach().double().cpu(), p.grad.double().cpu(),
                          *((opt.state[p][n].double().cpu() for n in ("exp_avg", "exp_avg_sq")) if step > 1 and bits == 32 else
                            (torch.zeros_like(p, dtype=torch.float64).cpu(),) * 2)) for k, p in model.named_parameters()}
            norm = opt.step(max_grad_norm=1.0)
            coef = float(torch.tensor(min(1.0, 1.0 / (float(norm.double()) + 1e-6)), dtype=FP))
            if step == 1 or bits == 32:                # in 8 bits the second step starts from rounded moments
                for name, p in model.named_parameters():
                    # the norm was rounded to 32 bits on its way here: one unit of the factor more
                    (val, e), _, _ = SO.adamw(*before[name], step, coef, kw["lr"], kw["betas"], kw["eps"], kw["weight_decay"])
                    _hold(name, p, val, e + 4 * SO.U * kw["lr"] * 10)
            opt.zero_grad()
    with pytest.raises(ValueError):
        VisionTransformer(cfg, (48, 80), num_classes=7, vis=True)

"""The long-sequence operators where their paths change over: first tokens in chunks, many bands, values that are not finite,
odd layouts.  Bounds are those of oracle/seq_oracle.py, derived there."""
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


def _near(name, got, value, most):
    """The error's norm against the value's."""
    got = got.detach().double().cpu()
    off = float((got - value).norm() / value.norm().clamp_min(1e-300))
    assert off <= most, f"{name}: off by {off:.5f} of its norm, allowed {most:.5f}"


# Rounded once, a value is off by an error that is spread evenly over half a step of 2^-8 to either side: 2^-8 / sqrt(3) of it, root of
# the mean square, at most.  bf16 results are rounded once and one of their factors (P, dS) once before; inputs are
# random and independent, so both errors add as squares.
TWICE = 2.0 ** -8 * math.sqrt(2.0 / 3.0)


def _check_attention(B, N, Hq, Hkv, dh, causal, window, sinks, lengths, dt):
    from vitk import ops
    q, k, v = (_rand(B, N, h, dh, dtype=dt, seed=s) for s, h in ((1, Hq), (2, Hkv), (3, Hkv)))
    d_o = _rand(B, N, Hq, dh, dtype=dt, seed=4)
    want = SO.sliding_attention(q, k, v, window, sinks, causal, lengths, dh ** -0.5, R[dt], d_o)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    o = ops.sliding_attention(*leaves, window, sinks=sinks, causal=causal, lengths=n)
    o.backward(d_o.to(DEV))
    for name, got in (("o", o), ("dq", leaves[0].grad), ("dk", leaves[1].grad), ("dv", leaves[2].grad)):
        _hold(name, got, *want[name])
        if dt == BF:
            _near(name, got, want[name][0], TWICE)
    with torch.no_grad():
        assert torch.equal(ops.sliding_attention(*leaves, window, sinks=sinks, causal=causal, lengths=n), o)


# ----------------------------------------------------------------------------- first tokens in chunks
# Without a causal mask and with more than 48 tiles of 32 tokens, what the first QUERIES see beyond their band is cut into chunks
# whose records are added at the end (forward, dQ), like that of the first keys.
CHUNKED = [  # (B, N, Hq, Hkv, dh, window, sinks, lengths)
    (1, 1700, 2, 2, 64, 40, 3, None), (2, 1640, 2, 1, 64, 9, 40, (1640, 1601)), (3, 1600, 2, 2, 32, 100, 130, (1600, 70, 0)),
    (1, 1700, 4, 2, 128, 300, 3, None), (2, 1700, 1, 1, 64, 0, 33, (1700, 20)), (1, 2305, 3, 3, 64, 145, 1, None)]


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,N,Hq,Hkv,dh,window,sinks,lengths", CHUNKED)
def test_first_tokens_of_long_sequences_in_chunks(B, N, Hq, Hkv, dh, window, sinks, lengths, dt):
    _check_attention(B, N, Hq, Hkv, dh, False, window, sinks, lengths, dt)


# ----------------------------------------------------------------------------- values that are not finite
def _pairs(N, window, sinks, causal):
    return SO.visible(N, N, N if window is None else window, sinks, causal, N)


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,window,sinks,causal", [(150, 20, 3, False), (150, 20, 3, True), (1700, 40, 3, False), (90, None, 0, False)])
@pytest.mark.parametrize("place", ["q", "k", "v"])
def test_a_nan_reaches_every_query_that_sees_it(N, window, sinks, causal, dt, place):
    """No query that looks at a NaN may come out as a number, least of all as the 0 of one that sees nothing; a NaN in a query
    or a key leaves the others alone."""
    from vitk import ops
    B, H, dh, bad = 1, 2, 64, N - 40
    t = {n: _rand(B, N, H, dh, dtype=dt, seed=s) for s, n in enumerate(("q", "k", "v"))}
    d_o = _rand(B, N, H, dh, dtype=dt, seed=5)
    want = SO.sliding_attention(t["q"], t["k"], t["v"], N if window is None else window, sinks, causal, None, dh ** -0.5, R[dt])["o"]
    t[place][0, bad, 0, 7] = math.nan
    seen = _pairs(N, window, sinks, causal)
    hit = (torch.arange(N) == bad) if place == "q" else seen[:, bad]
    leaves = [t[n].to(DEV).requires_grad_(True) for n in ("q", "k", "v")]
    o = ops.sliding_attention(*leaves, window, sinks=sinks, causal=causal)
    dq, dk, dv = torch.autograd.grad(o, leaves, d_o.to(DEV))
    got = o.detach().cpu()[0, :, 0]
    if place == "v":
        assert got[hit, 7].isnan().all()
    else:
        assert got[hit].isnan().all()
        _hold("others", o[:, ~hit, 0], want[0][:, ~hit, 0], want[1][:, ~hit, 0])
        assert dq.cpu()[0, hit, 0].isnan().all()
        of = seen[hit].any(0)                       # the keys that such a query sees
        assert dk.cpu()[0, of, 0].isnan().all() and dv.cpu()[0, of, 0].isnan().all()
    _hold("the other head", o[:, :, 1], want[0][:, :, 1], want[1][:, :, 1])


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,bad", [(1700, slice(1000, 1700)), (1700, slice(200, 1700)), (400, slice(128, 256))])
def test_a_run_of_nan_keys_is_not_dropped(N, bad, dt):
    """First tokens see everything: also where all that one chunk, or one wave, of them looks at is NaN."""
    from vitk import ops
    q, k, v = (_rand(1, N, 1, 64, dtype=dt, seed=s) for s in range(3))
    k[:, bad] = math.nan
    o = ops.sliding_attention(q.to(DEV), k.to(DEV), v.to(DEV), 20, sinks=3).cpu()
    hit = _pairs(N, 20, 3, False)[:, bad].any(1)
    assert o[0, hit].isnan().all() and torch.isfinite(o[0, ~hit]).all()


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("N,bad,clean", [(1700, slice(1600, 1601), slice(3, 1499)), (1700, slice(300, 1700), slice(3, 199)), (1700, slice(1500, 1501), slice(1602, 1700)),
                                         (500, slice(300, 301), slice(32, 199)), (500, slice(300, 301), slice(402, 500))])
def test_a_nan_in_v_stays_near_those_that_look_at_it(N, bad, clean, dt):
    """Queries further than 62 tokens (31 of a tile of keys and 31 of one of queries) from one that looks at it are clean; in long
    sequences, where chunks are records of their own, those beside a first token too."""
    from vitk import ops
    q, k, v = (_rand(1, N, 1, 64, dtype=dt, seed=s) for s in range(3))
    want = SO.sliding_attention(q, k, v, 40, 3, False, None, 0.125, R[dt])["o"]
    v[:, bad] = math.nan
    o = ops.sliding_attention(q.to(DEV), k.to(DEV), v.to(DEV), 40, sinks=3).cpu()
    assert o[0, _pairs(N, 40, 3, False)[:, bad].any(1)].isnan().all()
    _hold("o", o[:, clean], want[0][:, clean], want[1][:, clean])


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_infinite_keys(dt, causal):
    """A score of minus infinity is a weight of 0, one of plus infinity leaves no number."""
    from vitk import ops
    N, bad = 150, 60
    q, k, v = (_rand(1, N, 1, 64, dtype=dt, seed=s) for s in range(3))
    q[0, :2, 0, 0] = torch.tensor([1.0, -1.0])      # of the first tokens, which see it without a causal mask, one of each
    want = SO.sliding_attention(q, k, v, 20, 3, causal, None, 0.125, R[dt])["o"]
    without = SO.attention(q[0, :, 0].double(), k[0, :, 0].double(), v[0, :, 0].double(),
                           _pairs(N, 20, 3, causal) & (torch.arange(N) != bad), 0.125, R[dt])["o"]
    k[0, bad, 0, 0] = math.inf
    o = ops.sliding_attention(q.to(DEV), k.to(DEV), v.to(DEV), 20, sinks=3, causal=causal).cpu()[0, :, 0]
    seen, up = _pairs(N, 20, 3, causal)[:, bad], q[0, :, 0, 0].float() > 0
    assert o[seen & up].isnan().all() and (seen & up).any()
    for rows, (val, e) in ((~seen, (want[0][0, :, 0], want[1][0, :, 0])), (seen & ~up, without)):
        _hold("rows", o[rows], val[rows], e[rows])


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("cap,window", [(90, 50), (6000, 5000)])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_decode_of_values_that_are_not_finite(cap, window, value, dt):
    from vitk import ops
    B, Hq, Hkv, dh = 2, 4, 2, 64
    q, k, v = _rand(B, Hq, dh, dtype=dt).abs(), _rand(B, cap, Hkv, dh, dtype=dt, seed=1), _rand(B, cap, Hkv, dh, dtype=dt, seed=2)
    n = torch.tensor([cap, cap - 7], dtype=torch.int32, device=DEV)

    def call(q, k):
        return ops.sliding_attention_decode(q.to(DEV), k.to(DEV), v.to(DEV), n, window, sinks=2).cpu()

    clean = call(q, k)
    bad = q.clone()
    bad[0, 1, 3] = value
    o = call(bad, k)
    assert o[0, 1].isnan().all() and torch.equal(o[0, 0], clean[0, 0]) and torch.equal(o[:, 2:], clean[:, 2:])
    for at, hit in ((cap - 9, True), (1, True), (cap - window - 10, False)):
        bad = k.clone()
        bad[1, at, 0, 3] = value
        o = call(q, bad)
        assert o[1, :2].isnan().all() if hit else torch.equal(o, clean), at
        assert torch.equal(o[0], clean[0]) and torch.equal(o[:, 2:], clean[:, 2:])
    bad = k.clone()
    bad[1, cap - window - 7:cap - 8] = value                  # all that some workgroups look at
    assert call(q, bad)[1].isnan().all()


# ----------------------------------------------------------------------------- AdamW
def _pair_of_optimizers(n, **kw):
    from utils.optim import FusedAdamW
    out = []
    for _ in range(2):
        p = torch.nn.Parameter(_rand(n).to(DEV))
        out.append((p, FusedAdamW([p], lr=1e-2, state_bits=8, **kw)))
    return out


def _moments(p, opt):
    st = opt.state[p]
    return [st[x].view(torch.uint8).cpu() for x in ("exp_avg", "exp_avg_sq")] + [st[x + "_scale"].cpu() for x in ("exp_avg", "exp_avg_sq")]


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_adamw_8_bit_holds_what_is_not_finite_where_it_is(value):
    """One gradient that is no number: its own element shows it from here on, as in 32 bits; its 255 neighbours keep their moments."""
    (p, a), (q, b) = _pair_of_optimizers(700)
    at, others = 300, torch.arange(700) != 300
    for t in range(5):
        g = _rand(700, seed=10 + t)
        g[at] = 0.01
        q.grad = g.to(DEV)
        if t == 2:
            g = g.clone()
            g[at] = value
        p.grad = g.to(DEV)
        a.step()
        b.step()
        assert torch.equal(p.cpu()[others], q.cpu()[others]), t
        (m, v, ms, vs), (m2, v2, ms2, vs2) = _moments(p, a), _moments(q, b)
        assert torch.equal(m[others], m2[others]) and torch.equal(v[others], v2[others]) and torch.equal(ms, ms2) and torch.equal(vs, vs2), t
        assert bool(p.cpu()[at].isnan()) == (t >= 2)
        assert bool((m[at] & 127) == 127) == (t >= 2) and bool((v[at] & 127) == 127) == (t >= 2)


def test_adamw_8_bit_second_moment_that_overflows_is_not_forgotten():
    (p, a), _ = _pair_of_optimizers(700)
    for t in range(3):
        g = _rand(700, seed=10 + t)
        if t == 1:
            g[300] = 1e20                           # its square is beyond 32 bits
        was = p.detach().clone()
        p.grad = g.to(DEV)
        a.step()
        if t:
            _, v, _, vs = _moments(p, a)
            assert (v[300] & 127) == 127            # from now on no number, where 32 bits hold an infinity
            others = torch.arange(700) != 300
            assert (v[others] > 0).all() and (vs > 0).all() and torch.isfinite(vs).all()
            # a step of ordinary size: |m| / sqrt(v) of up to three steps is sqrt(3) at most, codes off by 1/8 twice each; and the decay
            assert ((p - was).abs().cpu()[others] <= 1e-2 * (4 + 0.01 * 5)).all()
    assert p[300].isnan()


# ----------------------------------------------------------------------------- rotary positions
def test_axial_rope_in_place_is_seen_by_autograd():
    from vitk import ops
    x = _rand(1, 5, 2, 64).to(DEV)
    w = _rand(1, 5, 2, 64, seed=1).to(DEV).requires_grad_(True)
    y = (w * x).sum()                                # its backward pass needs x
    before = x._version
    ops.axial_rope(x, torch.arange(5, device=DEV)[:, None], (32,), out=x)
    assert x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    with torch.inference_mode():                     # such tensors have no versions
        z = torch.ones(1, 5, 2, 64, device=DEV)
        assert ops.axial_rope(z, torch.arange(5, device=DEV)[:, None], (32,), out=z) is z


ODD = ["pointer", "tokens", "heads", "sequence of one", "gradient"]


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("odd", ODD)
def test_axial_rope_takes_rows_at_odd_places(odd, inter, dt):
    from vitk import ops
    B, N, H, dh, pairs = 2, 5, 3, 64, (7, 20)
    pos = torch.randint(0, 50, (N, 2), generator=torch.Generator().manual_seed(1))
    x, dy = _rand(B, N, H, dh, dtype=dt), _rand(B, N, H, dh, dtype=dt, seed=1)
    if odd == "sequence of one":
        x, dy = x[:1], dy[:1]

    def place(t):
        t = t.to(DEV)
        if odd == "pointer":
            return torch.zeros(t.numel() + 1, dtype=dt, device=DEV)[1:].view(t.shape).copy_(t)
        if odd == "tokens":
            return torch.zeros(B, N, H * dh + 1, dtype=dt, device=DEV)[:, :, :H * dh].unflatten(2, (H, dh)).copy_(t)
        if odd == "heads":
            return torch.zeros(B, N, H, dh + 3, dtype=dt, device=DEV)[..., :dh].copy_(t)
        if odd == "sequence of one":
            return t.as_strided(t.shape, (7, *t.stride()[1:]))
        return t

    xd = place(x).detach().requires_grad_(True)
    y = ops.axial_rope(xd, pos.to(DEV), pairs, interleaved=inter)
    if odd == "gradient":                            # the slice of a wider one
        wide = torch.cat([y, torch.ones(B, N, H, 1, dtype=dt, device=DEV)], -1)
        wide.backward(torch.cat([dy, torch.ones(B, N, H, 1, dtype=dt)], -1).to(DEV))
    else:
        y.backward(place(dy))
    for name, got, src, inv in (("y", y, x, False), ("dx", xd.grad, dy, True)):
        val, e = SO.rope(src, pos, pairs, 10000.0, inter, inv)
        _hold(name, got, val, e + (R[dt] + SO.U) * val.abs())
    to = place(torch.zeros_like(x))
    assert ops.axial_rope(x.to(DEV), pos.to(DEV), pairs, interleaved=inter, out=to) is to
    assert torch.equal(to, y)


@pytest.mark.parametrize("inter", [False, True])
def test_axial_rope_into_a_place_that_overlaps_its_input(inter):
    from vitk import ops
    cache = _rand(2, 4000, 6, 64, dtype=BF).to(DEV)
    pos = torch.arange(3999, device=DEV)[:, None]
    want = ops.axial_rope(cache[:, :-1, :4], pos, (32,), interleaved=inter)
    for to in (lambda c: c[:, 1:, :4], lambda c: c[:, :-1, 1:5], lambda c: c[:, :-1, 2:], lambda c: c[:, :-1, :4]):
        work = cache.clone()
        out = to(work)
        rest = torch.ones_like(work, dtype=torch.bool)
        to(rest).fill_(False)
        ops.axial_rope(work[:, :-1, :4], pos, (32,), interleaved=inter, out=out)
        assert torch.equal(out, want) and torch.equal(work[rest], cache[rest])


@pytest.mark.parametrize("N", [2 ** 25 + 5, 2 ** 26 + 3])
def test_axial_rope_of_more_tokens_than_a_launch_counts_threads_for(N):
    from vitk import ops
    x = torch.randn(1, N, 1, 2, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    pos = torch.arange(N, device=DEV, dtype=torch.int32)[:, None]
    y = ops.axial_rope(x, pos, (1,))[0, :, 0]
    for lo in range(0, N, 1 << 23):
        a, b = x[0, lo:lo + (1 << 23), 0].double().unbind(1)
        turn = pos[lo:lo + (1 << 23), 0].double()
        for got, val in ((y[lo:lo + (1 << 23), 0], a * turn.cos() - b * turn.sin()), (y[lo:lo + (1 << 23), 1], b * turn.cos() + a * turn.sin())):
            # the bound of the oracle; 2^26 radians are 2^-26 of one off in 64 bits
            assert ((got.double() - val).abs() <= 11 * SO.U * (a.abs() + b.abs())).all(), lo


# ----------------------------------------------------------------------------- no query heads
def test_key_heads_without_queries_have_gradients_of_zero():
    from vitk import ops
    junk = [torch.full((2, 50, 2, 64), math.nan, device=DEV) for _ in range(4)]
    del junk
    q, k, v = (torch.ones(2, 50, h, 64, device=DEV, requires_grad=True) for h in (0, 2, 2))
    junk = [torch.full((2, 50, 2, 64), math.nan, device=DEV) for _ in range(4)]
    del junk
    o = ops.sliding_attention(q, k, v, 5)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), torch.ones_like(o))
    assert o.shape == dq.shape == q.shape and not dk.any() and not dv.any()


# ----------------------------------------------------------------------------- AdamW: parameters written through raw pointers
def test_adamw_update_is_seen_by_autograd():
    """A parameter that a graph has kept is not silently another one in its backward pass."""
    from utils.optim import FusedAdamW
    for bits in (8, 32):
        p = torch.nn.Parameter(_rand(300).to(DEV))
        x = _rand(300, seed=1).to(DEV).requires_grad_(True)
        opt = FusedAdamW([p], state_bits=bits)
        y = (p * x).sum()
        p.grad = torch.ones_like(p)
        before = p._version
        opt.step()
        assert p._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


def test_adamw_update_of_a_weight_whose_operands_another_one_holds():
    """Query, key and value share one pair of GEMM operands, kept with the query's weight: also when only the key's is trained."""
    from utils.optim import FusedAdamW
    from vitk import ops
    ws = [torch.nn.Parameter(_rand(64, 64, seed=i).to(DEV)) for i in range(3)]
    bs = [torch.nn.Parameter(torch.zeros(64, device=DEV)) for _ in range(3)]
    x = _rand(64, 64, dtype=BF).to(DEV)
    opt = FusedAdamW([ws[1]], lr=0.1)
    with torch.no_grad():
        before = ops.linear(x, tuple(ws), tuple(bs)).clone()
        ws[1].grad = torch.ones_like(ws[1])
        opt.step()
        after = ops.linear(x, tuple(ws), tuple(bs)).clone()
        ops.invalidate_operands(ws)
        assert torch.equal(after, ops.linear(x, tuple(ws), tuple(bs)))
    assert not torch.equal(after[:, 64:128], before[:, 64:128]) and torch.equal(after[:, :64], before[:, :64])


def test_adamw_copies_step_on():
    import copy
    import io
    from utils.optim import FusedAdamW
    for bits in (8, 32):
        p = torch.nn.Parameter(_rand(300).to(DEV))
        opt = FusedAdamW([p], state_bits=bits, seed=7)
        p.grad = _rand(300, seed=2).to(DEV)
        opt.step()
        opt.step()                                   # the gradients' addresses are known to the table by now
        file = io.BytesIO()                          # (torch's tensors of 8-bit floats are not taken by `pickle` itself)
        torch.save((p, opt), file)
        file.seek(0)
        others = [copy.deepcopy((p, opt)), torch.load(file, weights_only=False)]
        for q, _ in others:
            q.grad = p.grad.clone()
        opt.step(max_grad_norm=1.0)
        for q, o in others:
            o.step(max_grad_norm=1.0)
            assert torch.equal(p, q)
            assert all(torch.equal(opt.state[p][n].float(), o.state[q][n].float()) for n in ("exp_avg", "exp_avg_sq"))


# ----------------------------------------------------------------------------- decode: alone, shared, replayed
@pytest.mark.parametrize("dt,dh,window", [(BF, 64, 1500), (BF, 64, 1700), (BF, 64, 1024), (FP, 32, 700), (BF, 128, 700), (BF, 128, 900), (FP, 64, 4000)])
def test_decode_replays_what_it_gives_eagerly(dt, dh, window):
    """On both sides of the size from which workgroups share a stream's keys."""
    from vitk import ops
    B, Hq, Hkv, cap = 2, 4, 2, window + 40
    q, k, v = _rand(B, Hq, dh, dtype=dt).to(DEV), _rand(B, cap, Hkv, dh, dtype=dt, seed=1).to(DEV), _rand(B, cap, Hkv, dh, dtype=dt, seed=2).to(DEV)
    n = torch.tensor([cap, cap - 30], dtype=torch.int32, device=DEV)
    ops.sliding_attention_decode(q, k, v, n, window, sinks=3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = ops.sliding_attention_decode(q, k, v, n, window, sinks=3)
    for turn in range(3):
        q.copy_(_rand(B, Hq, dh, dtype=dt, seed=10 + turn))
        n.fill_(cap - turn)
        want = ops.sliding_attention_decode(q, k, v, n, window, sinks=3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want), turn
        for b in range(B):
            L = cap - turn
            seen = torch.zeros(1, L, dtype=torch.bool)
            seen[:, L - window:] = seen[:, :3] = True
            for h in range(Hq):
                val, e = SO.attention(q[b, h:h + 1].double().cpu(), k[b, :L, h // 2].double().cpu(), v[b, :L, h // 2].double().cpu(), seen, dh ** -0.5, R[dt])["o"]
                _hold(f"{turn} {b} {h}", want[b, h:h + 1], val, e)


@pytest.mark.parametrize("B,Hq,Hkv,dh,cap,window,sinks", [(4, 12, 12, 64, 1100, 1024, 4), (8, 8, 2, 128, 3000, 2900, 0), (16, 8, 4, 32, 300, 200, 3), (32, 12, 12, 64, 40, 9, 2)])
def test_decode_is_off_by_the_rounding_of_its_result(B, Hq, Hkv, dh, cap, window, sinks):
    """bf16: probabilities are held in 16 bits behind the leading one, so the error's norm is that of the exact result rounded once,
    but for 2^-8 of it and the 32-bit sums: a tenth more at most, where probabilities of 8 bits would make it sqrt(2) of that."""
    from vitk import ops
    q, k, v = _rand(B, Hq, dh, dtype=BF), _rand(B, cap, Hkv, dh, dtype=BF, seed=1), _rand(B, cap, Hkv, dh, dtype=BF, seed=2)
    n = torch.full((B,), cap, dtype=torch.int32, device=DEV)
    o = ops.sliding_attention_decode(q.to(DEV), k.to(DEV), v.to(DEV), n, window, sinks=sinks)
    at = torch.cat([torch.arange(sinks), torch.arange(cap - window, cap)])
    qd, kd, vd = q.double().view(B, Hkv, -1, dh), k[:, at].double().transpose(1, 2).contiguous(), v[:, at].double().transpose(1, 2).contiguous()
    want = (torch.softmax(qd @ kd.transpose(2, 3).contiguous() * dh ** -0.5, -1) @ vd).view(B, Hq, dh)
    _near("o", o, want, 1.1 * float((want.to(BF).double() - want).norm() / want.norm()))


# ----------------------------------------------------------------------------- many bands
# Bands of 128 keys want 512 of them; with 1024 bands one item does first tokens of up to 96 tiles.  (B, N, Hq, Hkv, dh, causal, window,
# sinks): the last two rows reach 1024.
MANY = [(16, 130, 16, 16, 64, False, 40, 1), (16, 130, 16, 16, 32, True, 20, 0), (8, 150, 64, 32, 64, False, 9, 3), (13, 257, 14, 14, 128, False, 70, 5),
        (16, 200, 32, 16, 64, True, 200, 0), (8, 2305, 12, 12, 64, False, 145, 1), (16, 385, 64, 16, 32, False, 12, 40)]


@pytest.mark.parametrize("dt", [FP, BF], ids=["fp32", "bf16"])
@pytest.mark.parametrize("B,N,Hq,Hkv,dh,causal,window,sinks", MANY)
def test_attention_of_many_heads(B, N, Hq, Hkv, dh, causal, window, sinks, dt):
    """Some heads of a launch with many: first, last and in between, each with its neighbours' memory around it."""
    from vitk import ops
    G = Hq // Hkv
    g = torch.Generator(device=DEV).manual_seed(N)
    q, k, v, d_o = (torch.randn(B, N, h, dh, device=DEV, generator=g).to(dt) for h in (Hq, Hkv, Hkv, Hq))
    n = torch.full((B,), N, dtype=torch.int32, device=DEV)
    n[B // 2] = N - 77
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    o = ops.sliding_attention(*leaves, window, sinks=sinks, causal=causal, lengths=n)
    got = (o, *torch.autograd.grad(o, leaves, d_o))
    for b, h in ((0, 0), (B // 2, Hkv // 2), (B - 1, Hkv - 1)):
        qs, ks = slice(h * G, (h + 1) * G), slice(h, h + 1)
        at = [t.detach()[b:b + 1, :, s].cpu() for t, s in ((q, qs), (k, ks), (v, ks), (d_o, qs))]
        want = SO.sliding_attention(*at[:3], window, sinks, causal, (int(n[b]),), dh ** -0.5, R[dt], at[3])
        for name, t, s in zip(("o", "dq", "dk", "dv"), got, (qs, qs, ks, ks)):
            _hold(f"{name} {b} {h}", t[b:b + 1, :, s], *want[name])
            if dt == BF:
                _near(f"{name} {b} {h}", t[b:b + 1, :, s], want[name][0], TWICE)
    assert all(not t[B // 2, N - 77:].any() for t in got)


# ----------------------------------------------------------------------------- short windows
@pytest.mark.parametrize("N,Hq,Hkv,dh,causal,window,sinks", [(700, 4, 2, 64, False, 9, 0), (700, 2, 2, 128, True, 16, 0), (1700, 2, 2, 64, False, 16, 3),
                                                             (500, 4, 4, 32, True, 3, 2)])
def test_short_windows_are_off_by_the_rounding_of_their_results(N, Hq, Hkv, dh, causal, window, sinks):
    """bf16, windows of up to 16 keys: what goes into the products is held in 16 bits, so an error's norm is nearer to that of the exact result
    rounded once than to that and another rounding of probabilities or score gradients, sqrt(2) of it; the limit lies half way."""
    from vitk import ops
    q, k, v, d_o = (_rand(1, N, h, dh, dtype=BF, seed=s) for s, h in enumerate((Hq, Hkv, Hkv, Hq)))
    want = SO.sliding_attention(q, k, v, window, sinks, causal, None, dh ** -0.5, R[BF], d_o)
    leaves = [t.to(DEV).requires_grad_(True) for t in (q, k, v)]
    o = ops.sliding_attention(*leaves, window, sinks=sinks, causal=causal)
    for name, got in zip(("o", "dq", "dk", "dv"), (o, *torch.autograd.grad(o, leaves, d_o.to(DEV)))):
        val = want[name][0]
        _near(name, got, val, (1 + math.sqrt(2.0)) / 2 * float((val.to(BF).double() - val).norm() / val.norm()))


def test_decode_reads_a_cache_of_far_apart_tokens_where_it_is():
    """Tokens outermost, with room between them: no copy of the cache, whatever the stride."""
    from vitk import ops
    cap, dh, apart = 40, 64, (1 << 23) + 64
    cache = torch.zeros(cap, apart, dtype=BF, device=DEV)
    k, v = (cache[:, at:at + dh].unflatten(1, (1, dh))[None] for at in (0, dh))
    k.copy_(_rand(1, cap, 1, dh, dtype=BF, seed=1))
    v.copy_(_rand(1, cap, 1, dh, dtype=BF, seed=2))
    q, n = _rand(1, 2, dh, dtype=BF).to(DEV), torch.tensor([cap], dtype=torch.int32, device=DEV)
    want = ops.sliding_attention_decode(q, k.contiguous(), v.contiguous(), n, 30, sinks=2)
    assert k.stride(1) == apart
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    got = ops.sliding_attention_decode(q, k, v, n, 30, sinks=2)
    assert torch.equal(got, want) and torch.cuda.max_memory_allocated() - before < 2 * k.numel()

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

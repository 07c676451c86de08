"""What the long-sequence operators refuse or keep, without a GPU, beyond tests/test_seq_cpu.py."""
import pytest
import torch
from torch.autograd import forward_ad

from vitk import VitkError, ops


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_derivatives_are_refused(which, grad):
    """Inputs with a tangent and without `requires_grad` look like constants to a call that records nothing."""
    pos = torch.zeros(5, 2, dtype=torch.int64)
    n = torch.zeros(2, dtype=torch.int32)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        def dual(*ts):
            return [forward_ad.make_dual(t, torch.ones_like(t)) if i == which else t for i, t in enumerate(ts)]

        q, k, v = dual(_t(2, 5, 4, 64), _t(2, 5, 2, 64), _t(2, 5, 2, 64))
        calls = [lambda: ops.sliding_attention(q, k, v, 3),
                 lambda: ops.sliding_attention_decode(*dual(_t(2, 4, 64), _t(2, 9, 2, 64), _t(2, 9, 2, 64)), n, 3)]
        if which == 0:
            x, qkv = dual(_t(2, 5, 3, 64)), dual(_t(10, 3 * 128))
            calls += [lambda: ops.axial_rope(*x, pos, (16, 16)), lambda: ops.axial_rope(*x, pos, (16, 16), out=_t(2, 5, 3, 64)),
                      lambda: ops.axial_rope(_t(2, 5, 3, 64), pos, (16, 16), out=x[0]),
                      lambda: ops.sliding_attention_qkv(*qkv, 2, 5, 2, window=3)]
        for call in calls:
            with pytest.raises(VitkError, match="forward-mode"):
                call()
    with pytest.raises(VitkError, match="GPU only"):
        ops.sliding_attention(_t(2, 5, 4, 64), _t(2, 5, 2, 64), _t(2, 5, 2, 64), 3)

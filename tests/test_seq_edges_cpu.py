"""What the long-sequence operators refuse or keep, without a GPU, beyond tests/test_seq_cpu.py."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

import vitk
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


def _views():
    """(x, out, whether they share an element at different indices) of one buffer, told element by element."""
    for shape in ((1, 4, 2, 2), (2, 3, 1, 4), (1, 1, 3, 2), (2, 2, 2, 2)):
        for st in ((16, 4, 2, 1), (2, 8, 4, 1), (24, 8, 4, 1), (3, 5, 2, 1), (0, 4, 2, 1)):
            for to in (st, (16, 4, 2, 1)):
                for at in range(-9, 10):
                    base = torch.arange(200)
                    x, out = base.as_strided(shape, st, 20), base.as_strided(shape, to, 20 + at)
                    if out.unique().numel() == out.numel():
                        yield x, out, bool(((x.reshape(-1, 1) == out.reshape(1, -1)) & ~torch.eye(x.numel(), dtype=torch.bool)).any())


def test_axial_rope_knows_where_out_meets_x():
    from vitk.seq_ops import _meets
    said = known = 0
    for x, out, shares in _views():
        if shares:
            assert _meets(x, out), (x.shape, x.stride(), out.stride(), out.storage_offset())
        said, known = said + (not _meets(x, out)), known + (not shares)
    assert said > known // 3                           # and does not always copy
    packed = torch.zeros(2, 5, 6, 8)
    assert not _meets(packed[:, :, :3], packed[:, :, 3:]) and not _meets(packed, packed) and not _meets(packed, packed.clone())
    assert _meets(packed[:, :-1], packed[:, 1:]) and _meets(packed[:, :, :4], packed[:, :, 2:])


def test_axial_rope_refuses_what_its_counters_do_not_hold():
    one, at = _t(1, 1, 1, 2), torch.zeros(1, 1, dtype=torch.int64)
    for shape in ((1, 1 << 31, 1, 2), (1 << 16, 1 << 16, 1, 2), (1, (1 << 32) + 5, 1, 2), (1, 1, 1 << 27, 2)):
        with pytest.raises(VitkError, match="tokens"):
            ops.axial_rope(one.expand(shape), at.expand(shape[1], 1), (1,))


@pytest.mark.parametrize("scale", [3.4e38, 1e39, 1e300, 1e-40, 1e-300, float("inf"), float("nan"), 0.0, -1.0])
def test_scales_that_32_bits_do_not_hold_are_refused(scale):
    n = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.sliding_attention(_t(2, 5, 4, 64), _t(2, 5, 2, 64), _t(2, 5, 2, 64), 3, scale=scale),
                 lambda: ops.sliding_attention_decode(_t(2, 4, 64), _t(2, 9, 2, 64), _t(2, 9, 2, 64), n, 3, scale=scale)):
        with pytest.raises(VitkError, match="scale"):
            call()


@pytest.mark.parametrize("scale", [3.4e38, float("inf")])
def test_c_entries_refuse_scales_that_overflow(scale):
    a = dict(q=4096, k=4096, v=4096, o=4096, B=1, Hq=2, Hkv=2, dh=64, window=3, scale=scale)
    assert vitk.lib.vitk_slide_attn_fwd(ctypes.byref(vitk.SlideAttn(**a, N=5)), 0, None) == -1
    assert vitk.lib.vitk_slide_decode(ctypes.byref(vitk.SlideCache(**a, cap=5, splits=1, lengths=4096)), 0, None) == -1


def test_adamw_copies_keep_their_settings():
    import copy
    import pickle
    from utils.optim import FusedAdamW
    opt = FusedAdamW([torch.nn.Parameter(torch.zeros(3))], lr=1e-2, state_bits=8, seed=5)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert (other.state_bits, other.seed, other.param_groups[0]["lr"]) == (8, 5, 1e-2)
        assert other.step() is None                   # no gradients
        other.param_groups[0]["params"][0].grad = torch.zeros(3)
        with pytest.raises(ValueError, match="GPU"):
            other.step()


@pytest.mark.parametrize("asked", [dict(attention_window=4), dict(rope_pairs=(8, 8)), dict(attention_window=4, rope_pairs=(8, 8))])
@pytest.mark.parametrize("name", ["RKR", "PB", "PBG", "RKRPB", "RKRPBG", "RKRTSN"])
def test_models_without_a_window_refuse_one(name, asked):
    """The task-conditioned models have full attention only: a configuration that asks for more is no silent full attention."""
    import importlib
    from models.config import get_tiny_config
    Attention = importlib.import_module(f"models.ViT.modeling_{name}").Attention
    cfg = get_tiny_config()
    cfg.transformer.update(asked)
    args = (cfg, False) + ((0,) if "PBG" in name else ())
    with pytest.raises(ValueError, match="|".join(asked)):
        Attention(*args)

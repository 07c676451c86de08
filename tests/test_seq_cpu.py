"""What the long-sequence operators refuse, without a GPU: arguments at the Python entry points and at the C entries
(which check before they launch anything), and the optimizer's settings."""
import ctypes

import pytest
import torch

import vitk
from vitk import VitkError, ops


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


ROPE = dict(x=_t(2, 5, 3, 64), positions=torch.zeros(5, 2, dtype=torch.int64), pairs=(16, 16))
ATTN = dict(q=_t(2, 5, 4, 64), k=_t(2, 5, 2, 64), v=_t(2, 5, 2, 64), window=3)
DECODE = dict(q=_t(2, 4, 64), k_cache=_t(2, 9, 2, 64), v_cache=_t(2, 9, 2, 64), lengths=torch.zeros(2, dtype=torch.int32), window=3)


@pytest.mark.parametrize("change", [
    {}, dict(x=_t(5, 3, 64)), dict(x=_t(2, 5, 3, 64, dtype=torch.float16)), dict(x=_t(2, 5, 3, 258)), dict(x=_t(2, 5, 3, 63)),
    dict(pairs=(16, 17)), dict(pairs=(16, 0)), dict(pairs=()), dict(pairs=(16,)), dict(pairs=(1,) * 9),
    dict(positions=torch.zeros(4, 2)), dict(positions=torch.zeros(5, 3)), dict(positions=torch.zeros(3, 5, 2)),
    dict(positions=torch.zeros(5, 2, dtype=torch.float16)), dict(positions=torch.zeros(5, 2, requires_grad=True)),
    dict(base=0.0), dict(base=float("inf")), dict(out=_t(2, 5, 3, 32)), dict(out=_t(2, 5, 3, 64, dtype=torch.float32)),
    dict(out=_t(2, 5, 64, 3).transpose(2, 3)), dict(out=_t(2, 5, 1, 64).expand(2, 5, 3, 64)),
])
def test_axial_rope_refuses(change):
    with pytest.raises(VitkError, match="axial_rope|unsupported dtype" if change else "GPU only"):
        ops.axial_rope(**{**ROPE, **change})


@pytest.mark.parametrize("change", [
    {}, dict(q=_t(2, 5, 64)), dict(q=_t(2, 5, 3, 64)), dict(q=_t(2, 6, 4, 64)), dict(q=_t(3, 5, 4, 64)), dict(q=_t(2, 5, 4, 32)),
    dict(v=_t(2, 5, 1, 64)), dict(k=_t(2, 5, 2, 64, dtype=torch.float32)), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
    dict(scale=float("nan")), dict(lengths=torch.zeros(2, dtype=torch.int64)), dict(lengths=torch.zeros(3, dtype=torch.int32)),
    dict(q=_t(2, 5, 4, 48), k=_t(2, 5, 2, 48), v=_t(2, 5, 2, 48)),
    dict(q=_t(2, 5, 4, 64, dtype=torch.float16), k=_t(2, 5, 2, 64, dtype=torch.float16), v=_t(2, 5, 2, 64, dtype=torch.float16)),
])
def test_sliding_attention_refuses(change):
    with pytest.raises(VitkError, match="sliding_attention|unsupported dtype" if change else "GPU only"):
        ops.sliding_attention(**{**ATTN, **change})


@pytest.mark.parametrize("change", [
    {}, dict(q=_t(2, 1, 4, 64)), dict(q=_t(2, 3, 64)), dict(q=_t(3, 4, 64)), dict(k_cache=_t(2, 9, 2, 32)), dict(v_cache=_t(2, 8, 2, 64)),
    dict(lengths=torch.zeros(2)), dict(window=-1), dict(sinks=-2), dict(scale=-1.0), dict(q=_t(2, 4, 64, dtype=torch.float32)),
    dict(q=_t(2, 4, 64).requires_grad_(True)),
])
def test_sliding_attention_decode_refuses(change):
    with pytest.raises(VitkError, match="sliding_attention_decode" if change else "GPU only"):
        ops.sliding_attention_decode(**{**DECODE, **change})


def test_sliding_attention_qkv_refuses():
    qkv = _t(10, 3 * 128)
    for args in ((2, 4, 2), (2, 5, 5), (0, 5, 2)):
        with pytest.raises(VitkError, match="sliding_attention_qkv"):
            ops.sliding_attention_qkv(qkv, *args, window=3)
    with pytest.raises(VitkError, match="go together"):
        ops.sliding_attention_qkv(qkv, 2, 5, 2, window=3, pairs=(16, 16))
    with pytest.raises(VitkError, match="GPU only"):
        ops.sliding_attention_qkv(qkv, 2, 5, 2, window=3)


def _attn(**change):
    a = dict(q=4096, k=4096, v=4096, o=4096, q_b=640, q_n=128, q_h=64, k_b=640, k_n=128, k_h=64, v_b=640, v_n=128, v_h=64, B=1, N=5,
             Hq=2, Hkv=2, dh=64, window=3, sinks=1, scale=0.125)
    return vitk.SlideAttn(**{**a, **change})


@pytest.mark.parametrize("change,dtype,code", [
    (dict(q=None), 0, -3), (dict(o=None), 0, -3), ({}, 2, -2), (dict(dh=48), 0, -4), (dict(Hq=3), 0, -1), (dict(N=0), 0, -1),
    (dict(B=0), 0, -1), (dict(B=65536), 0, -1), (dict(window=-1), 0, -1), (dict(sinks=-1), 0, -1), (dict(scale=0.0), 0, -1),
    (dict(q=4098), 0, -1), (dict(k_n=129), 0, -1), (dict(v_h=65), 1, -1), (dict(o=4100), 0, -1)])
def test_c_entry_of_the_forward_pass_refuses(change, dtype, code):
    assert vitk.lib.vitk_slide_attn_fwd(ctypes.byref(_attn(**change)), dtype, None) == code


@pytest.mark.parametrize("change,dtype,code", [
    (dict(d_o=None), 0, -3), (dict(lse=None), 0, -3), (dict(delta=None), 0, -3), (dict(o_rest=None), 0, -3), (dict(o=None), 0, -3), (dict(o=None), 1, -3),
    (dict(dk=None), 0, -3), (dict(dq=None, dk=None, dv=None), 0, -3), (dict(do_n=4), 0, -1), (dict(dq=4104), 0, -1)])
def test_c_entry_of_the_backward_pass_refuses(change, dtype, code):
    a = dict(d_o=4096, lse=4096, delta=4096, o_rest=4096, dq=4096, dk=4096, dv=4096)
    assert vitk.lib.vitk_slide_attn_bwd(ctypes.byref(_attn(**{**a, **change})), dtype, None) == code


@pytest.mark.parametrize("change,code", [
    (dict(lengths=None), -3), (dict(workspace=None), -3), (dict(splits=0), -1), (dict(splits=1025), -1), (dict(cap=0), -1),
    (dict(dh=96), -4), (dict(Hkv=3), -1), (dict(q=4097), -1), (dict(k_b=1), -1), (dict(window=-1), -1)])
def test_c_entry_of_decode_refuses(change, code):
    a = dict(q=4096, k=4096, v=4096, o=4096, lengths=4096, workspace=4096, B=1, cap=9, Hq=2, Hkv=2, dh=64, window=3, splits=2, scale=1.0)
    assert vitk.lib.vitk_slide_decode(ctypes.byref(vitk.SlideCache(**{**a, **change})), 0, None) == code


@pytest.mark.parametrize("change,code", [
    (dict(pos=None), -3), (dict(dh=63), -1), (dict(dh=258), -1), (dict(axes=0), -1), (dict(axes=9), -1), (dict(pos_kind=4), -1),
    (dict(base=0.0), -1), (dict(pairs=(ctypes.c_int * 8)(20, 20)), -1), (dict(pairs=(ctypes.c_int * 8)(20, 0)), -1),
    (dict(pairs=(ctypes.c_int * 8)(2 ** 31 - 1, 2 ** 31 - 1)), -1), (dict(x=4097), -1), (dict(interleaved=1, x_h=65), -1)])
def test_c_entry_of_axial_rope_refuses(change, code):
    a = dict(x=4096, y=4096, pos=4096, x_h=64, y_h=64, B=1, N=1, H=1, dh=64, axes=2, base=100.0, pairs=(ctypes.c_int * 8)(16, 16))
    assert vitk.lib.vitk_axial_rope(ctypes.byref(vitk.Rope(**{**a, **change})), 0, None) == code


def test_c_entries_of_adamw_refuse():
    lib = vitk.lib
    good = [4096, 4096, 1, 1.0, 4096, None, None]
    for at, value, code in ((0, None, -3), (1, None, -3), (2, 0, -1), (3, -1.0, -1), (4, None, -3)):
        assert lib.vitk_adamw_norm(*(good[:at] + [value] + good[at + 1:])) == code, at
    good = [4096, 4096, 0, 1, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, 32, 0, None]
    for at, value, code in ((0, None, -3), (1, None, -3), (2, -1, -1), (3, 0, -1), (6, 1.0, -1), (7, -0.1, -1), (8, -1.0, -1),
                            (10, 0, -1), (11, 16, -4)):
        assert lib.vitk_adamw_step(*(good[:at] + [value] + good[at + 1:])) == code, at


@pytest.mark.parametrize("settings", [dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-1.0), dict(betas=(0.9, 1.0)),
                                      dict(betas=(-0.1, 0.9)), dict(state_bits=16)])
def test_adamw_refuses_settings(settings):
    from utils.optim import FusedAdamW
    with pytest.raises(ValueError):
        FusedAdamW([torch.nn.Parameter(torch.zeros(3))], **settings)


def test_adamw_refuses_what_it_cannot_update():
    from utils.optim import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(3))
    opt = FusedAdamW([p])
    assert opt.step() is None                       # no gradients
    p.grad = torch.zeros(3)
    with pytest.raises((ValueError, RuntimeError)):
        opt.step()
    with pytest.raises(ValueError):
        opt.step(closure=lambda: 0)
    with pytest.raises(ValueError):
        opt.step(max_grad_norm=-1.0)


def test_adamw_refuses_states_of_other_parameters():
    from utils.optim import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(300))
    moments = {name: torch.zeros(300) for name in ("exp_avg", "exp_avg_sq")}
    groups = torch.optim.AdamW([p]).state_dict()["param_groups"]

    def load(bits=32, groups=groups, **change):
        st = {k: v for k, v in {"step": 1, **moments, **change}.items() if v is not None}
        FusedAdamW([p], state_bits=bits).load_state_dict(dict(state={0: st}, param_groups=groups))

    load()
    scales = dict(exp_avg_scale=torch.zeros(2), exp_avg_sq_scale=torch.zeros(2))
    load(8, **scales)
    for bits, change in ((32, dict(exp_avg=torch.zeros(299))), (32, dict(exp_avg_sq=torch.zeros(1, 300))), (32, dict(exp_avg=None)),
                         (8, dict(scales, exp_avg_scale=torch.zeros(1))), (8, dict(scales, exp_avg_sq_scale=None)), (32, scales), (8, {})):
        with pytest.raises(ValueError):
            load(bits, **change)
    for name in ("amsgrad", "maximize"):
        with pytest.raises(ValueError):
            load(groups=[dict(groups[0], **{name: True})])


def test_adamw_refused_step_leaves_no_states():
    from utils.optim import FusedAdamW
    p = torch.nn.Parameter(torch.zeros(3))
    opt = FusedAdamW([p])
    p.grad = torch.zeros(3)
    with pytest.raises(ValueError):
        opt.step()
    assert not opt.state[p]


def test_grid_positions():
    pos = ops.grid_positions((2, 3), lead=1, device="cpu")
    assert pos.tolist() == [[0, 0], [0, 0], [0, 1], [0, 2], [1, 0], [1, 1], [1, 2]]

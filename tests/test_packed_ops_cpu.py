"""CPU: what rope_axes and attention_varlen refuse, in Python and at the C entries, before anything touches a device."""
import ctypes
import math

import pytest
import torch


def _rope(**kw):
    from diffusion_pipe_amd import ops
    args = dict(q=torch.zeros(6, 4, 64), k=torch.zeros(6, 2, 64), positions=torch.zeros(6, 3), axes_dim=(8, 28, 28))
    args.update(kw)
    return ops.rope_axes(**args)


@pytest.mark.parametrize('kw,match', [
    ({}, 'device tensors'),
    ({'q': torch.zeros(6, 64)}, 'one dtype'),
    ({'k': torch.zeros(5, 2, 64)}, 'one dtype'),
    ({'k': torch.zeros(6, 2, 64, dtype=torch.bfloat16)}, 'one dtype'),
    ({'q': torch.zeros(6, 4, 64, dtype=torch.float16), 'k': None}, 'unsupported dtype'),
    ({'q': torch.zeros(6, 4, 60), 'k': None}, 'multiple of 8'),
    ({'q': torch.zeros(6, 4, 264), 'k': None}, 'multiple of 8'),
    ({'q': torch.zeros(6, 0, 64), 'k': None}, 'at least one head'),
    ({'axes_dim': (8, 28, 30)}, 'even axis sizes'),
    ({'axes_dim': (7, 29, 28)}, 'even axis sizes'),
    ({'axes_dim': ()}, 'even axis sizes'),
    ({'axes_dim': (8, 28, 0)}, 'even axis sizes'),
    ({'axes_dim': (8, 10, 10), 'interleaved': False}, 'even axis sizes'),
    ({'theta': 0.0}, 'theta'),
    ({'theta': (10.0, 10.0)}, 'theta'),
    ({'theta': math.nan}, 'theta'),
    ({'theta': (10.0, 20.0, 10.0), 'shared': True}, 'theta'),
    ({'positions': torch.zeros(6, 3, dtype=torch.float64)}, 'positions'),
    ({'positions': torch.zeros(6, 3, dtype=torch.bfloat16)}, 'positions'),
    ({'positions': torch.zeros(6, 3, requires_grad=True)}, 'positions'),
    ({'positions': torch.zeros(6, 2)}, 'do not fit'),
    ({'positions': torch.zeros(5, 3)}, 'do not fit'),
    ({'positions': torch.zeros(3)}, 'do not fit'),
    ({'positions': torch.zeros(2, 6, 3)}, 'do not fit'),
    ({'q_weight': torch.ones(63)}, 'norm weights'),
    ({'k': None, 'k_weight': torch.ones(64)}, 'needs k'),
])
def test_rope_axes_refuses(kw, match):
    from diffusion_pipe_amd.hip import DpipeHipError
    with pytest.raises(DpipeHipError, match=match):
        _rope(**kw)


def _varlen(**kw):
    from diffusion_pipe_amd import ops
    bf = torch.bfloat16
    args = dict(q=torch.zeros(6, 4, 64, dtype=bf), k=torch.zeros(6, 2, 64, dtype=bf), v=torch.zeros(6, 2, 64, dtype=bf), cu_q=torch.tensor([0, 2, 6], dtype=torch.int32))
    args.update(kw)
    return ops.attention_varlen(**args)


_Z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)


@pytest.mark.parametrize('kw,match', [
    ({}, 'device tensors'),
    ({'q': _Z(1, 6, 4, 64)}, 'attention_varlen: q'),
    ({'q': _Z(6, 3, 64)}, 'multiple of Hk'),
    ({'v': _Z(6, 1, 64)}, 'multiple of Hk'),
    ({'v': _Z(5, 2, 64)}, 'multiple of Hk'),
    ({'k': _Z(6, 0, 64), 'v': _Z(6, 0, 64)}, 'multiple of Hk'),
    ({'q': _Z(6, 4, 32), 'k': _Z(6, 2, 32), 'v': _Z(6, 2, 32)}, 'head dim 64 or 128'),
    ({'q': _Z(6, 4, 64, dt=torch.float32)}, 'bf16 or fp32'),
    ({'v': _Z(6, 2, 64, dt=torch.float32)}, 'bf16 or fp32'),
    ({n: _Z(6, h, 64, dt=torch.float16) for n, h in (('q', 4), ('k', 2), ('v', 2))}, 'bf16 or fp32'),
    ({'cu_q': torch.tensor([0.0, 6.0])}, 'offsets'),
    ({'cu_q': torch.tensor([0], dtype=torch.int32)}, 'offsets'),
    ({'cu_q': torch.tensor([[0, 6]], dtype=torch.int32)}, 'offsets'),
    ({'cu_k': torch.tensor([0, 6], dtype=torch.int32)}, 'offsets'),
    ({'k': _Z(7, 2, 64), 'v': _Z(7, 2, 64)}, 'as many keys'),
    ({'scale': 0.0}, 'scale'),
    ({'scale': -1.0}, 'scale'),
    ({'scale': math.inf}, 'scale'),
])
def test_attention_varlen_refuses(kw, match):
    from diffusion_pipe_amd.hip import DpipeHipError
    with pytest.raises(DpipeHipError, match=match):
        _varlen(**kw)


def _rope_c(**kw):
    from diffusion_pipe_amd import hip
    a = dict(q=256, k=256, pos=256, pos_type=0, freq=(ctypes.c_double * 32)(), axis=(ctypes.c_int * 32)(), wq=None, wk=None, yq=256, yk=256, tokens=6, period=6, axes=1, pairs=32, hq=2,
             hk=1, D=64, q_ss=128, q_sh=64, k_ss=64, k_sh=64, eps=1e-6, half=0, dtype=1, wq_dt=1, wk_dt=1)
    a.update(kw)
    rc = hip.lib().dpipe_rope_axes_fwd(*a.values(), None)
    return rc, hip.lib().dpipe_last_error().decode()


@pytest.mark.parametrize('kw', [{'q': None}, {'k': None}, {'pos': None}, {'pos_type': 3}, {'freq': None}, {'axis': (ctypes.c_int * 32)(*[1] * 32)}, {'axis': (ctypes.c_int * 32)(*[-1] * 32)},
                                {'tokens': 0}, {'period': 0}, {'axes': 0}, {'pairs': 0}, {'pairs': 33}, {'half': 1, 'pairs': 30}, {'hq': 0}, {'hk': -1}, {'D': 60}, {'D': 264}, {'q': 264},
                                {'q_ss': 132}, {'k_sh': 4}, {'wq': 8}, {'wq': 256, 'wq_dt': 2}, {'dtype': 2}, {'yq': None}, {'yk': None}, {'yq': 8}, {'hq': 5000}])
def test_rope_axes_c_entry_refuses(kw):
    rc, msg = _rope_c(**kw)
    assert rc < 0 and 'dpipe_rope_axes_fwd' in msg, (rc, msg)


def _varlen_c(name='fwd', **kw):
    from diffusion_pipe_amd import hip
    a = dict(q=256, k=256, v=256, cu_q=256, cu_k=256)
    if name == 'fwd':
        a.update(o=256, o_lo=256, lse=256)
    else:
        a.update(o=256, o_lo=256, do=256, lse=256, delta=256, dq=256, dk=256, dv=256)
    a.update(ws=None, floats=0, tq=6, tk=6, n=1, hq=2, hk=1, D=64, q_ss=128, q_sh=64, k_ss=64, k_sh=64, v_ss=64, v_sh=64)
    if name == 'bwd':
        a.update(do_ss=128, do_sh=64)
    a.update(scale=0.125, causal=0, dtype=0)
    a.update(kw)
    rc = getattr(hip.lib(), f'dpipe_attn_varlen_{name}')(*a.values(), None)
    return rc, hip.lib().dpipe_last_error().decode()


@pytest.mark.parametrize('name', ['fwd', 'bwd'])
@pytest.mark.parametrize('kw', [{'q': None}, {'cu_k': None}, {'tq': 0}, {'tk': -1}, {'n': 0}, {'hq': 3, 'hk': 2}, {'D': 96}, {'D': 256}, {'scale': 0.0}, {'scale': math.nan},
                                {'scale': math.inf}, {'q': 264}, {'q_ss': 132}, {'k_ss': 32}, {'v_ss': 2 ** 23}, {'k_sh': -64}, {'tq': 2 ** 31}, {'n': 2 ** 23}, {'dtype': 2}, {'tk': 2 ** 18}])
def test_attention_varlen_c_entries_refuse(name, kw):
    """(the last: few rows and long keys -- or few keys' gradients -- need the workspace, which is missing)"""
    if name == 'bwd' and kw == {'tk': 2 ** 18}:
        kw = {'tq': 2 ** 18}
    rc, msg = _varlen_c(name, **kw)
    assert rc < 0 and f'dpipe_attn_varlen_{name}' in msg, (rc, msg)


def test_workspace_is_asked_for_where_few_tiles_meet_a_long_axis():
    from diffusion_pipe_amd import hip
    fwd, bwd = hip.lib().dpipe_attn_varlen_fwd_workspace_floats, hip.lib().dpipe_attn_varlen_bwd_workspace_floats
    assert fwd(4, 20000, 2, 8, 2, 128) > 0 and bwd(20000, 77, 1, 8, 8, 128) > 0
    assert bwd(500, 7000, 2, 8, 8, 128) > 0 and bwd(500, 7000, 2, 8, 8, 128) % (500 * 8 * 128) == 0      # (dQ's parts)
    assert fwd(8000, 512, 1, 4, 4, 128) == 0 and fwd(77, 77, 1, 12, 12, 64) == 0 == bwd(77, 77, 1, 12, 12, 64)
    assert fwd(20000, 20000, 2, 24, 24, 128) == 0 and bwd(20000, 20000, 2, 24, 24, 128) == 0
    assert fwd(4, 100, 2, 8, 2, 128) == 0 and fwd(0, 5, 1, 1, 1, 64) == 0 and bwd(5, 5, 1, 3, 2, 64) == 0

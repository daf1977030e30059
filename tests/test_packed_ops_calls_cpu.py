"""CPU: calls of rope_axes and attention_varlen that are refused, or not, before anything touches a device."""
import pytest
import torch
import torch.autograd.forward_ad as fw

ROPE = {'q': (6, 4, 64), 'k': (6, 2, 64), 'positions': (6, 3), 'q_weight': (64,), 'k_weight': (64,)}
ATTENTION = {'q': (6, 4, 64), 'k': (6, 2, 64), 'v': (6, 2, 64)}


def _rope(t):
    from diffusion_pipe_amd import ops
    return ops.rope_axes(t['q'], t['k'], t['positions'], (8, 28, 28), q_weight=t['q_weight'], k_weight=t['k_weight'])


def _attention(t):
    from diffusion_pipe_amd import ops
    return ops.attention_varlen(t['q'], t['k'], t['v'], torch.tensor([0, 2, 6], dtype=torch.int32))


@pytest.mark.parametrize('call,shapes,name', [(c, s, n) for c, s in ((_rope, ROPE), (_attention, ATTENTION)) for n in s], ids=lambda x: x.strip('_') if isinstance(x, str) else '')
def test_forward_mode_tangents_are_refused(call, shapes, name):
    """a dual tensor does not require a gradient: its tangent must not vanish on the path without autograd"""
    from diffusion_pipe_amd.hip import DpipeHipError
    t = {n: torch.zeros(*s) for n, s in shapes.items()}
    with fw.dual_level():
        with pytest.raises(DpipeHipError, match='device tensors'):           # no tangent: as outside
            call(t)
        whole = fw.make_dual(torch.zeros(2, *shapes[name]), torch.ones(2, *shapes[name]))
        for dual in (fw.make_dual(t[name], torch.ones_like(t[name])), whole[1]):       # (a view of a dual tensor is one)
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(DpipeHipError, match='forward-mode'):
                    call({**t, name: dual})
    with pytest.raises(DpipeHipError, match='device tensors'):
        call(t)


def test_the_same_offsets_given_for_both_sides_allow_buffers_of_two_sizes():
    """what is allowed goes by the offsets' values, not by which object holds them: rows behind the last sequence may differ in number"""
    from diffusion_pipe_amd import ops
    from diffusion_pipe_amd.hip import DpipeHipError
    cu, (q, k) = torch.tensor([0, 2, 6], dtype=torch.int32), (torch.zeros(n, 2, 64) for n in (6, 9))
    for cu_k in (cu, cu.clone()):
        with pytest.raises(DpipeHipError, match='device tensors'):
            ops.attention_varlen(q, k, k, cu, cu_k)
    with pytest.raises(DpipeHipError, match='as many keys'):
        ops.attention_varlen(q, k, k, cu)


@pytest.mark.parametrize('n', [2, 4, 8, 16, 32, 64])
def test_an_axis_is_cut_however_many_sequences_stand_beside_the_long_one(n):
    """few rows against a long axis leave most of the card idle unless the axis is cut: neither empty sequences (offsets of a fixed capacity) nor short neighbours may talk the rule out
    of it, and equal short sequences are left whole"""
    from diffusion_pipe_amd import hip
    fwd, bwd = hip.lib().dpipe_attn_varlen_fwd_workspace_floats, hip.lib().dpipe_attn_varlen_bwd_workspace_floats
    for rows, keys, hq, hk, D in ((1, 8191, 32, 8, 128), (64, 30063, 32, 8, 128), (n, 16384 + 100 * n, 32, 8, 128), (8, 16384, 12, 12, 64)):
        assert fwd(rows, keys, n, hq, hk, D) // (rows * hq * (D + 1)) >= 4, (rows, keys)
        assert bwd(rows, keys, n, hq, hk, D) >= 4 * rows * hq * D, (rows, keys)
    for rows, keys, heads, D in ((8000, 512, 4, 128), (4096, 512, 10, 64)):
        assert bwd(rows, keys, n, heads, heads, D) >= 2 * 2 * keys * heads * D, (rows, keys)
    assert fwd(77 * n, 77 * n, n, 12, 12, 64) == 0 == bwd(77 * n, 77 * n, n, 12, 12, 64)
    assert fwd(1000 * n, 1000 * n, n, 24, 24, 128) == 0 == bwd(1000 * n, 1000 * n, n, 24, 24, 128)


@pytest.mark.parametrize('sizes', [(1, 2584, 245673, 24, 24, 128), (1, 39237, 104819, 4, 4, 128), (100, 2 ** 21, 20000, 40, 40, 128), (2 ** 21, 100, 20000, 40, 40, 128), (64, 2 ** 22, 200000, 8, 8, 64)])
def test_cutting_refuses_no_call_that_fits_whole(sizes):
    """offsets for very many sequences: the parts are as many as the grid allows, one if need be.  (o is missing, so nothing is launched)"""
    from diffusion_pipe_amd import hip
    tq, tk, n, hq, hk, D = sizes
    strides = (hq * D, D, hk * D, D, hk * D, D)
    lib = hip.lib()
    assert lib.dpipe_attn_varlen_fwd(256, 256, 256, 256, 256, None, None, None, None, 0, *sizes, *strides, 0.125, 0, hip.BF16, None) < 0
    assert 'bad output or workspace' in lib.dpipe_last_error().decode()
    assert lib.dpipe_attn_varlen_bwd(256, 256, 256, 256, 256, None, None, 256, 256, 256, 256, 256, 256, None, 0, *sizes, *strides, hq * D, D, 0.125, 0, hip.BF16, None) < 0
    assert 'bad gradient or workspace' in lib.dpipe_last_error().decode()


def test_rope_axes_c_entry_refuses_an_axis_that_it_cannot_hold():
    """the launch keeps an axis in 8 bits: a position column from the 257th on is refused, not taken for another"""
    import ctypes
    from diffusion_pipe_amd import hip
    a = dict(q=256, k=None, pos=256, pos_type=0, freq=(ctypes.c_double * 32)(), axis=(ctypes.c_int * 32)(*[256] * 32), wq=None, wk=None, yq=None, yk=None, tokens=6, period=6, axes=400, pairs=32,
             hq=2, hk=0, D=64, q_ss=128, q_sh=64, k_ss=0, k_sh=0, eps=1e-6, half=0, dtype=1, wq_dt=1, wk_dt=1)
    for column, message in ((256, 'axis index'), (255, 'bad output')):        # (no output is given, so nothing is launched)
        a['axis'] = (ctypes.c_int * 32)(*[column] * 32)
        assert hip.lib().dpipe_rope_axes_fwd(*a.values(), None) < 0 and message in hip.lib().dpipe_last_error().decode(), column

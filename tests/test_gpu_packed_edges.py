"""ops.attention_varlen and ops.rope_axes at their edges: rows that see no key and hold NaN, short sequences beside long ones, axes that are cut where a sequence has several row tiles,
rows behind the last sequence where an axis is cut, and every buffer between guards.  Bounds: those of test_gpu_attention_varlen, element by element."""
import math

import pytest
import torch

import test_gpu_attention_varlen as av

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
NAN = float('nan')


# ------------------------------------------------------------------------------------------------ rows that see no key
@BOTH
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('case', [([257, 200, 33, 130], [40, 77, 512, 0], 4, 2), ([1, 300], [9001, 70], 4, 1), ([3000, 65], [77, 64], 4, 4)], ids=['ragged', 'long_keys', 'many_queries'])
def test_rows_that_see_no_key_neither_take_nor_give(gpu, case, D, dtype):
    """causal with more queries than keys: the first queries see nothing.  Whatever they and their gradients hold, they get zeros and leave every other output and gradient bit for bit"""
    lens_q, lens_k, H, Hk = case
    q, k, v, do, cu_q, cu_k = av._inputs(gpu, lens_q, lens_k, H, Hk, D, dtype=dtype)
    clean = av._run(q, k, v, do, cu_q, cu_k, True)
    av._check(clean, av._exact(q, k, v, do, lens_q, lens_k, True, 1.0 / math.sqrt(D)), f'{case} D={D}', dtype)
    blind = torch.cat([torch.arange(n, device=gpu) < n - m for n, m in zip(lens_q, lens_k)])
    assert blind.any() and not blind.all()
    q[blind], do[blind] = NAN, float('inf')
    for _ in range(2):
        got = av._run(q, k, v, do, cu_q, cu_k, True)
        for n in got:
            assert torch.equal(got[n], clean[n]), n
        assert (got['o'][blind] == 0).all() and (got['dq'][blind] == 0).all()
        q[blind], do[blind] = -float('inf'), NAN


@BOTH
@pytest.mark.parametrize('lens_k', [[70], [5000]], ids=['whole', 'cut'])
def test_rows_that_see_no_key_are_zero_beside_keys_that_are_not_finite(gpu, lens_k, dtype):
    """the same rows where the keys and values that others see are NaN: still zeros"""
    lens_q = [lens_k[0] + 20]
    q, k, v, do, cu_q, cu_k = av._inputs(gpu, lens_q, lens_k, 2, 1, 128, dtype=dtype)
    k[:], v[:] = NAN, NAN
    got = av._run(q, k, v, do, cu_q, cu_k, True)
    assert (got['o'][:20] == 0).all() and (got['dq'][:20] == 0).all() and got['o'][20:].isnan().all()


# ------------------------------------------------------------------------------------------------ short sequences in any company
SHORT = [1, 2, 1, 9, 5, 64, 1, 12, 40, 2]


@pytest.mark.parametrize('H,Hk,D', [(4, 2, 128), (4, 2, 64), (2, 2, 128)])
@pytest.mark.parametrize('company', ['tail', 'long', 'cross'])
def test_short_sequences_are_rounded_once_in_any_company(gpu, company, H, Hk, D, monkeypatch):
    """a sequence of one tile of queries and keys (64) is rounded once (h for its results, h^2 for P and dS: see test_sequences_of_one_tile_are_rounded_once), whatever rows lie behind
    the last sequence and however long its neighbours are"""
    lens_q = SHORT + ([3000] if company == 'long' else [1500, 70] if company == 'cross' else [])
    lens_k = SHORT + ([3000] if company == 'long' else [70, 900] if company == 'cross' else [])
    tail = 4096 if company == 'tail' else 0
    q, k, v, do, cu_q, cu_k = av._inputs(gpu, lens_q, lens_k, H, Hk, D, tail_q=tail, tail_k=tail)
    got = av._run(q, k, v, do, cu_q, cu_k, True)
    n, scale = sum(SHORT), 1.0 / math.sqrt(D)
    rows = [t[:n] for t in (q, k, v, do)]
    av._check({x: t[:n] for x, t in got.items()}, av._exact(*rows, SHORT, SHORT, True, scale), company)
    h = av.H_BF16
    monkeypatch.setattr(av, 'H_BF16', 2.0 ** -16)
    once = av._exact(*rows, SHORT, SHORT, True, scale)
    for x, t in got.items():
        value, bound = once[x]
        worst = ((t[:n].detach().double() - value).abs() / (bound + h * (value.abs() + bound))).max().item()
        print(f'{company} {x}: worst error / bound {worst:.3f}')
        assert worst <= 1.0, x


# ------------------------------------------------------------------------------------------------ cut axes
@BOTH
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('case', [([300, 200], [4000, 3000], 8, 8), ([129, 70, 1], [2500, 70, 3000], 8, 2), ([4096], [4096], 4, 4)], ids=['two_sequences', 'grouped', 'one_sequence'])
def test_cut_axes_with_several_row_tiles(gpu, case, D, dtype):
    """several tiles of rows and several parts of the keys at once, forward and dQ; causal: parts that begin behind everything a tile sees"""
    from diffusion_pipe_amd import hip
    lens_q, lens_k, H, Hk = case
    data = av._inputs(gpu, lens_q, lens_k, H, Hk, D, dtype=dtype)
    sizes = (sum(lens_q), sum(lens_k), len(lens_q), H, Hk, D)
    assert hip.lib().dpipe_attn_varlen_fwd_workspace_floats(*sizes) > 0 and hip.lib().dpipe_attn_varlen_bwd_workspace_floats(*sizes) >= 2 * sum(lens_q) * H * D
    for causal in (False, True):
        first = av._run(*data, causal)
        av._check(first, av._exact(*data[:4], lens_q, lens_k, causal, 1.0 / math.sqrt(D)), f'{case} D={D} causal={causal}', dtype)
        again = av._run(*data, causal)
        assert all(torch.equal(first[n], again[n]) for n in first)


@BOTH
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('case', [([1, 3] + [0] * 30, [9001, 500] + [0] * 30, 16, 4), ([2] + [1] * 39, [16001] + [50, 0, 130] * 13, 8, 2), ([5000] + [10, 0, 1] * 13, [200] + [0, 70, 3] * 13, 4, 4)],
                         ids=['empty', 'short', 'long_queries'])
def test_a_long_sequence_among_empty_and_short_ones(gpu, case, D, dtype):
    """the axis is cut for the long one; the parts that the others do not need leave nothing behind"""
    from diffusion_pipe_amd import hip
    lens_q, lens_k, H, Hk = case
    data = av._inputs(gpu, lens_q, lens_k, H, Hk, D, dtype=dtype)
    sizes = (sum(lens_q), sum(lens_k), len(lens_q), H, Hk, D)
    assert hip.lib().dpipe_attn_varlen_bwd_workspace_floats(*sizes) > 0 and (lens_q[0] > 100 or hip.lib().dpipe_attn_varlen_fwd_workspace_floats(*sizes) > 0)
    for causal in (False, True):
        av._check(av._run(*data, causal), av._exact(*data[:4], lens_q, lens_k, causal, 1.0 / math.sqrt(D)), f'{case} D={D} causal={causal}', dtype)


@BOTH
@pytest.mark.parametrize('case', [([1, 3, 2], [9001, 4096, 63], 16, 4, 128), ([3000, 1500], [77, 20], 4, 4, 64), ([300, 200], [4000, 3000], 8, 8, 128)],
                         ids=['few_rows', 'few_keys', 'several_row_tiles'])
def test_rows_behind_the_last_sequence_where_axes_are_cut(gpu, case, dtype):
    lens_q, lens_k, H, Hk, D = case
    q, k, v, do, cu_q, cu_k = av._inputs(gpu, lens_q, lens_k, H, Hk, D, tail_q=150, tail_k=300, dtype=dtype)
    nq, nk = sum(lens_q), sum(lens_k)
    for t, n in ((q, nq), (do, nq), (k, nk), (v, nk)):
        t[n:] = NAN
    for causal in (False, True):
        got = av._run(q, k, v, do, cu_q, cu_k, causal)
        for name, t in got.items():
            assert (t[(nq if name in ('o', 'dq') else nk):] == 0).all(), name
        want = av._exact(q[:nq], k[:nk], v[:nk], do[:nq], lens_q, lens_k, causal, 1.0 / math.sqrt(D))
        av._check({n: t[:(nq if n in ('o', 'dq') else nk)] for n, t in got.items()}, want, f'{case} causal={causal}', dtype)


# ------------------------------------------------------------------------------------------------ guards
GUARD, MARK = 40, 2.0 ** 100            # rows (floats: 64 of them) on either side; a value that no result takes


class _Guarded:
    """an operand inside a larger buffer: NaN around what is read, a mark around (and in) what is written"""

    def __init__(self, shape, dtype, device, data=None):
        rows, rest = shape[0], tuple(shape[1:])
        self.guard = GUARD if rest else 64
        self.read = data is not None
        self.whole = torch.full((rows + 2 * self.guard, *rest), NAN if self.read else MARK, dtype=dtype, device=device)
        self.t = self.whole[self.guard:self.guard + rows]
        if self.read:
            self.t.copy_(data)
        assert self.t.data_ptr() % 16 == 0

    def ptr(self):
        return self.t.data_ptr()

    def check(self, name):
        outside = torch.cat([self.whole[:self.guard].flatten(), self.whole[self.guard + self.t.shape[0]:].flatten()])
        assert (outside.isnan() if self.read else outside == MARK).all(), f'{name}: written outside'
        assert self.t.isfinite().all(), f'{name}: what lies outside an operand was read'


PLANS = [  # (query rows, key rows, query offsets, key offsets, H, Hk)
    (200, 200, [0, 100, 200], None, 2, 2),
    (290, 290, [0, 70, 200], None, 4, 2),
    (200, 200, [0, 150, 100], None, 2, 1),                 # (from here on offsets that do not ascend from 0 to the end)
    (200, 200, [0, -5, 900], None, 2, 2),
    (200, 200, [0, 2000000000, -2000000000], None, 2, 2),
    (200, 200, [50, 20, 200], None, 4, 1),
    (200, 330, [0, 150, 100], [0, 400, 90], 2, 2),
    (300, 300, [0] + [250, 3, -7, 300, 310, 120] * 8, None, 2, 1),
    (7, 9100, [0, 1, 4], [0, 9001, 9050], 16, 4),          # cut keys
    (7, 9100, [0, 9, 4], [0, 9001, 50], 16, 4),
    (500, 7000, [0, 300, 500], [0, 4000, 7000], 8, 8),
    (500, 7000, [0, 300, 200], [0, 8000, -1], 8, 8),
    (4600, 97, [0, 3000, 4500], [0, 77, 97], 4, 4),        # cut queries
    (4600, 97, [0, 3000, 100], [0, 100, -3], 4, 4),
]


@BOTH
@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('plan', PLANS, ids=lambda p: f'{p[0]}x{p[1]}_{"_".join(map(str, p[2][:4]))}')
def test_attention_stays_inside_its_buffers(gpu, plan, D, dtype):
    """the C entries on operands, outputs and workspaces with guards on both sides, also where the offsets are wrong (their rows' values are then unspecified, their places are not)"""
    from diffusion_pipe_amd import hip
    tq, tk, cu_q, cu_k, H, Hk = plan
    g = torch.Generator().manual_seed(tq + tk)
    f32, lib = torch.float32, hip.lib()
    make = lambda *s: _Guarded(s, dtype, gpu, torch.randn(*s, generator=g))
    out = lambda *s, dt=dtype: _Guarded(s, dt, gpu)
    cu_q, cu_k = (torch.tensor([0] * 8 + cu + [0] * 8, dtype=torch.int32, device=gpu)[8:8 + len(cu)] for cu in (cu_q, cu_k or cu_q))
    sizes = (tq, tk, cu_q.shape[0] - 1, H, Hk, D)
    b = {'q': make(tq, H, D), 'k': make(tk, Hk, D), 'v': make(tk, Hk, D), 'do': make(tq, H, D), 'o': out(tq, H, D), 'o_lo': out(tq, H, D), 'lse': out(H * tq, dt=f32),
         'delta': out(H * tq, dt=f32), 'dq': out(tq, H, D), 'dk': out(tk, Hk, D), 'dv': out(tk, Hk, D)}
    need = lib.dpipe_attn_varlen_fwd_workspace_floats(*sizes), lib.dpipe_attn_varlen_bwd_workspace_floats(*sizes)
    ws = [out(max(x, 4), dt=f32) for x in need]
    p = {x: t.ptr() for x, t in b.items()}
    strides = (H * D, D, Hk * D, D, Hk * D, D)
    for causal in (0, 1):
        for x in b.values():
            if not x.read:
                x.t.fill_(MARK)
        code = hip.BF16 if dtype == torch.bfloat16 else hip.F32
        hip.check(lib.dpipe_attn_varlen_fwd(p['q'], p['k'], p['v'], cu_q.data_ptr(), cu_k.data_ptr(), p['o'], p['o_lo'], p['lse'], ws[0].ptr(), need[0], *sizes, *strides,
                                            1.0 / math.sqrt(D), causal, code, hip.stream()), 'fwd')
        hip.check(lib.dpipe_attn_varlen_bwd(p['q'], p['k'], p['v'], cu_q.data_ptr(), cu_k.data_ptr(), p['o'], p['o_lo'], p['do'], p['lse'], p['delta'], p['dq'], p['dk'], p['dv'],
                                            ws[1].ptr(), need[1], *sizes, *strides, H * D, D, 1.0 / math.sqrt(D), causal, code, hip.stream()), 'bwd')
        torch.cuda.synchronize()
        for name, x in b.items():
            if name != 'lse':
                x.check(name)
        assert not b['lse'].t.isnan().any()
        b['lse'].t.fill_(0.0)                              # (+inf for a row that sees nothing)
        b['lse'].check('lse')
        for i, x in enumerate(ws):
            x.t.fill_(0.0)
            x.check(f'workspace {i}')


@BOTH
@pytest.mark.parametrize('tokens,H,Hk,D,axes', [(1, 1, 1, 64, (8, 28, 28)), (133, 5, 2, 128, (16, 56, 56)), (37, 3, 0, 80, (16, 24, 24)), (2100, 4, 1, 256, (64,))])
def test_rotary_positions_stay_inside_their_buffers(gpu, tokens, H, Hk, D, axes, dtype):
    from diffusion_pipe_amd import hip, ops
    g = torch.Generator().manual_seed(tokens)
    f32, lib = torch.float32, hip.lib()
    make = lambda *s, dt=dtype: _Guarded(s, dt, gpu, torch.randn(*s, generator=g))
    hk = max(Hk, 1)
    b = {'q': make(tokens, H, D), 'k': make(tokens, hk, D), 'gq': make(tokens, H, D), 'gk': make(tokens, hk, D), 'pos': make(tokens, len(axes), dt=f32), 'wq': make(D), 'wk': make(D),
         'yq': _Guarded((tokens, H, D), dtype, gpu), 'yk': _Guarded((tokens, hk, D), dtype, gpu), 'dq': _Guarded((tokens, H, D), dtype, gpu), 'dk': _Guarded((tokens, hk, D), dtype, gpu),
         'dwq': _Guarded((D,), dtype, gpu), 'dwk': _Guarded((D,), dtype, gpu), 'ws': _Guarded((lib.dpipe_rope_axes_workspace_floats(D),), f32, gpu)}
    p = {n: x.ptr() for n, x in b.items()}
    if not Hk:
        p.update(k=None, gk=None, yk=None, dk=None, dwk=None, wk=None)
    code = hip.BF16 if dtype == torch.bfloat16 else hip.F32
    for half in (0, 1):
        freq, axis, pairs = ops._rope_axes_tables(axes, 10000.0, False, D, half == 0)
        for normed in (True, False):
            wq, wk = (p['wq'], p['wk']) if normed else (None, None)
            meta, strides = (tokens, tokens, len(axes), pairs, H, Hk, D), (H * D, D, Hk * D, D)
            hip.check(lib.dpipe_rope_axes_fwd(p['q'], p['k'], p['pos'], 0, freq, axis, wq, wk, p['yq'], p['yk'], *meta, *strides, 1e-6, half, code, code, code, hip.stream()), 'fwd')
            hip.check(lib.dpipe_rope_axes_bwd(p['q'], p['k'], p['gq'], p['gk'], p['pos'], 0, freq, axis, wq, wk, p['dq'], p['dk'], p['dwq'] if normed else None,
                                              p['dwk'] if normed else None, p['ws'], *meta, *strides, *strides, 1e-6, half, code, code, code, 0, 0, hip.stream()), 'bwd')
            torch.cuda.synchronize()
            for name, x in b.items():
                x.check(name)


# ------------------------------------------------------------------------------------------------ derivatives of derivatives
def test_a_graph_of_the_gradient_is_refused(gpu):
    """a gradient of a gradient has no formula here: the term must not vanish from a sum whose other terms have one"""
    from diffusion_pipe_amd import ops
    from diffusion_pipe_amd.hip import DpipeHipError
    q, k, v, do, cu, _ = av._inputs(gpu, [40, 30], [40, 30], 2, 1, 64)
    q.requires_grad_(True)
    pos = torch.arange(70, device=gpu).unsqueeze(-1)
    for y in (ops.attention_varlen(q, k, v, cu), ops.attention_varlen(q, k[:0], v[:0], cu, torch.zeros_like(cu)), ops.rope_axes(q, None, pos, (64,))[0],
              ops.rope_axes(q, k, pos, (64,), q_weight=torch.ones(64, device=gpu))[0]):
        with pytest.raises(DpipeHipError, match='differentiable once'):
            dq, = torch.autograd.grad(y, q, do, create_graph=True)
            torch.autograd.grad(q.sum() + dq.square().sum(), q)
        assert torch.autograd.grad(y, q, do, retain_graph=True)[0].isfinite().all()


# ------------------------------------------------------------------------------------------------ layouts
@BOTH
def test_any_layout_gives_the_bits_of_the_contiguous_one(gpu, dtype):
    """heads before tokens, heads interleaved with other tensors, one head, one token, a gradient in either order, rows that overlap a wider buffer"""
    from diffusion_pipe_amd import ops
    lens, H, Hk, D = [70, 1, 59], 4, 2, 64
    q, k, v, do, cu, _ = av._inputs(gpu, lens, lens, H, Hk, D, dtype=dtype)
    base = av._run(q, k, v, do, cu, None, True)
    heads_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    interleaved = lambda t: torch.stack([t, t + 1, t - 1], dim=2)[:, :, 0]
    wide = lambda t: torch.cat([t.flatten(1), t.flatten(1)[:, :8]], dim=1)[:, :t.shape[1] * D].unflatten(1, (t.shape[1], D))
    for layout in (heads_first, interleaved, wide):
        got = av._run(*(layout(t) for t in (q, k, v, do)), cu, None, True)
        assert all(torch.equal(got[n], base[n]) for n in base)
        pos = torch.arange(130, device=gpu).unsqueeze(-1) % 70
        w = torch.linspace(0.5, 1.5, D, device=gpu)
        for weight in (w, None):
            want = ops.rope_axes(q, k, pos, (48,), q_weight=weight, k_weight=weight)
            got = ops.rope_axes(layout(q), layout(k), pos, (48,), q_weight=weight, k_weight=weight)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            batch = lambda t: torch.stack([t[:65], t[65:]])                  # [2, 65, H, D], heads first inside a sample
            got = ops.rope_axes(batch(q).transpose(1, 2).contiguous().transpose(1, 2), batch(k), pos.view(2, 65, 1), (48,), q_weight=weight, k_weight=weight)
            assert all(torch.equal(a.flatten(0, 1), b) for a, b in zip(got, want))
    one = av._run(q[:, :1], k[:, :1], v[:, :1], do[:, :1], cu, None, True)
    same = av._run(*(t[:, :1].contiguous() for t in (q, k, v, do)), cu, None, True)
    assert all(torch.equal(one[n], same[n]) for n in one)
    cu1 = torch.tensor([0, 1], dtype=torch.int32, device=gpu)
    one = av._run(*(heads_first(t)[5:6] for t in (q, k, v, do)), cu1, None, False)
    same = av._run(*(t[5:6].contiguous() for t in (q, k, v, do)), cu1, None, False)
    assert all(torch.equal(one[n], same[n]) for n in one)

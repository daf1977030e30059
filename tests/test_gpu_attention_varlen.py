"""ops.attention_varlen against softmax attention in 64 bits, sequence by sequence.

Bounds, element by element, from the roundings the kernels make (h = 2^-8: half a step of bf16; everything else is fp32):
    o   = sum_j P_j v_j        P rounded to bf16, o rounded:                     h sum P |v| + h |o|
    dV  = P^T dO               likewise:                                          h P^T |dO| + h |dV|
    dS  = P (dP - delta)       rounded, dP and delta fp32 sums of D terms:        h |dS| + g P (|dO| |V|^T + rowsum |dO| |O|)
                               delta = rowsum dO O of the O the forward formed,
                               each term off by |dO| times o's first bound above:  + P rowsum |dO| (h + r) sum P |V|                    =: E
    dQ  = scale dS K           dS as above, result rounded:                       scale E |K| + h |dQ|;      dK: scale E^T |Q| + h |dK|
fp32 parts: a sum of D <= 128 products is off by at most 2^7 2^-24 of its terms' absolute sum (g = 2^-16 with room for both sums); a score's error moves P by
|error| relatively: |scale q . k| 2^-16 <= 2^-10 for the |scores| <= 64 of these inputs, and sums over keys add 2^-24 a term: P itself carries r = 2^-10 relatively.
In fp32 (h = 2^-24, nothing rounded but results) r is taken row by row: a row's scores are off by 2^-16 of scale |q| . |k| at most, P and its normalizer each by the largest of
these, and every sum over n queries of g heads or m keys adds 2^-24 a term, the exponential and the joins less than 2^7 2^-24:  r = 2^-15 max_j scale |q| . |k_j| + (g n + m + 2^7) 2^-24."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H_BF16, G_DOT, R_P = 2.0 ** -8, 2.0 ** -16, 2.0 ** -10


def _inputs(gpu, lens_q, lens_k, H, Hk, D, seed=0, tail_q=0, tail_k=0, spread=1.0, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed + 31 * sum(lens_q) + sum(lens_k) + H)
    tq, tk = sum(lens_q) + tail_q, sum(lens_k) + tail_k
    q, k, v, do = (torch.randn(n, h, D, generator=g) for n, h in ((tq, H), (tk, Hk), (tk, Hk), (tq, H)))
    q, k, v, do = ((t * s).to(gpu, dtype) for t, s in ((q, spread), (k, spread), (v + 0.5, 1.0), (do, 1.0)))
    cu = [torch.tensor([0] + [sum(lens[:i + 1]) for i in range(len(lens))], dtype=torch.int32, device=gpu) for lens in (lens_q, lens_k)]
    return q, k, v, do, cu[0], cu[1]


def _exact(q, k, v, do, lens_q, lens_k, causal, scale):
    """{name: (value, bound)} in fp64"""
    fp32 = q.dtype == torch.float32
    u = 2.0 ** -24 if fp32 else H_BF16
    q, k, v, do = (t.detach().double() for t in (q, k, v, do))
    H, Hk = q.shape[1], k.shape[1]
    val = {n: torch.zeros_like(t) for n, t in (('o', q), ('dq', q), ('dk', k), ('dv', v))}
    err = {n: torch.zeros_like(t) for n, t in val.items()}
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        for h in range(H):
            kh = h // (H // Hk)
            Q, K, V, G = q[a:a + n, h], k[b:b + m, kh], v[b:b + m, kh], do[a:a + n, h]
            S = (Q @ K.t()) * scale
            if causal:
                i, j = torch.arange(n, device=q.device)[:, None], torch.arange(m, device=q.device)[None, :]
                S = S.masked_fill(j - m > i - n, -math.inf)
            P = torch.nan_to_num(torch.softmax(S, dim=-1), nan=0.0) if m else S
            O = P @ V
            dP, delta = G @ V.t(), (G * O).sum(-1, keepdim=True)
            dS = P * (dP - delta)
            r = R_P
            if fp32:
                r = 2.0 ** -24 * (H // Hk * n + m + 128) + (2.0 ** -15 * scale * (Q.abs() @ K.abs().t()).amax(-1, keepdim=True) if m else 0.0)
            E = (u + r) * dS.abs() + G_DOT * P * (G.abs() @ V.abs().t() + (G.abs() * O.abs()).sum(-1, keepdim=True))
            E = E + P * (G.abs() * ((u + r) * (P @ V.abs()))).sum(-1, keepdim=True)
            val['o'][a:a + n, h], err['o'][a:a + n, h] = O, (u + r) * (P @ V.abs())
            val['dq'][a:a + n, h], err['dq'][a:a + n, h] = scale * dS @ K, scale * E @ K.abs()
            val['dk'][b:b + m, kh] += scale * dS.t() @ Q
            err['dk'][b:b + m, kh] += scale * E.t() @ Q.abs()
            val['dv'][b:b + m, kh] += P.t() @ G
            err['dv'][b:b + m, kh] += ((u + r) * P).t() @ G.abs()
        a, b = a + n, b + m
    return {n: (val[n], err[n] + u * (val[n].abs() + err[n]) + 1e-30) for n in val}


def _check(got, want, label, dtype=torch.bfloat16):
    for name, t in got.items():
        value, bound = want[name]
        assert t.shape == value.shape and t.dtype == dtype
        ratio = ((t.detach().double() - value).abs() / bound).max().item() if t.numel() else 0.0
        print(f'{label} {name}: worst error / bound {ratio:.3f}')
        assert ratio <= 1.0, (label, name, ratio)          # (a NaN fails too)


def _run(q, k, v, do, cu_q, cu_k, causal, scale=None):
    from diffusion_pipe_amd import ops
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    o = ops.attention_varlen(q, k, v, cu_q, cu_k, scale=scale, causal=causal)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    return {'o': o, 'dq': dq, 'dk': dk, 'dv': dv}


CASES = [  # (queries, keys (None: the same), H, Hk, causal)
    ([1], None, 1, 1, False),
    ([1], None, 4, 2, True),
    ([64, 1, 63, 65], None, 2, 2, True),
    ([300], None, 3, 3, False),
    ([5, 0, 129, 31, 0], None, 4, 2, True),
    ([5, 0, 129, 31, 0], None, 4, 4, False),
    ([257, 200, 33], [40, 77, 512], 4, 4, False),
    ([257, 200, 33], [40, 77, 512], 6, 2, True),          # causal with fewer keys than queries: rows that see nothing
    ([100, 7], [0, 50], 2, 1, False),                      # a sequence without keys
    ([0, 70], [33, 64], 2, 1, True),                       # a sequence without queries
    ([1, 1, 2, 1], [700, 64, 65, 1], 8, 1, True),          # single tokens, eight heads to a key head
    ([130] * 70, None, 2, 1, True),                        # more sequences than a wave has lanes
    ([5, 70, 1, 128, 33, 64, 65, 2] * 5, None, 6, 2, True),      # more sequences than are ordered by length
    ([129, 1, 64] * 11 , [7, 300, 65] * 11, 2, 2, False),
    ([1000, 600], None, 24, 24, False),                    # 8-wave tiles
    ([900, 1100], None, 32, 8, True),
]


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{"_".join(map(str, c[0][:5]))}x{len(c[0])}_{c[2]}h{c[3]}{"_causal" if c[4] else ""}{"_cross" if c[1] else ""}')
def test_forward_and_gradients(gpu, case, D):
    lens_q, lens_k, H, Hk, causal = case
    data = _inputs(gpu, lens_q, lens_k or lens_q, H, Hk, D)
    got = _run(*data[:5], data[5] if lens_k else None, causal)
    _check(got, _exact(*data[:4], lens_q, lens_k or lens_q, causal, 1.0 / math.sqrt(D)), f'{case} D={D}')


@pytest.mark.parametrize('D', [64, 128])
@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{"_".join(map(str, c[0][:5]))}x{len(c[0])}_{c[2]}h{c[3]}{"_causal" if c[4] else ""}{"_cross" if c[1] else ""}')
def test_fp32_forward_and_gradients(gpu, case, D):
    lens_q, lens_k, H, Hk, causal = case
    data = _inputs(gpu, lens_q, lens_k or lens_q, H, Hk, D, dtype=torch.float32)
    got = _run(*data[:5], data[5] if lens_k else None, causal)
    _check(got, _exact(*data[:4], lens_q, lens_k or lens_q, causal, 1.0 / math.sqrt(D)), f'fp32 {case} D={D}', torch.float32)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('D', [64, 128])
def test_few_rows_against_long_keys(gpu, D, dtype):
    """the key range is split over workgroups and joined, in the forward and in dQ; some sequences are shorter than the parts"""
    lens_q, lens_k = [1, 3, 1, 1], [9001, 4096, 63, 1]
    data = _inputs(gpu, lens_q, lens_k, 16, 4, D, dtype=dtype)
    from diffusion_pipe_amd import hip
    assert hip.lib().dpipe_attn_varlen_fwd_workspace_floats(data[0].shape[0], data[1].shape[0], 4, 16, 4, D) > 0
    assert hip.lib().dpipe_attn_varlen_bwd_workspace_floats(data[0].shape[0], data[1].shape[0], 4, 16, 4, D) > 0
    for causal in (True, False):
        _check(_run(*data, causal), _exact(*data[:4], lens_q, lens_k, causal, 1.0 / math.sqrt(D)), f'few rows D={D} causal={causal}', dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_single_tokens_against_very_long_keys(gpu, dtype):
    """parts enough for three workgroups on a CU: tiles of 32 keys at head size 128 in bf16; a sequence that ends inside the first tile, one of no keys at all"""
    lens_q, lens_k, H, Hk, D = [2, 1, 3, 1], [40001, 37, 30015, 0], 32, 8, 128
    data = _inputs(gpu, lens_q, lens_k, H, Hk, D, dtype=dtype)
    from diffusion_pipe_amd import hip
    floats = hip.lib().dpipe_attn_varlen_fwd_workspace_floats(7, sum(lens_k), 4, H, Hk, D)
    assert floats // (7 * H * (D + 1)) * 4 * Hk >= 512
    for causal in (True, False):
        _check(_run(*data, causal), _exact(*data[:4], lens_q, lens_k, causal, 1.0 / math.sqrt(D)), f'very long keys causal={causal}', dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
@pytest.mark.parametrize('D', [64, 128])
def test_few_keys_against_many_queries(gpu, D, dtype):
    """the query range of dK / dV is split over workgroups and summed in order"""
    lens_q, lens_k = [3000, 1500], [77, 20]
    data = _inputs(gpu, lens_q, lens_k, 4, 4, D, dtype=dtype)
    from diffusion_pipe_amd import hip
    assert hip.lib().dpipe_attn_varlen_bwd_workspace_floats(data[0].shape[0], data[1].shape[0], 2, 4, 4, D) > 0
    _check(_run(*data, False), _exact(*data[:4], lens_q, lens_k, False, 1.0 / math.sqrt(D)), f'few keys D={D}', dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_rows_behind_the_last_sequence(gpu, dtype):
    """a buffer of fixed size: what lies behind the last sequence (NaN here) is not read into anything; its outputs and gradients are zero"""
    lens = [70, 130]
    q, k, v, do, cu, _ = _inputs(gpu, lens, lens, 4, 2, 128, tail_q=90, tail_k=90, dtype=dtype)
    for t in (q, k, v, do):
        t[200:] = float('nan')
    for causal in (False, True):
        got = _run(q, k, v, do, cu, None, causal)
        for t in got.values():
            assert (t[200:] == 0).all()
        want = _exact(q[:200], k[:200], v[:200], do[:200], lens, lens, causal, 1.0 / math.sqrt(128))
        _check({n: t[:200] for n, t in got.items()}, want, f'tail causal={causal}', dtype)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_neighbouring_sequences_do_not_leak(gpu, dtype):
    """infinities and NaN in one sequence leave the others' outputs and gradients bit for bit as they were"""
    lens = [40, 65, 50]
    q, k, v, do, cu, _ = _inputs(gpu, lens, lens, 2, 1, 64, dtype=dtype)
    clean = _run(q, k, v, do, cu, None, True)
    for t, x in zip((q, k, v, do), (float('nan'), float('inf'), -float('inf'), float('nan'))):
        t[40:105] = x
    dirty = _run(q, k, v, do, cu, None, True)
    for n in clean:
        assert torch.equal(clean[n][:40], dirty[n][:40]) and torch.equal(clean[n][105:], dirty[n][105:]), n


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_large_scores(gpu, dtype):
    """scores whose exponentials span the whole range of fp32: the running maximum moves far and often.  A score error moves P relatively by |score| 2^-16: the bound's r grows with it."""
    lens = [200, 90]
    q, k, v, do, cu, _ = _inputs(gpu, lens, lens, 2, 2, 64, spread=6.0, dtype=dtype)
    from diffusion_pipe_amd import ops
    o = ops.attention_varlen(q, k, v, cu, causal=True)
    value, bound = _exact(q, k, v, do, lens, lens, True, 0.125)['o']
    top = (q.double().norm(dim=-1).max() * k.double().norm(dim=-1).max() * 0.125).item() * 2.0 ** -16
    assert ((o.double() - value).abs() <= bound + 2 * top * v.double().abs().max()).all()


def test_strided_operands_and_broadcast_heads(gpu):
    """column blocks of a fused projection are read in place; a key head expanded over heads gets its heads' summed gradient; a misaligned view and an expanded gradient are copied"""
    from diffusion_pipe_amd import ops
    lens, H, Hk, D = [100, 33], 4, 2, 64
    q, k, v, do, cu, _ = _inputs(gpu, lens, lens, H, Hk, D)
    base = _run(q, k, v, do, cu, None, True)
    qkv = torch.cat([q, k, v], dim=1).requires_grad_(True)
    o = ops.attention_varlen(qkv[:, :H], qkv[:, H:H + Hk], qkv[:, H + Hk:], cu, causal=True)
    assert torch.equal(o, base['o'])
    g, = torch.autograd.grad(o, qkv, do)
    assert torch.equal(g, torch.cat([base['dq'], base['dk'], base['dv']], dim=1))
    odd = torch.empty(q.numel() + 3, device=gpu, dtype=q.dtype)[3:].view(q.shape).copy_(q)
    assert odd.data_ptr() % 16 and torch.equal(ops.attention_varlen(odd, k, v, cu, causal=True), base['o'])
    one_k, one_v = (t[:, :1].contiguous().requires_grad_(True) for t in (k, v))
    o = ops.attention_varlen(q, one_k.expand(-1, H, -1), one_v.expand(-1, H, -1), cu, causal=True)
    want = _run(q, one_k, one_v, do, cu, None, True)
    assert torch.equal(o, want['o'])
    dk, dv = torch.autograd.grad(o, (one_k, one_v), do)
    exact = _exact(q, one_k, one_v, do, lens, lens, True, 0.125)
    for got, name in ((dk, 'dk'), (dv, 'dv')):           # each head's gradient is rounded once more before the heads' sum is
        value, bound = exact[name]
        slack = H_BF16 * sum(_exact(q[:, h:h + 1], one_k, one_v, do[:, h:h + 1], lens, lens, True, 0.125)[name][0].abs() for h in range(H)) * (H + 1)
        assert ((got.double() - value).abs() <= bound + slack).all(), name
    lone = q.detach().requires_grad_(True)
    ops.attention_varlen(lone, k, v, cu, causal=True).sum().backward()          # (an expanded gradient)
    assert torch.equal(lone.grad, _run(q, k, v, torch.ones_like(do), cu, None, True)['dq'])


def test_gradients_against_differences(gpu):
    """the directional derivative of sum(o * do) by central differences in fp64"""
    lens_q, lens_k, H, Hk, D = [33, 70], [90, 65], 4, 2, 64
    q, k, v, do, cu_q, cu_k = _inputs(gpu, lens_q, lens_k, H, Hk, D)
    got = _run(q, k, v, do, cu_q, cu_k, True)
    exact = _exact(q, k, v, do, lens_q, lens_k, True, 0.125)
    g = torch.Generator().manual_seed(5)
    for i, name in enumerate(('dq', 'dk', 'dv')):
        d = torch.randn(got[name].shape, generator=g, dtype=torch.float64).to(gpu)
        def loss(step):
            args = [q.double(), k.double(), v.double()]
            args[i] = args[i] + step * d
            return (_exact(*args, do, lens_q, lens_k, True, 0.125)['o'][0] * do.double()).sum().item()
        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        bound = (exact[name][1] * d.abs()).sum().item()
        assert abs((got[name].double() * d).sum().item() - slope) <= bound + 1e-5 * abs(slope)


def test_same_bits_every_time_and_no_gradient_wanted(gpu):
    from diffusion_pipe_amd import ops
    lens_q, lens_k = [3000, 1500], [77, 20]
    data = _inputs(gpu, lens_q, lens_k, 4, 2, 128)
    a, b = _run(*data, False), _run(*data, False)
    assert all(torch.equal(a[n], b[n]) for n in a)
    with torch.no_grad():
        assert torch.equal(ops.attention_varlen(*data[:3], data[4], data[5]), a['o'])
    assert torch.equal(ops.attention_varlen(*data[:3], data[4].long(), data[5].long()), a['o'])
    v = data[2].detach().requires_grad_(True)
    dv, = torch.autograd.grad(ops.attention_varlen(data[0], data[1], v, data[4], data[5]), v, data[3])
    assert torch.equal(dv, a['dv'])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_captured_and_replayed_with_other_offsets(gpu, dtype):
    """forward and backward in one graph; the lengths are data: two graphs, replayed in turn with offsets changed between replays, equal the eager results"""
    from diffusion_pipe_amd import ops
    plans = ([150, 50, 100], [10, 280, 10], [300, 0, 0])
    q, k, v, do, cu, _ = _inputs(gpu, plans[0], plans[0], 4, 2, 128, dtype=dtype)
    few = _inputs(gpu, [1, 2], [5000, 3000], 4, 2, 128, dtype=dtype)

    def step(q, k, v, do, cu_q, cu_k):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = ops.attention_varlen(*leaves, cu_q, cu_k, causal=True)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    graphs = []
    for args in ((q, k, v, do, cu, None), few):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*args)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*args)
        graphs.append((graph, out, args))
    for turn in range(4):
        lens = plans[turn % 3]
        cu.copy_(torch.tensor([0, lens[0], lens[0] + lens[1], 300], dtype=torch.int32))
        few[4].copy_(torch.tensor([0, 1 + turn % 2, 3], dtype=torch.int32))
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out, args in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, step(*args))), turn


def test_on_another_stream(gpu):
    lens = [500, 300]
    q, k, v, do, cu, _ = _inputs(gpu, lens, lens, 4, 4, 64)
    want = _run(q, k, v, do, cu, None, False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, cu, None, False)
    side.synchronize()
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_two_threads_on_two_streams_at_once(gpu):
    """calls in flight at the same time share nothing: parts of split axes, statistics and outputs are each call's own"""
    import threading
    cases = [_inputs(gpu, [1, 2], [5000, 3000], 4, 2, 128), _inputs(gpu, [3000, 1500], [77, 20], 4, 4, 64)]
    want = [_run(*c, True) for c in cases]
    torch.cuda.synchronize()
    got, streams = [[], []], [torch.cuda.Stream(), torch.cuda.Stream()]

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(8):
                got[i].append(_run(*cases[i], True))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 8 and all(torch.equal(g[n], want[i][n]) for g in got[i] for n in g)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_offsets_that_do_not_ascend_stay_inside_the_tensors(gpu, dtype):
    """wrong offsets give wrong rows, never an access outside: every start and end is clamped by the kernels"""
    q, k, v, do, cu, _ = _inputs(gpu, [100, 100], [100, 100], 2, 2, 64, dtype=dtype)
    for bad in ([0, 150, 100], [0, -5, 900], [0, 2000000000, -2000000000], [50, 20, 200]):
        _run(q, k, v, do, torch.tensor(bad, dtype=torch.int32, device=gpu), None, True)
    torch.cuda.synchronize()


def test_sequences_of_one_tile_are_rounded_once(gpu):
    """sequences of up to 64 tokens multiply what the rounding of P and dS left as well: o, dQ, dK, dV are off by their own rounding (h) and by products of two roundings (h^2),
    the same terms as the bounds above with h^2 for h, and fp32's"""
    lens, H, Hk, D = [1, 2, 1, 9, 5, 64, 1, 12, 40, 2], 4, 2, 128
    q, k, v, do, cu, _ = _inputs(gpu, lens, lens, H, Hk, D)
    got = _run(q, k, v, do, cu, None, True)
    global H_BF16, R_P
    keep = H_BF16, R_P
    want = _exact(q, k, v, do, lens, lens, True, 1.0 / math.sqrt(D))
    try:
        H_BF16, R_P = 2.0 ** -16, 2.0 ** -10
        once = _exact(q, k, v, do, lens, lens, True, 1.0 / math.sqrt(D))
    finally:
        H_BF16, R_P = keep
    for n, t in got.items():
        value, bound = once[n]
        assert ((t.detach().double() - value).abs() <= bound + H_BF16 * (value.abs() + bound)).all(), n
    _check(got, want, 'one tile')


def test_empty_tensors(gpu):
    from diffusion_pipe_amd import ops
    q, k, v, do, cu, _ = _inputs(gpu, [3], [3], 2, 2, 64)
    none = torch.zeros(2, dtype=torch.int32, device=gpu)
    e = torch.empty(0, 2, 64, device=gpu, dtype=torch.bfloat16)
    assert ops.attention_varlen(e, k, v, none, cu).shape == e.shape
    got = _run(q, e, e, do, cu, none, False)
    assert all((t == 0).all() for t in got.values())


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32], ids=['bf16', 'fp32'])
def test_long_sequence_past_32_bit_offsets(gpu, dtype):
    """keys and values 2^32 bytes apart within one sequence: a token stride of 2^22 elements"""
    D, n, stride = 64, 700, 2 ** 22
    buf = torch.zeros(n * stride, dtype=dtype, device=gpu)
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(n, 1, D, generator=g).to(gpu, dtype) for _ in range(4))
    kv = torch.as_strided(buf, (n, 2, D), (stride, D, 1))
    kv[:, :1], kv[:, 1:] = k, v
    cu = torch.tensor([0, n], dtype=torch.int32, device=gpu)
    want = _run(q, k, v, do, cu, None, True)
    got = _run(q, kv[:, :1], kv[:, 1:], do, cu, None, True)
    assert all(torch.equal(got[x], want[x]) for x in want)

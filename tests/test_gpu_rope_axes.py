"""ops.rope_axes against the rotation in 64 bits.

Bounds, element by element (f = 2^-24: half a step of fp32; h: half a step of the stored type).  The remainder of the turns is <= 1/2 and kept in fp32, off by 2^-26 turns = 1.6 f in
radians; sine and cosine add 2 units in the last place of values <= 1: a table entry is off by at most 6 f, a rotated value by 6 f (|a| + |b|) + 3 roundings: 9 f (|a| + |b|).
A norm's sum of squares takes at most 8 + 5 additions in sequence, halved by the root, 2 f for rsqrt, 2 f for the products: 11 f of the value, 24 f (|a| + |b|) with the rotation.
Storing adds h |y|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _turn(x, angles, interleaved, back=False):
    R = 2 * angles.shape[-1]
    c, s = angles.cos().unsqueeze(-2), angles.sin().unsqueeze(-2) * (-1 if back else 1)
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    ya, yb = a * c - b * s, b * c + a * s
    y = torch.stack([ya, yb], -1).flatten(-2) if interleaved else torch.cat([ya, yb], -1)
    return torch.cat([y, x[..., R:]], -1)


def _pair_size(x, R, interleaved):
    """|a| + |b| of every channel's pair (the channel itself where nothing rotates)"""
    x = x.abs()
    if interleaved:
        s = (x[..., 0:R:2] + x[..., 1:R:2]).repeat_interleave(2, -1)
    else:
        s = (x[..., :R // 2] + x[..., R // 2:R]).repeat(*([1] * (x.dim() - 1)), 2)
    return torch.cat([s, x[..., R:]], -1)


def _angles(positions, axes, theta, shared=False):
    theta = theta if isinstance(theta, tuple) else (theta,) * len(axes)
    out, at = [], 0
    for a, dim in enumerate(axes):
        j = torch.arange(dim // 2, dtype=torch.float64, device=positions.device)
        e = -2 * (at + j) / sum(axes) if shared else -2 * j / dim
        out.append(positions[..., a:a + 1].double() * theta[a] ** e)
        at += dim // 2
    return torch.cat(out, -1)


def _exact(x, w, gy, angles, eps, interleaved, depth):
    """{y, dx, dw: (value, bound)}; depth: additions in sequence of the weight gradient's sum"""
    h, R = HALF_STEP[x.dtype], 2 * angles.shape[-1]
    x, gy = x.detach().double(), gy.double()
    w = w.detach().double() if w is not None else None
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) if w is not None else 1.0
    xh = x * r
    n = xh * w if w is not None else x
    y = _turn(n, angles, interleaved)
    g = _turn(gy, angles, interleaved, back=True)
    eg = 9 * F * _pair_size(gy, R, interleaved)
    out = {'y': (y, 24 * F * _pair_size(n, R, interleaved) + h * y.abs())}
    if w is None:
        return {**out, 'dx': (g, eg + h * g.abs())}
    u = g * w
    m = (u * xh).mean(-1, keepdim=True)
    em = ((eg * w.abs() + 24 * F * u.abs()) * xh.abs()).mean(-1, keepdim=True)
    dx = r * (u - xh * m)
    e = r * (eg * w.abs() + 24 * F * (u.abs() + (xh * m).abs()) + xh.abs() * em)
    dims = tuple(range(x.dim() - 1))
    dw = (g * xh).sum(dims)
    ew = ((eg + 24 * F * g.abs()) * xh.abs()).sum(dims) + depth * F * (g * xh).abs().sum(dims)
    return {**out, 'dx': (dx, e + h * dx.abs()), 'dw': (dw, ew + h * dw.abs())}


def _check(got, want, label):
    value, bound = want
    assert got.shape == value.shape
    ratio = ((got.detach().double() - value).abs() / (bound + 1e-30)).max().item()
    print(f'{label}: worst error / bound {ratio:.3f}')
    assert ratio <= 1.0, (label, ratio)


def _positions(gpu, lead, axes, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == 'fraction':
        return (torch.rand(*lead, axes, generator=g) * 60 - 30).to(gpu)
    return torch.randint(0, 2 ** 20 if kind == torch.int64 else 90, (*lead, axes), generator=g).to(gpu, kind)


CASES = [  # (tokens, H, Hk, D, axes, theta, positions, interleaved, shared)
    ((1,), 1, 1, 64, (8, 28, 28), 10000.0, torch.int32, True, False),
    ((7,), 3, 1, 64, (64,), 1000000.0, torch.int64, False, False),
    ((129,), 24, 24, 128, (16, 56, 56), 256.0, torch.float32, True, False),
    ((50,), 5, 0, 128, (44, 42, 42), 10000.0, 'fraction', True, False),
    ((2, 33), 4, 2, 128, (16, 24, 24), (10000.0, 100.0, 300.0), torch.int32, False, False),      # channels behind the axes are not rotated
    ((3, 20), 2, 2, 80, (16, 24, 30), 10000.0, torch.int64, True, False),                        # the last pairs end inside a vector of 8
    ((65,), 40, 8, 128, (32, 48, 48), 1000000.0, torch.int64, False, True),
    ((17,), 2, 1, 256, (64, 96, 96), 10000.0, torch.float32, False, False),
    ((31,), 3, 3, 8, (4,), 10000.0, torch.int32, True, False),
    ((3000,), 10, 2, 96, (32, 32, 32), 10000.0, torch.float32, True, False),
]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16], ids=['f32', 'bf16'])
@pytest.mark.parametrize('norm', ['none', 'both', 'query'])
@pytest.mark.parametrize('case', CASES, ids=lambda c: f'{"x".join(map(str, c[0]))}_{c[1]}h{c[2]}_d{c[3]}_{"".join("i" if c[7] else "h")}')
def test_forward_and_gradients(gpu, case, norm, dtype):
    from diffusion_pipe_amd import ops
    lead, H, Hk, D, axes, theta, kind, interleaved, shared = case
    g = torch.Generator().manual_seed(D + H)
    pos = _positions(gpu, lead[1:] if lead[0] == 2 else lead, len(axes), kind)               # (two samples: one run of positions for both)
    make = lambda *s: torch.randn(*s, generator=g).to(gpu, dtype)
    q, gq = make(*lead, H, D), make(*lead, H, D)
    k, gk = (make(*lead, Hk, D), make(*lead, Hk, D)) if Hk else (None, None)
    wq = (1 + 0.3 * make(D)) if norm != 'none' else None
    wk = (1 + 0.3 * make(D)).float() if norm == 'both' and Hk else None                      # (a weight of another type)
    leaves = [t.requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    yq, yk = ops.rope_axes(q, k, pos, axes, theta=theta, q_weight=wq, k_weight=wk, eps=1e-6, interleaved=interleaved, shared=shared)
    assert (yk is None) == (k is None) and yq.dtype == dtype
    grads = iter(torch.autograd.grad([t for t in (yq, yk) if t is not None], leaves, [t for t in (gq, gk) if t is not None]))
    got = {n: next(grads) for n, t in (('q', q), ('k', k), ('wq', wq), ('wk', wk)) if t is not None}
    angles = _angles(pos, axes, theta, shared)
    for n, x, y, gy, w in (('q', q, yq, gq, wq), ('k', k, yk, gk, wk)):
        if x is None:
            continue
        want = _exact(x, w, gy, angles, 1e-6, interleaved, depth=x[..., 0].numel() // 32 + 256)
        _check(y, want['y'], n)
        _check(got[n], want['dx'], 'd' + n)
        if w is not None:
            assert got['w' + n].dtype == w.dtype
            value, bound = want['dw']
            _check(got['w' + n], (value, bound + HALF_STEP[w.dtype] * value.abs()), 'dw' + n)


def test_channels_behind_the_axes_keep_their_bits(gpu):
    """not rotated and without a norm: copied, also next to an infinity or NaN"""
    from diffusion_pipe_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(9, 2, 40, generator=torch.Generator().manual_seed(1)).to(gpu, dtype)
        x[3, 0, 35], x[4, 1, 31] = float('inf'), float('nan')
        for interleaved, axes in ((True, (12, 10)), (False, (8, 16))):
            y, _ = ops.rope_axes(x, None, _positions(gpu, (9,), 2, torch.int32), axes, interleaved=interleaved)
            assert torch.equal(torch.nan_to_num(y[..., sum(axes):], nan=7.0), torch.nan_to_num(x[..., sum(axes):], nan=7.0))
            ok = torch.isfinite(x[..., :sum(axes)]).all(-1)
            assert torch.isfinite(y[..., :sum(axes)])[ok].all()


def test_matches_the_table_operator(gpu):
    """the same rotation as ops.rms_norm_rope with tables, per head, on one axis after the other"""
    from diffusion_pipe_amd import ops
    x = torch.randn(1, 60, 4, 64, generator=torch.Generator().manual_seed(2)).to(gpu)
    w = torch.rand(64, generator=torch.Generator().manual_seed(3)).to(gpu) + 0.5
    pos = _positions(gpu, (60,), 3, torch.int32)
    angles = _angles(pos, (8, 28, 28), 256.0)
    want = ops.rms_norm_rope(x, w, angles.cos().float(), angles.sin().float(), eps=1e-6)
    got, _ = ops.rope_axes(x, None, pos, (8, 28, 28), theta=256.0, q_weight=w)
    assert (got - want).abs().max() <= 64 * F * want.abs().max()


def test_far_positions_keep_their_angle(gpu):
    """positions of a million and more, whose angle in fp32 would be off by a tenth of a radian"""
    from diffusion_pipe_amd import ops
    x = torch.randn(40, 1, 64, generator=torch.Generator().manual_seed(4)).to(gpu)
    pos = (torch.arange(40, dtype=torch.int64, device=gpu) * 104729 + 2 ** 31).unsqueeze(-1)
    y, _ = ops.rope_axes(x, None, pos, (64,), interleaved=False)
    # fp64 angles up to 4e9: off by 4e9 2^-53 2 = 1e-6 in the reference and the kernel alike
    value, bound = _exact(x, None, x, _angles(pos, (64,), 10000.0), 1e-6, False, 0)['y']
    assert ((y.double() - value).abs() <= bound + 2e-6 * _pair_size(x.double(), 64, False)).all()


def test_views_gradients_and_accumulation(gpu):
    """column blocks of a fused projection, expanded and missing gradients, and the fused accumulation into an existing .grad"""
    from diffusion_pipe_amd import ops
    g = torch.Generator().manual_seed(6)
    qkv = torch.randn(70, 10, 64, generator=g).to(gpu, torch.bfloat16)
    pos = _positions(gpu, (70,), 3, torch.int32)
    wq, wk = (torch.nn.Parameter((1 + 0.2 * torch.randn(64, generator=g)).to(gpu, torch.bfloat16)) for _ in range(2))
    call = lambda q, k: ops.rope_axes(q, k, pos, (8, 28, 28), q_weight=wq, k_weight=wk)
    a, b = call(qkv[:, :6], qkv[:, 6:8]), call(qkv[:, :6].contiguous(), qkv[:, 6:8].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    odd = torch.empty(qkv.numel() + 1, device=gpu, dtype=qkv.dtype)[1:].view(qkv.shape).copy_(qkv)
    assert torch.equal(call(odd[:, :6], odd[:, 6:8])[0], a[0])
    leaf = qkv.detach().requires_grad_(True)
    yq, yk = call(leaf[:, :6], leaf[:, 6:8])
    first = torch.autograd.grad(yq.sum(), (leaf, wq), retain_graph=True)                       # an expanded gradient, none for yk
    second = torch.autograd.grad(yq, (leaf, wq), torch.ones_like(yq), retain_graph=True)
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1]) and (first[0][:, 6:] == 0).all()
    wq.grad = torch.full_like(wq, 3.0)
    ops.FUSE_GRAD_ACCUM = True
    try:
        torch.autograd.backward((yq, yk), (torch.ones_like(yq), torch.ones_like(yk)))
    finally:
        ops.FUSE_GRAD_ACCUM = False
    f = torch.float32
    assert ((wq.grad.to(f) - 3.0 - second[1].to(f)).abs() <= 2.0 ** -7 * (3.0 + second[1].to(f).abs())).all()


def test_one_weight_for_queries_and_keys(gpu):
    """a shared, strided weight gets the sum of both gradients, also where the parameter gradients are accumulated inside the kernels"""
    from diffusion_pipe_amd import ops
    g = torch.Generator().manual_seed(7)
    q, k = (torch.randn(300, h, 64, generator=g).to(gpu) for h in (4, 2))
    gq, gk = torch.randn(300, 4, 64, generator=g).to(gpu), torch.randn(300, 2, 64, generator=g).to(gpu)
    pos = _positions(gpu, (300,), 1, torch.int64)
    wide = torch.nn.Parameter(1 + 0.2 * torch.randn(128, generator=g).to(gpu))
    w = torch.nn.Parameter(wide.detach()[::2].contiguous())
    angles = _angles(pos, (64,), 10000.0)
    (vq, bq), (vk, bk) = (_exact(x, w, gy, angles, 1e-6, True, 300)['dw'] for x, gy in ((q, gq), (k, gk)))
    y = ops.rope_axes(q, k, pos, (64,), q_weight=wide[::2], k_weight=wide[::2])
    got, = torch.autograd.grad(y, wide, (gq, gk))
    assert ((got[::2].double() - vq - vk).abs() <= bq + bk + F * (vq + vk).abs()).all() and (got[1::2] == 0).all()
    for fuse in (False, True):
        w.grad = torch.full_like(w, 5.0)
        y = ops.rope_axes(q, k, pos, (64,), q_weight=w, k_weight=w)
        ops.FUSE_GRAD_ACCUM = fuse
        try:
            torch.autograd.backward(y, (gq, gk))
        finally:
            ops.FUSE_GRAD_ACCUM = False
        assert ((w.grad.double() - 5.0 - vq - vk).abs() <= bq + bk + 4 * F * (5.0 + vq.abs() + vk.abs())).all(), fuse


def test_gradients_against_differences(gpu):
    from diffusion_pipe_amd import ops
    g = torch.Generator().manual_seed(8)
    x, gy = (torch.randn(20, 3, 64, generator=g).to(gpu).requires_grad_(r) for r in (True, False))
    w = (1 + 0.2 * torch.randn(64, generator=g)).to(gpu).requires_grad_(True)
    pos = _positions(gpu, (20,), 3, 'fraction')
    angles = _angles(pos, (8, 28, 28), 10000.0)
    y, _ = ops.rope_axes(x, None, pos, (8, 28, 28), q_weight=w)
    grads = torch.autograd.grad(y, (x, w), gy)
    want = _exact(x, w, gy, angles, 1e-6, True, 300)
    for i, name in enumerate(('dx', 'dw')):
        d = torch.randn(grads[i].shape, generator=g).to(gpu).double()
        def loss(step):
            args = [x.detach().double(), w.detach().double()]
            args[i] = args[i] + step * d
            n = args[0] * torch.rsqrt((args[0] ** 2).mean(-1, keepdim=True) + 1e-6) * args[1]
            return (_turn(n, angles, True) * gy.double()).sum().item()
        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        # differences: third derivatives are O(1) in the step, 1e-8 of the terms' absolute sum
        assert abs((grads[i].double() * d).sum().item() - slope) <= (want[name][1] * d.abs()).sum().item() + 1e-7 * (grads[i].double() * d).abs().sum().item()


def test_captured_and_replayed_with_other_positions(gpu):
    from diffusion_pipe_amd import ops
    g = torch.Generator().manual_seed(9)
    q, k, gq, gk = (torch.randn(500, h, 128, generator=g).to(gpu, torch.bfloat16) for h in (6, 2, 6, 2))
    w = torch.ones(128, device=gpu, dtype=torch.bfloat16)
    pos = _positions(gpu, (500,), 3, torch.float32)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, w)]
        y = ops.rope_axes(leaves[0], leaves[1], pos, (16, 56, 56), q_weight=leaves[2], k_weight=leaves[2])
        return [y[0].detach(), y[1].detach(), *torch.autograd.grad(y, leaves, (gq, gk))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for turn in range(3):
        pos.copy_(_positions(gpu, (500,), 3, torch.float32, seed=turn))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, step())), turn


@pytest.mark.parametrize('dtype,interleaved', [(torch.bfloat16, True), (torch.bfloat16, False), (torch.float32, True), (torch.float32, False)], ids=['bf16', 'bf16_halves', 'f32', 'f32_halves'])
def test_more_than_the_caches_hold(gpu, dtype, interleaved):
    """heads of more than 256 MB take the kernels that stream past the caches: the same bits as the two halves of the tokens by themselves; the weight's gradient is the sum of the halves'
    (each fp32 sum off by at most depth F of its terms' absolute sum, see _exact)"""
    from diffusion_pipe_amd import ops
    n = 24000 if dtype == torch.bfloat16 else 12000
    g = torch.Generator(device=gpu).manual_seed(13)
    q, gq = (torch.randn(n, 40, 128, device=gpu, generator=g).to(dtype) for _ in range(2))
    k, gk = (torch.randn(n, 8, 128, device=gpu, generator=g).to(dtype) for _ in range(2))
    assert (q.numel() + k.numel()) * q.element_size() > 2 ** 28 > (q[:n // 2].numel() + k[:n // 2].numel()) * q.element_size()
    w = (1 + 0.2 * torch.randn(128, device=gpu, generator=g)).requires_grad_(True)
    pos = _positions(gpu, (n,), 3, torch.float32)

    def step(rows, weight):
        leaves = [q[rows].detach().requires_grad_(True), k[rows].detach().requires_grad_(True)]
        y = ops.rope_axes(*leaves, pos[rows], (16, 56, 56), q_weight=weight, k_weight=weight, interleaved=interleaved)
        return [y[0].detach(), y[1].detach(), *torch.autograd.grad(y, leaves + ([weight] if weight is not None else []), (gq[rows], gk[rows]))]
    for weight in (w, None):
        whole, first, second = (step(r, weight) for r in (slice(None), slice(0, n // 2), slice(n // 2, n)))
        for i in range(4):
            assert torch.equal(whole[i], torch.cat([first[i], second[i]])), (weight is None, i)
    whole, first, second = (step(r, w)[4].double() for r in (slice(None), slice(0, n // 2), slice(n // 2, n)))
    xh = q.float() * torch.rsqrt((q.float() ** 2).mean(-1, keepdim=True) + 1e-6)
    terms = 2.0 * _pair_size(gq.float(), 128, interleaved).mul_(xh.abs()).sum((0, 1)).double()          # queries' terms, and the fewer keys' within as much again
    assert ((whole - first - second).abs() <= (n * 40 // 16 // 256 + 600) * F * terms).all()


def test_no_tokens(gpu):
    from diffusion_pipe_amd import ops
    q = torch.empty(0, 4, 64, device=gpu).requires_grad_(True)
    w = torch.ones(64, device=gpu, requires_grad=True)
    y, _ = ops.rope_axes(q, None, torch.empty(0, 1, device=gpu), (64,), q_weight=w)
    y.sum().backward()
    assert y.shape == q.shape and (w.grad == 0).all()


def test_rotary_positions_then_packed_attention(gpu):
    """the two operators in the order a packed image-text batch runs them: norm and rotation of query and key heads, attention per sequence, gradients back to the fused projection and
    the norm weights.  The composition is held to the same composition with the rotated heads rounded to bf16 as the first operator stores them; gradients that pass the second
    operator are rounded to bf16 between the two (half a step each), which the bound adds through the rotation and the norm (an orthogonal map and a projection, |r w| <= rw)."""
    from diffusion_pipe_amd import ops
    import test_gpu_attention_varlen as av
    g = torch.Generator().manual_seed(12)
    lens, H, Hk, D = [90, 200], 4, 2, 64
    T = sum(lens)
    qkv = torch.randn(T, H + 2 * Hk, D, generator=g).to(gpu, torch.bfloat16).requires_grad_(True)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).to(gpu, torch.bfloat16).requires_grad_(True) for _ in range(2))
    do = torch.randn(T, H, D, generator=g).to(gpu, torch.bfloat16)
    pos = torch.cat([torch.stack([torch.zeros(n), torch.arange(n) // 10, torch.arange(n) % 10], -1) for n in lens]).to(gpu)
    cu = torch.tensor([0, 90, 290], dtype=torch.int32, device=gpu)
    q, k = ops.rope_axes(qkv[:, :H], qkv[:, H:H + Hk], pos, (8, 28, 28), q_weight=wq, k_weight=wk)
    o = ops.attention_varlen(q, k, qkv[:, H + Hk:], cu)
    dqkv, dwq, dwk = torch.autograd.grad(o, (qkv, wq, wk), do)
    attn = av._exact(q, k, qkv[:, H + Hk:], do, lens, lens, False, 0.125)
    av._check({'o': o, 'dv': dqkv[:, H + Hk:]}, attn, 'composed')
    angles = _angles(pos, (8, 28, 28), 10000.0)
    for n, x, w, dx, dw in (('dq', qkv[:, :H], wq, dqkv[:, :H], dwq), ('dk', qkv[:, H:H + Hk], wk, dqkv[:, H:H + Hk], dwk)):
        value, bound = attn[n]
        want = _exact(x, w, value, angles, 1e-6, True, 300)
        xd = x.detach().double()
        r = torch.rsqrt((xd * xd).mean(-1, keepdim=True) + 1e-6)
        xh, rot = xd * r, 1.5 * _pair_size(bound, 64, True)                       # |cos|, |sin| <= 1
        u = rot * w.detach().double().abs()
        extra = r * (u + xh.abs() * (u * xh.abs()).mean(-1, keepdim=True))
        _check(dx, (want['dx'][0], want['dx'][1] + extra), n)
        _check(dw, (want['dw'][0], want['dw'][1] + (rot * xh.abs()).sum((0, 1))), n + ' weight')

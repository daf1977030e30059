"""Rotary positions over several axes and attention over packed sequences: the work that is timed, in plain form and through the kernels.

The two operators follow each other in a transformer block that trains on images and videos of different sizes, or on prompts of different
lengths, packed back to back without padding: the query and key heads are normalised and turned by their tokens' positions (time, height,
width), then every sequence attends to itself (or a packed image to its packed prompt).

    rope        y = R(position) (x / rms(x) * weight),  R turns channel pair p of axis a by  position[a] * theta ** (-2 j / dim_a)
    attention   o_i = sum_j softmax_j(scale q_i . k_j) v_j  over the keys of the token's own sequence; query head h reads key head h // group;
                causal: key j is seen from query i where  j - len_k <= i - len_q; a query that sees nothing gives zero

`own` selects the plain form (elementary torch operations in 32 bits, angles in 64) or the framework's kernels.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {'bfloat16': torch.bfloat16, 'float32': torch.float32}


# ------------------------------------------------------------------------------------------------------------------------- cases
def _rope(name, tokens, q_heads, kv_heads, head_dim, axes, theta, dtype='bfloat16', norm=True, half=False, train=False, positions='float32'):
    return {'name': name, 'op': 'rope', 'tokens': tokens, 'q_heads': q_heads, 'kv_heads': kv_heads, 'head_dim': head_dim, 'axes': axes, 'theta': theta,
            'dtype': dtype, 'norm': norm, 'half': half, 'train': train, 'positions': positions}


def _attention(name, lens_q, lens_k, q_heads, kv_heads, head_dim, causal, train, tail=0):
    return {'name': name, 'op': 'attention', 'lens_q': ','.join(map(str, lens_q)), 'lens_k': ','.join(map(str, lens_k)) if lens_k else '',
            'q_heads': q_heads, 'kv_heads': kv_heads, 'head_dim': head_dim, 'causal': causal, 'train': train, 'tail': tail}


def listed():
    return [
        # one small image's tokens behind the fused projection: a call of a few microseconds, where the launch counts
        _rope('rope_small', 256, 10, 10, 64, '8,28,28', 10000.0),
        # a 1024 x 1024 image and its prompt, 24 heads of 128 (text tokens sit at position zero), query and key norms, evaluation
        _rope('rope_image', 4608, 24, 24, 128, '16,56,56', 10000.0),
        # the same heads over a long video, one training pass: gradients of queries, keys and both norm weights
        _rope('rope_video_train', 61456, 24, 24, 128, '16,56,56', 256.0, train=True),
        # packed prompts with grouped heads, channels paired across the halves of the head, one axis, far positions, exact arithmetic
        _rope('rope_prompt_f32', 9001, 28, 4, 128, '128', 1000000.0, dtype='float32', norm=False, half=True, train=True, positions='int64'),
        # two prompts of a text encoder: 77 tokens and 12 heads of 64, causal; latency
        _attention('prompts_small', [77, 77], None, 12, 12, 64, True, False),
        # a batch of ragged prompts, causal, four query heads to a key head
        _attention('prompts_ragged', [1, 17, 4096, 333, 1, 1025, 77, 2050, 512, 64, 129, 1300], None, 32, 8, 128, True, False),
        # the same kind of batch, trained on, in a buffer of fixed size whose end no sequence fills
        _attention('prompts_train', [2049, 1500, 700, 4096, 31, 1, 900], None, 32, 8, 128, True, True, tail=100),
        # images of three sizes with their prompts in one batch, 24 heads of 128, trained on
        _attention('images_train', [4608, 2560, 1311], None, 24, 24, 128, False, True),
        # images of two sizes at 10 heads of 64, trained on
        _attention('images_d64_train', [4096, 1024, 2501], None, 10, 10, 64, False, True),
        # image tokens reading their prompts (ragged, 77 tokens up to 512), 40 heads of 128, trained on
        _attention('cross_train', [9216, 4080], [512, 77], 40, 40, 128, False, True),
        # single new tokens behind long cached prompts: few rows, long keys
        _attention('new_tokens', [1, 1, 1, 1, 3, 1], [30000, 8191, 1, 16385, 5000, 777], 32, 8, 128, True, False),
        # one long video next to a short one, 24 heads of 128, trained on: the largest
        _attention('videos_train', [15000, 6001], None, 24, 24, 128, False, True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _ragged(rng, total, count):
    """`count` lengths from one token up, spread over their logarithm, that come to about `total`"""
    raw = [math.exp(rng.uniform(0.0, math.log(max(total, 2)))) for _ in range(count)]
    return [max(1, int(r * total / sum(raw))) for r in raw]


def draw(rng):
    if rng.random() < 0.35:
        head_dim, axes = rng.choice([(64, '8,28,28'), (128, '16,56,56'), (128, '44,42,42'), (96, '32,32,32'), (128, '128'), (64, '64'), (80, '16,24,24')])
        kv_heads = rng.choice([1, 2, 4, 8, 10, 12, 24])
        q_heads = kv_heads * rng.choice([1, 1, 2, 4] if kv_heads <= 10 else [1])
        dtype = rng.choice(['bfloat16', 'bfloat16', 'float32'])
        room = 61456 * 48 * 128 // (2 if dtype == 'float32' else 1) // ((q_heads + kv_heads) * head_dim)
        return {k: v for k, v in _rope('', _spread(rng, 1, min(61456, room)), q_heads, kv_heads, head_dim, axes, rng.choice([256.0, 10000.0, 1000000.0]), dtype,
                                       norm=rng.random() < 0.6, half=rng.random() < 0.4 and head_dim != 80, train=rng.random() < 0.5,
                                       positions=rng.choice(['float32', 'int64', 'int32'])).items() if k != 'name'}
    head_dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8, 10])
    q_heads = kv_heads * rng.choice([1, 2, 3, 4])
    most = min(16000, int(math.sqrt(1e13 / (14 * head_dim * q_heads))))       # one sequence of all tokens stays below the largest listed case
    kind, lens_k = rng.choice(['prompts', 'images', 'cross', 'new_tokens']), None
    if kind == 'prompts':
        lens_q = _ragged(rng, _spread(rng, 16, most), rng.randint(1, 24))
    elif kind == 'images':
        lens_q = _ragged(rng, _spread(rng, 64, most), rng.randint(1, 5))
    elif kind == 'cross':
        lens_q = _ragged(rng, _spread(rng, 64, most), rng.randint(1, 5))
        lens_k = [rng.randint(1, 512) for _ in lens_q]
    else:
        lens_k = _ragged(rng, _spread(rng, 64, 60000), rng.randint(1, 16))
        lens_q = [rng.choice([1, 1, 1, 2, 5]) for _ in lens_k]
    return {k: v for k, v in _attention('', lens_q, lens_k, q_heads, kv_heads, head_dim, kind in ('prompts', 'new_tokens') or rng.random() < 0.2,
                                        kind != 'new_tokens' and rng.random() < 0.6, rng.choice([0, 0, 0, 37])).items() if k != 'name'}


def _lens(case):
    lens_q = [int(n) for n in case['lens_q'].split(',')]
    lens_k = [int(n) for n in case['lens_k'].split(',')] if case['lens_k'] else lens_q
    return lens_q, lens_k


def _axes(case):
    return tuple(int(a) for a in case['axes'].split(','))


# ------------------------------------------------------------------------------------------------------------------------ inputs
def _grid_positions(case, seed):
    """[tokens, axes]: prompts at position zero followed by a grid of (time, height, width), or plain counting with one axis"""
    r, n, axes = np.random.RandomState((seed + 17) % 2 ** 32), case['tokens'], len(_axes(case))
    pos = np.zeros((n, axes))
    at = 0
    while at < n:
        length = min(n - at, int(r.randint(max(1, n // 8), n + 1)))
        if axes == 1:
            pos[at:at + length, 0] = r.randint(0, 100000) + np.arange(length)
        else:
            text, (h, w) = min(length, int(r.randint(0, 513))), r.randint(16, 97, size=2)
            i = np.arange(length - text)
            pos[at + text:at + length] = np.stack([i // (h * w), i // w % h, i % w], axis=1)
        at += length
    return pos


def prepare(case, seed):
    dev = torch.device('cuda')
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed * 2 + 1)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, device=dev, generator=gen) * scale).to(dtype)

    hq, hk, d = case['q_heads'], case['kv_heads'], case['head_dim']
    if case['op'] == 'rope':
        dt = _DTYPES[case['dtype']]
        n = case['tokens']
        qkv = normal(n, hq + 2 * hk, d, scale=1.5, dtype=dt)          # the fused projection: queries and keys are views of its rows
        s = {'case': case, 'q': qkv[:, :hq], 'k': qkv[:, hq:hq + hk], 'wq': None, 'wk': None,
             'positions': torch.from_numpy(_grid_positions(case, seed)).to(dev, {'float32': torch.float32, 'int64': torch.int64, 'int32': torch.int32}[case['positions']])}
        if case['norm']:
            s['wq'], s['wk'] = ((1.0 + 0.2 * torch.randn(d, device=dev, generator=gen)).to(dt) for _ in range(2))
        if case['train']:
            s['gq'], s['gk'] = normal(n, hq, d, scale=0.02, dtype=dt), normal(n, hk, d, scale=0.02, dtype=dt)
            s['leaves'] = [t.requires_grad_(True) for t in (s['q'].detach(), s['k'].detach(), s['wq'], s['wk']) if t is not None]
            s['q'], s['k'] = s['leaves'][:2]
        return s
    lens_q, lens_k = _lens(case)
    nq, nk = sum(lens_q) + case['tail'], sum(lens_k) + (case['tail'] if not case['lens_k'] else 0)
    s = {'case': case, 'q': normal(nq, hq, d)}
    kv = normal(nk, 2 * hk, d)                                        # keys are rotated tensors of their own, values a view of the projection
    s['k'], s['v'] = kv[:, :hk].contiguous(), kv[:, hk:]
    s['cu_q'] = torch.tensor([0] + list(np.cumsum(lens_q)), dtype=torch.int32, device=dev)
    s['cu_k'] = torch.tensor([0] + list(np.cumsum(lens_k)), dtype=torch.int32, device=dev) if case['lens_k'] else None
    if case['train']:
        s['do'] = normal(nq, hq, d, scale=0.1)
        s['q'], s['k'], s['v'] = s['leaves'] = [t.detach().requires_grad_(True) for t in (s['q'], s['k'], s['v'])]
    return s


# -------------------------------------------------------------------------------------------------------------- the plain forms
def _rope_plain(s):
    case = s['case']
    pos, dims = s['positions'].double(), _axes(case)
    rot = sum(dims)
    angles = torch.cat([pos[:, a:a + 1] * torch.pow(case['theta'], torch.arange(0, dim, 2, device=pos.device, dtype=torch.float64) / -dim)
                        for a, dim in enumerate(dims)], dim=1)
    cos, sin = angles.cos().float()[:, None], angles.sin().float()[:, None]

    def turn(x, sin):
        y = x.clone()
        a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if case['half'] else (x[..., 0:rot:2], x[..., 1:rot:2])
        ya, yb = a * cos - b * sin, b * cos + a * sin
        if case['half']:
            y[..., :rot // 2], y[..., rot // 2:rot] = ya, yb
        else:
            y[..., 0:rot:2], y[..., 1:rot:2] = ya, yb
        return y

    outs, grads, weight_grads = [], [], []
    for x, w, name in ((s['q'], s['wq'], 'gq'), (s['k'], s['wk'], 'gk')):
        x = x.detach()
        dt, x = x.dtype, x.float()
        if w is not None:
            w = w.detach().float()
            r = torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + 1e-6)
            x = x * r
        outs.append(turn(x if w is None else x * w, sin).to(dt))
        if case['train']:
            g = turn(s[name].float(), -sin)
            if w is not None:
                weight_grads.append((g * x).sum(dim=(0, 1), dtype=torch.float64).to(dt))
                g = g * w
                g = r * (g - x * (g * x).mean(dim=-1, keepdim=True))
            grads.append(g.to(dt))
    return outs + grads + weight_grads


def _attention_plain(s):
    case = s['case']
    hq, hk, d = case['q_heads'], case['kv_heads'], case['head_dim']
    lens_q, lens_k = _lens(case)
    q, k, v = (s[n].detach() for n in 'qkv')
    scale = 1.0 / math.sqrt(d)
    o = torch.zeros_like(q, memory_format=torch.contiguous_format)
    grads = [torch.zeros_like(t, memory_format=torch.contiguous_format) for t in (q, k, v)] if case['train'] else []
    a = b = 0
    for n, m in zip(lens_q, lens_k):
        step = max(1, min(hk, 2 ** 28 // (n * m * (hq // hk))))       # key heads at a time: scores of at most about a gigabyte
        for h in range(0, hk, step):
            hs = slice(h * (hq // hk), min(h + step, hk) * (hq // hk))
            qs = q[a:a + n, hs].float().transpose(0, 1).contiguous()
            ks, vs = (t[b:b + m, h:h + step].float().transpose(0, 1).repeat_interleave(hq // hk, dim=0) for t in (k, v))
            p = torch.matmul(qs, ks.transpose(1, 2)) * scale
            if case['causal']:
                hidden = torch.arange(m, device=q.device)[None, :] - m > torch.arange(n, device=q.device)[:, None] - n
                p = p.masked_fill(hidden, -math.inf)
            top = p.amax(dim=-1, keepdim=True)
            p = torch.exp(p - torch.where(top == -math.inf, 0.0, top))
            total = p.sum(dim=-1, keepdim=True)
            p = p / torch.where(total == 0.0, 1.0, total)
            os = torch.matmul(p, vs)
            o[a:a + n, hs] = os.transpose(0, 1).to(o.dtype)
            if case['train']:
                dos = s['do'][a:a + n, hs].float().transpose(0, 1).contiguous()
                dvs = torch.matmul(p.transpose(1, 2), dos)
                ds = torch.matmul(dos, vs.transpose(1, 2))
                ds = p * (ds - (dos * os).sum(dim=-1, keepdim=True)) * scale
                grads[0][a:a + n, hs] = torch.matmul(ds, ks).transpose(0, 1).to(q.dtype)
                dks = torch.matmul(ds.transpose(1, 2), qs)
                for out, g in ((grads[1], dks), (grads[2], dvs)):     # a shared key head collects its query heads' gradients
                    out[b:b + m, h:h + step] = g.view(-1, hq // hk, m, d).sum(dim=1).transpose(0, 1).to(q.dtype)
        a, b = a + n, b + m
    return [o] + grads


# --------------------------------------------------------------------------------------------------------------------- one pass
def run(state):
    case = state['case']
    if not own:
        return _rope_plain(state) if case['op'] == 'rope' else _attention_plain(state)
    from diffusion_pipe_amd import ops
    if case['op'] == 'rope':
        outs = ops.rope_axes(state['q'], state['k'], state['positions'], _axes(case), theta=case['theta'], q_weight=state['wq'], k_weight=state['wk'],
                             eps=1e-6, interleaved=not case['half'])
        if not case['train']:
            return list(outs)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, state['leaves'], (state['gq'], state['gk'])))
    o = ops.attention_varlen(state['q'], state['k'], state['v'], state['cu_q'], state['cu_k'], causal=case['causal'])
    if not case['train']:
        return [o]
    return [o.detach()] + list(torch.autograd.grad(o, state['leaves'], state['do']))


def _pairs(case):
    total = 0
    for n, m in zip(*_lens(case)):
        if not case['causal']:
            total += n * m
        else:                                                         # query i sees clamp(m - n + i + 1, 0, m) keys
            first = max(0, n - m)
            rows = n - first
            total += rows * (m - n + first + 1) + rows * (rows - 1) // 2
    return total


def work(case):
    hq, hk, d = case['q_heads'], case['kv_heads'], case['head_dim']
    if case['op'] == 'rope':
        size = 4 if case['dtype'] == 'float32' else 2
        elements = case['tokens'] * (hq + hk) * d
        position = {'float32': 4, 'int32': 4, 'int64': 8}[case['positions']]
        passes = 4 if case['train'] else 2                            # x and y, and the gradients of both
        per = (3 + (4 if case['norm'] else 0)) + ((3 + (10 if case['norm'] else 0)) if case['train'] else 0)
        return {'bytes': passes * elements * size + case['tokens'] * len(_axes(case)) * position, 'flops': per * elements}
    lens_q, lens_k = _lens(case)
    nq, nk = sum(lens_q) + case['tail'], sum(lens_k)
    passes = 2 if case['train'] else 1                                # training: the gradient of every tensor as well
    return {'bytes': 2 * d * passes * (2 * nq * hq + 2 * nk * hk), 'flops': (14 if case['train'] else 4) * d * hq * _pairs(case)}


# ------------------------------------------------------------------------------------------------- the definitions in 64 bits
def _rope_exact(case, s):
    dims, half = _axes(case), case['half']
    rot, pos = sum(dims), s['positions'].to(torch.float64)
    outs, leaves = [], []
    for x, w in ((s['q'], s['wq']), (s['k'], s['wk'])):
        x = x.detach().to(torch.float64).requires_grad_(True)
        w = w.detach().to(torch.float64).requires_grad_(True) if w is not None else None
        leaves.append((x, w))
        y = x if w is None else x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + 1e-6).sqrt() * w
        first, second = (y[..., :rot // 2], y[..., rot // 2:rot]) if half else y[..., :rot].unflatten(-1, (rot // 2, 2)).unbind(-1)
        pair, at, parts = torch.complex(first.contiguous(), second.contiguous()), 0, []
        for a, dim in enumerate(dims):
            j = torch.arange(dim // 2, device=x.device, dtype=torch.float64)
            angle = pos[:, a].unsqueeze(1) * torch.exp(j * (-2.0 * math.log(case['theta']) / dim)).unsqueeze(0)
            parts.append(pair[..., at:at + dim // 2] * torch.polar(torch.ones_like(angle), angle).unsqueeze(1))
            at += dim // 2
        z = torch.cat(parts, dim=-1)
        turned = torch.cat([z.real, z.imag], dim=-1) if half else torch.view_as_real(z).flatten(-2)
        outs.append(torch.cat([turned, y[..., rot:]], dim=-1))
    result = [o.detach() for o in outs]
    if case['train']:
        grads = torch.autograd.grad(outs, [t for pair in leaves for t in pair if t is not None], (s['gq'].to(torch.float64), s['gk'].to(torch.float64)))
        result += [grads[0], grads[2], grads[1], grads[3]] if case['norm'] else list(grads)
    return result


def _attention_exact(case, s):
    group = case['q_heads'] // case['kv_heads']
    q, k, v = (s[n].detach().to(torch.float64) for n in 'qkv')
    results = [torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in ((q, q, k, v) if case['train'] else (q,))]
    starts, rows_at_once = [0, 0], 8192
    for n, m in zip(*_lens(case)):
        for h in range(case['q_heads']):
            kh = h // group
            key, value = k[starts[1]:starts[1] + m, kh].contiguous(), v[starts[1]:starts[1] + m, kh].contiguous()
            for r in range(0, n, rows_at_once):
                rows = slice(starts[0] + r, starts[0] + min(r + rows_at_once, n))
                query = q[rows, h].contiguous()
                score = query @ key.T / math.sqrt(case['head_dim'])
                if case['causal']:
                    i = torch.arange(r, min(r + rows_at_once, n), device=q.device) + (m - n)
                    score[torch.arange(m, device=q.device)[None] > i[:, None]] = -math.inf
                weight = torch.nan_to_num(torch.exp(score - torch.logsumexp(score, dim=1, keepdim=True)), nan=0.0)
                del score
                out = weight @ value
                results[0][rows, h] = out
                if case['train']:
                    do = s['do'][rows, h].to(torch.float64)
                    results[3][starts[1]:starts[1] + m, kh] += weight.T @ do
                    slope = do @ value.T
                    slope -= (weight * slope).sum(dim=1, keepdim=True)
                    slope *= weight
                    results[1][rows, h] = slope @ key / math.sqrt(case['head_dim'])
                    results[2][starts[1]:starts[1] + m, kh] += slope.T @ query / math.sqrt(case['head_dim'])
        starts = [starts[0] + n, starts[1] + m]
    return results


def exact(case, seed):
    if case['op'] == 'attention' and work(case)['flops'] > 3e13:
        return None
    s = prepare(case, seed)
    return _rope_exact(case, s) if case['op'] == 'rope' else _attention_exact(case, s)

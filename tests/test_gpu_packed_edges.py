"""ops.attention_varlen at its edges: rows that see no key and hold NaN, short sequences beside long ones.  Bounds: those of test_gpu_attention_varlen, element by element."""
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

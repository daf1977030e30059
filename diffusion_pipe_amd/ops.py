"""Autograd operators of the training hot path, each a thin host wrapper over the C-ABI HIP layer.

Every function here launches gfx950 kernels from libdpipe_hip.so on the current HIP stream; there is no PyTorch /
CPU fallback (a CPU tensor or a missing library raises `DpipeHipError`).  Reference semantics are cited per op.
"""
import contextlib
import ctypes
import functools
import math
import os as _os_mod

import torch
from torch.autograd import Function, forward_ad

from . import hip
from .hip import ACT, DpipeHipError, check, dtype_code, lib, ptr, require_cuda, stream


def _contig(t):
    return t if t.is_contiguous() else t.contiguous()


def _al(t):
    """Read-only per-column operand (norm weight / bias, modulation row, gate, bypass gradient) at a 16-byte aligned address: the kernels read these as
    16-byte vectors (csrc/dpipe_common.h, PVec).  Parameters and fresh tensors are aligned already; an odd view (a slice at an offset that is not a multiple
    of 8 elements) is copied once."""
    return t if t is None or t.data_ptr() % 16 == 0 else t.clone()


def _rows2d(x):
    """View x as [rows, cols] with a contiguous last dim and uniform row stride."""
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) != x2.shape[1]):
        x2 = x2.contiguous()
    return x2


# --------------------------------------------------------------------------------------------- GEMM (K1/K6)
# bench.py sets this to a list for one eager step: the full call descriptor (shapes, leading dimensions, batch strides, epilogue
# flags -- no pointers) of every GEMM launch is appended; tools/gemm_replay.py re-issues that launch list as a GEMM-only
# hipGraph over scratch operands and times it with HIP events for the `roofline` object.
GEMM_TRACE = None

# Split-K workspace of the pipelined bf16 GEMM: [4 KiB ticket counters][640 fp32 slabs of 64 KiB], zero-filled once and
# private to one (device, stream) -- launches on one stream are ordered, so slices of two GEMMs never share counters.
_SPLITK_WS = {}
_SPLITK_WS_BYTES = 4096 + 640 * 65536
# Set by the engine while it captures / runs one of several concurrent micro-batch lanes: graphs captured on the same
# capture stream but replayed on different streams must not share ticket counters, so the lane id replaces the stream key.
WS_LANE = None


def _splitk_workspace(device):
    cur = torch.cuda.current_stream(device)
    if WS_LANE is not None:
        key = (device.index, ('lane', WS_LANE))
    else:
        key = (device.index, cur.cuda_stream)
    ws = _SPLITK_WS.get(key)
    if ws is None:
        ws = torch.zeros(_SPLITK_WS_BYTES, dtype=torch.uint8, device=device)
        _SPLITK_WS[key] = ws
    return ws


def gemm(a, b, trans_a, trans_b, M, N, K, out, *, lda, ldb, ldc, batch_outer=1, batch_inner=1,
         stride_a=(0, 0), stride_b=(0, 0), stride_c=(0, 0), bias=None, act=None, alpha=1.0, accumulate=False,
         tile_hint=0, residual=None, ldr=0, colsum=None, colsum_accumulate=False):
    """Raw strided, batched MFMA GEMM:  out = act(alpha * op(a) @ op(b) + bias) (+ out)."""
    require_cuda(a, b, out, bias)
    if a.dtype != b.dtype:
        raise DpipeHipError(f'gemm operand dtypes differ: {a.dtype} vs {b.dtype}')
    dt = dtype_code(a.dtype)
    out_f32 = int(out.dtype == torch.float32 and a.dtype == torch.bfloat16)
    if not out_f32 and out.dtype != a.dtype:
        raise DpipeHipError('gemm output dtype must be the operand dtype or fp32')
    if bias is not None and bias.dtype != a.dtype:
        bias = bias.to(a.dtype)
    ws = _splitk_workspace(a.device) if dt == hip.BF16 else None
    if residual is not None and (residual.dtype != out.dtype or residual.stride(-1) != 1):
        raise DpipeHipError('gemm residual must have the output dtype and a contiguous last dim')
    rc = lib().dpipe_gemm_ex(dt, int(trans_a), int(trans_b), M, N, K, ptr(a), lda, ptr(b), ldb, ptr(out), ldc,
                             batch_outer, batch_inner, stride_a[0], stride_a[1], stride_b[0], stride_b[1],
                             stride_c[0], stride_c[1], ptr(bias), ACT[act], float(alpha), int(accumulate), out_f32,
                             tile_hint, ptr(ws), ws.numel() if ws is not None else 0, ptr(residual), ldr,
                             ptr(colsum), int(colsum_accumulate), stream())
    if rc == -2 and colsum is not None:
        return None                      # not eligible for the fused column sum: the caller takes the two-kernel route
    check(rc, 'dpipe_gemm')
    if GEMM_TRACE is not None:
        GEMM_TRACE.append({'dt': dt, 'ta': int(trans_a), 'tb': int(trans_b), 'M': M, 'N': N, 'K': K, 'lda': lda, 'ldb': ldb, 'ldc': ldc,
                           'bo': batch_outer, 'bi': batch_inner, 'sa': tuple(stride_a), 'sb': tuple(stride_b), 'sc': tuple(stride_c),
                           'bias': bias is not None, 'act': act, 'alpha': float(alpha), 'acc': bool(accumulate), 'out_f32': out_f32,
                           'tile': tile_hint, 'res': residual is not None, 'ldr': ldr, 'colsum': colsum is not None,
                           'colsum_acc': bool(colsum_accumulate)})
    return out


def mm(a, b, trans_a=False, trans_b=False, bias=None, act=None, out=None, out_dtype=None, tile_hint=0, accumulate=False,
       residual=None, colsum=None, colsum_accumulate=False):
    """2-D product of row-major matrices (last dim contiguous): op(a) [M,K] @ op(b) [K,N]."""
    assert a.dim() == 2 and b.dim() == 2
    if a.stride(1) != 1:
        a = a.contiguous()
    if b.stride(1) != 1:
        b = b.contiguous()
    M, K = (a.shape[1], a.shape[0]) if trans_a else a.shape
    Kb, N = (b.shape[1], b.shape[0]) if trans_b else b.shape
    if K != Kb:
        raise DpipeHipError(f'mm shape mismatch: K={K} vs {Kb}')
    if out is None:
        out = torch.empty((M, N), device=a.device, dtype=out_dtype or a.dtype)
    return gemm(a, b, trans_a, trans_b, M, N, K, out, lda=a.stride(0), ldb=b.stride(0), ldc=out.stride(0),
                bias=bias, act=act, tile_hint=tile_hint, accumulate=accumulate, residual=residual,
                ldr=residual.stride(0) if residual is not None else 0, colsum=colsum, colsum_accumulate=colsum_accumulate)


def mm_problem(a, b, trans_a=False, trans_b=False, out=None, bias=None, act=None, accumulate=False, residual=None, colsum=None, colsum_accumulate=False,
               out_dtype=None):
    """One problem of `gemm_group`: the arguments of `mm` (2-D row-major operands, last dim contiguous), resolved to the descriptor fields."""
    assert a.dim() == 2 and b.dim() == 2
    if a.stride(1) != 1:
        a = a.contiguous()
    if b.stride(1) != 1:
        b = b.contiguous()
    M, K = (a.shape[1], a.shape[0]) if trans_a else a.shape
    Kb, N = (b.shape[1], b.shape[0]) if trans_b else b.shape
    if K != Kb:
        raise DpipeHipError(f'mm shape mismatch: K={K} vs {Kb}')
    if out is None:
        out = torch.empty((M, N), device=a.device, dtype=out_dtype or a.dtype)
    return {'a': a, 'b': b, 'ta': int(trans_a), 'tb': int(trans_b), 'M': M, 'N': N, 'K': K, 'out': out, 'lda': a.stride(0), 'ldb': b.stride(0), 'ldc': out.stride(0),
            'bias': bias, 'act': act, 'alpha': 1.0, 'acc': bool(accumulate), 'res': residual, 'ldr': residual.stride(0) if residual is not None else 0,
            'colsum': colsum, 'colsum_acc': bool(colsum_accumulate)}


# A/B switch (bench / tests): 0 = every problem of a group as its own dpipe_gemm_ex launch (the round-3 launch list)
GROUP_GEMM = _os_mod.environ.get('DPIPE_GROUP_GEMM', '1') == '1'


def gemm_group(problems):
    """INDEPENDENT 2-D GEMMs (`mm_problem` dicts; none reads what another writes) as few kernel launches as possible: dpipe_gemm_group puts the problems that
    share a tile geometry into ONE launch of the pipelined kernel (the dgrad and the wgrad of a Linear fill the chip together).  Results are bit-identical to
    issuing the problems one by one WHENEVER the group keeps each problem's own plan (same tile, same split-K: tests/test_gpu_gemm_pipe.py holds that for 13 Linear
    shapes x 2 ring policies).  The one exception: a PAIR whose two plans name different tile geometries -- one big enough for 128^2, the other not --
    is re-planned as a whole onto 64^2 tiles so that it still leaves as one launch (`DPIPE_GEMM_GROUP_UNIFY=0`: two launches, own plans); its results then equal the
    64^2-forced single launches, i.e. differ from the own-plan results by fp32 summation order inside a split-K reduction only.  The register-staged and the DMA form
    of the 128^2 tile are ONE geometry (same LDS, same arithmetic order): they share a launch and stay bit-identical.  -> the list of outputs, or None (nothing launched) when a problem asking for a fused column sum cannot take the
    pipelined kernel (the caller then takes the separate-launch route, as with `mm(..., colsum=...)` returning None)."""
    if not GROUP_GEMM:
        outs = []
        for q in problems:
            r = gemm(q['a'], q['b'], q['ta'], q['tb'], q['M'], q['N'], q['K'], q['out'], lda=q['lda'], ldb=q['ldb'], ldc=q['ldc'], bias=q['bias'], act=q['act'],
                     alpha=q['alpha'], accumulate=q['acc'], residual=q['res'], ldr=q['ldr'], colsum=q['colsum'], colsum_accumulate=q['colsum_acc'])
            if r is None:
                if outs:
                    raise DpipeHipError('gemm_group (ungrouped A/B path): a fused column sum turned out ineligible after earlier problems were launched')
                return None
            outs.append(r)
        return outs
    n = len(problems)
    descs = (hip.GemmDesc * n)()
    any_bf16 = False
    for d, q in zip(descs, problems):
        a, b, out, bias, res = q['a'], q['b'], q['out'], q['bias'], q['res']
        require_cuda(a, b, out, bias, res, q['colsum'])
        if a.dtype != b.dtype:
            raise DpipeHipError(f'gemm operand dtypes differ: {a.dtype} vs {b.dtype}')
        dt = dtype_code(a.dtype)
        out_f32 = int(out.dtype == torch.float32 and a.dtype == torch.bfloat16)
        if not out_f32 and out.dtype != a.dtype:
            raise DpipeHipError('gemm output dtype must be the operand dtype or fp32')
        if bias is not None and bias.dtype != a.dtype:
            bias = q['bias'] = bias.to(a.dtype)
        if res is not None and (res.dtype != out.dtype or res.stride(-1) != 1):
            raise DpipeHipError('gemm residual must have the output dtype and a contiguous last dim')
        any_bf16 = any_bf16 or dt == hip.BF16
        d.dtype, d.transA, d.transB, d.M, d.N, d.K = dt, q['ta'], q['tb'], q['M'], q['N'], q['K']
        d.A, d.lda, d.B, d.ldb, d.C, d.ldc = a.data_ptr(), q['lda'], b.data_ptr(), q['ldb'], out.data_ptr(), q['ldc']
        d.bias, d.act, d.alpha, d.accumulate, d.out_f32 = (bias.data_ptr() if bias is not None else None), (q['act'] if isinstance(q['act'], int) else ACT[q['act']]), float(q['alpha']), int(q['acc']), out_f32
        d.residual, d.ldr = (res.data_ptr() if res is not None else None), q['ldr']
        d.colsum, d.colsum_accumulate = (q['colsum'].data_ptr() if q['colsum'] is not None else None), int(q['colsum_acc'])
        q['_dt'], q['_out_f32'] = dt, out_f32
    ws = _splitk_workspace(problems[0]['a'].device) if any_bf16 else None
    launches = hip.c_int(0)
    rc = lib().dpipe_gemm_group(descs, n, ptr(ws), ws.numel() if ws is not None else 0, hip.ctypes.byref(launches), stream())
    if rc == -2 and any(q['colsum'] is not None or (isinstance(q['act'], int) and q['act'] >= hip.ACT_GEGLU_BWD) for q in problems):
        return None          # (fused column sum / GEGLU epilogue not available for this problem: the caller takes the separate-launch route)
    check(rc, 'dpipe_gemm_group')
    if GEMM_TRACE is not None:
        for i, q in enumerate(problems):
            GEMM_TRACE.append({'dt': q['_dt'], 'ta': q['ta'], 'tb': q['tb'], 'M': q['M'], 'N': q['N'], 'K': q['K'], 'lda': q['lda'], 'ldb': q['ldb'], 'ldc': q['ldc'],
                               'bo': 1, 'bi': 1, 'sa': (0, 0), 'sb': (0, 0), 'sc': (0, 0), 'bias': q['bias'] is not None, 'act': q['act'], 'alpha': float(q['alpha']),
                               'acc': q['acc'], 'out_f32': q['_out_f32'], 'tile': 0, 'res': q['res'] is not None, 'ldr': q['ldr'], 'colsum': q['colsum'] is not None,
                               'colsum_acc': q['colsum_acc'], 'grp': i, 'grp_n': n, 'grp_l': int(launches.value)})
    return [q['out'] for q in problems]


# Gradient-accumulation fusion (set by the engine): when a parameter already owns a .grad buffer (micro-batch > 0 of a
# step, or the persistent buffers of the hipGraph path) the parameter-gradient kernels add into it in their epilogue
# (wgrad GEMM `accumulate`, column-sum / slab-sum `accumulate`) and autograd receives None -- this removes one
# elementwise add launch per parameter per micro-batch (DeepSpeed accumulates the same way into .grad in the
# parameter dtype).
FUSE_GRAD_ACCUM = False


# "First micro-batch of a step" graphs (engine config `store_first_micro_batch`): while the engine captures a lane's FIRST-micro-batch graph it sets GRAD_STORE to
# a dict; the first fused gradient write into a persistent .grad buffer inside that graph then STORES (accumulate flag off) and registers the buffer, later writes to
# the same buffer in the same micro-batch accumulate as usual.  The step end then has no accumulators to zero (16 GB of writes per SDXL step on four lanes).
GRAD_STORE = None


def _acc(tgt):
    """accumulate flag of a fused gradient write into `tgt` (a persistent .grad buffer, a packed view of several, or None = fresh output)"""
    if tgt is None:
        return False
    if GRAD_STORE is None:
        return True
    key = tgt.data_ptr()
    if key in GRAD_STORE:
        return True
    GRAD_STORE[key] = tgt.numel() * tgt.element_size()
    return False


def _acc_all(fused, *tgts):
    """accumulate flag shared by the parameter gradients one kernel writes together (gamma + beta): every buffer is registered, the first one's answer is returned
    (they are written by the same set of kernels, so they are first-touched together)"""
    if not fused:
        return 0
    flags = [_acc(t) for t in tgts if t is not None]
    return int(flags[0]) if flags else 0


def _accum_target(param):
    if not FUSE_GRAD_ACCUM or param is None or not param.is_leaf:
        return None
    g = param.grad
    if g is None or g.dtype != param.dtype or not g.is_contiguous() or g.shape != param.shape:
        return None
    return g


# (Round 2 / 3 negative result: wgrad forked onto a side stream next to dgrad -- `parallel_wgrad`, no gain at micro-batch 1 once the pair leaves as ONE grouped launch; removed
#  in round 5 together with its side streams.)
# Bias gradient inside the wgrad GEMM (dpipe_gemm_ex `colsum`) and residual add inside the output projection's epilogue.
# Same-box A/B on the SDXL step: +2.7 % and +0.3 % images/s (env switches kept for that measurement).
import os as _os
FUSE_BIAS_GRAD = _os.environ.get('DPIPE_FUSE_BIAS_GRAD', '1') == '1'
FUSE_RESIDUAL = _os.environ.get('DPIPE_FUSE_RESIDUAL', '1') == '1'
class _LinearFn(Function):
    """y = x W^T + b (+ residual)  (nn.Linear; reference: models/wan/model.py:120-122,138-142,270-272).  `residual` folds the
    transformer block's "x + proj(...)" add into the GEMM epilogue; its gradient is the incoming gradient itself."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual):
        x2 = _rows2d(x)
        if x2.dtype != weight.dtype:
            x2 = x2.to(weight.dtype)
        res2 = None
        if residual is not None:
            res2 = _rows2d(residual)
            if res2.dtype != weight.dtype:
                res2 = res2.to(weight.dtype)
        y = mm(x2, weight, False, True, bias=bias, residual=res2)
        ctx.save_for_backward(x2, weight, bias)
        ctx.has_bias = bias is not None
        ctx.has_res = residual is not None
        ctx.x_shape = x.shape
        ctx.x_dtype = x.dtype
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, gy):
        x2, weight, bias = ctx.saved_tensors
        gy2 = _rows2d(gy)
        if gy2.dtype != weight.dtype:
            gy2 = gy2.to(weight.dtype)
        gx = gw = gb = None
        need_w = ctx.needs_input_grad[1]
        need_b = ctx.has_bias and ctx.needs_input_grad[2]

        # accumulate flags: asked ONCE per target.  `_acc` registers a buffer in GRAD_STORE the first time it is asked (the first-micro-batch graphs store instead of
        # accumulating); a launch that is then refused (gemm_group / mm(colsum=...) returning None: rc -2, not pipe-eligible) falls through to the unfused kernels,
        # which must see the SAME answer -- a second `_acc` call would say "accumulate" and the store graph would add into a stale buffer, step after step
        tw = _accum_target(weight) if need_w else None
        tb = _accum_target(bias) if need_b else None
        acc_w = _acc(tw) if need_w else False
        acc_b = _acc(tb) if need_b else False

        def param_grads():
            gw_ = gb_ = None
            if FUSE_BIAS_GRAD and need_w and need_b and gy2.dtype == torch.bfloat16:
                # one launch: dW (+)= dy^T . x with db (+)= column sums of dy taken from the A fragments inside the GEMM
                w_out = tw if tw is not None else torch.empty(weight.shape, device=weight.device, dtype=weight.dtype)
                b_out = tb if tb is not None else torch.empty(bias.shape, device=bias.device, dtype=bias.dtype)
                if mm(gy2, x2, True, False, out=w_out, accumulate=acc_w, colsum=b_out, colsum_accumulate=acc_b) is not None:
                    return (None if tw is not None else w_out), (None if tb is not None else b_out)
            if need_w:
                if tw is not None:
                    mm(gy2, x2, True, False, out=tw, accumulate=acc_w)        # dW += dy^T . x  (fused accumulation)
                else:
                    gw_ = mm(gy2, x2, True, False)                            # dW = dy^T . x
            if need_b:
                gb_ = column_sum(gy2, out=tb, accumulate=acc_b)
                if tb is not None:
                    gb_ = None
            return gw_, gb_

        if ctx.needs_input_grad[0] and need_w and gy2.dtype == torch.bfloat16:
            # dgrad and wgrad (+ the bias column sums inside it) as ONE grouped launch: dx = dy . W next to dW (+)= dy^T . x -- independent problems that share
            # dy, each filling well under half of the chip at micro-batch 1
            w_out = tw if tw is not None else torch.empty(weight.shape, device=weight.device, dtype=weight.dtype)
            fuse_b = FUSE_BIAS_GRAD and need_b
            b_out = (tb if tb is not None else torch.empty(bias.shape, device=bias.device, dtype=bias.dtype)) if fuse_b else None
            gx2 = torch.empty((gy2.shape[0], weight.shape[1]), device=gy2.device, dtype=gy2.dtype)
            done = gemm_group([mm_problem(gy2, weight, False, False, out=gx2),
                               mm_problem(gy2, x2, True, False, out=w_out, accumulate=acc_w, colsum=b_out, colsum_accumulate=acc_b if fuse_b else False)])
            if done is not None:
                gx = gx2.view(ctx.x_shape)
                if gx.dtype != ctx.x_dtype:
                    gx = gx.to(ctx.x_dtype)
                gw = None if tw is not None else w_out
                if fuse_b:
                    gb = None if tb is not None else b_out
                elif need_b:
                    gb = column_sum(gy2, out=tb, accumulate=acc_b)
                    if tb is not None:
                        gb = None
                gres = gy if (ctx.has_res and ctx.needs_input_grad[3]) else None
                return gx, gw, gb, gres
        if ctx.needs_input_grad[0]:
            gx = mm(gy2, weight, False, False).view(ctx.x_shape)          # dx = dy . W
            if gx.dtype != ctx.x_dtype:
                gx = gx.to(ctx.x_dtype)
        gw, gb = param_grads()
        gres = gy if (ctx.has_res and ctx.needs_input_grad[3]) else None
        return gx, gw, gb, gres


def linear(x, weight, bias=None, residual=None):
    if residual is not None and not FUSE_RESIDUAL:
        return gated_residual(residual, _LinearFn.apply(x, weight, bias, None))
    return _LinearFn.apply(x, weight, bias, residual)


# ------------------------------------------------------------------------- fused projections (K1: fused QKV)
def packed_view(tensors):
    """[sum rows, ...] view over tensors that sit back to back in one storage (row blocks of one matrix), else None."""
    t0 = tensors[0]
    nxt = t0.data_ptr()
    for t in tensors:
        if t is None or not t.is_contiguous() or t.data_ptr() != nxt or t.shape[1:] != t0.shape[1:] or t.dtype != t0.dtype \
                or t.untyped_storage().data_ptr() != t0.untyped_storage().data_ptr():
            return None
        nxt += t.numel() * t.element_size()
    rows = sum(t.shape[0] for t in tensors)
    return torch.as_strided(t0.detach(), (rows, *t0.shape[1:]), t0.stride(), t0.storage_offset())


@torch.no_grad()
def pack_parameters(params):
    """Re-home parameters (row blocks: [N_i, K] weights or [N_i] biases) into one buffer, in order, keeping the Parameter
    objects (optimizers / state dicts keep working); existing gradients are packed the same way."""
    buf = torch.cat([p.data for p in params], dim=0)
    off = 0
    for p in params:
        n = p.shape[0]
        p.data = buf[off:off + n]
        off += n
    if all(p.grad is not None for p in params):
        gbuf = torch.cat([p.grad for p in params], dim=0)
        off = 0
        for p in params:
            n = p.shape[0]
            p.grad = gbuf[off:off + n]
            off += n


class _FusedLinearFn(Function):
    """y = x [W_1; ...; W_n]^T + [b_1; ...; b_n] -- several nn.Linear layers that share their input (to_q / to_k / to_v of
    self attention, to_k / to_v of cross attention, CLIP q/k/v_proj) as ONE GEMM each for forward, dgrad (K = sum N_i) and
    wgrad, on weights packed back to back (`pack_parameters`).  The layers stay separate Parameters (LoRA / checkpoints
    address them one by one: models/base.py:262-270)."""

    @staticmethod
    def forward(ctx, x, n, *params):
        ws, bs = params[:n], params[n:]
        x2 = _rows2d(x)
        if x2.dtype != ws[0].dtype:
            x2 = x2.to(ws[0].dtype)
        wcat = packed_view(ws)
        has_bias = bs[0] is not None
        bcat = packed_view(bs) if has_bias else None
        if wcat is None or (has_bias and bcat is None):
            raise DpipeHipError('fused_linear: parameters are not packed (call ops.pack_parameters first)')
        y = mm(x2, wcat, False, True, bias=bcat)
        ctx.save_for_backward(x2, *params)
        ctx.n, ctx.has_bias, ctx.x_shape, ctx.x_dtype = n, has_bias, x.shape, x.dtype
        return y.view(*x.shape[:-1], wcat.shape[0])

    @staticmethod
    def backward(ctx, gy):
        x2, *params = ctx.saved_tensors
        n = ctx.n
        ws, bs = params[:n], params[n:]
        gy2 = _rows2d(gy)
        if gy2.dtype != ws[0].dtype:
            gy2 = gy2.to(ws[0].dtype)
        wcat = packed_view(ws)
        need_dx = ctx.needs_input_grad[0]
        state = {'gx2': None}

        def dgrad():
            return mm(gy2, wcat, False, False)                                     # dx = dy . [W_1; ...; W_n], K = sum N_i

        def plan(group, first):
            """Where the packed gradient of a parameter group goes: -> (mode, out, accumulate).  'skip': nobody needs it; 'install': first micro-batch under
            fused accumulation, a fresh packed buffer becomes the parameters' .grad; 'accum': accumulate into the packed .grad in the epilogue; 'return':
            hand row-block views to autograd."""
            if not any(ctx.needs_input_grad[2 + first + i] for i in range(n)):
                return 'skip', None, False
            if FUSE_GRAD_ACCUM:
                grads = [p.grad for p in group]
                if all(g is None for g in grads):
                    return 'install', None, False
                if all(g is not None for g in grads):
                    gv = packed_view(grads)
                    if gv is not None:
                        return 'accum', gv, _acc(gv)
            return 'return', None, False

        def finish(group, mode, gcat):
            if mode in ('skip', 'accum'):
                return [None] * n
            out, off = [], 0
            for p in group:
                blk = gcat[off:off + p.shape[0]]
                off += p.shape[0]
                if mode == 'install':
                    p.grad = blk
                else:
                    out.append(blk)
            return out if mode == 'return' else [None] * n

        wmode, w_out, w_acc = plan(ws, 0)
        bmode, b_out, b_acc = plan(bs, n) if ctx.has_bias else ('skip', None, False)
        gwcat = gbcat = None
        if wmode != 'skip' and gy2.dtype == torch.bfloat16 and (need_dx or bmode != 'skip'):
            # ONE grouped launch: dgrad next to the packed wgrad, the packed bias gradient as column sums inside the wgrad
            if w_out is None:
                w_out = torch.empty(wcat.shape, device=wcat.device, dtype=wcat.dtype)
            fuse_b = FUSE_BIAS_GRAD and bmode != 'skip'
            if fuse_b and b_out is None:
                b_out = torch.empty((wcat.shape[0],), device=wcat.device, dtype=bs[0].dtype)
            probs = [mm_problem(gy2, x2, True, False, out=w_out, accumulate=w_acc, colsum=b_out if fuse_b else None, colsum_accumulate=b_acc)]
            if need_dx:
                state['gx2'] = torch.empty((gy2.shape[0], wcat.shape[1]), device=gy2.device, dtype=gy2.dtype)
                probs.insert(0, mm_problem(gy2, wcat, False, False, out=state['gx2']))
            if gemm_group(probs) is not None:
                gwcat = w_out
                gbcat = b_out if fuse_b else None
            else:
                state['gx2'] = None
        if need_dx and state['gx2'] is None:
            state['gx2'] = dgrad()
        gx = None
        if need_dx:
            gx = state['gx2'].view(ctx.x_shape)
            if gx.dtype != ctx.x_dtype:
                gx = gx.to(ctx.x_dtype)
        if wmode != 'skip' and gwcat is None:
            gwcat = mm(gy2, x2, True, False, out=w_out, accumulate=w_acc)
        if bmode != 'skip' and gbcat is None:
            gbcat = column_sum(gy2, out=b_out if bmode == 'accum' else None, accumulate=b_acc)
        gws = finish(ws, wmode, gwcat)
        gbs = finish(bs, bmode, gbcat) if ctx.has_bias else [None] * n
        return (gx, None, *gws, *gbs)


def fused_linear(x, weights, biases=None):
    """[.., K] -> [.., sum N_i].  weights: list of [N_i, K] Parameters; biases: matching list or None."""
    weights = list(weights)
    biases = list(biases) if biases is not None and biases[0] is not None else [None] * len(weights)
    if packed_view(weights) is None:
        pack_parameters(weights)
    if biases[0] is not None and packed_view(biases) is None:
        pack_parameters(biases)
    return _FusedLinearFn.apply(x, len(weights), *weights, *biases)


class _SplitColumnsFn(Function):
    """[..., sum w_i] -> column-block views (w_i wide each) with ONE concatenation as the backward -- torch's own slicing would give every consumer a
    zero-filled full-width gradient plus an add (3 launches per slice).  Used to hand the per-block K / V slices of one batched context projection
    (nn.Transformer cross attention: every block of a Transformer2DModel projects the same 77 text tokens) to their blocks."""

    @staticmethod
    def forward(ctx, x, widths):
        ctx.widths, ctx.shape, ctx.dtype = widths, x.shape, x.dtype
        ctx.set_materialize_grads(False)
        outs, off = [], 0
        for w in widths:
            outs.append(x[..., off:off + w])
            off += w
        return tuple(outs)

    @staticmethod
    def backward(ctx, *grads):
        parts = []
        for g, w in zip(grads, ctx.widths):
            parts.append(g if g is not None else torch.zeros(*ctx.shape[:-1], w, device=next(t for t in grads if t is not None).device, dtype=ctx.dtype))
        return torch.cat(parts, dim=-1), None


def split_columns(x, widths):
    return _SplitColumnsFn.apply(x, tuple(int(w) for w in widths))


def column_sum(x2, out=None, out_dtype=None, accumulate=None):
    """sum over the rows of a [rows, cols] matrix (fp32 accumulate, two-stage slab reduction).  `out` given: out += sum
    (the fused gradient-accumulation form; `accumulate=False`: out = sum); else a new [cols] tensor in x2's dtype (or out_dtype)."""
    require_cuda(x2, out)
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    rows, cols = x2.shape
    accumulate = (out is not None) if accumulate is None else bool(accumulate and out is not None)
    if out is None:
        out = torch.empty(cols, device=x2.device, dtype=out_dtype or x2.dtype)
    ws = torch.empty(lib().dpipe_norm_slabs(rows) * cols, device=x2.device, dtype=torch.float32)
    check(lib().dpipe_colsum(ptr(x2), rows, cols, x2.stride(0), ptr(out), ptr(ws), dtype_code(x2.dtype), dtype_code(out.dtype),
                             int(accumulate), stream()), 'colsum')
    return out


# ---------------------------------------------------------------------------- precise row linear (round 6: fp32 per-channel addends)
PRECISE_ADDENDS = _os.environ.get('DPIPE_PRECISE_ADDENDS', '1') == '1'      # A/B switch: 0 = the time-embedding rows in bf16 like every other activation (rounds 1 - 5)


class _PreciseRowLinearFn(Function):
    """y = act(x) W^T + bias (+ extra) for a FEW fp32 rows x [R, K] whose result is a per-channel addend (the SDXL time embedding: diffusers TimestepEmbedding and
    ResnetBlock2D.time_emb_proj behind models/sdxl.py:797-865, `hidden_states + temb[:, :, None, None]`).  W / bias / extra are the bf16 parameters; the row keeps fp32
    accuracy through the bf16 MFMA GEMM as a hi / lo bf16 row pair (csrc/elementwise.hip: rowsplit / rowcombine).  `pair` = False: fp32 [R, N]; True: the bf16 hi / lo
    pair [2, R, N] a convolution takes as its bias (`conv2d_nhwc(..., bias=pair)`: `extra` = that convolution's own bias vector, whose gradient is taken here).
    Why: a bf16 rounding of such a row shifts EVERY pixel of a channel together -- a coherent error the gradient norm of the network reacts to (tools/coherent_noise_probe.py:
    rounding these rows alone moves the norm by 2 - 3e-4, every other activation of the network together by 5e-5)."""

    @staticmethod
    def forward(ctx, x, weight, bias, extra, act, pair):
        require_cuda(x, weight, bias, extra)
        if weight.dtype != torch.bfloat16:
            raise DpipeHipError('precise_row_linear: bf16 parameters only (fp32 models take ops.linear)')
        x32 = _contig(x.reshape(-1, x.shape[-1]))
        if x32.dtype != torch.float32:
            x32 = x32.float()
        R, K = x32.shape
        N = weight.shape[0]
        hl = torch.empty((2 * R, K), device=x.device, dtype=torch.bfloat16)
        check(lib().dpipe_rowsplit_fwd(ptr(x32), ptr(hl), R * K, ACT[act], stream()), 'rowsplit_fwd')
        g = mm(hl, weight, False, True, out_dtype=torch.float32)
        out = torch.empty((2, R, N), device=x.device, dtype=torch.bfloat16) if pair else torch.empty((R, N), device=x.device, dtype=torch.float32)
        check(lib().dpipe_rowcombine_fwd(ptr(g), ptr(bias), ptr(extra), None if pair else ptr(out), ptr(out) if pair else None, R, N, stream()), 'rowcombine_fwd')
        ctx.save_for_backward(x32, hl, weight, bias, extra)
        ctx.act, ctx.pair, ctx.x_shape = act, pair, x.shape
        return out if pair else out.view(*x.shape[:-1], N)

    @staticmethod
    def backward(ctx, gout):
        x32, hl, weight, bias, extra = ctx.saved_tensors
        R, K = x32.shape
        N = weight.shape[0]
        g1 = gout[0] if ctx.pair else gout.reshape(R, N)            # a pair's two rows carry the same gradient (the convolution hands back an expanded view)
        g1 = _contig(g1)
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        tb = _accum_target(bias) if (bias is not None and ctx.needs_input_grad[2]) else None
        te = _accum_target(extra) if (extra is not None and ctx.needs_input_grad[3]) else None
        b_out = (tb if tb is not None else torch.empty_like(bias)) if (bias is not None and ctx.needs_input_grad[2]) else None
        e_out = (te if te is not None else torch.empty_like(extra)) if (extra is not None and ctx.needs_input_grad[3]) else None
        gy = torch.empty((2 * R, N), device=g1.device, dtype=torch.bfloat16)
        check(lib().dpipe_rowcombine_bwd(ptr(g1), dtype_code(g1.dtype), ptr(gy), ptr(b_out), int(_acc(tb)), ptr(e_out), int(_acc(te)), R, N, stream()), 'rowcombine_bwd')
        gx = gw = None
        tw = _accum_target(weight) if need_w else None
        acc_w = _acc(tw) if need_w else False
        w_out = (tw if tw is not None else torch.empty_like(weight)) if need_w else None
        ds = torch.empty((2 * R, K), device=g1.device, dtype=torch.bfloat16) if need_x else None
        done = None
        if need_x and need_w:
            done = gemm_group([mm_problem(gy, weight, False, False, out=ds), mm_problem(gy, hl, True, False, out=w_out, accumulate=acc_w)])
        if done is None:
            if need_x:
                mm(gy, weight, False, False, out=ds)
            if need_w:
                mm(gy, hl, True, False, out=w_out, accumulate=acc_w)          # dW (+)= gy^T (hi + lo): exact over the 2R rows
        if need_x:
            dx = torch.empty_like(x32)
            check(lib().dpipe_rowsplit_bwd(ptr(ds), ptr(x32), ptr(dx), R * K, ACT[ctx.act], stream()), 'rowsplit_bwd')
            gx = dx.view(ctx.x_shape)
        if need_w and tw is None:
            gw = w_out
        return gx, gw, (None if tb is not None else b_out), (None if te is not None else e_out), None, None


def precise_row_linear(x, weight, bias=None, extra=None, act=None, pair=False):
    """see _PreciseRowLinearFn.  x: [..., K] fp32 (a few rows); -> fp32 [..., N], or with `pair` the bf16 hi / lo pair [2, R, N]."""
    return _PreciseRowLinearFn.apply(x, weight, bias, extra, act, bool(pair))


# ------------------------------------------------------------------------------------------- activations (K6)
class _ActFn(Function):
    @staticmethod
    def forward(ctx, x, act):
        require_cuda(x)
        xc = _contig(x)
        y = torch.empty_like(xc)
        check(lib().dpipe_act_fwd(ptr(xc), ptr(y), xc.numel(), dtype_code(xc.dtype), ACT[act], stream()), 'act_fwd')
        ctx.save_for_backward(xc)
        ctx.act = act
        return y

    @staticmethod
    def backward(ctx, gy):
        (xc,) = ctx.saved_tensors
        gy = _contig(gy)
        gx = torch.empty_like(xc)
        check(lib().dpipe_act_bwd(ptr(xc), ptr(gy), ptr(gx), xc.numel(), dtype_code(xc.dtype), ACT[ctx.act], stream()), 'act_bwd')
        return gx, None


def gelu_tanh(x):
    return _ActFn.apply(x, 'gelu_tanh')


def gelu(x):
    return _ActFn.apply(x, 'gelu_erf')


def silu(x):
    return _ActFn.apply(x, 'silu')


def quick_gelu(x):
    return _ActFn.apply(x, 'quick_gelu')


class _GegluFn(Function):
    """diffusers GEGLU: h, gate = x.chunk(2, -1); h * gelu(gate)."""

    @staticmethod
    def forward(ctx, x, act):
        x2 = _contig(_rows2d(x))
        H = x2.shape[1] // 2
        y = torch.empty((x2.shape[0], H), device=x.device, dtype=x.dtype)
        check(lib().dpipe_geglu_fwd(ptr(x2), ptr(y), x2.shape[0], H, dtype_code(x.dtype), ACT[act], stream()), 'geglu_fwd')
        ctx.save_for_backward(x2)
        ctx.act = act
        ctx.shape = x.shape
        return y.view(*x.shape[:-1], H)

    @staticmethod
    def backward(ctx, gy):
        (x2,) = ctx.saved_tensors
        gy2 = _contig(_rows2d(gy))
        gx = torch.empty_like(x2)
        check(lib().dpipe_geglu_bwd(ptr(x2), ptr(gy2), ptr(gx), x2.shape[0], x2.shape[1] // 2, dtype_code(x2.dtype), ACT[ctx.act], stream()), 'geglu_bwd')
        return gx.view(ctx.shape), None


def geglu(x, act='gelu_erf'):
    return _GegluFn.apply(x, act)


# DPIPE_FUSE_GEGLU_BWD=1: the GEGLU backward in the epilogue of the output Linear's dgrad GEMM (DPIPE_ACT_GEGLU_BWD).  OFF by default -- measured, round 6, same box, two
# pairs (profiles/r6s_bench_geglu_bwd_epilogue_ab.jsonl): 355.5 / 355.0 ms per step fused against 353.0 / 352.7 with the separate pass (r6r, before the cheaper GELU:
# 358.1 / 358.0 against 355.9 / 356.3).  The fusion saves the dy round trip and a launch, but moves the GELU / GELU' arithmetic of 5 M elements per call from an element-wise
# kernel that the other lanes' GEMMs run NEXT TO (VALU work under their MFMA work) into the tail of GEMM workgroups, where it holds the CU's LDS and registers
# while the matrix pipe idles.  Parity-tested either way (tests/test_gpu_geglu_linear.py).
FUSE_GEGLU_BWD = _os_mod.environ.get('DPIPE_FUSE_GEGLU_BWD', '0') == '1'


class _GegluLinearFn(Function):
    """out = Linear(geglu(h)) (+ residual): diffusers FeedForward's [GEGLU's multiply, Dropout, Linear] tail as ONE autograd node, so that the backward of the
    GEGLU rides the epilogue of the Linear's dgrad GEMM (DPIPE_ACT_GEGLU_BWD): dy = dout . W never reaches memory, dh = [dy * act(gate) | dy * value * act'(gate)]
    is written by the GEMM itself -- the element-wise geglu_bwd pass (3 reads + 2 writes of [rows, H]-sized tensors) is gone.  Grouped with the wgrad
    dW (+)= dout^T . y as in _LinearFn.  Falls back to the two-pass route whenever the fused launch is refused (fp32 parity mode, odd shapes)."""

    @staticmethod
    def forward(ctx, h, weight, bias, residual, act):
        h2 = _contig(_rows2d(h))
        H = h2.shape[1] // 2
        y = torch.empty((h2.shape[0], H), device=h.device, dtype=h.dtype)
        check(lib().dpipe_geglu_fwd(ptr(h2), ptr(y), h2.shape[0], H, dtype_code(h.dtype), ACT[act], stream()), 'geglu_fwd')
        if y.dtype != weight.dtype:
            y = y.to(weight.dtype)
        res2 = None
        if residual is not None:
            res2 = _rows2d(residual)
            if res2.dtype != weight.dtype:
                res2 = res2.to(weight.dtype)
        out = mm(y, weight, False, True, bias=bias, residual=res2)
        ctx.save_for_backward(h2, y, weight, bias)
        ctx.act, ctx.h_shape, ctx.has_bias, ctx.has_res = act, h.shape, bias is not None, residual is not None
        return out.view(*h.shape[:-1], weight.shape[0])

    @staticmethod
    def backward(ctx, gout):
        h2, y, weight, bias = ctx.saved_tensors
        go2 = _rows2d(gout)
        if go2.dtype != weight.dtype:
            go2 = go2.to(weight.dtype)
        need_h, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[1]
        need_b = ctx.has_bias and ctx.needs_input_grad[2]
        gres = gout if (ctx.has_res and ctx.needs_input_grad[3]) else None
        tw = _accum_target(weight) if need_w else None
        tb = _accum_target(bias) if need_b else None
        acc_w = _acc(tw) if need_w else False
        acc_b = _acc(tb) if need_b else False
        H = h2.shape[1] // 2
        gh = gw = gb = None
        fused_ok = FUSE_GEGLU_BWD and need_h and go2.dtype == torch.bfloat16 and h2.dtype == torch.bfloat16
        if fused_ok:
            gh2 = torch.empty_like(h2)
            dgrad = mm_problem(go2, weight, False, False, out=gh2, residual=h2, act=ACT[ctx.act] | hip.ACT_GEGLU_BWD)
            if need_w:
                w_out = tw if tw is not None else torch.empty(weight.shape, device=weight.device, dtype=weight.dtype)
                fuse_b = FUSE_BIAS_GRAD and need_b
                b_out = (tb if tb is not None else torch.empty(bias.shape, device=bias.device, dtype=bias.dtype)) if fuse_b else None
                done = gemm_group([dgrad, mm_problem(go2, y, True, False, out=w_out, accumulate=acc_w, colsum=b_out, colsum_accumulate=acc_b if fuse_b else False)])
                if done is not None:
                    gw = None if tw is not None else w_out
                    if fuse_b:
                        gb = None if tb is not None else b_out
                    elif need_b:
                        gb = column_sum(go2, out=tb, accumulate=acc_b)
                        if tb is not None:
                            gb = None
                    return gh2.view(ctx.h_shape), gw, gb, gres, None
            else:
                done = gemm_group([dgrad])
                if done is not None:
                    gb = None
                    if need_b:
                        gb = column_sum(go2, out=tb, accumulate=acc_b)
                        if tb is not None:
                            gb = None
                    return gh2.view(ctx.h_shape), None, gb, gres, None
        # two-pass route: plain dgrad, then the element-wise GEGLU backward -- the dgrad still leaves in ONE grouped launch with the wgrad (as in _LinearFn)
        if need_h and need_w and go2.dtype == torch.bfloat16 and h2.dtype == torch.bfloat16:
            w_out = tw if tw is not None else torch.empty(weight.shape, device=weight.device, dtype=weight.dtype)
            fuse_b = FUSE_BIAS_GRAD and need_b
            b_out = (tb if tb is not None else torch.empty(bias.shape, device=bias.device, dtype=bias.dtype)) if fuse_b else None
            gy = torch.empty((go2.shape[0], H), device=go2.device, dtype=go2.dtype)
            done = gemm_group([mm_problem(go2, weight, False, False, out=gy),
                               mm_problem(go2, y, True, False, out=w_out, accumulate=acc_w, colsum=b_out, colsum_accumulate=acc_b if fuse_b else False)])
            if done is not None:
                gh2 = torch.empty_like(h2)
                check(lib().dpipe_geglu_bwd(ptr(h2), ptr(gy), ptr(gh2), h2.shape[0], H, dtype_code(h2.dtype), ACT[ctx.act], stream()), 'geglu_bwd')
                gw = None if tw is not None else w_out
                if fuse_b:
                    gb = None if tb is not None else b_out
                elif need_b:
                    gb = column_sum(go2, out=tb, accumulate=acc_b)
                    if tb is not None:
                        gb = None
                return gh2.view(ctx.h_shape), gw, gb, gres, None
        if need_h:
            gy = mm(go2, weight, False, False)
            if gy.dtype != h2.dtype:
                gy = gy.to(h2.dtype)
            gh2 = torch.empty_like(h2)
            check(lib().dpipe_geglu_bwd(ptr(h2), ptr(_contig(gy)), ptr(gh2), h2.shape[0], H, dtype_code(h2.dtype), ACT[ctx.act], stream()), 'geglu_bwd')
            gh = gh2.view(ctx.h_shape)
        if need_w:
            if FUSE_BIAS_GRAD and need_b and go2.dtype == torch.bfloat16:
                w_out = tw if tw is not None else torch.empty(weight.shape, device=weight.device, dtype=weight.dtype)
                b_out = tb if tb is not None else torch.empty(bias.shape, device=bias.device, dtype=bias.dtype)
                if mm(go2, y, True, False, out=w_out, accumulate=acc_w, colsum=b_out, colsum_accumulate=acc_b) is not None:
                    return gh, (None if tw is not None else w_out), (None if tb is not None else b_out), gres, None
            if tw is not None:
                mm(go2, y, True, False, out=tw, accumulate=acc_w)
            else:
                gw = mm(go2, y, True, False)
        if need_b:
            gb = column_sum(go2, out=tb, accumulate=acc_b)
            if tb is not None:
                gb = None
        return gh, gw, gb, gres, None


def geglu_linear(h, weight, bias=None, residual=None, act='gelu_erf'):
    """Linear(geglu(h)) (+ residual) with the GEGLU backward fused into the dgrad GEMM's epilogue (see _GegluLinearFn)."""
    if residual is not None and not FUSE_RESIDUAL:
        return gated_residual(residual, _GegluLinearFn.apply(h, weight, bias, None, act))
    return _GegluLinearFn.apply(h, weight, bias, residual, act)


# ----------------------------------------------------------------------------------------- gated residual (K5)
class _GatedResidualFn(Function):
    """out = x + y * gate  with gate [B, D] broadcast over the rows of each sample (models/wan/model.py:301,308)."""

    @staticmethod
    def forward(ctx, x, y, gate):
        require_cuda(x, y, gate)
        xc, yc = _contig(x), _contig(y)
        D = xc.shape[-1]
        rows = xc.numel() // D
        gc = None
        rows_per_gate = rows
        if gate is not None:
            gc = _contig(gate).reshape(-1, D)
            rows_per_gate = rows // gc.shape[0]
        out = torch.empty_like(xc)
        check(lib().dpipe_gated_residual_fwd(ptr(xc), ptr(yc), ptr(_al(gc)), ptr(out), rows, D, rows_per_gate,
                                             dtype_code(xc.dtype), dtype_code(gc.dtype) if gc is not None else dtype_code(xc.dtype),
                                             stream()), 'gated_residual_fwd')
        ctx.save_for_backward(yc, gc)
        ctx.gate_shape = None if gate is None else gate.shape
        ctx.rows_per_gate = rows_per_gate
        return out

    @staticmethod
    def backward(ctx, gout):
        yc, gc = ctx.saved_tensors
        gout = _contig(gout)
        if gc is None:
            return gout, gout, None
        D = yc.shape[-1]
        batches = gc.shape[0]
        slabs = lib().dpipe_gated_residual_slabs(ctx.rows_per_gate)
        ws = torch.empty(batches * slabs * D, device=yc.device, dtype=torch.float32)
        gy = torch.empty_like(yc)
        dgate = torch.empty_like(gc)
        check(lib().dpipe_gated_residual_bwd(ptr(gout), ptr(yc), ptr(gc), ptr(gy), ptr(dgate), ptr(ws), batches,
                                             ctx.rows_per_gate, D, dtype_code(yc.dtype), dtype_code(gc.dtype), stream()),
              'gated_residual_bwd')
        return gout, gy, dgate.view(ctx.gate_shape)


def gated_residual(x, y, gate=None):
    return _GatedResidualFn.apply(x, y, gate)


# ------------------------------------------------------------------------------------------------ norms (K2/K5)
class _RMSNormFn(Function):
    """WanRMSNorm: _norm(x.float()).type_as(x) * weight  (models/wan/model.py:70-86)."""

    @staticmethod
    def forward(ctx, x, weight, eps):
        require_cuda(x, weight)
        x2 = _contig(_rows2d(x))
        rows, cols = x2.shape
        y = torch.empty_like(x2)
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
        wd = dtype_code(weight.dtype) if weight is not None else dtype_code(x.dtype)
        check(lib().dpipe_rmsnorm_fwd(ptr(x2), ptr(_al(weight)), ptr(y), ptr(rstd), rows, cols, eps, dtype_code(x.dtype), wd, stream()), 'rmsnorm_fwd')
        ctx.save_for_backward(x2, weight, rstd)
        ctx.shape = x.shape
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, gy):
        x2, weight, rstd = ctx.saved_tensors
        rows, cols = x2.shape
        gy2 = _contig(_rows2d(gy))
        gx = torch.empty_like(x2)
        dw = ws = None
        fused = False
        if weight is not None and ctx.needs_input_grad[1]:
            dw = _accum_target(weight)
            fused = dw is not None
            if dw is None:
                dw = torch.empty_like(weight)
            ws = torch.empty(lib().dpipe_norm_slabs(rows) * cols, device=x2.device, dtype=torch.float32)
        wd = dtype_code(weight.dtype) if weight is not None else dtype_code(x2.dtype)
        check(lib().dpipe_rmsnorm_bwd(ptr(x2), ptr(_al(weight)), ptr(gy2), ptr(rstd), ptr(gx), ptr(dw), ptr(ws), rows, cols,
                                      dtype_code(x2.dtype), wd, _acc_all(fused, dw), stream()), 'rmsnorm_bwd')
        return gx.view(ctx.shape), (None if fused else dw), None


def rms_norm(x, weight=None, eps=1e-6):
    return _RMSNormFn.apply(x, weight, eps)


class _LNModFn(Function):
    """LayerNorm(x) [* gamma + beta] * (1 + scale) + shift, statistics in fp32 (models/wan/model.py:89-99,295-309)."""

    @staticmethod
    def forward(ctx, x, gamma, beta, scale, shift, eps, with_skip=False):
        require_cuda(x, gamma, beta, scale, shift)
        ctx.set_materialize_grads(False)
        ctx.with_skip = with_skip
        x2 = _contig(_rows2d(x))
        rows, cols = x2.shape
        sc = sh = None
        rows_per_mod = rows
        mdt = dtype_code(x.dtype)
        if scale is not None or shift is not None:
            ref = scale if scale is not None else shift
            sc = _contig(scale).reshape(-1, cols) if scale is not None else None
            sh = _contig(shift).reshape(-1, cols) if shift is not None else None
            rows_per_mod = rows // (ref.numel() // cols)
            mdt = dtype_code(ref.dtype)
            if sc is not None and sh is not None and sc.dtype != sh.dtype:
                raise DpipeHipError('scale and shift must share a dtype')
        wdt = dtype_code(gamma.dtype) if gamma is not None else dtype_code(x.dtype)
        y = torch.empty_like(x2)
        mean = torch.empty(rows, device=x.device, dtype=torch.float32)
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
        check(lib().dpipe_lnmod_fwd(ptr(x2), ptr(_al(gamma)), ptr(_al(beta)), ptr(_al(sc)), ptr(_al(sh)), ptr(y), ptr(mean), ptr(rstd), rows, cols,
                                    rows_per_mod, eps, dtype_code(x.dtype), wdt, mdt, stream()), 'lnmod_fwd')
        ctx.save_for_backward(x2, gamma, beta, sc, mean, rstd)
        ctx.meta = (x.shape, None if scale is None else scale.shape, None if shift is None else shift.shape,
                    rows_per_mod, wdt, mdt, shift is not None)
        if with_skip:
            # second output: x itself, for the residual branch that bypasses the norm.  x then has ONE consumer (this node), and
            # the branch's gradient arrives here as `gskip` and is added inside the dx kernel (no autograd accumulation kernel)
            return y.view(x.shape), x.view_as(x)
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, gy, gskip=None):
        x2, gamma, beta, sc, mean, rstd = ctx.saved_tensors
        x_shape, scale_shape, shift_shape, rows_per_mod, wdt, mdt, has_shift = ctx.meta
        rows, cols = x2.shape
        if gy is None:              # the normalised output was unused: only the bypass carries gradient
            return gskip, None, None, None, None, None, None
        gy2 = _contig(_rows2d(gy))
        gadd = None
        if gskip is not None:
            gadd = _contig(_rows2d(gskip))
            if gadd.dtype != x2.dtype:
                gadd = gadd.to(x2.dtype)
        gx = torch.empty_like(x2)
        groups = rows // rows_per_mod
        mod_dtype = torch.bfloat16 if mdt == hip.BF16 else torch.float32
        fused = False
        dgamma = dbeta = None
        if gamma is not None:
            tg, tb = _accum_target(gamma), _accum_target(beta)
            if tg is not None and (beta is None or tb is not None):
                dgamma, dbeta, fused = tg, tb, True
            else:
                dgamma = torch.empty_like(gamma)
                dbeta = torch.empty_like(beta) if beta is not None else None
        need_mod = sc is not None or has_shift
        dscale = torch.empty((groups, cols), device=x2.device, dtype=mod_dtype) if need_mod else None
        dshift = torch.empty((groups, cols), device=x2.device, dtype=mod_dtype) if need_mod else None
        ws = None
        if dgamma is not None or need_mod:
            ws = torch.empty(lib().dpipe_lnmod_workspace_floats(rows, cols, rows_per_mod), device=x2.device, dtype=torch.float32)
        check(lib().dpipe_lnmod_bwd(ptr(x2), ptr(gy2), ptr(_al(gamma)), ptr(_al(beta)), ptr(_al(sc)), ptr(mean), ptr(rstd), ptr(gx),
                                    ptr(dgamma), ptr(dbeta), ptr(dscale), ptr(dshift), ptr(ws), rows, cols, rows_per_mod,
                                    dtype_code(x2.dtype), wdt, mdt, _acc_all(fused, dgamma, dbeta), ptr(_al(gadd)), stream()), 'lnmod_bwd')
        g_scale = dscale.view(scale_shape) if scale_shape is not None else None
        g_shift = dshift.view(shift_shape) if shift_shape is not None else None
        if fused:
            dgamma = dbeta = None
        return gx.view(x_shape), dgamma, dbeta, g_scale, g_shift, None, None


def layer_norm_modulate(x, gamma=None, beta=None, scale=None, shift=None, eps=1e-6, with_skip=False):
    """scale/shift: [B, D] (or broadcastable [B, 1, D]) applied to the rows of sample b.  with_skip: -> (y, x') where x' aliases x and
    is what the residual branch around the norm should consume (its gradient is then added inside the backward kernel)."""
    return _LNModFn.apply(x, gamma, beta, scale, shift, eps, with_skip)


class _GroupNormFn(Function):
    """nn.GroupNorm(G, C) on NCHW (+ fused SiLU): diffusers ResnetBlock2D / Transformer2DModel norms behind models/sdxl.py:797-865."""

    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, eps, act, with_skip=False):
        require_cuda(x, weight, bias)
        ctx.set_materialize_grads(False)
        xc = _contig(x)
        N, C = xc.shape[0], xc.shape[1]
        HW = xc.numel() // (N * C)
        y = torch.empty_like(xc)
        mean = torch.empty(N * num_groups, device=x.device, dtype=torch.float32)
        rstd = torch.empty_like(mean)
        ws = torch.empty(lib().dpipe_groupnorm_workspace_floats(N, C, HW, num_groups), device=x.device, dtype=torch.float32)
        wdt = dtype_code(weight.dtype) if weight is not None else dtype_code(x.dtype)
        check(lib().dpipe_groupnorm_fwd(ptr(xc), ptr(weight), ptr(bias), ptr(y), ptr(mean), ptr(rstd), ptr(ws), N, C, HW, num_groups, float(eps),
                                        ACT[act], dtype_code(x.dtype), wdt, stream()), 'groupnorm_fwd')
        ctx.save_for_backward(xc, weight, bias, mean, rstd)
        ctx.meta = (num_groups, act, wdt)
        if with_skip:
            return y, x.view_as(x)              # see _LNModFn: the bypass branch's gradient is folded into the dx kernel
        return y

    @staticmethod
    def backward(ctx, gy, gskip=None):
        xc, weight, bias, mean, rstd = ctx.saved_tensors
        G, act, wdt = ctx.meta
        N, C = xc.shape[0], xc.shape[1]
        HW = xc.numel() // (N * C)
        if gy is None:
            return gskip, None, None, None, None, None, None
        gy = _contig(gy)
        gadd = None
        if gskip is not None:
            gadd = _contig(gskip)
            if gadd.dtype != xc.dtype:
                gadd = gadd.to(xc.dtype)
        gx = torch.empty_like(xc)
        fused = False
        dgamma = dbeta = None
        if weight is not None and (ctx.needs_input_grad[2] or ctx.needs_input_grad[3]):
            tg, tb = _accum_target(weight), _accum_target(bias)
            if tg is not None and (bias is None or tb is not None):
                dgamma, dbeta, fused = tg, tb, True
            else:
                dgamma = torch.empty_like(weight)
                dbeta = torch.empty_like(bias) if bias is not None else None
        ws = torch.empty(lib().dpipe_groupnorm_workspace_floats(N, C, HW, G), device=xc.device, dtype=torch.float32)
        check(lib().dpipe_groupnorm_bwd(ptr(xc), ptr(gy), ptr(weight), ptr(bias), ptr(mean), ptr(rstd), ptr(gx), ptr(dgamma), ptr(dbeta), ptr(ws),
                                        N, C, HW, G, ACT[act], dtype_code(xc.dtype), wdt, _acc_all(fused, dgamma, dbeta), ptr(gadd), stream()), 'groupnorm_bwd')
        if fused:
            dgamma = dbeta = None
        return gx, None, dgamma, dbeta, None, None, None


def group_norm(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, with_skip=False):
    """x: [N, C, *spatial] contiguous; act: None or 'silu' (applied to the normalised, affine-transformed value).
    with_skip: -> (y, x') as in layer_norm_modulate."""
    return _GroupNormFn.apply(x, num_groups, weight, bias, eps, act, with_skip)


# ------------------------------------------------------------------------- channels-last (NHWC) UNet ops: GroupNorm, Conv2d
class _AddSampleChannelBiasFn(Function):
    """y[b, c, h, w] = x[b, c, h, w] + t[b, c] on a channels-last x (the ResnetBlock's time-embedding addend at batch > 1: models/sdxl.py -> diffusers ResnetBlock2D,
    `hidden_states + temb[:, :, None, None]`).  The backward's dt[b, c] = sum_hw dy[b, c, h, w] is one deterministic `column_sum` per sample over the [H W, C] memory of
    that sample -- NOT autograd's broadcast reduction: ATen's reduce kernel returned garbage in single elements of exactly this sum under hipGraph REPLAY on MI355X
    (round 5: stacked micro-batches at full size went NaN from the second step on; tools/stack_debug_graph.py localised it to the dt of up_blocks.1.resnets.1)."""

    @staticmethod
    def forward(ctx, x, t):
        ctx.t_dtype = t.dtype
        return x + t[:, :, None, None].to(x.dtype)

    @staticmethod
    def backward(ctx, gy):
        gt = None
        if ctx.needs_input_grad[1]:
            B, C, H, W = gy.shape
            g = gy if is_channels_last(gy) else gy.contiguous(memory_format=torch.channels_last)
            rows = g.permute(0, 2, 3, 1).reshape(B, H * W, C)          # a view: channels-last memory is [B, H W, C]
            gt = torch.stack([column_sum(rows[b]) for b in range(B)], 0).to(ctx.t_dtype)
        return (gy if ctx.needs_input_grad[0] else None), gt


class _BiasPlusSampleFn(Function):
    """[B, C] = bias[C] + t[B, C]; the bias gradient is `column_sum` over the B rows (not autograd's broadcast reduction)."""

    @staticmethod
    def forward(ctx, bias, t):
        ctx.dtypes = (bias.dtype, t.dtype)
        return (bias[None, :].to(t.dtype) + t).contiguous()

    @staticmethod
    def backward(ctx, g):
        gbias = column_sum(g.contiguous()).to(ctx.dtypes[0]) if ctx.needs_input_grad[0] else None
        return gbias, (g.to(ctx.dtypes[1]) if ctx.needs_input_grad[1] else None)


def bias_plus_sample(bias, t):
    return t.contiguous() if bias is None else _BiasPlusSampleFn.apply(bias, t)


def add_sample_channel_bias(x, t):
    """x [B, C, H, W] (channels-last) + t [B, C] broadcast over the pixels; gradients without an ATen reduction (see _AddSampleChannelBiasFn)."""
    return _AddSampleChannelBiasFn.apply(x, t)


def is_channels_last(x):
    """4-D tensor with logical shape [N, C, H, W] whose memory is dense [N, H, W, C]."""
    return x.dim() == 4 and x.permute(0, 2, 3, 1).is_contiguous()


def nhwc_view(x):
    """[N, C, H, W] (any layout) -> contiguous [N, H, W, C] tensor; zero-copy for channels-last inputs."""
    v = x.permute(0, 2, 3, 1)
    return v if v.is_contiguous() else v.contiguous()


class _GroupNormNHWCFn(Function):
    """nn.GroupNorm(G, C) (+ fused SiLU) on a channels-last [N, C, H, W] tensor = [N, HW, C] memory (csrc/groupnorm_nhwc.hip)."""

    @staticmethod
    def forward(ctx, x, num_groups, weight, bias, eps, act, with_skip=False):
        require_cuda(x, weight, bias)
        ctx.set_materialize_grads(False)
        xv = nhwc_view(x)
        N, H, W, C = xv.shape
        HW = H * W
        y = torch.empty_like(xv)
        mean = torch.empty(N * num_groups, device=x.device, dtype=torch.float32)
        rstd = torch.empty_like(mean)
        ws = torch.empty(lib().dpipe_groupnorm_nhwc_workspace_floats(N, C, HW, num_groups), device=x.device, dtype=torch.float32)
        wdt = dtype_code(weight.dtype) if weight is not None else dtype_code(x.dtype)
        check(lib().dpipe_groupnorm_nhwc_fwd(ptr(xv), ptr(_al(weight)), ptr(_al(bias)), ptr(y), ptr(mean), ptr(rstd), ptr(ws), N, C, HW, num_groups, float(eps),
                                             ACT[act], dtype_code(x.dtype), wdt, stream()), 'groupnorm_nhwc_fwd')
        ctx.save_for_backward(xv, weight, bias, mean, rstd)
        ctx.meta = (num_groups, act, wdt)
        if with_skip:
            return y.permute(0, 3, 1, 2), x.view_as(x)     # see _LNModFn: the bypass branch's gradient is folded into the dx kernel
        return y.permute(0, 3, 1, 2)

    @staticmethod
    def backward(ctx, gy, gskip=None):
        xv, weight, bias, mean, rstd = ctx.saved_tensors
        G, act, wdt = ctx.meta
        N, H, W, C = xv.shape
        if gy is None:
            return gskip, None, None, None, None, None, None
        gyv = nhwc_view(gy)
        gadd = None
        if gskip is not None:
            gadd = nhwc_view(gskip)
            if gadd.dtype != xv.dtype:
                gadd = gadd.to(xv.dtype)
        gx = torch.empty_like(xv)
        fused = False
        dgamma = dbeta = None
        if weight is not None and (ctx.needs_input_grad[2] or ctx.needs_input_grad[3]):
            tg, tb = _accum_target(weight), _accum_target(bias)
            if tg is not None and (bias is None or tb is not None):
                dgamma, dbeta, fused = tg, tb, True
            else:
                dgamma = torch.empty_like(weight)
                dbeta = torch.empty_like(bias) if bias is not None else None
        ws = torch.empty(lib().dpipe_groupnorm_nhwc_workspace_floats(N, C, H * W, G), device=xv.device, dtype=torch.float32)
        check(lib().dpipe_groupnorm_nhwc_bwd(ptr(xv), ptr(gyv), ptr(_al(weight)), ptr(_al(bias)), ptr(mean), ptr(rstd), ptr(gx), ptr(dgamma), ptr(dbeta), ptr(ws),
                                             N, C, H * W, G, ACT[act], dtype_code(xv.dtype), wdt, _acc_all(fused, dgamma, dbeta), ptr(_al(gadd)), stream()), 'groupnorm_nhwc_bwd')
        if fused:
            dgamma = dbeta = None
        return gx.permute(0, 3, 1, 2), None, dgamma, dbeta, None, None, None


def group_norm_nhwc(x, num_groups, weight=None, bias=None, eps=1e-5, act=None, with_skip=False):
    """x: [N, C, H, W] channels-last; returns a channels-last tensor of the same logical shape.  with_skip: -> (y, x') as in layer_norm_modulate."""
    return _GroupNormNHWCFn.apply(x, num_groups, weight, bias, eps, act, with_skip)


# tools/conv_timing.py forces tile configurations through these (0 = the dispatcher's own choice): (forward, dgrad, wgrad) tile_hint codes of dpipe_gemm_ex
CONV_TILE_HINTS = (0, 0, 0)


def conv2d_eligible(x_dtype, weight, stride, padding, dilation=(1, 1), groups=1):
    """The implicit-GEMM convolution (csrc/conv_pipe.hip) takes bf16 -- or fp32 (exact-parity mode: three bf16 hi / lo split launches
    accumulated in fp32) --, stride 1 / 2, square padding, Cin % 64 == 0 and Cout % 64 == 0."""
    Cout, Cin, kh, kw = weight.shape
    return (x_dtype == weight.dtype and x_dtype in (torch.bfloat16, torch.float32) and groups == 1 and tuple(dilation) == (1, 1)
            and stride[0] == stride[1] and stride[0] in (1, 2) and padding[0] == padding[1] and Cin % 64 == 0 and Cout % 64 == 0)


def _dense_like(t, ref):
    return t is not None and t.dtype == ref.dtype and t.shape == ref.shape and t.stride() == ref.stride()


def _split_bf16(t):
    """fp32 -> (hi, lo) bf16 pair with hi + lo = t up to 2^-17 relative (strides preserved: channels-last stays channels-last)."""
    if t is None:
        return None, None
    hi = t.to(torch.bfloat16)
    return hi, (t - hi.float()).to(torch.bfloat16)


def _conv_fwd_launch(xv, Cin, weight, bias, rv, y, B, H, W, Cout, kh, kw, stride, pad, upsample, flags, ws):
    check(lib().dpipe_conv2d_fwd(ptr(xv), Cin, ptr(weight), ptr(bias), ptr(rv), Cout, ptr(y), Cout, B, H, W, Cin, Cout, kh, kw, stride, pad, upsample,
                                 0, flags, ptr(ws), ws.numel(), CONV_TILE_HINTS[0], stream()), 'conv2d_fwd')


class _Conv2dNHWCFn(Function):
    """nn.Conv2d on channels-last activations as implicit GEMM (forward, dgrad, wgrad + fused bias gradient); `upsample` = 2 folds the
    nearest-neighbour 2x up-sampling of diffusers' Upsample2D into the gather; `residual` rides the epilogue.  fp32 tensors (exact-parity
    mode) run the SAME bf16 MFMA kernels three times over hi / lo splits of the operands, accumulating in fp32 (include/dpipe_hip.h)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, stride, pad, upsample):
        require_cuda(x, weight, bias, residual)
        xv = nhwc_view(x)
        B, H, W, Cin = xv.shape
        Cout, Cin_w, kh, kw = weight.shape
        if Cin_w != Cin:
            raise DpipeHipError(f'conv2d: input has {Cin} channels, weight expects {Cin_w}')
        if not weight.permute(0, 2, 3, 1).is_contiguous():
            raise DpipeHipError('conv2d: weight must be stored channels-last ([Cout, kh, kw, Cin] memory); use nn.Conv2d of diffusion_pipe_amd.nn')
        Ho = (H * upsample + 2 * pad - kh) // stride + 1
        Wo = (W * upsample + 2 * pad - kw) // stride + 1
        y = torch.empty((B, Ho, Wo, Cout), device=x.device, dtype=x.dtype)
        rv = None
        if residual is not None:
            rv = nhwc_view(residual)
            if rv.shape != y.shape or rv.dtype != y.dtype:
                raise DpipeHipError('conv2d: residual must have the output shape and dtype')
        if bias is not None and bias.dtype != x.dtype:
            bias = bias.to(x.dtype)
        ws = _splitk_workspace(x.device)
        geo = (B, H, W, Cout, kh, kw, stride, pad, upsample)
        if x.dtype == torch.float32:
            if bias is not None and bias.dim() != 1:
                raise DpipeHipError('conv2d: the fp32 (exact-parity) mode takes a per-channel bias only')
            (xh, xl), (wh, wl), (bh, bl) = _split_bf16(xv), _split_bf16(weight), _split_bf16(bias)
            _conv_fwd_launch(xh, Cin, wh, bh, rv, y, *geo, hip.CONV_OUT_F32, ws)
            _conv_fwd_launch(xl, Cin, wh, bl, None, y, *geo, hip.CONV_OUT_F32 | hip.CONV_ACCUMULATE, ws)
            _conv_fwd_launch(xh, Cin, wl, None, None, y, *geo, hip.CONV_OUT_F32 | hip.CONV_ACCUMULATE, ws)
        else:
            hilo = bias is not None and bias.dim() == 3                # [2, R, Cout]: the bf16 hi / lo pair of an fp32 addend (precise_row_linear(..., pair=True)), R = 1 or B rows
            if hilo and (bias.shape[0] != 2 or bias.shape[1] not in (1, B) or bias.shape[2] != Cout or not bias.is_contiguous()):
                raise DpipeHipError('conv2d: a hi / lo bias pair must be a contiguous [2, 1 or B, Cout] tensor')
            per_sample = bias is not None and (bias.dim() == 2 or (hilo and bias.shape[1] > 1))       # a bias row per sample (the ResnetBlock's time-embedding addend at batch > 1)
            if per_sample and not hilo and (bias.shape != (B, Cout) or not bias.is_contiguous()):
                raise DpipeHipError('conv2d: a per-sample bias must be a contiguous [B, Cout] tensor')
            _conv_fwd_launch(xv, Cin, weight, bias, rv, y, *geo, (hip.CONV_BIAS_PER_SAMPLE if per_sample else 0) | (hip.CONV_BIAS_HILO if hilo else 0), ws)
        ctx.save_for_backward(xv, weight, bias)
        ctx.geom = (stride, pad, upsample, residual is not None)
        return y.permute(0, 3, 1, 2)

    @staticmethod
    def backward(ctx, gy):
        xv, weight, bias = ctx.saved_tensors
        stride, pad, upsample, has_res = ctx.geom
        B, H, W, Cin = xv.shape
        Cout, _, kh, kw = weight.shape
        gyv = nhwc_view(gy)
        if gyv.dtype != xv.dtype:
            gyv = gyv.to(xv.dtype)
        f32 = xv.dtype == torch.float32
        ws = _splitk_workspace(xv.device)
        gx = gw = gb = None
        if f32:
            (gh, gl), (wh, wl) = _split_bf16(gyv), _split_bf16(weight)
        if ctx.needs_input_grad[0]:
            Hi, Wi = H * upsample, W * upsample
            dxu = torch.empty((B, Hi, Wi, Cin), device=xv.device, dtype=xv.dtype)

            def dgrad(g, w, flags):
                check(lib().dpipe_conv2d_dgrad(ptr(g), Cout, ptr(w), ptr(dxu), Cin, B, Hi, Wi, Cin, Cout, kh, kw, stride, pad, flags,
                                               ptr(ws), ws.numel(), CONV_TILE_HINTS[1], stream()), 'conv2d_dgrad')
            if f32:
                dgrad(gh, wh, hip.CONV_OUT_F32)
                dgrad(gl, wh, hip.CONV_OUT_F32 | hip.CONV_ACCUMULATE)
                dgrad(gh, wl, hip.CONV_OUT_F32 | hip.CONV_ACCUMULATE)
            else:
                dgrad(gyv, weight, 0)
            if upsample > 1:       # adjoint of the nearest up-sampling: sum over each 2 x 2 block
                if upsample == 2 and Cin % (4 if f32 else 8) == 0:
                    dxs = torch.empty((B, H, W, Cin), device=xv.device, dtype=xv.dtype)
                    check(lib().dpipe_upsample2x_adjoint(ptr(dxu), ptr(dxs), B, H, W, Cin, dtype_code(xv.dtype), stream()), 'upsample2x_adjoint')
                    dxu = dxs
                else:
                    dxu = dxu.view(B, H, upsample, W, upsample, Cin).sum(dim=(2, 4))
            gx = dxu.permute(0, 3, 1, 2)
        need_w, need_b = ctx.needs_input_grad[1], bias is not None and ctx.needs_input_grad[2]
        gb_rows = None
        hilo = bias is not None and bias.dim() == 3
        if need_b and (bias.dim() == 2 or (hilo and bias.shape[1] > 1)):
            # per-sample bias: its gradient is one deterministic column sum per sample over that sample's [Ho Wo, Cout] rows of dy (no ATen reduction: see
            # _AddSampleChannelBiasFn); the wgrad launch below then carries no fused bias gradient
            rows = gyv.reshape(B, -1, Cout)
            gb_rows = torch.stack([column_sum(rows[b]) for b in range(B)], 0)
            need_b = False
        if need_w or need_b:
            tw = _accum_target_dense(weight)
            tb = _accum_target(bias) if need_b else None
            w_out = tw if tw is not None else torch.empty_like(weight)           # preserve_format: channels-last like the weight
            b_out = (tb if tb is not None else (torch.empty_like(bias[0, 0]) if hilo else torch.empty_like(bias))) if need_b else None

            def wgrad(g, xs, acc, bo, bacc, out_f32):
                check(lib().dpipe_conv2d_wgrad(ptr(g), Cout, ptr(xs), Cin, ptr(w_out), ptr(bo), B, H, W, Cin, Cout, kh, kw, stride, pad, upsample,
                                               int(acc), int(bacc), int(out_f32), ptr(ws), ws.numel(), CONV_TILE_HINTS[2], stream()), 'conv2d_wgrad')
            if f32:
                xh, xl = _split_bf16(xv)
                wgrad(gh, xh, _acc(tw), None, 0, 1)
                wgrad(gl, xh, True, None, 0, 1)
                wgrad(gh, xl, True, None, 0, 1)
                if need_b:                       # the fused bias gradient is written in the operand dtype: fp32 takes the column-sum kernel
                    g2 = gyv.reshape(-1, Cout)
                    if tb is not None:
                        column_sum(g2, out=tb, accumulate=_acc(tb))
                    else:
                        b_out = column_sum(g2)
            else:
                wgrad(gyv, xv, _acc(tw), b_out, _acc(tb), 0)
            gw = None if tw is not None else w_out
            gb = None if (tb is not None or not need_b) else b_out
        if gb_rows is not None:
            gb = gb_rows
        if hilo and gb is not None:
            gb = gb.reshape(1, -1, Cout).expand(2, -1, -1)          # both rows of the pair receive the gradient of their sum (a view: precise_row_linear reads row 0)
        gres = gy if (has_res and ctx.needs_input_grad[3]) else None
        return gx, gw, gb, gres, None, None, None


def _accum_target_dense(param):
    """like _accum_target for parameters that are dense but not row-major (channels-last conv weights): .grad must share the strides"""
    if not FUSE_GRAD_ACCUM or param is None or not param.is_leaf:
        return None
    g = param.grad
    return g if _dense_like(g, param) else None


def conv2d_nhwc(x, weight, bias=None, stride=1, padding=0, upsample=1, residual=None):
    """x: [B, Cin, H, W] channels-last bf16 (or fp32, see _Conv2dNHWCFn), weight: [Cout, Cin, kh, kw] channels-last -> [B, Cout, Ho, Wo] channels-last."""
    return _Conv2dNHWCFn.apply(x, weight, bias, residual, int(stride), int(padding), int(upsample))


# ------------------------------------------------------------------------------------------------- RoPE (K3)
class _RopeFn(Function):
    """Rotary embedding on [B, S, H, D] with fp32 cos/sin tables [S, D/2] (models/wan/model.py:40-67)."""

    @staticmethod
    def forward(ctx, x, cos, sin, interleaved):
        require_cuda(x, cos, sin)
        xc = _contig(x)
        B, S, H, D = xc.shape
        if cos.shape != (S, D // 2) or cos.dtype != torch.float32:
            raise DpipeHipError(f'rope tables must be fp32 [S, D/2]; got {tuple(cos.shape)} {cos.dtype}')
        cos, sin = _contig(cos), _contig(sin)
        y = torch.empty_like(xc)
        check(lib().dpipe_rope(ptr(xc), ptr(cos), ptr(sin), ptr(y), B, S, H, D, int(interleaved), 0, dtype_code(xc.dtype), stream()), 'rope')
        ctx.save_for_backward(cos, sin)
        ctx.interleaved = interleaved
        return y

    @staticmethod
    def backward(ctx, gy):
        cos, sin = ctx.saved_tensors
        gy = _contig(gy)
        B, S, H, D = gy.shape
        gx = torch.empty_like(gy)
        check(lib().dpipe_rope(ptr(gy), ptr(cos), ptr(sin), ptr(gx), B, S, H, D, int(ctx.interleaved), 1, dtype_code(gy.dtype), stream()), 'rope_bwd')
        return gx, None, None, None


def rope(x, cos, sin, interleaved=True):
    return _RopeFn.apply(x, cos, sin, interleaved)


# K2 + K3 fused: RMSNorm -> RoPE -> Q / K written once.  A/B switch DPIPE_FUSE_NORM_ROPE=0 restores the two-kernel route (+ the contiguous copy of a strided q / k).
FUSE_NORM_ROPE = _os_mod.environ.get('DPIPE_FUSE_NORM_ROPE', '1') == '1'


class _RMSNormRopeFn(Function):
    """y = rope(rms_norm(x) * weight) on [B, S, H, D] in ONE pass (models/wan/model.py:124-125,139-140 q = rope(norm_q(q(x))): the norm spans the whole token,
    weight [H D]; hunyuan_image_modeling.py:181-190 / diffusers FluxAttnProcessor: per-head norm, weight [D]).  x may be a strided view of a fused QKV projection
    (`qkv.view(B, S, 3, H, D).unbind(2)`): the kernel takes the token pitch, no contiguous copy is made.  cos / sin: fp32 [>= token_offset + S, D / 2], interleaved pairs;
    tokens s >= rope_tokens are normalised but not rotated (the text tokens of an [image ; text] sequence)."""

    @staticmethod
    def forward(ctx, x, weight, cos, sin, eps, per_head, token_offset, rope_tokens):
        require_cuda(x, weight, cos, sin)
        B, S, H, D = x.shape
        if x.stride(3) != 1 or x.stride(2) != D or x.stride(1) < H * D or (B > 1 and x.stride(0) != S * x.stride(1)) or x.stride(1) % 8:
            x = x.contiguous()
        rt = S if rope_tokens is None else min(int(rope_tokens), S)
        if cos.dtype != torch.float32 or cos.dim() != 2 or cos.shape[1] != D // 2 or cos.shape[0] < token_offset + rt or sin.shape != cos.shape:
            raise DpipeHipError(f'rms_norm_rope: tables must be fp32 [>= {token_offset + rt}, {D // 2}] (the rotated tokens); got {tuple(cos.shape)} {cos.dtype}')
        cos, sin = _contig(cos), _contig(sin)
        groups, cols = (H, D) if per_head else (1, H * D)
        if weight is not None and weight.numel() != cols:
            raise DpipeHipError(f'rms_norm_rope: weight has {weight.numel()} elements, the normalised row {cols}')
        rows = B * S * groups
        y = torch.empty((B, S, H, D), device=x.device, dtype=x.dtype)
        rstd = torch.empty(rows, device=x.device, dtype=torch.float32)
        wd = dtype_code(weight.dtype) if weight is not None else dtype_code(x.dtype)
        check(lib().dpipe_rmsnorm_rope_fwd(ptr(x), ptr(_al(weight)), ptr(cos), ptr(sin), ptr(y), ptr(rstd), rows, cols, D, S, groups, int(token_offset), rt, x.stride(1), float(eps),
                                           dtype_code(x.dtype), wd, stream()), 'rmsnorm_rope_fwd')
        ctx.save_for_backward(x, weight, rstd, cos, sin)
        ctx.meta = (rows, cols, D, S, groups, int(token_offset), rt)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight, rstd, cos, sin = ctx.saved_tensors
        rows, cols, D, S, groups, tok_off, rt = ctx.meta
        gy = _contig(gy)
        gx = torch.empty(gy.shape, device=gy.device, dtype=gy.dtype)
        dw = ws = None
        fused = False
        if weight is not None and ctx.needs_input_grad[1]:
            dw = _accum_target(weight)
            fused = dw is not None
            if dw is None:
                dw = torch.empty_like(weight)
            ws = torch.empty(lib().dpipe_norm_slabs(rows) * cols, device=gy.device, dtype=torch.float32)
        wd = dtype_code(weight.dtype) if weight is not None else dtype_code(x.dtype)
        check(lib().dpipe_rmsnorm_rope_bwd(ptr(x), ptr(_al(weight)), ptr(gy), ptr(rstd), ptr(cos), ptr(sin), ptr(gx), ptr(dw), ptr(ws), rows, cols, D, S, groups, tok_off, rt,
                                           x.stride(1), dtype_code(x.dtype), wd, _acc_all(fused, dw), stream()), 'rmsnorm_rope_bwd')
        return gx, (None if fused else dw), None, None, None, None, None, None


def rms_norm_rope(x, weight, cos, sin, eps=1e-6, per_head=True, token_offset=0, rope_tokens=None):
    """[B, S, H, D] -> rope(rms_norm(x) * weight); see _RMSNormRopeFn.  Falls back to the two-kernel composition when the fusion is switched off."""
    if not FUSE_NORM_ROPE:
        B, S, H, D = x.shape
        n = rms_norm(x if per_head else x.reshape(B, S, H * D), weight, eps).view(B, S, H, D)
        c, s_ = cos[token_offset:token_offset + S], sin[token_offset:token_offset + S]
        if rope_tokens is None or rope_tokens >= S:
            return rope(n, c, s_, interleaved=True)
        return torch.cat([rope(n[:, :rope_tokens].contiguous(), c[:rope_tokens], s_[:rope_tokens], interleaved=True), n[:, rope_tokens:]], dim=1)
    return _RMSNormRopeFn.apply(x, weight, cos, sin, eps, per_head, token_offset, rope_tokens)


# Rotary positions from the positions themselves: several axes, any position per token, query and key heads in one launch.
# (These operators and attention_varlen are also called where a call costs more than its kernels -- a prompt, one image's tokens: their host path passes plain
#  integers to the C entry, takes the raw stream handle, and enters autograd only when a gradient is wanted.)
def _head_rows(x):
    """x [..., H, D] as rows the kernels walk by (token stride, head stride): (tensor, tokens, H, D, token stride, head stride).  A view with one uniform token stride (a column block
    of a fused projection) is taken as it is; anything else, or an address that is not 16-byte aligned, is copied once."""
    shape, st = x.shape, x.stride()
    H, D = shape[-2:]
    ss = H * D
    ok = st[-1] == 1 and st[-2] % 8 == 0 and x.data_ptr() % 16 == 0
    if len(shape) == 3:
        tokens = shape[0]
        if tokens > 1:
            ss = st[0]
    else:
        tokens, first = 1, True
        for size, s in zip(shape[-3::-1], st[-3::-1]):
            if size != 1:
                if first:
                    ss, first = s, False
                elif s != ss * tokens:
                    ok = False
            tokens *= size
    if not ok or ss % 8 or not D <= ss < 2 ** 23 or st[-2] * H >= 2 ** 28:
        x = x.clone(memory_format=torch.contiguous_format)
        return x, tokens, H, D, H * D, D
    return x, tokens, H, D, ss, st[-2]


def _dense(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _addr(t):
    return None if t is None else t.data_ptr()


def _one_device(*tensors):
    """the operands' device; DpipeHipError for a CPU tensor or operands on different devices"""
    device = tensors[0].device
    for t in tensors:
        if t is not None and t.device != device:
            raise DpipeHipError(f'operands on different devices: {device} and {t.device}')
    require_cuda(tensors[0])
    return device


def _no_tangents(what, *tensors):
    """Forward-mode derivatives are refused, not dropped: a dual tensor does not ask for a gradient, so it would take the path without autograd.  (The level is read first: no dual
    level, no tangents, and nothing to unpack.)"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise DpipeHipError(f'{what}: forward-mode derivatives are not supported')


def _no_second_graph(what):
    """Called in a backward: the gradient has no gradient of its own here.  Asked to record one (create_graph), it refuses: a term of a second derivative would vanish from its sum."""
    if torch.is_grad_enabled():
        raise DpipeHipError(f'{what} is differentiable once: no graph of its gradient (create_graph)')


@contextlib.contextmanager
def _launching_on(device):
    """kernels are launched on the current device: make it the operands'"""
    with torch.cuda.device(device):
        yield


_HERE = contextlib.nullcontext()


def _on(device):
    return _HERE if device.index == torch.cuda.current_device() else _launching_on(device)


@functools.lru_cache(maxsize=64)
def _rope_axes_tables(axes_dim, theta, shared, D, interleaved):
    """host tables of the kernel: (turns per unit of position in fp64, axis) of every channel pair, and their count; the checks of what they are made from"""
    thetas = theta if isinstance(theta, tuple) else (theta,) * len(axes_dim)
    if not axes_dim or any(a <= 0 or a % 2 for a in axes_dim) or sum(axes_dim) > D or (not interleaved and sum(axes_dim) % 8) or len(thetas) != len(axes_dim) \
            or any(not (t > 0.0 and math.isfinite(t)) for t in thetas) or (shared and len(set(thetas)) > 1):
        raise DpipeHipError(f'rope_axes: even axis sizes that fit the head dim {D} (halves pairing: together a multiple of 8) and a positive theta (shared: one); got {axes_dim}, {theta}')
    total, freq, axis = sum(axes_dim), [], []
    for a, dim in enumerate(axes_dim):
        for j in range(dim // 2):
            e = -2.0 * len(freq) / total if shared else -2.0 * j / dim
            freq.append(thetas[a] ** e / (2.0 * math.pi))
            axis.append(a)
    return (ctypes.c_double * len(freq))(*freq), (ctypes.c_int * len(axis))(*axis), len(freq)


_POSITION_TYPES = {torch.float32: 0, torch.int32: 1, torch.int64: 2}


def _rope_axes_forward(q, k, positions, q_weight, k_weight, tables, eps, half):
    """-> (yq, yk, (q, k as read), what the backward's call repeats)"""
    device = q.device
    q, tokens, hq, D, q_ss, q_sh = _head_rows(q)
    yq = _dense(q)
    hk = k_ss = k_sh = 0
    yk = None
    if k is not None:
        k, _, hk, _, k_ss, k_sh = _head_rows(k)
        yk = _dense(k)
    freq, axis, pairs = tables
    axes = positions.shape[-1]
    meta = (tokens, positions.numel() // axes, axes, pairs, hq, hk, D)
    dt = dtype_code(q.dtype)
    tail = (eps, half, dt, dt if q_weight is None else dtype_code(q_weight.dtype), dt if k_weight is None else dtype_code(k_weight.dtype))
    strides = (q_ss, q_sh, k_ss, k_sh)
    if tokens:
        wq, wk = _al(q_weight), _al(k_weight)
        check(lib().dpipe_rope_axes_fwd(q.data_ptr(), _addr(k), positions.data_ptr(), _POSITION_TYPES[positions.dtype], freq, axis, _addr(wq), _addr(wk), yq.data_ptr(), _addr(yk),
                                        *meta, *strides, *tail, hip.raw_stream(device)), 'rope_axes_fwd')
    return yq, yk, q, k, (meta, strides, tail, tables)


class _RopeAxesFn(Function):
    """q', k' = R(positions) [rms_norm](q, k); see rope_axes.  The backward re-derives the norm's statistics from q / k: nothing but the inputs is kept."""

    @staticmethod
    def forward(ctx, q, k, positions, q_weight, k_weight, tables, eps, half):
        yq, yk, q, k, ctx.call = _rope_axes_forward(q, k, positions, q_weight, k_weight, tables, eps, half)
        normed = q_weight is not None or k_weight is not None
        ctx.save_for_backward(q if normed else None, k if normed else None, positions, q_weight, k_weight)
        return yq, yk

    @staticmethod
    def backward(ctx, gq, gk):
        _no_second_graph('rope_axes')
        q, k, positions, q_weight, k_weight = ctx.saved_tensors
        meta, strides, tail, (freq, axis, _) = ctx.call
        tokens, has_k, D, device = meta[0], meta[5] > 0, meta[6], gq.device
        with _on(device):
            gq, _, _, _, gq_ss, gq_sh = _head_rows(gq)
            dq = _dense(gq)
            dk, gk_ss, gk_sh = None, 0, 0
            if has_k:
                gk, _, _, _, gk_ss, gk_sh = _head_rows(gk)
                dk = _dense(gk)
            else:
                gk = None
            normed = q is not None
            if not normed:
                q, k, strides = gq, gk, (gq_ss, gq_sh, gk_ss, gk_sh)
            dw, fused = [None, None], [False, False]
            for i, w in enumerate((q_weight, k_weight)):
                if w is not None and ctx.needs_input_grad[3 + i]:
                    dw[i] = _accum_target(w)
                    if dw[i] is not None and i == 1 and fused[0] and dw[0].data_ptr() == dw[1].data_ptr():
                        dw[i] = None                      # one weight for queries and keys: the kernel must not add into its gradient from two workgroups at once
                    fused[i] = dw[i] is not None
                    if dw[i] is None:
                        dw[i] = torch.empty_like(w) if tokens else torch.zeros_like(w)
            if tokens:
                ws = torch.empty(lib().dpipe_rope_axes_workspace_floats(D), device=device, dtype=torch.float32) if normed else None
                wq, wk = _al(q_weight), _al(k_weight)
                check(lib().dpipe_rope_axes_bwd(q.data_ptr(), _addr(k), gq.data_ptr(), _addr(gk), positions.data_ptr(), _POSITION_TYPES[positions.dtype], freq, axis, _addr(wq), _addr(wk),
                                                dq.data_ptr(), _addr(dk), _addr(dw[0]), _addr(dw[1]), _addr(ws), *meta, *strides, gq_ss, gq_sh, gk_ss, gk_sh, *tail,
                                                _acc_all(fused[0], dw[0]), _acc_all(fused[1], dw[1]), hip.raw_stream(device)), 'rope_axes_bwd')
        return dq, dk, None, (None if fused[0] else dw[0]), (None if fused[1] else dw[1]), None, None, None


def rope_axes(q, k, positions, axes_dim, theta=10000.0, q_weight=None, k_weight=None, eps=1e-6, interleaved=True, shared=False):
    """Rotary positions with several axes on query and key heads, optionally behind their per-head RMS norms, in one launch; differentiable once in q, k and the weights (reverse mode).

    q [..., H, D], k [..., Hk, D] or None (bf16 or fp32, the same leading sizes; D a multiple of 8 up to 256; column blocks of a fused projection are read in place).
    positions [..., axes] (fp32, int32 or int64): one row per token, or one row per token of the innermost leading sizes, repeated over the outer ones ([S, axes] for q [B, S, H, D]).
    axes_dim: channels of every axis (even, together at most D; the channels behind them are not rotated), e.g. (16, 56, 56) for (time, height, width).
    theta: base of the frequencies theta ** (-2 j / dim), one number or one per axis; shared=True: one run of frequencies over all axes' channels together instead.
    q_weight, k_weight [D]: x * rsqrt(mean(x ** 2) + eps) * weight before the rotation (None: no norm).
    interleaved: pairs are neighbouring channels (2 p, 2 p + 1); False: the halves (p, p + sum(axes_dim) / 2) of the rotated channels, whose count is a multiple of 8.
    Angles are formed in fp64 from the positions: far positions keep their precision.  (models/wan/model.py:40-67; diffusers FluxPosEmbed; models/hunyuan_video.py:35-81)
    -> (q', k'), contiguous; k' is None without k."""
    qs, dtype = q.shape, q.dtype
    if len(qs) < 3 or (k is not None and (k.shape[:-2] != qs[:-2] or k.shape[-1] != qs[-1] or k.dtype != dtype)):
        raise DpipeHipError(f'rope_axes: q [..., H, D] and k [..., Hk, D] of one dtype; got {tuple(qs)} {dtype} and {(tuple(k.shape), k.dtype) if k is not None else None}')
    dtype_code(dtype)
    D = qs[-1]
    if D % 8 or not 0 < D <= 256 or qs[-2] == 0 or (k is not None and k.shape[-2] == 0):
        raise DpipeHipError(f'rope_axes: the head dim must be a multiple of 8 up to 256, with at least one head; got {tuple(qs)}')
    tables = _rope_axes_tables(tuple(axes_dim), tuple(theta) if isinstance(theta, list) else theta, bool(shared), D, bool(interleaved))
    ps = positions.shape
    if positions.dtype not in _POSITION_TYPES or positions.requires_grad:
        raise DpipeHipError(f'rope_axes: positions are fp32, int32 or int64 and have no gradient; got {positions.dtype}')
    if len(ps) < 2 or ps[-1] != len(axes_dim) or len(ps) > len(qs) - 1 or ps[:-1] != qs[len(qs) - 1 - len(ps):-2]:
        raise DpipeHipError(f'rope_axes: positions {tuple(ps)} do not fit tokens {tuple(qs[:-2])} and {len(axes_dim)} axes')
    for w in (q_weight, k_weight):
        if w is not None and tuple(w.shape) != (D,):
            raise DpipeHipError(f'rope_axes: norm weights have shape [{D}]; got {tuple(w.shape)}')
    if k is None and k_weight is not None:
        raise DpipeHipError('rope_axes: a key weight needs k')
    _no_tangents('rope_axes', q, k, positions, q_weight, k_weight)
    q_weight, k_weight = (w if w is None or w.is_contiguous() else w.contiguous() for w in (q_weight, k_weight))
    args = (q, k, _contig(positions), q_weight, k_weight, tables, float(eps), 0 if interleaved else 1)
    with _on(_one_device(q, k, positions, q_weight, k_weight)):
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad) or (q_weight is not None and q_weight.requires_grad)
                                        or (k_weight is not None and k_weight.requires_grad)):
            return _RopeAxesFn.apply(*args)
        return _rope_axes_forward(*args)[:2]


# -------------------------------------------------------------------------------------------- attention (K4)
def _bshd_strides(t):
    if t.stride(3) != 1:
        raise DpipeHipError('attention tensors need a contiguous head dim')
    return t.stride(0), t.stride(1), t.stride(2)


# The forward keeps O a second time in fp32 for the backward's delta = rowsum(dO . O) (csrc/attention.hip, AttnParams::out32: the bf16 rounding of O otherwise
# reaches dQ / dK amplified by the common component of the value rows).  Costs 4 bytes per output element of saved activation; DPIPE_ATTN_O32=0 for the A/B.
ATTN_SAVE_O32 = _os_mod.environ.get('DPIPE_ATTN_O32', '1') == '1'


def _flash_fwd(q, k, v, kv_len, scale, causal, want_o32=False):
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    if q.dtype != torch.bfloat16 or k.dtype != q.dtype or v.dtype != q.dtype:
        raise DpipeHipError('flash attention kernel computes in bf16')
    o = torch.empty((B, Sq, H, D), device=q.device, dtype=q.dtype)
    lse = torch.empty((B, H, Sq), device=q.device, dtype=torch.float32)
    o32 = torch.empty((B, Sq, H, D), device=q.device, dtype=torch.float32) if (want_o32 and ATTN_SAVE_O32) else None
    check(lib().dpipe_attn_fwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lse), ptr(kv_len), B, H, Sq, Sk, D,
                               *_bshd_strides(q), *_bshd_strides(k), *_bshd_strides(v), *_bshd_strides(o),
                               float(scale), int(causal), ptr(o32), stream()), 'attn_fwd')
    return o, lse, o32


def _flash_bwd(q, k, v, o, do, lse, kv_len, dq, dk, dv, scale, causal, o32=None):
    B, Sq, H, D = q.shape
    Sk = k.shape[1]
    if do.stride(3) != 1:
        do = do.contiguous()
    delta = torch.empty((B, H, Sq), device=q.device, dtype=torch.float32)
    npart = lib().dpipe_attn_bwd_partial_floats(B, H, Sq, Sk, D)
    part = torch.empty(npart, device=q.device, dtype=torch.float32) if npart > 0 else None
    check(lib().dpipe_attn_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(do), ptr(lse), ptr(delta), ptr(dq), ptr(dk), ptr(dv),
                               ptr(kv_len), B, H, Sq, Sk, D,
                               *_bshd_strides(q), *_bshd_strides(k), *_bshd_strides(v), *_bshd_strides(o), *_bshd_strides(do),
                               *_bshd_strides(dq), *_bshd_strides(dk), *_bshd_strides(dv), float(scale), int(causal),
                               ptr(part), npart, ptr(o32), stream()), 'attn_bwd')


class _FlashAttnFn(Function):
    """softmax(q k^T * scale) v on [B, S, H, D] bf16 tensors, flash style (models/wan/attention.py:91-122)."""

    @staticmethod
    def forward(ctx, q, k, v, kv_len, scale, causal):
        require_cuda(q, k, v, kv_len)
        o, lse, o32 = _flash_fwd(q, k, v, kv_len, scale, causal, want_o32=any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, k, v, o, lse, kv_len, o32)
        ctx.scale = scale
        ctx.causal = causal
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, kv_len, o32 = ctx.saved_tensors
        dq, dk, dv = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format), \
            torch.empty_like(v, memory_format=torch.contiguous_format)
        _flash_bwd(q, k, v, o, do, lse, kv_len, dq, dk, dv, ctx.scale, ctx.causal, o32)
        return dq, dk, dv, None, None, None


def _split_heads(packed, parts, H, D):
    """[B, S, parts * H * D] -> `parts` strided views [B, S, H, D] (no copies: the kernels take strides)."""
    B, S, _ = packed.shape
    return [torch.as_strided(packed, (B, S, H, D), (packed.stride(0), packed.stride(1), D, 1), packed.storage_offset() + i * H * D) for i in range(parts)]


class _FlashAttnPackedFn(Function):
    """The same kernels on the output of a fused projection: mode 'qkv' takes one [B, S, 3 H D] tensor, mode 'q_kv' a query
    [B, Sq, H D] and a packed [B, Sk, 2 H D] key/value tensor.  Backward writes dq / dk / dv straight into the packed
    gradient of the projection output (strided stores), so the fused dgrad / wgrad GEMMs consume it without any concat."""

    @staticmethod
    def forward(ctx, a, b, H, D, kv_len, scale, causal):
        require_cuda(a, b, kv_len)
        a = _contig(a)
        if b is None:
            q, k, v = _split_heads(a, 3, H, D)
        else:
            # a column block of a wider projection output (split_columns) is consumed in place: the kernels take the token stride
            if not (b.dim() == 3 and b.stride(2) == 1 and b.stride(1) % 8 == 0 and (b.shape[0] == 1 or b.stride(0) == b.shape[1] * b.stride(1))):
                b = _contig(b)
            q = a.view(a.shape[0], a.shape[1], H, D)
            k, v = _split_heads(b, 2, H, D)
        o, lse, o32 = _flash_fwd(q, k, v, kv_len, scale, causal, want_o32=any(ctx.needs_input_grad[:2]))
        ctx.save_for_backward(a, b, o, lse, kv_len, o32)
        ctx.meta = (H, D, scale, causal)
        return o.view(o.shape[0], o.shape[1], H * D)

    @staticmethod
    def backward(ctx, do):
        a, b, o, lse, kv_len, o32 = ctx.saved_tensors
        H, D, scale, causal = ctx.meta
        do = _contig(do).view(o.shape)
        da = torch.empty_like(a)
        if b is None:
            q, k, v = _split_heads(a, 3, H, D)
            dq, dk, dv = _split_heads(da, 3, H, D)
            db = None
        else:
            db = torch.empty_like(b)
            q, dq = a.view(a.shape[0], a.shape[1], H, D), da.view(a.shape[0], a.shape[1], H, D)
            k, v = _split_heads(b, 2, H, D)
            dk, dv = _split_heads(db, 2, H, D)
        _flash_bwd(q, k, v, o, do, lse, kv_len, dq, dk, dv, scale, causal, o32)
        return da, db, None, None, None, None, None


def attention_packed(qkv_or_q, kv=None, heads=1, head_dim=64, kv_len=None, scale=None, causal=False):
    """bf16 flash attention on fused-projection outputs; returns [B, Sq, H D].  See _FlashAttnPackedFn."""
    if scale is None:
        scale = 1.0 / math.sqrt(head_dim)
    if ATTN_TRACE is not None:
        Sk = qkv_or_q.shape[1] if kv is None else kv.shape[1]
        ATTN_TRACE.append((qkv_or_q.shape[0], qkv_or_q.shape[1], Sk, heads, head_dim, int(causal), int(torch.is_grad_enabled() and qkv_or_q.requires_grad)))
    if kv_len is not None and kv_len.dtype != torch.int32:
        kv_len = kv_len.to(torch.int32)
    return _FlashAttnPackedFn.apply(qkv_or_q, kv, heads, head_dim, kv_len, scale, causal)


def flash_eligible(dtype, head_dim):
    return dtype == torch.bfloat16 and head_dim in (64, 128)


class _UnfusedAttnFn(Function):
    """Same contraction built from the batched MFMA GEMM + row-softmax kernels (exact-fp32 parity path; also the
    on-device cross-check of the flash kernel).  Materialises the [B, H, Sq, Sk] score matrix."""

    @staticmethod
    def forward(ctx, q, k, v, scale, causal, kv_len=None):
        require_cuda(q, k, v)
        B, Sq, H, D = q.shape
        Sk = k.shape[1]
        q, k, v = _contig(q), _contig(k), _contig(v)
        Skp = (Sk + 7) // 8 * 8
        p = torch.zeros((B, H, Sq, Skp), device=q.device, dtype=q.dtype)
        o = torch.empty((B, Sq, H, D), device=q.device, dtype=q.dtype)
        sq, sk = (Sq * H * D, D), (Sk * H * D, D)
        sp = (H * Sq * Skp, Sq * Skp)
        gemm(q, k, False, True, Sq, Sk, D, p, lda=H * D, ldb=H * D, ldc=Skp, batch_outer=B, batch_inner=H,
             stride_a=sq, stride_b=sk, stride_c=sp)
        dt = dtype_code(q.dtype)
        if kv_len is not None:      # keys past the valid count leave the softmax (exact-parity mode only: one ATen fill on the score matrix)
            p.masked_fill_(torch.arange(Skp, device=q.device).view(1, 1, 1, Skp) >= kv_len.view(B, 1, 1, 1), float('-inf'))
        check(lib().dpipe_softmax_fwd(ptr(p), ptr(p), B * H * Sq, Sk, Skp, float(scale), Sq if causal else 0, dt, stream()), 'softmax_fwd')
        gemm(p, v, False, False, Sq, D, Sk, o, lda=Skp, ldb=H * D, ldc=H * D, batch_outer=B, batch_inner=H,
             stride_a=sp, stride_b=sk, stride_c=sq)
        ctx.save_for_backward(q, k, v, p)
        ctx.scale = scale
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, p = ctx.saved_tensors
        B, Sq, H, D = q.shape
        Sk, Skp = k.shape[1], p.shape[-1]
        do = _contig(do)
        sq, sk = (Sq * H * D, D), (Sk * H * D, D)
        sp = (H * Sq * Skp, Sq * Skp)
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dp = torch.zeros_like(p)
        kw = dict(batch_outer=B, batch_inner=H)
        gemm(p, do, True, False, Sk, D, Sq, dv, lda=Skp, ldb=H * D, ldc=H * D, stride_a=sp, stride_b=sq, stride_c=sk, **kw)
        gemm(do, v, False, True, Sq, Sk, D, dp, lda=H * D, ldb=H * D, ldc=Skp, stride_a=sq, stride_b=sk, stride_c=sp, **kw)
        check(lib().dpipe_softmax_bwd(ptr(p), ptr(dp), ptr(dp), B * H * Sq, Sk, Skp, float(ctx.scale), dtype_code(q.dtype), stream()), 'softmax_bwd')
        gemm(dp, k, False, False, Sq, D, Sk, dq, lda=Skp, ldb=H * D, ldc=H * D, stride_a=sp, stride_b=sk, stride_c=sq, **kw)
        gemm(dp, q, True, False, Sk, D, Sq, dk, lda=Skp, ldb=H * D, ldc=H * D, stride_a=sp, stride_b=sq, stride_c=sk, **kw)
        return dq, dk, dv, None, None, None


ATTN_TRACE = None     # like GEMM_TRACE: (B, Sq, Sk, H, D, causal, has_backward) of every attention call of a step


def attention(q, k, v, kv_len=None, scale=None, impl='auto', causal=False):
    """q: [B, Sq, H, D], k/v: [B, Sk, H, D] -> [B, Sq, H, D].  kv_len: optional int32 [B] of valid keys.
    impl: 'flash' (bf16 MFMA flash kernel), 'unfused' (GEMM + softmax kernels), 'auto' = flash for bf16."""
    D = q.shape[-1]
    if ATTN_TRACE is not None:
        ATTN_TRACE.append((q.shape[0], q.shape[1], k.shape[1], q.shape[2], D, int(causal), int(torch.is_grad_enabled() and q.requires_grad)))
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    if impl == 'auto':
        impl = 'flash' if (q.dtype == torch.bfloat16 and D in (64, 128)) else 'unfused'
    if impl == 'flash':
        if kv_len is not None and kv_len.dtype != torch.int32:
            kv_len = kv_len.to(torch.int32)
        return _FlashAttnFn.apply(q, k, v, kv_len, scale, causal)
    return _UnfusedAttnFn.apply(q, k, v, scale, causal, kv_len)


@functools.lru_cache(maxsize=1024)
def _varlen_floats(backward, sizes):
    """fp32 workspace of a call of these sizes"""
    return (lib().dpipe_attn_varlen_bwd_workspace_floats if backward else lib().dpipe_attn_varlen_fwd_workspace_floats)(*sizes)


def _varlen_forward(q, k, v, cu_q, cu_k, scale, causal, keep):
    """-> (o, what the backward reads, what its call repeats); keep: the row statistics and what the output's rounding left are stored for the backward's P and delta"""
    device = q.device
    (q, tq, hq, D, *qs), (k, tk, hk, _, *ks), (v, _, _, _, *vs) = _head_rows(q), _head_rows(k), _head_rows(v)
    if tq == 0 or tk == 0:                        # nothing to read: every row is empty
        return torch.zeros(q.shape, device=device, dtype=q.dtype), (), None
    sizes, strides = (tq, tk, cu_q.shape[0] - 1, hq, hk, D), (*qs, *ks, *vs)
    o = _dense(q)
    dt = dtype_code(q.dtype)
    o_lo, lse = (torch.empty_like(o) if dt == hip.BF16 else None, q.new_empty((hq, tq), dtype=torch.float32)) if keep else (None, None)
    need = _varlen_floats(False, sizes)
    ws = torch.empty(need, device=device, dtype=torch.float32) if need else None
    check(lib().dpipe_attn_varlen_fwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), o.data_ptr(), _addr(o_lo), _addr(lse), _addr(ws), need, *sizes,
                                      *strides, scale, causal, dt, hip.raw_stream(device)), 'attn_varlen_fwd')
    return o, (q, k, v, cu_q, cu_k, o, o_lo, lse), (sizes, strides, scale, causal, dt)


class _AttnVarlenFn(Function):
    """see attention_varlen; keeps the bf16 output to 16 bits of significand (o and what its rounding left) for the backward's delta, where _FlashAttnFn keeps an fp32 copy"""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, causal):
        ctx.shapes = (q.shape, k.shape, v.shape, q.dtype)
        o, saved, ctx.call = _varlen_forward(q, k, v, cu_q, cu_k, scale, causal, True)
        ctx.save_for_backward(*saved)
        return o

    @staticmethod
    def backward(ctx, do):
        _no_second_graph('attention_varlen')
        device = do.device
        if ctx.call is None:
            *shapes, dtype = ctx.shapes
            return (*(torch.zeros(sh, device=device, dtype=dtype) for sh in shapes), None, None, None, None)
        q, k, v, cu_q, cu_k, o, o_lo, lse = ctx.saved_tensors
        sizes, strides, scale, causal, dt = ctx.call
        with _on(device):
            do, _, _, _, *ds = _head_rows(do)
            dq, dk, dv = _dense(q), _dense(k), _dense(v)
            delta = torch.empty_like(lse)
            need = _varlen_floats(True, sizes)
            ws = torch.empty(need, device=device, dtype=torch.float32) if need else None
            check(lib().dpipe_attn_varlen_bwd(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), o.data_ptr(), _addr(o_lo), do.data_ptr(), lse.data_ptr(),
                                              delta.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _addr(ws), need, *sizes, *strides, *ds, scale, causal,
                                              dt, hip.raw_stream(device)), 'attn_varlen_bwd')
        return dq, dk, dv, None, None, None, None


def attention_varlen(q, k, v, cu_q, cu_k=None, scale=None, causal=False):
    """softmax(scale q k^T) v over sequences of different lengths packed back to back; bf16, or fp32 throughout, head dim 64 or 128, differentiable once in q, k, v (reverse mode).

    q [Tq, H, D], k / v [Tk, Hk, D] with H a multiple of Hk: query head h reads key head h // (H // Hk).  Column blocks of a fused projection are read in place.
    cu_q, cu_k: int32 offsets [N + 1] on the device, ascending from 0; sequence b holds query tokens cu_q[b] .. cu_q[b + 1] - 1 and key tokens cu_k[b] .. cu_k[b + 1] - 1, either
    of which may be empty.  cu_k None: the queries' offsets (Tk = Tq).  The lengths are never read on the host: the call can be captured and replayed with other offsets.
    (As with any operator: while its backward pass is captured, no eager graph of the same leaf tensors may be alive -- their accumulation nodes would run on that graph's stream.)
    causal: query i sees key j of its sequence when j - len_k <= i - len_q (the last query sees every key; with equal lengths j <= i).
    A query that sees no key, and the rows behind the last sequence, give zeros and take and give no gradient, whatever those rows hold (the other values of a sequence are expected
    to be finite: an infinity or NaN reaches its sequence's other rows, also where it is masked).  The same inputs give the same bits (no atomics).  (models/wan/attention.py:91-122)
    -> [Tq, H, D]"""
    qs, ks, dtype = q.shape, k.shape, q.dtype
    if len(qs) != 3 or len(ks) != 3 or ks != v.shape or ks[2] != qs[2] or ks[1] == 0 or qs[1] == 0 or qs[1] % ks[1]:
        raise DpipeHipError(f'attention_varlen: q [Tq, H, D], k and v [Tk, Hk, D] with H a multiple of Hk; got {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}')
    if dtype not in (torch.bfloat16, torch.float32) or qs[2] not in (64, 128) or k.dtype != dtype or v.dtype != dtype:
        raise DpipeHipError(f'attention_varlen computes in bf16 or fp32 at head dim 64 or 128; got {dtype}, {k.dtype}, {v.dtype}, head dim {qs[2]}')
    if cu_k is None:
        if ks[0] != qs[0]:
            raise DpipeHipError(f'attention_varlen: shared offsets need as many keys as queries; got {qs[0]} and {ks[0]}')
        cu_k = cu_q
    for cu in (cu_q, cu_k):
        if cu.dtype not in (torch.int32, torch.int64) or cu.dim() != 1 or cu.shape[0] < 2 or cu.shape[0] != cu_q.shape[0]:
            raise DpipeHipError(f'attention_varlen: offsets are int32 [N + 1], N >= 1, for queries and keys alike; got {cu.dtype} {tuple(cu.shape)}, {tuple(cu_q.shape)}')
    scale = 1.0 / math.sqrt(qs[2]) if scale is None else float(scale)
    if not (scale > 0.0 and math.isfinite(scale)):
        raise DpipeHipError(f'attention_varlen: scale must be positive and finite, got {scale}')
    _no_tangents('attention_varlen', q, k, v)
    device = _one_device(q, k, v, cu_q, cu_k)
    cu_q, cu_k = (cu if cu.dtype == torch.int32 and cu.is_contiguous() else cu.to(torch.int32).contiguous() for cu in (cu_q, cu_k))
    with _on(device):
        if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
            return _AttnVarlenFn.apply(q, k, v, cu_q, cu_k, scale, int(causal))
        return _varlen_forward(q, k, v, cu_q, cu_k, scale, int(causal), False)[0]


# ------------------------------------------------------------------------------------------------- loss (K9)
class _LossFn(Function):
    @staticmethod
    def forward(ctx, out, target, mask, row_weight, rows, kind, param):
        require_cuda(out, target, mask, row_weight)
        oc = _contig(out)
        tc = _contig(target.to(device=out.device, dtype=torch.float32))
        mc = None
        if mask is not None and mask.numel() > 0:
            mc = mask.to(device=out.device, dtype=torch.float32)
            if mc.shape != oc.shape:
                mc = mc.expand_as(oc)
            mc = _contig(mc)
        cols = oc.numel() // rows
        ws = torch.empty(lib().dpipe_loss_workspace_floats(rows, cols), device=out.device, dtype=torch.float32)
        loss = torch.empty((), device=out.device, dtype=torch.float32)
        rw = _contig(row_weight.to(device=out.device, dtype=torch.float32)) if row_weight is not None else None
        check(lib().dpipe_loss_fwd(ptr(oc), dtype_code(oc.dtype), ptr(tc), ptr(mc), ptr(rw), rows, cols, hip.LOSS_KIND[kind],
                                   float(param), ptr(ws), ptr(loss), None, stream()), 'loss_fwd')
        ctx.save_for_backward(oc, tc, mc, rw)
        ctx.meta = (rows, cols, kind, param, out.shape)
        return loss

    @staticmethod
    def backward(ctx, gl):
        oc, tc, mc, rw = ctx.saved_tensors
        rows, cols, kind, param, shape = ctx.meta
        gl = gl.to(dtype=torch.float32).contiguous()
        go = torch.empty_like(oc)
        check(lib().dpipe_loss_bwd(ptr(oc), dtype_code(oc.dtype), ptr(tc), ptr(mc), ptr(rw), ptr(gl), rows, cols,
                                   hip.LOSS_KIND[kind], float(param), ptr(go), stream()), 'loss_bwd')
        return go.view(shape), None, None, None, None, None, None


def fused_loss(output, target, mask=None, row_weight=None, per_sample=False, kind='mse', param=0.0):
    """mean(elem(output - target) * mask); with per_sample: mean_b(row_weight[b] * mean_chw(...)).
    Reference: models/base.py:418-436 (default), models/sdxl.py:632-651 (per-sample x SNR weights)."""
    rows = output.shape[0] if per_sample else 1
    return _LossFn.apply(output, target, mask, row_weight, rows, kind, param)


# ------------------------------------------------------------------------------- grad-norm + clip (K10)
_CHUNK = 1 << 16
_table_cache = {}


def _chunk_table(tensors):
    key = tuple((t.data_ptr(), t.numel()) for t in tensors)
    hit = _table_cache.get(key)
    if hit is not None:
        return hit
    ptrs, ctens, coff, clen = [], [], [], []
    for i, t in enumerate(tensors):
        ptrs.append(t.data_ptr())
        n = t.numel()
        for off in range(0, n, _CHUNK):
            ctens.append(i); coff.append(off); clen.append(min(_CHUNK, n - off))
    dev = tensors[0].device
    table = (torch.tensor(ptrs, dtype=torch.int64, device=dev), torch.tensor(ctens, dtype=torch.int32, device=dev),
             torch.tensor(coff, dtype=torch.int64, device=dev), torch.tensor(clen, dtype=torch.int32, device=dev), len(ctens))
    if len(_table_cache) > 64:
        _table_cache.clear()
    _table_cache[key] = table
    return table


def grads_sumsq(grads):
    """fp32 device scalar: sum over all tensors of sum(g^2) (utils/patches.py:211-221)."""
    dev = grads[0].device
    total = torch.zeros((), device=dev, dtype=torch.float32)
    for dt in (torch.bfloat16, torch.float32):
        group = [g for g in grads if g.dtype == dt]
        if not group:
            continue
        for g in group:
            if not (g.is_contiguous() or (g.dim() == 4 and g.is_contiguous(memory_format=torch.channels_last))):
                raise DpipeHipError('gradients must be dense (row-major or channels-last)')
        ptrs, ctens, coff, clen, n = _chunk_table(group)
        partials = torch.empty(max(n, 1), device=dev, dtype=torch.float32)
        out = torch.empty((), device=dev, dtype=torch.float32)
        check(lib().dpipe_multi_sumsq(ptr(ptrs), ptr(ctens), ptr(coff), ptr(clen), n, dtype_code(dt), ptr(partials), ptr(out), stream()), 'multi_sumsq')
        total = total + out
    rest = [g for g in grads if g.dtype not in (torch.bfloat16, torch.float32)]
    if rest:
        raise DpipeHipError(f'unsupported gradient dtype {rest[0].dtype}')
    return total


def grads_clip_scale_(grads, total_sumsq, max_norm):
    """g *= min(1, max_norm / (sqrt(total_sumsq) + 1e-6)) in place, no host sync (utils/patches.py:240-245)."""
    for dt in (torch.bfloat16, torch.float32):
        group = [g for g in grads if g.dtype == dt]
        if not group:
            continue
        ptrs, ctens, coff, clen, n = _chunk_table(group)
        check(lib().dpipe_multi_clip_scale(ptr(ptrs), ptr(ctens), ptr(coff), ptr(clen), n, dtype_code(dt), ptr(total_sumsq),
                                           float(max_norm), stream()), 'multi_clip_scale')


# ------------------------------------------------------------------------ fused step end (lane sum + clip + AdamW + zero)
_adam_tables = {}


def _adam_table(params, exp_avgs, exp_avg_sqs, lane_grads, shifts=None):
    """Device pointer / chunk tables of one (dtype, param group); cached on the parameter / state addresses.  The gradient pointer table is
    rebuilt whenever the gradient buffers moved (eager path: autograd allocates fresh .grad tensors every step; graph path: persistent) --
    the cache keeps only the CURRENT gradient tensors alive, never those of earlier steps."""
    L = len(lane_grads)
    key = (L,) + tuple(t.data_ptr() for t in params) + tuple(t.data_ptr() for t in exp_avgs) + (tuple(t.data_ptr() for t in shifts) if shifts is not None else ())
    gkey = tuple(g.data_ptr() for lane in lane_grads for g in lane)
    dev = params[0].device
    i64 = lambda xs: torch.tensor(xs, dtype=torch.int64, device=dev)
    hit = _adam_tables.get(key)
    if hit is not None:
        if hit['gkey'] != gkey:
            hit['g'] = i64([lane_grads[l][i].data_ptr() for i in range(len(params)) for l in range(L)])
            hit['gkey'] = gkey
        hit['keep'] = (params, exp_avgs, exp_avg_sqs, lane_grads, shifts)
        return hit
    ctens, coff, clen = [], [], []
    for i, t in enumerate(params):
        n = t.numel()
        for off in range(0, n, _CHUNK):
            ctens.append(i); coff.append(off); clen.append(min(_CHUNK, n - off))
    table = {'p': i64([t.data_ptr() for t in params]), 'm': i64([t.data_ptr() for t in exp_avgs]), 'v': i64([t.data_ptr() for t in exp_avg_sqs]),
             'g': i64([lane_grads[l][i].data_ptr() for i in range(len(params)) for l in range(L)]), 'gkey': gkey,
             'ctens': torch.tensor(ctens, dtype=torch.int32, device=dev), 'coff': i64(coff),
             'clen': torch.tensor(clen, dtype=torch.int32, device=dev), 'n': len(ctens),
             'partials': torch.empty(max(len(ctens), 1), device=dev, dtype=torch.float32), 'keep': (params, exp_avgs, exp_avg_sqs, lane_grads, shifts),
             's': i64([t.data_ptr() for t in shifts]) if shifts is not None else None}
    if len(_adam_tables) > 64:
        _adam_tables.clear()
    _adam_tables[key] = table
    return table


def _adam_check(params, exp_avgs, exp_avg_sqs, lane_grads):
    require_cuda(*params)
    dt = params[0].dtype
    if dt not in (torch.bfloat16, torch.float32):
        raise DpipeHipError(f'fused AdamW: unsupported dtype {dt}')
    if not 1 <= len(lane_grads) <= 8:
        raise DpipeHipError('fused AdamW: 1..8 gradient lanes')
    for group in (params, exp_avgs, exp_avg_sqs, *lane_grads):
        if len(group) != len(params):
            raise DpipeHipError('fused AdamW: ragged tensor lists')
        for t, p in zip(group, params):
            dense = p.is_contiguous() or (p.dim() == 4 and p.is_contiguous(memory_format=torch.channels_last))
            if t.dtype != dt or t.shape != p.shape or not dense or t.stride() != p.stride():
                raise DpipeHipError('fused AdamW: parameters, states and gradients must be dense tensors of one dtype, shape and memory layout')
    return dt


def adamw_grads_sumsq(params, exp_avgs, exp_avg_sqs, lane_grads, out, accumulate=False):
    """out (+)= sum over elements of (sum over lanes g)^2 for one same-dtype tensor group (fp32 device scalar)."""
    dt = _adam_check(params, exp_avgs, exp_avg_sqs, lane_grads)
    t = _adam_table(params, exp_avgs, exp_avg_sqs, lane_grads)
    check(lib().dpipe_adamw_sumsq(ptr(t['g']), len(lane_grads), ptr(t['ctens']), ptr(t['coff']), ptr(t['clen']), t['n'], dtype_code(dt),
                                  ptr(t['partials']), ptr(out), int(accumulate), stream()), 'adamw_sumsq')
    return out


def adamw_step(params, exp_avgs, exp_avg_sqs, lane_grads, *, lr, beta1, beta2, eps, weight_decay, step, total_sumsq=None, max_norm=0.0,
               zero_grads=True, shifts=None):
    """One fused pass over a same-dtype group: g = clip * sum_lanes g; AdamW update in fp32; lanes zeroed.  shifts: the parameters' Kahan
    compensation buffers (optimizers/generic_optim.py:486-497) -> compensated application of the update."""
    dt = _adam_check(params, exp_avgs, exp_avg_sqs, lane_grads)
    t = _adam_table(params, exp_avgs, exp_avg_sqs, lane_grads, shifts)
    tail = (len(lane_grads), ptr(t['ctens']), ptr(t['coff']), ptr(t['clen']), t['n'], dtype_code(dt), float(lr), float(beta1), float(beta2), float(eps),
            float(weight_decay), float(1.0 - beta1 ** step), float(1.0 - beta2 ** step), ptr(total_sumsq), float(max_norm), int(zero_grads), stream())
    if shifts is not None:
        for sft, p in zip(shifts, params):
            if sft.dtype != dt or sft.shape != p.shape or sft.stride() != p.stride():
                raise DpipeHipError('fused AdamW: Kahan shift buffers must match their parameters')
        check(lib().dpipe_adamw_step_kahan(ptr(t['p']), ptr(t['m']), ptr(t['v']), ptr(t['s']), ptr(t['g']), *tail), 'adamw_step_kahan')
    else:
        check(lib().dpipe_adamw_step(ptr(t['p']), ptr(t['m']), ptr(t['v']), ptr(t['g']), *tail), 'adamw_step')


def release_caches():
    """Drop the module-level caches that keep device memory alive after an engine is gone: the fused step end's pointer tables hold references to the parameters,
    optimizer states and lane gradients they were built for (`keep`), the clip kernels' chunk tables to the gradients, the split-K workspaces to ~42 MB per lane.
    Call between two workloads of one process (bench.py's `other_configs` leg) before `torch.cuda.empty_cache()`; everything is rebuilt on demand."""
    _adam_tables.clear()
    _table_cache.clear()
    _SPLITK_WS.clear()


# ----------------------------------------------------------------------------------------- small helpers (K7/K8)
def sinusoidal_embedding(t, dim, max_period=10000.0, sin_first=False, downscale_shift=0.0, scale=1.0):
    """[cos | sin] (Wan, models/wan/model.py:15-25) or [sin | cos] (sin_first) timestep embedding, fp32."""
    require_cuda(t)
    tc = _contig(t.to(torch.float32).reshape(-1))
    out = torch.empty((tc.numel(), dim), device=t.device, dtype=torch.float32)
    check(lib().dpipe_sinusoidal_embed(ptr(tc), ptr(out), tc.numel(), dim, float(max_period), int(sin_first), float(downscale_shift),
                                       float(scale), stream()), 'sinusoidal_embed')
    return out


def flow_match_prep(x1, x0, t):
    """x_t = (1-t) x1 + t x0, target = x0 - x1  (models/flux.py:368-372).  fp32 tensors, t: [B]."""
    require_cuda(x1, x0, t)
    x1, x0, t = _contig(x1.float()), _contig(x0.float()), _contig(t.float())
    xt, target = torch.empty_like(x1), torch.empty_like(x1)
    B = x1.shape[0]
    check(lib().dpipe_flow_match_prep(ptr(x1), ptr(x0), ptr(t), ptr(xt), ptr(target), B, x1.numel() // B, stream()), 'flow_match_prep')
    return xt, target


def transpose2d(x):
    """[..., R, C] -> [..., C, R] materialised by the LDS tile-transpose kernel."""
    require_cuda(x)
    xc = _contig(x)
    R, C = xc.shape[-2:]
    batch = xc.numel() // (R * C)
    out = torch.empty(*xc.shape[:-2], C, R, device=x.device, dtype=x.dtype)
    check(lib().dpipe_transpose(ptr(xc), ptr(out), R, C, C, R, R * C, R * C, batch, dtype_code(x.dtype), stream()), 'transpose')
    return out

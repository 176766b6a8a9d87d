"""tune.py - losses over rows of logits that tune a trained model (csrc/tune.hip): a clipped policy loss with a KL term and
a paired preference loss, each with its gradient.

A row of logits is one decision (a token; an active pair of a graph, classes 0 / 1), `taken` what was chosen there (int64,
or uint8 as the sampler's bits are), and the rows of one sequence (an answer; a graph) are consecutive: sequence s is rows
seq_ptr[s] .. seq_ptr[s+1]-1, ascending from 0, empty ones allowed (`aptr` of the active pairs is a seq_ptr).  A row counts
unless its mask is False, its `taken` lies outside the classes (-100, say) or it lies in no sequence; what stands in the
logits of the others does not matter, and their gradient is 0.

`policy_loss` / `preference_loss` are differentiable in the logits; the `_grad` forms return the gradient of
sum(weight * loss) at once, without a graph (`logits.backward(r.dlogits)` goes on from it)."""
import ctypes as C
from collections import namedtuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import capi

lib = capi.lib
byref = C.byref
KINDS = {'sigmoid': 0, 'square': 1}
REDUCE = {'sum': 0, 'mean': 1}

PolicyLoss = namedtuple('PolicyLoss', 'loss kl clipped logp')
PolicyGrad = namedtuple('PolicyGrad', 'loss kl clipped logp dlogits')
PreferenceLoss = namedtuple('PreferenceLoss', 'loss margin')
PreferenceGrad = namedtuple('PreferenceGrad', 'loss margin dlogits')


def _vector(what, name, t, n, dtype, dev):
    if t is None:
        return None
    capi.same_device(what, name, t, dev)
    if t.dtype != dtype or t.shape != (n,):
        raise ValueError(f'{what}: {name} must be [{n}] of {dtype}, got {tuple(t.shape)} of {t.dtype}')
    return t.contiguous()


def _describe(what, logits, taken, seq_ptr, mask):
    """(C description, the tensors it points to)"""
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f'{what}: logits must be [rows, classes], got {tuple(logits.shape)}')
    code = capi.dtype_code(what, 'logits', logits)
    rows, classes = logits.shape
    if classes > 1 << 30 or seq_ptr is not None and seq_ptr.numel() > 1 << 24:
        raise ValueError(f'{what}: up to 2^30 classes and 2^24 - 1 sequences')
    dev = logits.device
    if classes > 1 and logits.stride(1) != 1 or rows > 1 and logits.stride(0) < classes:
        logits = logits.contiguous()
    small = taken.dtype == torch.uint8
    taken = _vector(what, 'taken', taken, rows, torch.uint8 if small else torch.int64, dev)
    if mask is not None:
        if mask.dtype not in (torch.bool, torch.uint8):
            raise ValueError(f'{what}: mask must be bool or uint8, got {mask.dtype}')
        mask = _vector(what, 'mask', mask, rows, mask.dtype, dev)
    if seq_ptr is not None:
        capi.same_device(what, 'seq_ptr', seq_ptr, dev)
        if seq_ptr.dtype != torch.int64 or seq_ptr.dim() != 1 or seq_ptr.numel() < 2:
            raise ValueError(f'{what}: seq_ptr must be an int64 vector of sequences + 1 offsets')
        seq_ptr = seq_ptr.contiguous()
    Q = capi.LogitRows()
    Q.rows, Q.classes, Q.dtype = rows, classes, code
    Q.row_stride = logits.stride(0) if rows > 1 else classes
    Q.taken_type = int(small)
    Q.num_seqs = 0 if seq_ptr is None else seq_ptr.numel() - 1
    Q.logits, Q.taken, Q.mask, Q.seq_ptr = logits.data_ptr(), taken.data_ptr(), capi.ptr(mask), capi.ptr(seq_ptr)
    return Q, (logits, taken, mask, seq_ptr)


def _workspace(Q, dev):
    nbytes = lib.edgehip_tune_workspace_bytes(byref(Q))
    if nbytes == 0:
        raise capi.EdgeHipError('edgehip_tune_workspace_bytes: unsupported configuration')
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def row_logp(logits, taken, mask=None):
    """[rows] fp32: the log-probability of what each row took (0 where the row does not count).  For the log-probabilities
    of the policy that generated and of a reference model; not differentiable."""
    Q, keep = _describe('row_logp', logits, taken, None, mask)
    capi.on_gpu('row_logp', logits)
    out = torch.empty(Q.rows, dtype=torch.float32, device=logits.device)
    with capi.on_device_of(logits) as stream:
        capi.check(lib.edgehip_row_logp(byref(Q), out.data_ptr(), stream), 'row_logp')
    return out


def _policy_args(what, logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask, weight, clip, kl_coef, reduce):
    if seq_ptr is None:
        raise ValueError(f'{what}: seq_ptr is needed')
    Q, keep = _describe(what, logits, taken, seq_ptr, mask)
    dev, rows, seqs = logits.device, Q.rows, Q.num_seqs
    if reduce not in REDUCE:
        raise ValueError(f'{what}: reduce must be one of {sorted(REDUCE)}, got {reduce!r}')
    lo, hi = (clip, clip) if isinstance(clip, (int, float)) else clip
    if not (lo >= 0 and hi >= 0):
        raise ValueError(f'{what}: clip must not be negative, got {clip}')
    if kl_coef and ref_logp is None:
        raise ValueError(f'{what}: a KL term needs ref_logp')
    old_logp = _vector(what, 'old_logp', old_logp, rows, torch.float32, dev)
    ref_logp = _vector(what, 'ref_logp', ref_logp, rows, torch.float32, dev)
    if advantage.shape not in ((seqs,), (rows,)):
        raise ValueError(f'{what}: advantage must be [{seqs}] (per sequence) or [{rows}] (per row), got {tuple(advantage.shape)}')
    per_row = advantage.shape != (seqs,)
    advantage = _vector(what, 'advantage', advantage, advantage.shape[0], torch.float32, dev)
    weight = _vector(what, 'weight', weight, seqs, torch.float32, dev)
    O = capi.Policy(capi.ptr(old_logp), capi.ptr(advantage), capi.ptr(ref_logp), capi.ptr(weight), float(lo), float(hi),
                    float(kl_coef), int(per_row), REDUCE[reduce])
    capi.on_gpu(what, logits)
    return Q, O, keep + (old_logp, advantage, ref_logp, weight)


def _policy_out(Q, dev):
    f = dict(dtype=torch.float32, device=dev)
    return (torch.empty(Q.num_seqs, **f), torch.empty(Q.num_seqs, **f), torch.empty(Q.num_seqs, dtype=torch.int32, device=dev),
            torch.empty(Q.rows, **f))


def policy_loss_grad(logits, taken, old_logp, advantage, seq_ptr, *, ref_logp=None, mask=None, weight=None, clip=(0.2, 0.2),
                     kl_coef=0.0, reduce='mean'):
    """PolicyGrad(loss [S], kl [S], clipped [S], logp [rows], dlogits): the policy loss and, from the same pass over the
    logits, the gradient of sum(weight * loss) (weight None: the mean over the sequences).

    With rho = exp(logp - old_logp) and gap = ref_logp - logp a counted row adds
        -min(rho A, clip(rho, 1 - clip[0], 1 + clip[1]) A) + kl_coef (exp(gap) - gap - 1)
    to its sequence, which is divided by its counted rows (reduce 'mean') or not ('sum').  advantage: per sequence [S] or per
    row [rows] ([S] where the two are one number).  kl: the same reduction of exp(gap) - gap - 1; clipped: rows whose clip
    binds (their gradient is the KL term's alone; a ratio on the very edge still counts as inside)."""
    Q, O, keep = _policy_args('policy_loss_grad', logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask, weight, clip,
                              kl_coef, reduce)
    dev = logits.device
    loss, kl, clipped, logp = _policy_out(Q, dev)
    dlogits = torch.empty((Q.rows, Q.classes), dtype=logits.dtype, device=dev)
    ws = _workspace(Q, dev)
    with capi.on_device_of(logits) as stream:
        capi.check(lib.edgehip_policy_loss_grad(byref(Q), byref(O), loss.data_ptr(), kl.data_ptr(), clipped.data_ptr(),
                                                logp.data_ptr(), dlogits.data_ptr(), ws.data_ptr(), ws.numel(),
                                                stream), 'policy_loss_grad')
    return PolicyGrad(loss, kl, clipped, logp, dlogits)


class _PolicyLoss(Function):
    @staticmethod
    def forward(ctx, logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask, opts):
        Q, O, keep = _policy_args('policy_loss', logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask, None, **opts)
        loss, kl, clipped, logp = _policy_out(Q, logits.device)
        ws = _workspace(Q, logits.device)
        with capi.on_device_of(logits) as stream:
            capi.check(lib.edgehip_policy_loss_fwd(byref(Q), byref(O), loss.data_ptr(), kl.data_ptr(), clipped.data_ptr(),
                                                   logp.data_ptr(), ws.data_ptr(), ws.numel(), stream),
                       'policy_loss_fwd')
        ctx.save_for_backward(logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask, ws)
        ctx.opts = opts
        ctx.mark_non_differentiable(kl, clipped, logp)
        return loss, kl, clipped, logp

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, *_):
        logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask, ws = ctx.saved_tensors
        Q, O, keep = _policy_args('policy_loss', logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask,
                                  dloss.float().contiguous(), **ctx.opts)
        dlogits = torch.empty((Q.rows, Q.classes), dtype=logits.dtype, device=logits.device)
        with capi.on_device_of(logits) as stream:
            capi.check(lib.edgehip_policy_loss_bwd(byref(Q), byref(O), dlogits.data_ptr(), ws.data_ptr(), ws.numel(),
                                                   stream), 'policy_loss_bwd')
        return (dlogits,) + (None,) * 7


def policy_loss(logits, taken, old_logp, advantage, seq_ptr, *, ref_logp=None, mask=None, clip=(0.2, 0.2), kl_coef=0.0,
                reduce='mean'):
    """PolicyLoss(loss [S], kl [S], clipped [S], logp [rows]) of `policy_loss_grad`, `loss` differentiable in the logits."""
    opts = dict(clip=clip, kl_coef=kl_coef, reduce=reduce)
    return PolicyLoss(*_PolicyLoss.apply(logits, taken, old_logp, advantage, seq_ptr, ref_logp, mask, opts))


def _preference_args(what, logits, taken, seq_ptr, ref_logp, mask, weight, beta, label_smoothing, kind, reduce):
    if seq_ptr is None:
        raise ValueError(f'{what}: seq_ptr is needed')
    Q, keep = _describe(what, logits, taken, seq_ptr, mask)
    if Q.num_seqs % 2:
        raise ValueError(f'{what}: as many preferred sequences as others are needed, got {Q.num_seqs} in all')
    if kind not in KINDS or reduce not in REDUCE:
        raise ValueError(f'{what}: kind must be one of {sorted(KINDS)} and reduce one of {sorted(REDUCE)}, got {kind!r}, {reduce!r}')
    if not beta > 0 or not 0 <= label_smoothing < 0.5 or (label_smoothing and kind != 'sigmoid'):
        raise ValueError(f'{what}: beta > 0 and, for the sigmoid kind, label_smoothing in [0, 0.5) are needed')
    ref_logp = _vector(what, 'ref_logp', ref_logp, Q.rows, torch.float32, logits.device)
    weight = _vector(what, 'weight', weight, Q.num_seqs // 2, torch.float32, logits.device)
    O = capi.Preference(capi.ptr(ref_logp), capi.ptr(weight), float(beta), float(label_smoothing), KINDS[kind], REDUCE[reduce])
    capi.on_gpu(what, logits)
    return Q, O, keep + (ref_logp, weight)


def _preference_fwd(Q, O, dev, stream):
    loss = torch.empty(Q.num_seqs // 2, dtype=torch.float32, device=dev)
    margin = torch.empty_like(loss)
    ws = _workspace(Q, dev)
    capi.check(lib.edgehip_preference_loss_fwd(byref(Q), byref(O), loss.data_ptr(), margin.data_ptr(), ws.data_ptr(), ws.numel(),
                                               stream), 'preference_loss_fwd')
    return loss, margin, ws


def _preference_bwd(Q, O, logits, ws, stream):
    dlogits = torch.empty((Q.rows, Q.classes), dtype=logits.dtype, device=logits.device)
    capi.check(lib.edgehip_preference_loss_bwd(byref(Q), byref(O), dlogits.data_ptr(), ws.data_ptr(), ws.numel(),
                                               stream), 'preference_loss_bwd')
    return dlogits


def preference_loss_grad(logits, taken, seq_ptr, *, ref_logp=None, mask=None, weight=None, beta=0.1, label_smoothing=0.0,
                         kind='sigmoid', reduce='sum'):
    """PreferenceGrad(loss [P], margin [P], dlogits): the preference loss of P pairs and the gradient of sum(weight * loss)
    (weight None: the mean over the pairs).  Of the 2 P sequences, p was preferred to P + p.

    margin = m_p - m_{P+p}, m the sum (reduce 'mean': the mean) of logp - ref_logp over a sequence's counted rows.
    'sigmoid': -(1 - label_smoothing) ln sigmoid(beta margin) - label_smoothing ln sigmoid(-beta margin);
    'square': (margin - 1 / (2 beta))^2."""
    Q, O, keep = _preference_args('preference_loss_grad', logits, taken, seq_ptr, ref_logp, mask, weight, beta, label_smoothing,
                                  kind, reduce)
    dev = logits.device
    loss = torch.empty(Q.num_seqs // 2, dtype=torch.float32, device=dev)
    margin = torch.empty_like(loss)
    dlogits = torch.empty((Q.rows, Q.classes), dtype=logits.dtype, device=dev)
    ws = _workspace(Q, dev)
    with capi.on_device_of(logits) as stream:
        capi.check(lib.edgehip_preference_loss_grad(byref(Q), byref(O), loss.data_ptr(), margin.data_ptr(), dlogits.data_ptr(),
                                                    ws.data_ptr(), ws.numel(), stream), 'preference_loss_grad')
    return PreferenceGrad(loss, margin, dlogits)


class _PreferenceLoss(Function):
    @staticmethod
    def forward(ctx, logits, taken, seq_ptr, ref_logp, mask, opts):
        Q, O, keep = _preference_args('preference_loss', logits, taken, seq_ptr, ref_logp, mask, None, **opts)
        with capi.on_device_of(logits) as stream:
            loss, margin, ws = _preference_fwd(Q, O, logits.device, stream)
        ctx.save_for_backward(logits, taken, seq_ptr, ref_logp, mask, ws)
        ctx.opts = opts
        ctx.mark_non_differentiable(margin)
        return loss, margin

    @staticmethod
    @once_differentiable
    def backward(ctx, dloss, _):
        logits, taken, seq_ptr, ref_logp, mask, ws = ctx.saved_tensors
        Q, O, keep = _preference_args('preference_loss', logits, taken, seq_ptr, ref_logp, mask, dloss.float().contiguous(),
                                      **ctx.opts)
        with capi.on_device_of(logits) as stream:
            return (_preference_bwd(Q, O, logits, ws, stream),) + (None,) * 5


def preference_loss(logits, taken, seq_ptr, *, ref_logp=None, mask=None, beta=0.1, label_smoothing=0.0, kind='sigmoid',
                    reduce='sum'):
    """PreferenceLoss(loss [P], margin [P]) of `preference_loss_grad`, `loss` differentiable in the logits."""
    opts = dict(beta=beta, label_smoothing=label_smoothing, kind=kind, reduce=reduce)
    return PreferenceLoss(*_PreferenceLoss.apply(logits, taken, seq_ptr, ref_logp, mask, opts))

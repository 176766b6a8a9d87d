"""block.py - the step between two blocks of a deep network as one forward and one backward kernel (csrc/block.hip):

    u = N_post(z);   h' = res_scale h + gate u;   y = N_pre(h')

with root-mean-square or mean-and-variance norms.  `gate_norm` is the differentiable form; `gate_norm_fwd` /
`gate_norm_bwd` are its two halves for callers that order their own backward pass."""
import ctypes as C

import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import capi

lib = capi.lib
byref = C.byref
KINDS = {'rms': 0, 'layer': 1}
GATE_NONE, GATE_VECTOR, GATE_GROUP, GATE_ROW = range(4)
MAX_DIM = 8192


def _params(what, dim, branch, dev, **tensors):
    """The common type code of the parameters that are given (fp32 or the branch's)."""
    code = None
    for name, t in tensors.items():
        if t is None:
            continue
        capi.same_device(what, name, t, dev)
        if t.shape != (dim,) or not t.is_contiguous():
            raise ValueError(f'{what}: {name} must be a dense vector of {dim} values, got {tuple(t.shape)}')
        c = capi.dtype_code(what, name, t)
        if c != capi.F32 and c != branch:
            raise ValueError(f'{what}: {name} must be fp32 or of the type of z')
        if code is not None and c != code:
            raise ValueError(f'{what}: weights and biases must share one type')
        code = c
    return capi.F32 if code is None else code


def _describe(what, h, z, w_pre, b_pre, w_post, b_post, gate, row_ptr, kind, pre, post, res_scale, eps):
    """Checks the arguments and returns (the C description, h and z as dense [rows, dim] tensors, the dense gate)."""
    if kind not in KINDS:
        raise ValueError(f'{what}: kind must be one of {sorted(KINDS)}, got {kind!r}')
    if h.shape != z.shape or h.dim() < 1:
        raise ValueError(f'{what}: h and z must have one shape, got {tuple(h.shape)} and {tuple(z.shape)}')
    dim = h.shape[-1]
    if not 1 <= dim <= MAX_DIM:
        raise ValueError(f'{what}: rows of 1 to {MAX_DIM} values, got {dim}')
    dev = h.device
    capi.same_device(what, 'z', z, dev)
    hc, zc = capi.dtype_code(what, 'h', h), capi.dtype_code(what, 'z', z)
    if hc != zc and hc != capi.F32:
        raise ValueError(f'{what}: h must be fp32 or of the type of z')
    if kind == 'rms' and (b_pre is not None or b_post is not None):
        raise ValueError(f'{what}: the root-mean-square norm has no bias')
    if not pre and (w_pre is not None or b_pre is not None) or not post and (w_post is not None or b_post is not None):
        raise ValueError(f'{what}: parameters of a norm that is switched off')
    G = capi.GateNorm()
    G.param_dtype = _params(what, dim, zc, dev, w_pre=w_pre, b_pre=b_pre, w_post=w_post, b_post=b_post)
    rows = h.numel() // dim
    G.rows, G.dim, G.stream_dtype, G.branch_dtype, G.kind = rows, dim, hc, zc, KINDS[kind]
    G.pre, G.post, G.res_scale, G.eps = int(pre), int(post), float(res_scale), float(eps)
    G.w_pre, G.b_pre, G.w_post, G.b_post = capi.ptr(w_pre), capi.ptr(b_pre), capi.ptr(w_post), capi.ptr(b_post)
    G.gate_kind = GATE_NONE
    if row_ptr is not None and gate is None:
        raise ValueError(f'{what}: row_ptr without a gate')
    if gate is not None:
        capi.same_device(what, 'gate', gate, dev)
        G.gate_dtype = capi.dtype_code(what, 'gate', gate)
        if G.gate_dtype not in (capi.F32, zc):
            raise ValueError(f'{what}: gate must be fp32 or of the type of z')
        if row_ptr is not None:
            capi.same_device(what, 'row_ptr', row_ptr, dev)
            if row_ptr.dtype != torch.int32 or row_ptr.dim() != 1 or not row_ptr.is_contiguous() or row_ptr.numel() < 2:
                raise ValueError(f'{what}: row_ptr must be a dense int32 vector of groups + 1 offsets')
            if row_ptr.numel() > 65536:
                raise ValueError(f'{what}: up to 65535 groups, got {row_ptr.numel() - 1}')
            G.groups = row_ptr.numel() - 1
            if gate.shape != (G.groups, dim):
                raise ValueError(f'{what}: a gate per group must be [{G.groups}, {dim}], got {tuple(gate.shape)}')
            G.gate_kind, G.row_ptr = GATE_GROUP, row_ptr.data_ptr()
        elif gate.shape == (dim,) and h.dim() > 1:
            G.gate_kind = GATE_VECTOR
        elif gate.shape == h.shape:
            G.gate_kind = GATE_ROW
        else:
            raise ValueError(f'{what}: gate must be [{dim}], {list(h.shape)}, or [groups, {dim}] with row_ptr; got '
                             f'{tuple(gate.shape)}')
        gate = gate.contiguous()
        G.gate = gate.data_ptr()
    capi.on_gpu(what, h)
    return G, h.contiguous(), z.contiguous(), gate


def _fwd(G, h, z, want_stats):
    h_out = torch.empty_like(h)
    y = torch.empty_like(z) if G.pre else None
    stats = torch.empty((G.rows, 4), dtype=torch.float32, device=h.device) if want_stats else None
    with capi.on_device_of(h) as stream:
        capi.check(lib.edgehip_gate_norm_fwd(byref(G), h.data_ptr(), z.data_ptr(), h_out.data_ptr(), capi.ptr(y),
                                             capi.ptr(stats), stream), 'gate_norm_fwd')
    return h_out, y, stats


def gate_norm_fwd(h, z, *, w_pre=None, b_pre=None, w_post=None, b_post=None, gate=None, row_ptr=None, kind='rms', pre=True,
                  post=True, res_scale=1.0, eps=1e-6, want_stats=False):
    """(h', y, stats): h' = res_scale h + gate N_post(z), y = N_pre(h').  Not differentiable by itself.

    h, z: [..., dim], z fp32 / bf16 / fp16, h of the same type or fp32 (h' like h, y like z).  gate: None, [dim], one row
    per group of rows [groups, dim] (65535 groups at most) with row_ptr [groups + 1] int32 (a batch's node_ptr), or one per
    row, shaped like h.
    w_*, b_*: [dim], fp32 or of z's type; None: ones / zeros.  post=False: z itself is gated; pre=False: y is None.
    stats [rows, 4] (want_stats) is what `gate_norm_bwd` needs besides h and z."""
    G, h, z, gate = _describe('gate_norm', h, z, w_pre, b_pre, w_post, b_post, gate, row_ptr, kind, pre, post, res_scale, eps)
    return _fwd(G, h, z, want_stats)


def _bwd(G, dh_out, dy, h, z, stats, gate, like, want):
    """Gradients by name; `want`: names of the parameters whose gradient is asked for."""
    dev = h.device
    out = dict(dh=torch.empty_like(h), dz=torch.empty_like(z))
    for k in ('w_pre', 'b_pre', 'w_post', 'b_post'):
        if k in want:
            out['d' + k] = torch.empty_like(like[k])
    if 'gate' in want:
        out['dgate'] = torch.empty_like(gate)
    nbytes = lib.edgehip_gate_norm_workspace_bytes(byref(G))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    p = {k: v.data_ptr() for k, v in out.items()}
    with capi.on_device_of(h) as stream:
        capi.check(lib.edgehip_gate_norm_bwd(byref(G), capi.ptr(dh_out), capi.ptr(dy), h.data_ptr(), z.data_ptr(),
                                             stats.data_ptr(), p['dh'], p['dz'], p.get('dgate'), p.get('dw_pre'),
                                             p.get('db_pre'), p.get('dw_post'), p.get('db_post'), ws.data_ptr(), nbytes,
                                             stream), 'gate_norm_bwd')
    return out


def _grad_like(what, name, g, t):
    if g is None:
        return None
    capi.same_device(what, name, g, t.device)
    if g.shape != t.shape or g.dtype != t.dtype:
        raise ValueError(f'{what}: {name} must be {list(t.shape)} of {t.dtype}, got {tuple(g.shape)} of {g.dtype}')
    return g.contiguous()


def gate_norm_bwd(dh_out, dy, h, z, stats, *, w_pre=None, b_pre=None, w_post=None, b_post=None, gate=None, row_ptr=None,
                  kind='rms', pre=True, post=True, res_scale=1.0, eps=1e-6):
    """Gradients of `gate_norm_fwd` (same arguments) as a dict: dh, dz, and d<name> of every parameter that was given.
    dh_out / dy: gradients of h' and y; None: zero.  Sums over rows are made in a fixed order."""
    what = 'gate_norm_bwd'
    G, h, z, gate = _describe(what, h, z, w_pre, b_pre, w_post, b_post, gate, row_ptr, kind, pre, post, res_scale, eps)
    capi.same_device(what, 'stats', stats, h.device)
    if stats.shape != (G.rows, 4) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f'{what}: stats must be the dense fp32 [{G.rows}, 4] of the forward')
    if not pre and dy is not None:
        raise ValueError(f'{what}: dy without y')
    like = dict(w_pre=w_pre, b_pre=b_pre, w_post=w_post, b_post=b_post)
    want = {k for k, v in like.items() if v is not None} | ({'gate'} if gate is not None else set())
    return _bwd(G, _grad_like(what, 'dh_out', dh_out, h), _grad_like(what, 'dy', dy, z), h, z, stats, gate, like, want)


class _GateNorm(Function):
    @staticmethod
    def forward(ctx, h, z, w_pre, b_pre, w_post, b_post, gate, row_ptr, opts):
        G, hc, zc, gc = _describe('gate_norm', h, z, w_pre, b_pre, w_post, b_post, gate, row_ptr, **opts)
        h_out, y, stats = _fwd(G, hc, zc, True)
        ctx.save_for_backward(hc, zc, w_pre, b_pre, w_post, b_post, gc, row_ptr, stats)
        ctx.opts = opts
        ctx.set_materialize_grads(False)
        return h_out, y

    @staticmethod
    @once_differentiable
    def backward(ctx, dh_out, dy):
        h, z, w_pre, b_pre, w_post, b_post, gate, row_ptr, stats = ctx.saved_tensors
        G, h, z, gate = _describe('gate_norm', h, z, w_pre, b_pre, w_post, b_post, gate, row_ptr, **ctx.opts)
        like = dict(w_pre=w_pre, b_pre=b_pre, w_post=w_post, b_post=b_post)
        names = ('w_pre', 'b_pre', 'w_post', 'b_post', 'gate')
        want = {k for k, need in zip(names, ctx.needs_input_grad[2:7]) if need}
        g = _bwd(G, None if dh_out is None else dh_out.contiguous(), None if dy is None else dy.contiguous(), h, z, stats,
                 gate, like, want)
        return (g['dh'], g['dz']) + tuple(g.get('d' + k) for k in names) + (None, None)


def gate_norm(h, z, *, w_pre=None, b_pre=None, w_post=None, b_post=None, gate=None, row_ptr=None, kind='rms', pre=True,
              post=True, res_scale=1.0, eps=1e-6):
    """(h', y) of `gate_norm_fwd`, differentiable in h, z, the norms' parameters and the gate."""
    opts = dict(kind=kind, pre=pre, post=post, res_scale=res_scale, eps=eps)
    inputs = (h, z, w_pre, b_pre, w_post, b_post, gate)
    if forward_ad._current_level >= 0:
        capi.no_tangents('gate_norm', *inputs)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in inputs):
        return _GateNorm.apply(*inputs, row_ptr, opts)
    return gate_norm_fwd(h, z, w_pre=w_pre, b_pre=b_pre, w_post=w_post, b_post=b_post, gate=gate, row_ptr=row_ptr, **opts)[:2]

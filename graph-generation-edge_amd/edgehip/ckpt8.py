"""ckpt8.py - activations kept for the backward pass in 8 bits (csrc/ckpt8.hip).

A row is cut into groups of 64 values; a group keeps whole numbers of [-127, 127] and the power of two they are multiples
of: 1 + 1/64 bytes a value, off by at most 1/127 of the largest value of the group (half that at best; by up to 2^-121 in
groups of values below 2^-113, whose step ends there, and values above 127 2^121 are held to that).  `act8` and `linear8`
are torch's activation and linear layer with such a checkpoint in place of their input; their forward results are those of
the exact input, only the gradients (of the activation's input, of the weight) read the kept values."""
import torch
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import capi

lib = capi.lib
GROUP = 64
MAX_GROUPS = (1 << 29) - 32
KINDS = {'silu': 1, 'mish': 2}
_TORCH_TYPE = {capi.F32: torch.float32, capi.BF16: torch.bfloat16, capi.F16: torch.float16}


class Packed8:
    """A kept activation: `codes` int8 shaped like it, `exps` int8 [rows, ceil(K / 64)] (-128: the group held a value that
    was not finite, all of it stands for NaN), `dtype`: the type of what was kept."""

    __slots__ = ('codes', 'exps', 'dtype')

    def __init__(self, codes, exps, dtype):
        if codes.dim() < 1 or codes.shape[-1] < 1 or codes.dtype != torch.int8 or exps.dtype != torch.int8:
            raise ValueError(f'Packed8: int8 codes [..., K] and exps, got {tuple(codes.shape)} {codes.dtype}, {exps.dtype}')
        rows, k = _rows(codes)
        if exps.shape != (rows, -(-k // GROUP)) or exps.device != codes.device:
            raise ValueError(f'Packed8: exps must be [{rows}, {-(-k // GROUP)}] beside codes {tuple(codes.shape)}, got {tuple(exps.shape)}')
        self.codes, self.exps, self.dtype = codes.contiguous(), exps.contiguous(), dtype

    @classmethod
    def _of(cls, codes, exps, dtype):
        """Of tensors that fit each other by their making."""
        self = cls.__new__(cls)
        self.codes, self.exps, self.dtype = codes, exps, dtype
        return self

    @property
    def shape(self):
        return self.codes.shape

    @property
    def nbytes(self):
        return self.codes.numel() + self.exps.numel()

    def unpack(self, dtype=None):
        """The values the checkpoint stands for, in `dtype` (the kept tensor's own by default)."""
        x = torch.empty(self.codes.shape, dtype=dtype or self.dtype, device=self.codes.device)
        code = capi.dtype_code('unpack8', 'dtype', x)
        capi.on_gpu('unpack8', x)
        if x.numel():
            rows, k = _rows(x)
            with capi.on_device_of(x) as stream:
                capi.check(lib.edgehip_unpack8(code, self.codes.data_ptr(), self.exps.data_ptr(), rows, k, x.data_ptr(),
                                               stream), 'unpack8')
        return x


def _rows(x):
    return (x.numel() // x.shape[-1], x.shape[-1]) if x.shape[-1] else (0, 0)


def _input(what, x, kept=True):
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f'{what}: rows of at least one value, got {tuple(x.shape)}')
    code = capi.dtype_code(what, 'x', x)
    if kept and x.numel() > MAX_GROUPS and x.numel() // x.shape[-1] * -(-x.shape[-1] // GROUP) > MAX_GROUPS:
        raise ValueError(f'{what}: up to {MAX_GROUPS} groups of {GROUP} values, got {tuple(x.shape)}')
    capi.on_gpu(what, x)
    return x.contiguous(), code


def _kind(what, kind):
    if kind not in KINDS:
        raise ValueError(f'{what}: kind must be one of {sorted(KINDS)}, got {kind!r}')
    return KINDS[kind]


def _new(x):
    rows, k = _rows(x)
    return Packed8._of(torch.empty(x.shape, dtype=torch.int8, device=x.device),
                       torch.empty((rows, -(-k // GROUP)), dtype=torch.int8, device=x.device), x.dtype)


def pack8(x):
    """Keeps x ([..., K], fp32 / bf16 / fp16)."""
    x, code = _input('pack8', x)
    kept = _new(x)
    if x.numel():
        rows, k = _rows(x)
        with capi.on_device_of(x) as stream:
            capi.check(lib.edgehip_pack8(code, x.data_ptr(), rows, k, kept.codes.data_ptr(), kept.exps.data_ptr(),
                                         stream), 'pack8')
    return kept


def act8_fwd(x, kind='silu'):
    """(act(x), the checkpoint of x) in one pass over x; kind 'silu' or 'mish'."""
    what = 'act8_fwd'
    kc = _kind(what, kind)
    x, code = _input(what, x)
    y, kept = torch.empty_like(x), _new(x)
    if x.numel():
        rows, k = _rows(x)
        with capi.on_device_of(x) as stream:
            capi.check(lib.edgehip_act8_fwd(code, kc, x.data_ptr(), rows, k, y.data_ptr(), kept.codes.data_ptr(),
                                            kept.exps.data_ptr(), stream), what)
    return y, kept


def _against(what, dy, kept):
    if not isinstance(kept, Packed8):
        raise ValueError(f'{what}: kept must be what pack8 or act8_fwd returned')
    code = capi.dtype_code(what, 'dy', dy)
    capi.same_device(what, 'dy', dy, kept.codes.device)
    return code


def act8_bwd(dy, kept, kind='silu'):
    """dy act'(kept x), of dy's type."""
    what = 'act8_bwd'
    kc = _kind(what, kind)
    code = _against(what, dy, kept)
    if dy.shape != kept.shape:
        raise ValueError(f'{what}: dy must be {list(kept.shape)}, got {tuple(dy.shape)}')
    capi.on_gpu(what, dy)
    dy = dy.contiguous()
    dx = torch.empty_like(dy)
    if dy.numel():
        rows, k = _rows(dy)
        with capi.on_device_of(dy) as stream:
            capi.check(lib.edgehip_act8_bwd(code, kc, dy.data_ptr(), kept.codes.data_ptr(), kept.exps.data_ptr(), rows, k,
                                            dx.data_ptr(), stream), what)
    return dx


def linear8_bwd_weight(dy, kept, bias=True):
    """(dW [N, K], db [N]) of y = x W^T + b in fp32, x as it was kept: dW = dy^T x, db = column sums of dy (None with
    bias=False).  dy: [..., N] over the same rows as the kept [..., K].  The rows are summed in a fixed order."""
    what = 'linear8_bwd_weight'
    code = _against(what, dy, kept)
    if dy.dim() < 1 or dy.shape[:-1] != kept.shape[:-1] or dy.shape[-1] < 1:
        raise ValueError(f'{what}: dy must be {list(kept.shape[:-1])} x [outputs], got {tuple(dy.shape)}')
    n, k = dy.shape[-1], kept.shape[-1]
    if max(n, k) > 1 << 22:
        raise ValueError(f'{what}: layers of up to {1 << 22} inputs and outputs, got {k} and {n}')
    capi.on_gpu(what, dy)
    dy = dy.contiguous()
    m = dy.numel() // n
    nbytes = lib.edgehip_linear8_workspace_bytes(code, m, n, k)
    if nbytes == 0:
        raise ValueError(f'{what}: a gradient of {n} x {k} is too large')
    dw = torch.empty((n, k), dtype=torch.float32, device=dy.device)
    db = torch.empty(n, dtype=torch.float32, device=dy.device) if bias else None
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dy.device)
    with capi.on_device_of(dy) as stream:
        capi.check(lib.edgehip_linear8_bwd_weight(code, dy.data_ptr(), kept.codes.data_ptr(), kept.exps.data_ptr(), m, n, k,
                                                  dw.data_ptr(), capi.ptr(db), ws.data_ptr(), nbytes, stream), what)
    return dw, db


class _Act8(Function):
    @staticmethod
    def forward(ctx, x, kind):
        y, kept = act8_fwd(x, kind)
        ctx.save_for_backward(kept.codes, kept.exps)
        ctx.kept = (x.dtype, kind)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dtype, kind = ctx.kept
        return act8_bwd(dy, Packed8._of(*ctx.saved_tensors, dtype), kind), None


def act8(x, kind='silu'):
    """act(x), keeping x in 8 bits for the backward pass."""
    if forward_ad._current_level >= 0:
        capi.no_tangents('act8', x)
    if torch.is_grad_enabled() and x.requires_grad:
        return _Act8.apply(x, kind)
    return act8_fwd(x, kind)[0]


def _own_products(x, w):
    """Whether the package's fp32 products (edgehip_linear_fwd / _bwd_input) take this layer."""
    n, k = w.shape
    return x.dtype == torch.float32 and x.dim() == 2 and k % 64 == 0 and n % 64 == 0


def _aligned(t):
    """t as the package's products read it: dense, from a 16-byte boundary."""
    t = t.contiguous()
    return t.clone() if t.data_ptr() & 15 else t


class _Linear8(Function):
    @staticmethod
    def forward(ctx, x, w, b, kept):
        x, _ = _input('linear8', x, kept is not None)
        ctx.own = _own_products(x, w)
        if ctx.own:
            y = torch.empty((x.shape[0], w.shape[0]), dtype=x.dtype, device=x.device)
            if x.shape[0]:
                xc, wc, bc = _aligned(x), _aligned(w), None if b is None else _aligned(b)
                with capi.on_device_of(x) as stream:
                    capi.check(lib.edgehip_linear_fwd(xc.data_ptr(), x.shape[0], w.shape[1], wc.data_ptr(), capi.ptr(bc),
                                                      w.shape[0], 0, y.data_ptr(), stream), 'linear_fwd')
        else:
            with torch.autocast(x.device.type, enabled=False):   # y is of x's type, whatever surrounds the call
                y = torch.nn.functional.linear(x, w, b)
        ctx.save_for_backward(w, kept and kept.codes, kept and kept.exps)
        ctx.has_bias, ctx.dtype = b is not None, x.dtype
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w, codes, exps = ctx.saved_tensors
        dy = dy.contiguous()
        dx = dw = db = None
        if ctx.needs_input_grad[0]:
            if ctx.own:
                n, k = w.shape
                dx = torch.empty((dy.shape[0], k), dtype=dy.dtype, device=dy.device)
                if dy.shape[0]:
                    wt = torch.empty(k * n, dtype=torch.float32, device=dy.device)
                    yc, wc = _aligned(dy), _aligned(w)
                    with capi.on_device_of(dy) as stream:
                        capi.check(lib.edgehip_linear_bwd_input(yc.data_ptr(), dy.shape[0], n, wc.data_ptr(), k, wt.data_ptr(),
                                                                dx.data_ptr(), stream), 'linear_bwd_input')
            else:
                with torch.autocast(dy.device.type, enabled=False):
                    dx = torch.matmul(dy, w)
        want_db = ctx.has_bias and ctx.needs_input_grad[2]
        if ctx.needs_input_grad[1]:
            dw, db = linear8_bwd_weight(dy, Packed8._of(codes, exps, ctx.dtype), bias=want_db)
            dw = dw.to(w.dtype)
            db = db.to(w.dtype) if want_db else None
        elif want_db:
            # (no library sum: a captured one can hold a memory-set node; the checkpoint of an input of one zero is a stand-in)
            none = torch.zeros(dy.shape[:-1] + (1,), dtype=torch.int8, device=dy.device)
            db = linear8_bwd_weight(dy, Packed8._of(none, none.reshape(-1, 1), ctx.dtype))[1].to(w.dtype)
        return dx, dw, db, None


def linear8(x, w, b=None, kept=None):
    """x W^T + b, keeping x in 8 bits for the weight's gradient (nothing is kept of it when W needs none).  kept: pack8(x),
    for an input that several layers read (it is then kept once).  fp32 layers whose sizes are multiples of 64 run on the
    package's own products, others on the library's."""
    if w.dim() != 2 or x.dim() < 1 or x.shape[-1] != w.shape[1] or x.dtype != w.dtype:
        raise ValueError(f'linear8: x [..., K] and W [N, K] of one type, got {tuple(x.shape)} {x.dtype}, {tuple(w.shape)} {w.dtype}')
    if b is not None and (b.shape != (w.shape[0],) or b.dtype != w.dtype):
        raise ValueError(f'linear8: b must be [{w.shape[0]}] of the type of W')
    for name, t in (('W', w), ('b', b)):
        if t is not None:
            capi.same_device('linear8', name, t, x.device)
    if kept is not None and (not isinstance(kept, Packed8) or kept.shape != x.shape):
        raise ValueError('linear8: kept must be pack8(x)')
    if kept is not None:
        capi.same_device('linear8', 'kept', kept.codes, x.device)
    if not (torch.is_grad_enabled() and w.requires_grad):
        kept = None
    elif kept is None:
        kept = pack8(x.detach())
    return _Linear8.apply(x, w, b, kept)

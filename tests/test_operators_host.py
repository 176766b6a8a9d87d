"""CPU: what the operators for deeper networks and tuning refuse (edgehip.block, ckpt8, tune), at both levels."""
import ctypes

import pytest
import torch

byref = ctypes.byref
vec = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)
i64 = lambda *v: torch.tensor(v, dtype=torch.int64)


def test_struct_sizes():
    from edgehip import capi
    assert ctypes.sizeof(capi.GateNorm) == 8 + 10 * 4 + 6 * 8 + 2 * 4
    assert ctypes.sizeof(capi.LogitRows) == 2 * 8 + 4 * 4 + 4 * 8
    assert ctypes.sizeof(capi.Policy) == 4 * 8 + 3 * 8 + 2 * 4
    assert ctypes.sizeof(capi.Preference) == 2 * 8 + 2 * 8 + 2 * 4


H, Z, D = vec(6, 8), vec(6, 8), 8


@pytest.mark.parametrize('args,kw,text', [
    ((H, Z), {}, 'on a GPU'),
    ((H, vec(6, 9)), {}, 'one shape'),
    ((H, Z), dict(kind='batch'), 'kind must be'),
    ((H.double(), Z), {}, 'must be fp32, bf16 or fp16'),
    ((H.bfloat16(), Z), {}, 'h must be fp32 or of the type of z'),
    ((H, Z), dict(b_pre=vec(8)), 'no bias'),
    ((H, Z), dict(w_pre=vec(8), pre=False), 'switched off'),
    ((H, Z), dict(b_post=vec(8), post=False, kind='layer'), 'switched off'),
    ((H, Z), dict(w_pre=vec(7)), 'dense vector of 8'),
    ((H, Z), dict(w_pre=vec(8, t=torch.float16)), 'w_pre must be fp32 or of the type of z'),
    ((H.half(), Z.half()), dict(w_pre=vec(8), w_post=vec(8, t=torch.float16)), 'share one type'),
    ((H, Z), dict(gate=vec(7)), 'gate must be'),
    ((H, Z), dict(gate=vec(3, 8)), 'gate must be'),
    ((H, Z), dict(gate=vec(8, t=torch.float16)), 'gate must be fp32 or of the type of z'),
    ((H, Z), dict(gate=vec(3, 8), row_ptr=i64(0, 1, 2, 6)), 'int32'),
    ((H, Z), dict(gate=vec(2, 8), row_ptr=torch.tensor([0, 1, 2, 6], dtype=torch.int32)), r'\[3, 8\]'),
    ((H, Z), dict(row_ptr=torch.tensor([0, 6], dtype=torch.int32)), 'row_ptr without a gate'),
    ((vec(2, 8200), vec(2, 8200)), {}, '1 to 8192'),
])
def test_gate_norm_refusals(args, kw, text):
    import edgehip
    with pytest.raises(ValueError, match=text):
        edgehip.gate_norm(*args, **kw)


def test_gate_norm_backward_refusals():
    from edgehip import block
    with pytest.raises(ValueError, match='on a GPU'):
        block.gate_norm_bwd(H, Z, H, Z, vec(6, 4))


def test_gate_norm_c_refusals():
    from edgehip import capi
    f, b, n = capi.lib.edgehip_gate_norm_fwd, capi.lib.edgehip_gate_norm_bwd, capi.lib.edgehip_gate_norm_workspace_bytes

    def desc(**kw):
        G = capi.GateNorm(rows=4, dim=8, pre=1, post=1)
        for k, v in kw.items():
            setattr(G, k, v)
        return byref(G)
    fwd = lambda G: f(G, None, None, None, None, None, None)
    assert fwd(None) == capi.ERR_ARG and fwd(desc()) == capi.ERR_ARG
    for bad in (dict(rows=-1), dict(dim=0), dict(stream_dtype=3), dict(branch_dtype=-1), dict(kind=2), dict(gate_kind=4),
                dict(gate_kind=1), dict(gate=64), dict(gate=64, gate_kind=2), dict(b_pre=64), dict(param_dtype=1),
                dict(gate=64, gate_kind=1, gate_dtype=2)):
        assert fwd(desc(**bad)) == capi.ERR_ARG, bad
        assert n(desc(**bad)) == 0, bad
    assert fwd(desc(stream_dtype=1, branch_dtype=0)) == capi.ERR_UNSUPPORTED
    assert fwd(desc(dim=8193)) == capi.ERR_UNSUPPORTED and n(desc(dim=8193)) == 0
    assert fwd(desc(rows=1 << 31)) == capi.ERR_TOO_LARGE
    assert fwd(desc(rows=0)) == capi.OK
    need = n(desc())
    p = ctypes.c_void_p(4096)
    args = lambda ws, nb: (desc(), None, None, p, p, p, p, p, None, None, None, None, None, ws, nb, None)
    assert need > 0 and b(*args(p, need - 1)) == capi.ERR_WORKSPACE and b(*args(None, need)) == capi.ERR_ARG
    assert b(desc(), None, None, p, p, p, p, p, p, None, None, None, None, p, need, None) == capi.ERR_ARG      # gradient of no gate
    assert b(desc(), None, None, p, p, p, p, p, None, None, p, None, None, p, need, None) == capi.ERR_ARG      # bias of the rms kind
    assert b(desc(pre=0), None, None, p, p, p, p, p, None, p, None, None, None, p, need, None) == capi.ERR_ARG


def test_ckpt8_refusals():
    import edgehip
    from edgehip import ckpt8
    x = vec(4, 64)
    kept = ckpt8.Packed8(vec(4, 64, t=torch.int8), vec(4, 1, t=torch.int8), torch.float32)
    for f, text in ((lambda: edgehip.pack8(x), 'on a GPU'), (lambda: edgehip.pack8(x.double()), 'fp32, bf16 or fp16'),
                    (lambda: edgehip.pack8(vec(4, 0)), 'at least one value'), (lambda: edgehip.act8(x, 'tanh'), 'kind must be'),
                    (lambda: edgehip.act8(x), 'on a GPU'), (lambda: ckpt8.act8_bwd(vec(4, 63), kept), r'\[4, 64\]'),
                    (lambda: ckpt8.act8_bwd(x, x), 'what pack8'), (lambda: ckpt8.linear8_bwd_weight(vec(5, 3), kept), 'outputs'),
                    (lambda: ckpt8.linear8_bwd_weight(vec(4, 3), kept), 'on a GPU'), (lambda: kept.unpack(torch.float64), 'fp32, bf16 or fp16'),
                    (lambda: kept.unpack(), 'on a GPU'),
                    (lambda: edgehip.linear8(x, vec(3, 63)), 'one type'), (lambda: edgehip.linear8(x, vec(3, 64, t=torch.float16)), 'one type'),
                    (lambda: edgehip.linear8(x, vec(3, 64), vec(4)), 'b must be'), (lambda: edgehip.linear8(x, vec(3, 64)), 'on a GPU'),
                    (lambda: edgehip.linear8(vec(2, 64), vec(3, 64), None, kept), 'kept must be')):
        with pytest.raises(ValueError, match=text):
            f()


def test_ckpt8_c_refusals():
    from edgehip import capi
    L = capi.lib
    p = ctypes.c_void_p(4096)
    assert L.edgehip_pack8(3, p, 1, 1, p, p, None) == capi.ERR_ARG and L.edgehip_pack8(0, None, 1, 1, p, p, None) == capi.ERR_ARG
    assert L.edgehip_pack8(0, p, -1, 1, p, p, None) == capi.ERR_ARG and L.edgehip_pack8(0, p, 1, 0, p, p, None) == capi.ERR_ARG
    assert L.edgehip_pack8(0, p, 1 << 31, 64, p, p, None) == capi.ERR_TOO_LARGE
    assert L.edgehip_pack8(0, None, 0, 5, None, None, None) == capi.OK
    assert L.edgehip_act8_fwd(0, 3, p, 1, 1, p, p, p, None) == capi.ERR_ARG and L.edgehip_act8_bwd(0, 1, None, p, p, 1, 1, p, None) == capi.ERR_ARG
    assert L.edgehip_unpack8(0, p, None, 1, 1, p, None) == capi.ERR_ARG
    n = L.edgehip_linear8_workspace_bytes
    assert n(0, -1, 1, 1) == 0 and n(0, 1, 0, 1) == 0 and n(5, 1, 1, 1) == 0 and n(0, 1, 1 << 23, 1) == 0
    need = n(0, 100000, 64, 64)
    assert need > 64 * 64 * 4
    go = lambda ws, nb, dy=p, dw=p: L.edgehip_linear8_bwd_weight(0, dy, p, p, 100000, 64, 64, dw, p, ws, nb, None)
    assert go(p, need - 1) == capi.ERR_WORKSPACE and go(None, need) == capi.ERR_ARG
    assert go(p, need, dy=None) == capi.ERR_ARG and go(p, need, dw=None) == capi.ERR_ARG


X, A, OLD, ADV, PTR = vec(6, 5), i64(0, 1, 2, 3, 4, 0), vec(6), vec(2), i64(0, 2, 6)


@pytest.mark.parametrize('args,kw,text', [
    ((X, A, OLD, ADV, PTR), {}, 'on a GPU'),
    ((vec(6), A, OLD, ADV, PTR), {}, 'rows, classes'),
    ((X.long(), A, OLD, ADV, PTR), {}, 'fp32, bf16 or fp16'),
    ((X, A[:5], OLD, ADV, PTR), {}, 'taken must be'),
    ((X, A.int(), OLD, ADV, PTR), {}, 'taken must be'),
    ((X, A, OLD.half(), ADV, PTR), {}, 'old_logp must be'),
    ((X, A, OLD, vec(3), PTR), {}, 'advantage must be'),
    ((X, A, OLD, ADV, PTR.int()), {}, 'seq_ptr must be'),
    ((X, A, OLD, ADV, None), {}, 'seq_ptr is needed'),
    ((X, A, OLD, ADV, PTR), dict(mask=vec(6)), 'mask must be bool'),
    ((X, A, OLD, ADV, PTR), dict(mask=vec(5, t=torch.bool)), 'mask must be'),
    ((X, A, OLD, ADV, PTR), dict(kl_coef=0.1), 'needs ref_logp'),
    ((X, A, OLD, ADV, PTR), dict(clip=(-0.1, 0.2)), 'clip must not be negative'),
    ((X, A, OLD, ADV, PTR), dict(reduce='max'), 'reduce must be'),
])
def test_policy_refusals(args, kw, text):
    import edgehip
    for f in (edgehip.policy_loss, edgehip.policy_loss_grad):
        with pytest.raises(ValueError, match=text):
            f(*args, **kw)


@pytest.mark.parametrize('ptr,kw,text', [
    (PTR, {}, 'on a GPU'), (i64(0, 1, 2, 6), {}, 'as many preferred'), (PTR, dict(beta=0.0), 'beta > 0'),
    (PTR, dict(label_smoothing=0.5), 'label_smoothing'), (PTR, dict(kind='square', label_smoothing=0.1), 'label_smoothing'),
    (PTR, dict(kind='hinge'), 'kind must be'), (PTR, dict(ref_logp=vec(5)), 'ref_logp must be'),
])
def test_preference_refusals(ptr, kw, text):
    import edgehip
    for f in (edgehip.preference_loss, edgehip.preference_loss_grad):
        with pytest.raises(ValueError, match=text):
            f(X, A, ptr, **kw)
    with pytest.raises(ValueError, match='on a GPU'):
        edgehip.row_logp(X, A)


def test_tune_c_refusals():
    from edgehip import capi
    L, p = capi.lib, ctypes.c_void_p(4096)

    def rows(**kw):
        Q = capi.LogitRows(rows=4, row_stride=8, classes=8, num_seqs=2, logits=4096, taken=4096, seq_ptr=4096)
        for k, v in kw.items():
            setattr(Q, k, v)
        return byref(Q)
    n = L.edgehip_tune_workspace_bytes
    for bad in (dict(rows=-1), dict(classes=0), dict(dtype=3), dict(num_seqs=0), dict(seq_ptr=None), dict(logits=None), dict(taken=None),
                dict(row_stride=7), dict(rows=1 << 31)):
        assert n(rows(**bad)) == 0, bad
    need = n(rows())
    O = lambda **kw: byref(capi.Policy(**{**dict(old_logp=4096, advantage=4096), **kw}))
    go = lambda Q, o, ws=p, nb=need: L.edgehip_policy_loss_grad(Q, o, p, p, p, p, p, ws, nb, None)
    assert go(rows(), O(), nb=need - 1) == capi.ERR_WORKSPACE and go(rows(), O(), ws=None) == capi.ERR_ARG
    assert go(rows(), None) == capi.ERR_ARG and go(rows(), O(old_logp=None)) == capi.ERR_ARG
    assert go(rows(), O(clip_lo=-1.0)) == capi.ERR_ARG and go(rows(), O(kl_coef=1.0)) == capi.ERR_ARG
    R = lambda **kw: byref(capi.Preference(**{**dict(beta=0.1), **kw}))
    pf = lambda Q, o, nb=need: L.edgehip_preference_loss_fwd(Q, o, p, p, p, nb, None)
    assert pf(rows(), R(beta=0.0)) == capi.ERR_ARG and pf(rows(), R(kind=2)) == capi.ERR_ARG and pf(rows(), R(label_smoothing=0.6)) == capi.ERR_ARG
    assert pf(rows(num_seqs=3), R(), nb=1 << 20) == capi.ERR_ARG and pf(rows(), R(), nb=need - 1) == capi.ERR_WORKSPACE
    assert L.edgehip_row_logp(rows(num_seqs=0), p, None) == capi.ERR_ARG and L.edgehip_row_logp(rows(), None, None) == capi.ERR_ARG


def test_sizes_that_would_not_fit_their_field():
    """Wider than 32 bits: refused, never cut off.  (Expanded views: nothing of that size is allocated.)"""
    import edgehip
    from edgehip import capi, ckpt8
    wide = vec(1, 1).expand(1, (1 << 32) + 5)
    with pytest.raises(ValueError, match='2\\^30 classes'):
        edgehip.row_logp(wide, i64(0))
    with pytest.raises(ValueError, match='inputs and outputs'):
        ckpt8.linear8_bwd_weight(wide, ckpt8.Packed8(vec(1, 64, t=torch.int8), vec(1, 1, t=torch.int8), torch.float32))
    with pytest.raises(ValueError, match='65535 groups'):
        edgehip.gate_norm(H, Z, gate=vec(65536, 8), row_ptr=torch.zeros(65537, dtype=torch.int32))
    Q = capi.LogitRows(rows=1, row_stride=(1 << 30) + 1, classes=(1 << 30) + 1, num_seqs=1, logits=4096, taken=4096, seq_ptr=4096)
    assert capi.lib.edgehip_row_logp(byref(Q), ctypes.c_void_p(4096), None) == capi.ERR_TOO_LARGE

"""CPU: calls of the operators for deeper networks and tuning (edgehip.block, ckpt8, tune) that are refused, or taken, before any
kernel runs."""
import pytest
import torch
from torch.autograd import forward_ad

vec = lambda *s, t=torch.float32: torch.zeros(*s, dtype=t)


@pytest.mark.parametrize('grad', [True, False])
def test_forward_mode_derivatives_are_refused(grad):
    """A tangent is never lost silently, whichever input has it; without one the call goes on to its other checks."""
    import edgehip
    h, z, w, g = vec(6, 8), vec(6, 8), vec(8), vec(6, 8)
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))
        for args, kw in (((dual(h), z), {}), ((h, dual(z)), {}), ((h, z), dict(w_pre=dual(w))), ((h, z), dict(w_post=dual(w))),
                         ((h, z), dict(gate=dual(g))), ((h, z), dict(b_pre=dual(w), kind='layer')), ((h, z), dict(b_post=dual(w), kind='layer'))):
            with pytest.raises(NotImplementedError, match='gate_norm: no forward-mode derivative'):
                edgehip.gate_norm(*args, **kw)
        with pytest.raises(NotImplementedError, match='act8: no forward-mode derivative'):
            edgehip.act8(dual(h))
        for f in (lambda: edgehip.gate_norm(h, z, w_pre=w), lambda: edgehip.act8(h)):
            with pytest.raises(ValueError, match='on a GPU'):
                f()


def test_types_of_choices():
    """taken: int64 or uint8 (the sampler's bits); other types are refused, at both levels."""
    import ctypes
    import edgehip
    from edgehip import capi
    x, ptr = vec(6, 5), torch.tensor([0, 2, 6])
    for t in (torch.uint8, torch.int64):
        with pytest.raises(ValueError, match='on a GPU'):
            edgehip.policy_loss(x, vec(6, t=t), vec(6), vec(2), ptr)
    for t in (torch.bool, torch.int16, torch.int32, torch.float32):
        with pytest.raises(ValueError, match='taken must be'):
            edgehip.policy_loss(x, vec(6, t=t), vec(6), vec(2), ptr)
    with pytest.raises(ValueError, match='taken must be'):
        edgehip.row_logp(x, vec(5, t=torch.uint8))
    Q = capi.LogitRows(rows=4, row_stride=8, classes=8, num_seqs=2, logits=4096, taken=4096, seq_ptr=4096)
    assert capi.lib.edgehip_tune_workspace_bytes(ctypes.byref(Q)) > 0
    Q.taken_type = 1
    assert capi.lib.edgehip_tune_workspace_bytes(ctypes.byref(Q)) > 0
    for bad in (-1, 2):
        Q.taken_type = bad
        assert capi.lib.edgehip_tune_workspace_bytes(ctypes.byref(Q)) == 0
        assert capi.lib.edgehip_row_logp(ctypes.byref(Q), ctypes.c_void_p(4096), None) == capi.ERR_ARG


def test_sizes_past_a_launch():
    """A launch is a 32-bit number of threads along an axis: more are refused as too large, never handed to the runtime (which
    would report a failed launch).  Nothing of that size is allocated here."""
    import ctypes
    import edgehip
    from edgehip import capi, ckpt8
    L, p, big = capi.lib, ctypes.c_void_p(4096), 1 << 60
    byref = ctypes.byref
    for m, k in ((1 << 29, 1), (1 << 29, 64), (1 << 28, 65), (1, 1 << 31)):
        assert L.edgehip_pack8(1, p, m, k, p, p, None) == capi.ERR_TOO_LARGE
        assert L.edgehip_unpack8(1, p, p, m, k, p, None) == capi.ERR_TOO_LARGE
        assert L.edgehip_act8_fwd(1, 1, p, m, k, p, p, p, None) == capi.ERR_TOO_LARGE
        assert L.edgehip_act8_bwd(1, 1, p, p, p, m, k, p, None) == capi.ERR_TOO_LARGE
    assert L.edgehip_linear8_workspace_bytes(1, 64, 1 << 22, 1 << 22) == 0
    assert L.edgehip_linear8_bwd_weight(1, p, p, p, 64, 1 << 22, 1 << 22, p, p, p, big, None) == capi.ERR_TOO_LARGE
    wide = vec(1, 1).expand(1 << 29, 1)
    for f in (edgehip.pack8, edgehip.act8):
        with pytest.raises(ValueError, match='groups of 64'):
            f(wide)
    with pytest.raises(ValueError, match='too large'):
        ckpt8.linear8_bwd_weight(_Gpu(vec(1, 1).expand(1, 1 << 22)), _kept(1 << 22))
    # rows x threads of a row, and a block a sequence
    O, R = capi.Policy(old_logp=4096, advantage=4096), capi.Preference(beta=0.1)

    def codes(rows, classes, dtype, seqs=2):
        Q = byref(capi.LogitRows(rows=rows, row_stride=classes, classes=classes, dtype=dtype, num_seqs=seqs, logits=4096, taken=4096, seq_ptr=4096))
        return dict(logp=L.edgehip_row_logp(Q, p, None), fwd=L.edgehip_policy_loss_fwd(Q, byref(O), p, p, p, p, p, big, None),
                    bwd=L.edgehip_policy_loss_bwd(Q, byref(O), p, p, big, None), grad=L.edgehip_policy_loss_grad(Q, byref(O), p, p, p, p, p, p, big, None),
                    pfwd=L.edgehip_preference_loss_fwd(Q, byref(R), p, p, p, big, None), pbwd=L.edgehip_preference_loss_bwd(Q, byref(R), p, p, big, None),
                    pgrad=L.edgehip_preference_loss_grad(Q, byref(R), p, p, p, p, big, None))
    for rows, classes, dtype in ((1 << 30, 70, 0), (1 << 30, 70, 1), (1 << 28, 1025, 2), (1 << 22, 131073, 1), ((1 << 31) - 1, 1 << 20, 0)):
        assert set(codes(rows, classes, dtype).values()) == {capi.ERR_TOO_LARGE}, (rows, classes, dtype)
    assert set(codes(100, 4, 0, 1 << 24).values()) == {capi.ERR_TOO_LARGE}
    with pytest.raises(ValueError, match='2\\^24 - 1 sequences'):
        edgehip.preference_loss(vec(4, 3), torch.zeros(4, dtype=torch.int64), torch.zeros(1, dtype=torch.int64).expand((1 << 24) + 1))
    with pytest.raises(ValueError, match='fixed capacity'):      # (too large an argument is a ValueError wherever C finds it)
        capi.check(capi.ERR_TOO_LARGE, 'x')


class _Gpu:
    """A CPU tensor that says it is on a GPU: for checks that come behind that one."""
    is_cuda = True

    def __init__(self, t):
        self.t = t

    def contiguous(self):
        return self

    def __getattr__(self, name):
        return getattr(self.t, name)


def _kept(k):
    from edgehip import ckpt8
    return ckpt8.Packed8(vec(1, k, t=torch.int8), vec(1, -(-k // 64), t=torch.int8), torch.float32)


def test_a_checkpoint_put_together_by_hand():
    """What the kernels read of a Packed8 is fixed when it is made: shapes and types that do not fit are refused (its exponents
    would be read past their end), a strided part is made dense."""
    from edgehip import ckpt8
    i8 = lambda *s: vec(*s, t=torch.int8)
    for codes, exps in ((i8(4, 130), i8(4, 2)), (i8(4, 130), i8(3, 3)), (i8(4, 130), i8(12)), (i8(4, 130), vec(4, 3, t=torch.uint8)),
                        (vec(4, 130), i8(4, 3)), (i8(4, 0), i8(4, 0)), (torch.zeros((), dtype=torch.int8), i8(1, 1))):
        with pytest.raises(ValueError, match='Packed8'):
            ckpt8.Packed8(codes, exps, torch.float32)
    for codes, exps in ((i8(4, 130), i8(4, 3)), (i8(130), i8(1, 3)), (i8(2, 3, 64), i8(6, 1)), (i8(0, 70), i8(0, 2))):
        ckpt8.Packed8(codes, exps, torch.float32)
    whole = torch.arange(8 * 128).to(torch.int8).view(8, 128)
    part = ckpt8.Packed8(whole[::2, :64], i8(8, 2)[::2, :1], torch.float32)
    assert part.codes.is_contiguous() and part.exps.is_contiguous() and torch.equal(part.codes, whole[::2, :64])


def test_a_layer_that_keeps_nothing_takes_any_number_of_rows():
    import edgehip
    x, w = vec(1, 1).expand(1 << 29, 1), vec(3, 1)
    with pytest.raises(ValueError, match='on a GPU'):
        edgehip.linear8(x, w)
    with pytest.raises(ValueError, match='groups of 64'):
        edgehip.linear8(x, w.requires_grad_(True))

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

"""GPU: values at which the losses' formulas (edgehip.tune) are finite although a part of them is not.

Gradients are coef (onehot - p).  Tolerance: coef is made of A rho and kl_coef (exp(gap) - 1), each off by at most 16 half steps of
fp32 (the log-probability's 2^-24, two exponentials', their products'), p by as many: 32 x 2^-24 of the sizes."""
import math

import pytest
import torch

from test_gpu_tune import logp64, make, policy64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
INF = float('inf')


def policy(s, ref, kl_coef, mean=True, adv=None, old=None):
    """Both forms against autograd of the formula in fp64 (kl_coef 0: without the term); returns the one-pass form."""
    import edgehip
    s = dict(s, adv=s['adv'] if adv is None else adv, old=s['old'] if old is None else old)
    x = s['x'].double().requires_grad_(True)
    lp = logp64(s, x)
    loss, _, clipped, A, rho = policy64(s, lp, s['adv'], (0.2, 0.3), kl_coef, ref if kl_coef else None, mean)
    S = len(loss)
    (want,) = torch.autograd.grad(loss.sum() / S, x)
    assert bool(torch.isfinite(want).all())
    with torch.no_grad():
        gap = ref.double() - lp
        n = torch.stack([s['counts'][a:b].sum() for a, b in zip(s['ptr'].tolist(), s['ptr'].tolist()[1:])]).clamp(min=1) if mean else torch.ones(S, device='cuda')
        own = torch.repeat_interleave(torch.arange(S, device='cuda'), s['ptr'][1:] - s['ptr'][:-1])
        size = A.abs() * rho + (kl_coef * (torch.exp(gap) + 1) if kl_coef else 0.0)      # (of what the formula has: no term with kl_coef 0)
        size = torch.where(s['counts'], size / (n[own] * S), 0.0)
        p = torch.softmax(torch.where(s['counts'][:, None], s['x'].double(), 0.0), 1)
        hot = torch.zeros_like(p).scatter_(1, s['taken'].clamp(0, p.shape[1] - 1)[:, None], 1.0)
        tol = 32 * U * size[:, None] * (p + hot) + 1e-30
    kw = dict(ref_logp=ref, mask=s['mask'], clip=(0.2, 0.3), kl_coef=kl_coef, reduce='mean' if mean else 'sum')
    r = edgehip.policy_loss_grad(s['x'], s['taken'], s['old'], s['adv'], s['ptr'], **kw)
    leaf = s['x'].clone().requires_grad_(True)
    f = edgehip.policy_loss(leaf, s['taken'], s['old'], s['adv'], s['ptr'], **kw)
    (g,) = torch.autograd.grad(f.loss.mean(), leaf)
    for got in (r.dlogits, g):
        assert bool(((got.double() - want).abs() <= tol).all()), float(((got.double() - want).abs() / tol).max())
    for got in (r.loss, f.loss):
        assert torch.equal(torch.isinf(got), torch.isinf(loss)) and not bool(got.isnan().any())
        fin = torch.isfinite(loss)
        assert bool(((got.double() - loss).abs()[fin] <= 1e-5 * (1 + loss.abs()[fin])).all())
    assert torch.equal(r.clipped.cpu().long(), clipped) and torch.equal(f.clipped, r.clipped)
    return r


@pytest.mark.parametrize('classes', [2, 5, 40, 300])
@pytest.mark.parametrize('mean', [True, False])
def test_a_class_the_reference_forbids(classes, mean):
    """ref_logp = -inf where the class was taken all the same: the loss is infinite, its derivative is not; with kl_coef 0
    the term is only reported.  Finite gaps far below zero: exp(gap) - 1 is -1 to the last bit."""
    s = make(90, classes, 3, seed=classes, masked=classes != 5)
    live = s['counts'].nonzero()[:, 0]
    for gap in (-INF, -1e30, -1e6, -1000.0, -60.0):
        ref = s['ref'].clone()
        ref[live[4]] = gap
        ref[live[-3]] = gap
        r = policy(s, ref, 0.1, mean)
        assert int(torch.isinf(r.loss).sum()) == (0 if math.isfinite(gap) else len({int((s['ptr'][1:] <= int(live[k])).sum()) for k in (4, -3)}))
        r = policy(s, ref, 0.0, mean)
        assert bool(torch.isfinite(r.loss).all()) and bool((r.kl[:1] >= 0).all())
        if gap == -INF:
            assert bool(torch.isinf(r.kl).any())
    ref = s['ref'].clone()
    ref[live[4]] = float('nan')                                  # only watched: in kl alone
    r = policy(s, ref, 0.0, mean)
    assert bool(r.kl.isnan().any())


@pytest.mark.parametrize('classes', [3, 40, 300])
def test_an_advantage_of_nothing_and_a_ratio_past_the_range(classes):
    """old_logp so low that exp(logp - old_logp) leaves fp32: 0 where the advantage is 0, bounded where the clip binds."""
    s = make(80, classes, 4, seed=classes)
    live = s['counts'].nonzero()[:, 0]
    for old in (-120.0, -500.0):
        adv = torch.tensor([0.0, 1.5, 0.0, 0.25], device='cuda')
        far = s['old'].clone()
        far[live[::3]] = old
        r = policy(s, s['ref'], 0.1, adv=adv, old=far)
        assert bool(torch.isfinite(r.loss).all())


@pytest.mark.parametrize('smooth', [0.0, 0.1])
@pytest.mark.parametrize('mean', [False, True])
@pytest.mark.parametrize('classes', [3, 100])
def test_margins_without_end(classes, mean, smooth):
    """A taken class of logit -inf: the preferred sequence's margin is -inf (loss inf), the other's +inf (loss 0, or inf where
    smoothing asks for it), and the gradient is that of the formula's limit: beta (smooth - sigmoid(-x)), x = -inf, inf, 1.7."""
    import edgehip
    g = torch.Generator(device='cuda').manual_seed(classes)
    x = torch.randn(12, classes, generator=g, device='cuda')
    taken = torch.randint(0, classes, (12,), generator=g, device='cuda')
    for row in (1, 8):                                           # in sequence 0 (preferred) and in 4 (the other of pair 1)
        x[row, taken[row]] = -INF
    ptr = torch.arange(0, 13, 2, device='cuda')
    beta = 0.3
    leaf = x.clone().requires_grad_(True)
    f = edgehip.preference_loss(leaf, taken, ptr, beta=beta, label_smoothing=smooth, reduce='mean' if mean else 'sum')
    r = edgehip.preference_loss_grad(x, taken, ptr, beta=beta, label_smoothing=smooth, reduce='mean' if mean else 'sum')
    assert torch.equal(f.loss, r.loss) and torch.equal(f.margin, r.margin)
    assert r.margin[:2].tolist() == [-INF, INF] and r.loss[:2].tolist() == [INF, INF if smooth else 0.0]
    assert bool(torch.isfinite(r.loss[2]))
    (grad,) = torch.autograd.grad(f.loss.mean(), leaf)
    m = beta * r.margin.double()
    slope = beta * (smooth - torch.sigmoid(-m)) / 3 / (2 if mean else 1)
    coef = torch.cat([slope, -slope]).repeat_interleave(2)[:, None]
    hot = torch.zeros_like(x, dtype=torch.float64).scatter_(1, taken[:, None], 1.0)
    p = torch.softmax(x.double(), 1)
    want = coef * (hot - p)
    for got in (grad, r.dlogits):
        # coef: the margin's 2^-24 (its size, 6 at most, in units of 1) and four roundings; p: eight
        assert bool(((got.double() - want).abs() <= 32 * U * coef.abs() * (hot + p) + 1e-30).all())


@pytest.mark.parametrize('classes', [2, 9, 40, 200, 300, 9000])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_choices_of_one_byte(classes, dtype):
    """taken as uint8: the same bits as with the same choices in int64, classes out of range among them."""
    import edgehip
    s = make(700, classes, 4, dtype, seed=classes)
    small = s['taken'].clamp(min=0) % 256                        # (-100: another row's 0; 255 and the like lie outside of few classes)
    small[5] = 255
    small = small.to(torch.uint8)
    for f in (lambda t: edgehip.policy_loss_grad(s['x'], t, s['old'], s['adv'], s['ptr'], ref_logp=s['ref'], mask=s['mask'], kl_coef=0.1),
              lambda t: edgehip.preference_loss_grad(s['x'], t, s['ptr'], ref_logp=s['ref'], mask=s['mask']),
              lambda t: edgehip.policy_loss(s['x'], t, s['old'], s['adv'], s['ptr']), lambda t: edgehip.preference_loss(s['x'], t, s['ptr']),
              lambda t: [edgehip.row_logp(s['x'], t, s['mask'])]):
        got, want = f(small), f(small.long())
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(got, want))
    leaf = s['x'].clone().requires_grad_(True)
    a, b = (torch.autograd.grad(edgehip.policy_loss(leaf, t, s['old'], s['adv'], s['ptr'], mask=s['mask']).loss.sum(), leaf)[0] for t in (small, small.long()))
    assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_the_samplers_own_decisions():
    """A reverse step's logits and bits, as it hands them out, with `aptr` as the sequences."""
    import numpy as np

    import cases
    import edgehip
    import helpers as H
    from edgehip.model import _state
    from oracle import edge_oracle as orc
    graphs = cases.ragged_graphs(5)
    model = H.build_model(orc.random_tgnn_params(4), 48, cases.max_degree_of(graphs))
    b = H.graph_batch(graphs)
    rng, want = np.random.default_rng(1), {}
    draw = lambda n: cases.uniforms(rng, n, 2).cuda()
    H.set_state_from_pair_indices(b, torch.arange(0, sum(q['n'] * (q['n'] - 1) // 2 for q in graphs), 5))
    model.p_sample(b, 9, draw(b.num_nodes), draw, None, None, want)
    logits, bits, aptr = want['logits'], want['bits'], _state(b)['aptr']
    assert bits.dtype == torch.uint8 and bits.numel() > 50 and int(aptr[-1]) == bits.numel()
    old = edgehip.row_logp(logits, bits)
    lp = torch.log_softmax(logits.double(), 1).gather(1, bits.long()[:, None])[:, 0]
    assert bool(((old.double() - lp).abs() <= 2 * U * (1 + lp.abs())).all())
    adv = torch.linspace(-1, 1, b.num_graphs, device='cuda')
    r = edgehip.policy_loss_grad(logits, bits, old, adv, aptr)
    n = (aptr[1:] - aptr[:-1]).clamp(min=1)
    has = aptr[1:] > aptr[:-1]
    assert bool(((r.loss + adv)[has].abs() <= 1e-6).all())       # ratio 1 everywhere
    own = torch.repeat_interleave(torch.arange(b.num_graphs, device='cuda'), aptr[1:] - aptr[:-1])
    hot = torch.nn.functional.one_hot(bits.long(), 2).double()
    coef = -(adv.double() / n / b.num_graphs)[own][:, None]
    p = torch.softmax(logits.double(), 1)
    assert bool(((r.dlogits.double() - coef * (hot - p)).abs() <= 32 * U * coef.abs() * (hot + p) + 1e-30).all())


def test_no_operator_loses_a_tangent():
    """Forward mode: refused by every differentiable form."""
    import edgehip
    from torch.autograd import forward_ad
    x, w, ptr = torch.randn(8, 64, device='cuda'), torch.randn(64, 64, device='cuda'), torch.tensor([0, 3, 8], device='cuda')
    taken, old, adv = torch.zeros(8, dtype=torch.int64, device='cuda'), torch.zeros(8, device='cuda'), torch.ones(2, device='cuda')
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for f in (lambda: edgehip.gate_norm(d, x), lambda: edgehip.gate_norm(x, d), lambda: edgehip.act8(d), lambda: edgehip.linear8(d, w),
                  lambda: edgehip.policy_loss(d, taken, old, adv, ptr), lambda: edgehip.preference_loss(d, taken, ptr)):
            with pytest.raises(NotImplementedError):
                f()

"""GPU: the policy and preference losses (edgehip.tune) against their formulas in fp64 under automatic differentiation.

Tolerances.  A row's sum of C exponentials: each off by (2 + |x - max|) 2^-24 of itself (difference, product, exponential),
weighted by itself - the mean of |x - max| under the softmax, at most ln C + 1 - plus at most C / (8 threads) + 16
additions of positive terms: LSE below bounds ln(sum).  Everything after it is fp64.  A loss is rounded once; a gradient is
coef (onehot - p): p is off by LSE + (4 + |x - max|) 2^-24 of itself, coef by the derivative of its formula in logp times
LSE and by three roundings; then one rounding to the logits' type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]
CLASSES = [1, 2, 3, 7, 8, 9, 31, 32, 33, 63, 64, 65, 257, 500, 512, 513, 1000, 1025, 2049, 4096, 4097, 8193, 16385, 32769, 40001, 65537, 70000]


def step(t):
    return torch.finfo(t).eps / 2 if t != F32 else 0.0


def lse_error(c):
    return (6 + math.log(c + 1) + 16 + min(c, 512) / 8) * U


def make(rows, classes, seqs, dtype=F32, seed=0, masked=True, behind=0, edge=(0.2, 0.3)):
    """Rows of logits, what they took, ragged sequences (some empty), a mask with rows that hold rubbish, out-of-range
    choices, and log-probabilities whose ratios keep 1e-3 away from the clip's edges."""
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = (2 * torch.randn(rows, classes, generator=g, device='cuda')).to(dtype)
    taken = torch.randint(0, classes, (rows,), generator=g, device='cuda')
    if classes > 16:
        x[:, 3::7] = float('-inf')
        x[torch.arange(rows, device='cuda'), taken] = 1.0
    cut = torch.randint(0, rows - behind + 1, (seqs - 1,), generator=g, device='cuda').sort().values
    ptr = torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), rows - behind)])
    logp = torch.log_softmax(x.double(), 1).gather(1, taken[:, None])[:, 0]
    drift = 0.3 * torch.randn(rows, generator=g, device='cuda', dtype=torch.float64)
    for e in (math.log(1 - edge[0]), math.log(1 + edge[1])):
        drift = torch.where((drift - e).abs() < 1e-3, drift + 3e-3, drift)
    old = (logp - drift).float()
    ref = (logp + 0.2 * torch.randn(rows, generator=g, device='cuda', dtype=torch.float64)).float()
    mask = None
    counts = torch.arange(rows, device='cuda') < rows - behind
    if masked and rows > 4:
        mask = torch.rand(rows, generator=g, device='cuda') > 0.2
        taken[1], taken[2] = -100, classes
        x[~mask, 0] = float('nan')
        x[2] = float('inf')
        counts = counts & mask & (taken >= 0) & (taken < classes)
    adv = torch.randn(seqs, generator=g, device='cuda')
    return dict(x=x, taken=taken, ptr=ptr, old=old, ref=ref, mask=mask, counts=counts, adv=adv,
                adv_rows=torch.randn(rows, generator=g, device='cuda'))


def logp64(s, x):
    """Log-probabilities of counted rows, differentiable; 0 elsewhere."""
    rows = s['counts'].nonzero()[:, 0]
    lp = torch.log_softmax(x[rows], 1).gather(1, s['taken'][rows, None])[:, 0]
    return torch.zeros(len(s['counts']), dtype=torch.float64, device='cuda').index_put((rows,), lp)


def per_seq(s, v, mean):
    ptr = s['ptr'].tolist()
    v = torch.where(s['counts'], v, 0.0)
    out = [v[a:b].sum() / (max(1, int(s['counts'][a:b].sum())) if mean else 1) for a, b in zip(ptr, ptr[1:])]
    return torch.stack(out)


def policy64(s, lp, adv, clip, kl_coef, ref, mean):
    own = torch.zeros(len(lp), dtype=torch.long, device='cuda')
    n = int(s['ptr'][-1])
    own[:n] = torch.repeat_interleave(torch.arange(len(s['ptr']) - 1, device='cuda'), s['ptr'][1:] - s['ptr'][:-1])
    A = (adv if adv.shape == lp.shape and adv is s['adv_rows'] else adv[own]).double()
    rho = torch.exp(lp - s['old'].double())
    gain = torch.minimum(rho * A, rho.clamp(1 - clip[0], 1 + clip[1]) * A)
    kl = torch.zeros_like(lp)
    if ref is not None:
        gap = ref.double() - lp
        kl = torch.expm1(gap) - gap
    cut = ((A > 0) & (rho > 1 + clip[1]) | (A < 0) & (rho < 1 - clip[0])) & s['counts']
    ptr = s['ptr'].tolist()
    return per_seq(s, kl_coef * kl - gain, mean), per_seq(s, kl, mean), torch.tensor([int(cut[a:b].sum()) for a, b in zip(ptr, ptr[1:])]), A, rho


def near_gradient(s, got, want, coef_size, dtype):
    """coef_size: per row, the size of what coef is made of."""
    p = torch.softmax(s['x'].double(), 1)
    c = s['x'].shape[1]
    dist = (s['x'].double() - s['x'].double().amax(1, keepdim=True)).abs().clamp(max=200)
    hot = torch.zeros_like(p).scatter_(1, s['taken'].clamp(0, c - 1)[:, None], 1.0)
    tol = coef_size[:, None] * ((p * (2 * lse_error(c) + (8 + dist) * U)) + (p + hot) * (4 * lse_error(c) + 8 * U))
    tol = tol + step(dtype) * want.abs() + (2.0 ** -25 if dtype == F16 else 0.0) + 1e-42
    bad = (got.double() - want).abs() > tol
    bad[~s['counts']] = got[~s['counts']] != 0                     # exactly nothing, whatever their logits hold
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() / tol)[s['counts']].max()))


def check_policy(s, per_row=False, clip=(0.2, 0.3), kl_coef=0.1, ref=True, mean=True, weight=None):
    import edgehip
    x = s['x'].double().requires_grad_(True)
    adv = s['adv_rows'] if per_row else s['adv']
    ref_t = s['ref'] if ref else None
    lp = logp64(s, x)
    loss, kl, clipped, A, rho = policy64(s, lp, adv, clip, kl_coef, ref_t, mean)
    S = len(loss)
    w = torch.full((S,), 1.0 / S, device='cuda') if weight is None else weight
    (want,) = torch.autograd.grad((loss * w.double()).sum(), x)
    kw = dict(ref_logp=ref_t, mask=s['mask'], clip=clip, kl_coef=kl_coef, reduce='mean' if mean else 'sum')
    r = edgehip.policy_loss_grad(s['x'], s['taken'], s['old'], adv, s['ptr'], weight=weight, **kw)
    # sizes: |A| rho + kl's, times the number of rows summed
    c = s['x'].shape[1]
    gap = (s['ref'].double() - lp).abs() if ref else torch.zeros_like(lp)
    size = torch.where(s['counts'], A.abs() * rho + kl_coef * (torch.exp(gap) + 1), 0.0).detach()
    tol = per_seq(s, size, mean) * (2 * lse_error(c) + 4 * U) + U * loss.abs() + 1e-12
    assert bool(((r.loss.double() - loss).abs() <= tol).all()), (r.loss, loss)
    tol = per_seq(s, torch.exp(gap).detach() + 1, mean) * (2 * lse_error(c) + 4 * U) + 1e-12
    assert bool(((r.kl.double() - kl).abs() <= tol).all())
    assert torch.equal(r.clipped.cpu().long(), clipped)
    assert bool(((r.logp.double() - lp).abs() <= lse_error(c) + U * lp.abs() + 1e-12).all())
    n = torch.ones(S, dtype=torch.float64, device='cuda')
    if mean:
        n = per_seq(s, torch.ones_like(lp), False).clamp_min(1)
    own = torch.zeros(len(lp), dtype=torch.long, device='cuda')
    m = int(s['ptr'][-1])
    own[:m] = torch.repeat_interleave(torch.arange(S, device='cuda'), s['ptr'][1:] - s['ptr'][:-1])
    coef_size = size * (w.double().abs() / n)[own]
    near_gradient(s, r.dlogits, torch.where(s['counts'][:, None], want, 0.0), coef_size, s['x'].dtype)
    # the differentiable form: the same losses to the bit; its gradient for the same weights
    leaf = s['x'].clone().requires_grad_(True)
    f = edgehip.policy_loss(leaf, s['taken'], s['old'], adv, s['ptr'], **kw)
    assert torch.equal(f.loss, r.loss) and torch.equal(f.kl, r.kl) and torch.equal(f.clipped, r.clipped) and torch.equal(f.logp, r.logp)
    (g,) = torch.autograd.grad(f.loss, leaf, w.float())
    near_gradient(s, g, torch.where(s['counts'][:, None], want, 0.0), coef_size, s['x'].dtype)
    return r


@pytest.mark.parametrize('classes', CLASSES)
def test_policy_classes(classes):
    rows = 300 if classes <= 1000 else 23
    check_policy(make(rows, classes, 7, seed=classes))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('classes', [2, 20, 50, 700, 1500, 5001, 20000, 40000])
def test_policy_types_and_options(dtype, classes):
    rows = 200 if classes < 1000 else 40
    for k, opt in enumerate((dict(per_row=True), dict(ref=False, kl_coef=0.0), dict(mean=False, weight=torch.tensor([0.5, -1.0, 0.0, 2.0], device='cuda')),
                             dict(clip=(0.0, 0.0)), dict(clip=(0.9, 5.0)))):
        s = make(rows, classes, 4, dtype, seed=classes + k, masked=k % 2 == 0)
        check_policy(s, **opt)


def test_policy_sequences():
    """One sequence over many blocks' rows, one row each, more sequences than rows, rows behind the last one."""
    check_policy(make(5000, 2, 1, seed=1))
    check_policy(make(5000, 3, 2, seed=2, masked=False))
    check_policy(make(50, 5, 300, seed=3))
    check_policy(make(6200, 4, 2500, seed=4))
    s = make(4500, 4, 6, seed=5, behind=2300)
    r = check_policy(s)
    assert not bool(r.dlogits[2200:].any()) and not bool(r.logp[2200:].any())


def test_policy_without_a_row_that_counts():
    import edgehip
    s = make(40, 10, 3, masked=False)
    s['mask'] = torch.zeros(40, dtype=torch.bool, device='cuda')
    s['x'][:] = float('nan')
    r = edgehip.policy_loss_grad(s['x'], s['taken'], s['old'], s['adv'], s['ptr'], ref_logp=s['ref'], mask=s['mask'], kl_coef=0.1)
    for v in r:
        assert not bool(v.any())
    z = torch.zeros(0, 10, device='cuda')
    e = torch.zeros(0, dtype=torch.int64, device='cuda')
    f = torch.zeros(0, device='cuda')
    r = edgehip.policy_loss_grad(z, e, f, torch.ones(2, device='cuda'), torch.zeros(3, dtype=torch.int64, device='cuda'))
    assert r.loss.tolist() == [0.0, 0.0] and r.dlogits.shape == (0, 10)


def test_rows_of_the_lowest_values_and_single_choices():
    """All classes at the type's lowest value, one finite class, a huge logit; a row of -inf alone is NaN, as its formula is."""
    import edgehip
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        x = torch.zeros(5, 70, dtype=dtype, device='cuda')
        x[0], x[1], x[2] = low, float('-inf'), low
        x[1, 9], x[2, 9], x[3, 9] = 2.0, 60000.0, 60000.0
        x[4] = float('-inf')
        lp = edgehip.row_logp(x, torch.full((5,), 9, device='cuda'))
        assert abs(float(lp[0]) + math.log(70)) < 1e-6 and lp[1:4].tolist() == [0.0, 0.0, 0.0] and bool(lp[4].isnan())
        s = make(5, 70, 1, dtype, masked=False)
        r = edgehip.policy_loss_grad(x[:4], s['taken'][:4] * 0 + 9, lp[:4].contiguous(), torch.ones(1, device='cuda'),
                                     torch.tensor([0, 4], device='cuda'))
        assert float(r.loss[0]) == -1.0 and bool(torch.isfinite(r.dlogits).all())
        p = torch.softmax(x[:4].double(), 1)
        p[:, 9] -= 1
        assert bool(((r.dlogits.double() - p / 4).abs() <= 1e-6 + step(dtype) * p.abs() / 4 + (2.0 ** -25 if dtype == F16 else 0)).all())


def pref64(s, lp, beta, smooth, kind, mean, ref):
    m = per_seq(s, lp - (ref.double() if ref is not None else 0.0), mean)
    P = len(m) // 2
    margin = m[:P] - m[P:]
    if kind == 'sigmoid':
        f = torch.nn.functional.logsigmoid
        return -(1 - smooth) * f(beta * margin) - smooth * f(-beta * margin), margin
    return (margin - 1 / (2 * beta)) ** 2, margin


def check_pref(s, beta=0.1, smooth=0.0, kind='sigmoid', mean=False, ref=True, weight=None):
    import edgehip
    x = s['x'].double().requires_grad_(True)
    ref_t = s['ref'] if ref else None
    lp = logp64(s, x)
    loss, margin = pref64(s, lp, beta, smooth, kind, mean, ref_t)
    P = len(loss)
    w = torch.full((P,), 1.0 / P, device='cuda') if weight is None else weight
    (want,) = torch.autograd.grad((loss * w.double()).sum(), x)
    kw = dict(ref_logp=ref_t, mask=s['mask'], beta=beta, label_smoothing=smooth, kind=kind, reduce='mean' if mean else 'sum')
    r = edgehip.preference_loss_grad(s['x'], s['taken'], s['ptr'], weight=weight, **kw)
    c = s['x'].shape[1]
    cnt = per_seq(s, torch.ones_like(lp.detach()), mean)
    off = (cnt[:P] + cnt[P:]) * lse_error(c)                       # of the margin
    assert bool(((r.margin.double() - margin).abs() <= off + U * margin.abs() + 1e-12).all())
    slope = beta if kind == 'sigmoid' else 2 * (margin.detach().abs() + 1 / (2 * beta) + off)
    assert bool(((r.loss.double() - loss).abs() <= slope * off + U * loss.abs() + 1e-12).all())
    n = per_seq(s, torch.ones_like(lp.detach()), False).clamp_min(1) if mean else torch.ones(2 * P, dtype=torch.float64, device='cuda')
    # d loss / d margin: its size, and how far the margin's error moves it (curvature <= beta^2, or 2)
    bend = (beta * beta if kind == 'sigmoid' else 2.0) * off
    size = (slope + torch.zeros(P, dtype=torch.float64, device='cuda')) * w.double().abs() + bend * w.double().abs() / (4 * lse_error(c))
    own = torch.zeros(len(lp), dtype=torch.long, device='cuda')
    m = int(s['ptr'][-1])
    own[:m] = torch.repeat_interleave(torch.arange(2 * P, device='cuda'), s['ptr'][1:] - s['ptr'][:-1])
    coef_size = (torch.cat([size, size]) / n)[own]
    near_gradient(s, r.dlogits, torch.where(s['counts'][:, None], want, 0.0), coef_size, s['x'].dtype)
    leaf = s['x'].clone().requires_grad_(True)
    f = edgehip.preference_loss(leaf, s['taken'], s['ptr'], **kw)
    assert torch.equal(f.loss, r.loss) and torch.equal(f.margin, r.margin)
    (g,) = torch.autograd.grad(f.loss, leaf, w.float())
    near_gradient(s, g, torch.where(s['counts'][:, None], want, 0.0), coef_size, s['x'].dtype)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('classes', [2, 9, 100, 5001, 66000])
def test_preference(dtype, classes):
    rows = 400 if classes < 1000 else 40
    for k, opt in enumerate((dict(), dict(smooth=0.1, beta=0.5), dict(kind='square', beta=0.2), dict(mean=True, ref=False),
                             dict(weight=torch.tensor([1.0, 0.0, -3.0], device='cuda')))):
        check_pref(make(rows, classes, 6, dtype, seed=classes + k, masked=k % 2 == 0), **opt)


def test_preference_sequences():
    check_pref(make(5000, 3, 2, seed=1))
    check_pref(make(30, 3, 200, seed=2))
    check_pref(make(4500, 3, 8, seed=3, behind=2400))


def test_large_margins_do_not_overflow():
    import edgehip
    x = torch.zeros(2, 4, device='cuda')
    for gap in (1e4, -1e4):
        ref = torch.tensor([-gap, gap], device='cuda')
        r = edgehip.preference_loss_grad(x, torch.zeros(2, dtype=torch.int64, device='cuda'), torch.tensor([0, 1, 2], device='cuda'),
                                         ref_logp=ref, beta=1.0)
        assert abs(float(r.loss[0]) - max(0.0, -2 * gap)) <= 1e-3 and bool(torch.isfinite(r.dlogits).all())


def test_row_stride_offsets_and_mask_types():
    import edgehip
    s = make(60, 130, 4, BF16)
    wide = torch.zeros(60, 301, dtype=BF16, device='cuda')
    wide[:, 7:137] = s['x']
    view = wide[:, 7:137]
    kw = dict(ref_logp=s['ref'], kl_coef=0.1)
    a = edgehip.policy_loss_grad(s['x'], s['taken'], s['old'], s['adv'], s['ptr'], mask=s['mask'], **kw)
    b = edgehip.policy_loss_grad(view, s['taken'], s['old'], s['adv'], s['ptr'], mask=s['mask'].to(torch.uint8), **kw)
    c = edgehip.policy_loss_grad(s['x'].t().contiguous().t(), s['taken'], s['old'], s['adv'], s['ptr'], mask=s['mask'], **kw)
    for other in (b, c):
        assert all(torch.equal(u, v) for u, v in zip(a, other))
    lp = edgehip.row_logp(view, s['taken'], s['mask'])
    assert torch.equal(lp, a.logp)


def test_offsets_beyond_32_bits():
    """More than 2^31 logits: the last rows are where they should be."""
    import edgehip
    rows, classes = 33000, 66000
    x = torch.zeros(rows, classes, dtype=BF16, device='cuda')
    x[-1] = torch.randn(classes, device='cuda').to(BF16)
    taken = torch.zeros(rows, dtype=torch.int64, device='cuda')
    taken[-1] = classes - 1
    ptr = torch.tensor([0, rows - 1, rows], device='cuda')
    lp = edgehip.row_logp(x, taken)
    want = torch.log_softmax(x[-1].double(), 0)[-1]
    assert abs(float(lp[-1]) - float(want)) <= lse_error(classes) + U * abs(float(want))
    r = edgehip.policy_loss_grad(x, taken, lp, torch.ones(2, device='cuda'), ptr)
    p = torch.softmax(x[-1].double(), 0)
    p[-1] -= 1
    assert bool(((r.dlogits[-1].double() - p / 2).abs() <= 2.0 ** -8 * p.abs() / 2 + 1e-6 * p.abs()).all())
    assert float(r.dlogits[0, 0]) != 0 and torch.equal(r.dlogits[0, 1:], r.dlogits[0, 1].expand(classes - 1))


def test_against_differences():
    """d loss along a direction, step 2^-6 in fp32 logits: third derivatives are O(kl + A) per row, the difference is off by
    ~2^-12 of the direction's size, the losses' rounding adds 2^-24 x 2^6: 0.5 % of the product."""
    import edgehip
    s = make(60, 12, 3, masked=False, edge=(0.9, 9.0))
    d = torch.randn_like(s['x'])
    d = d / d.norm()
    for f in (lambda x: edgehip.policy_loss(x, s['taken'], s['old'], s['adv'], s['ptr'], ref_logp=s['ref'], kl_coef=0.3, clip=(0.9, 9.0)).loss,
              lambda x: edgehip.preference_loss(x, s['taken'], torch.tensor([0, 30, 60], device='cuda'), ref_logp=s['ref'], beta=0.3).loss):
        leaf = s['x'].clone().requires_grad_(True)
        (g,) = torch.autograd.grad(f(leaf).sum(), leaf)
        e = 2.0 ** -6
        diff = sum(sg * float(f(s['x'] + sg * e * d).double().sum()) for sg in (1, -1)) / (2 * e)
        assert abs(diff - float((g * d).sum())) <= 0.005 * float(g.norm()), (diff, float((g * d).sum()))


def test_same_bits_on_other_streams_and_in_a_graph():
    import edgehip
    s = make(3000, 300, 6, BF16)

    def both():
        a = edgehip.policy_loss_grad(s['x'], s['taken'], s['old'], s['adv'], s['ptr'], ref_logp=s['ref'], mask=s['mask'], kl_coef=0.1)
        b = edgehip.preference_loss_grad(s['x'], s['taken'], s['ptr'], ref_logp=s['ref'], mask=s['mask'])
        return list(a) + list(b)
    ref = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for k in range(3):
        s['old'].add_(0.05)
        s['x'].copy_(torch.randn(s['x'].shape, device='cuda') * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, both())), k


@pytest.mark.parametrize('rows,seqs,behind', [(16384, 512, 0), (16385, 512, 100), (16384, 514, 0), (20011, 4, 0), (3000, 700, 2000)])
@pytest.mark.parametrize('classes,dtype', [(70, F32), (40, BF16), (5, F16)])
def test_few_and_many_rows(rows, seqs, behind, classes, dtype):
    """On both sides of where the sequences' sums are taken from the rows themselves."""
    s = make(rows, classes, seqs, dtype, seed=rows + seqs, behind=behind)
    check_policy(s)
    check_pref(s, mean=True)

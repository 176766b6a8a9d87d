"""GPU: how exact a row's log-probability is where the losses add up many of them (edgehip.tune).

A preference's margin is the difference of two sums over rows, so what counts is a row's error before it is rounded, and
what all rows' errors have in common.  `ref_logp` is set to the log-probability rounded to fp32: margins are then of the size
of 1e-7 and their own rounding does not show.

Tolerances.  A term of a row's sum is off by at most 3.5e-8 of itself (the fp32 part of an exponential is below 0.42; its
rounding and its polynomial's: rms 5.8e-9), a partial sum's scaling by as much again, once or twice
on the way; the sum is fp64 and the logarithm 1e-9.  Independent, and the largest term exact: rms sqrt(3) x 5.8e-9 for a row
that one other term makes up, less for more terms.  Differences of fp32 logits are rounded before: a term e^-x by 2^-25 x at
most (rms / sqrt(3)), weighted with itself: x e^-x <= 0.37, 2^-25 0.37 / sqrt(3) = 6.4e-9.  In rows of more than 64 threads eight
terms are added up in fp32: 2^-25 / sqrt(3) = 1.7e-8 of a piece that is at most half of such a row here: 8.6e-9.  Together
under 2^-26 = 1.5e-8 a row.  What is common to the terms is the mean error of the hardware's exponential, 3.3e-9 at most."""
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ROW, COMMON = 2.0 ** -26, 3.5e-9


def rows_of(rows, classes, dtype, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = (2.5 * torch.randn(rows, classes, generator=g, device='cuda')).to(dtype)
    if classes >= 64:
        x[:, ::97] = float('-inf')
    taken = (x.float() + torch.randn(rows, classes, generator=g, device='cuda')).argmax(1)
    logp = torch.empty(rows, dtype=torch.float64, device='cuda')
    for a in range(0, rows, 1024):
        y = x[a:a + 1024].double()
        logp[a:a + 1024] = y.gather(1, taken[a:a + 1024, None])[:, 0] - torch.logsumexp(y, 1)
    return x, taken, logp


@pytest.mark.parametrize('dtype', [F32, BF16, F16])
@pytest.mark.parametrize('classes,rows', [(2, 1 << 17), (5, 1 << 16), (8, 1 << 16), (29, 1 << 16), (50, 1 << 16), (70, 1 << 15), (184, 1 << 15),
                                          (700, 1 << 14), (4777, 1 << 12), (30000, 1 << 11), (90486, 1 << 10)])
def test_margins_of_many_rows(dtype, classes, rows):
    import edgehip
    x, taken, logp = rows_of(rows, classes, dtype, seed=classes)
    ref = logp.float()
    left = logp - ref.double()                                   # what a row adds to its sequence
    pairs = rows // 2
    one = torch.arange(rows + 1, device='cuda')
    off = edgehip.preference_loss(x, taken, one, ref_logp=ref).margin.double() - (left[:pairs] - left[pairs:])
    assert float(off.square().mean().sqrt()) <= 2 ** 0.5 * ROW
    # one sequence of all rows: chance errors grow with the root of their number, common ones with it (5 sigma)
    for ptr in ([0, rows, rows], [0, 0, rows], [0, rows // 3, rows]):
        ptr = torch.tensor(ptr, device='cuda')
        r = edgehip.preference_loss_grad(x, taken, ptr, ref_logp=ref)
        want = left[:ptr[1]].sum() - left[ptr[1]:].sum()
        assert abs(float(r.margin[0]) - float(want)) <= 5 * ROW * rows ** 0.5 + COMMON * rows


def test_gradients_of_classes_far_below_the_largest():
    """Values of a gradient, coef p, are off by rounding x log2(e) to either side (2^-25 |x| log2(e) at most), never all to one: over
    10^6 values at |x| of 2 to 40 the mean relative error is the hardware exponential's own, 3.3e-9 at most, and chance: a value's
    8e-7 / 10^3, a row's three roundings 2^-24 / sqrt(10^3) (5 sigma: 1.4e-8).  A preference's coef is one fp32 number for all rows:
    its rounding, 2^-24 at most, is common to all values."""
    import edgehip
    rows, classes = 1024, 1024
    g = torch.Generator(device='cuda').manual_seed(3)
    x = -2 - 38 * torch.rand(rows, classes, generator=g, device='cuda')
    x[:, 5] = 0
    taken = torch.full((rows,), 5, device='cuda')
    old = torch.zeros(rows, device='cuda')
    p = torch.softmax(x.double(), 1)
    rho = p[:, 5:6]
    r = edgehip.policy_loss_grad(x, taken, old, torch.ones(1, device='cuda'), torch.tensor([0, rows], device='cuda'), reduce='sum', clip=(1.0, 9.0))
    f = edgehip.preference_loss_grad(x, taken, torch.tensor([0, rows, rows], device='cuda'), kind='square', beta=1.0)
    slope = 2 * (torch.log(p[:, 5]).sum() - 0.5)
    off = torch.arange(classes, device='cuda') != 5
    for got, coef, common in ((r.dlogits, rho, 0.0), (f.dlogits, -slope, 2.0 ** -24)):
        rel = got.double()[:, off] / (coef * p)[:, off] - 1
        assert abs(float(rel.mean())) <= 2e-8 + common, float(rel.mean())
        assert float(rel.abs().max()) <= 45 * 2.0 ** -24

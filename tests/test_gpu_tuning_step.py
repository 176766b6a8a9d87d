"""GPU: the operators for deeper networks and tuning as they are used together, and in this package's own paths."""
import numpy as np
import pytest
import torch

import cases
import helpers as H
from oracle import edge_oracle as orc

pytestmark = pytest.mark.gpu


def block64(p, h, z, row_ptr, kept=None):
    """Norm, two layers with an activation between, gated back into the stream, in fp64.  kept: the 8-bit values the
    layers' inputs are replaced by where only their gradient reads them."""
    def norm(x, w):
        return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w
    own = torch.repeat_interleave(torch.arange(len(row_ptr) - 1, device=h.device), (row_ptr[1:] - row_ptr[:-1]).long())
    h = 0.9 * h + p['gate'][own] * norm(z, p['w_post'])
    return h, norm(h, p['w_pre'])


def test_a_tuning_step_of_a_two_layer_block():
    """Stream -> gated norms -> linear8 -> act8 -> linear8 -> logits -> policy loss, forward and backward, against the same
    step in fp64 with exact inputs everywhere: the loss to fp32, the gradients to what 8-bit checkpoints leave of them -
    a kept value is off by at most 1/127 of the largest of its 64, uniformly distributed, rms 1/127/sqrt(12) x 4 sigma: under
    1 % of the rms; a gradient reads one checkpoint in each of two layers: 3 % of its norm."""
    import edgehip
    g = torch.Generator(device='cuda').manual_seed(3)
    rows, dim, hid, seqs = 900, 128, 256, 12
    n = lambda *s: torch.randn(*s, generator=g, device='cuda')
    cut = torch.randint(0, rows, (seqs - 1,), generator=g, device='cuda').sort().values
    ptr = torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), rows)])
    p = dict(w_pre=1 + 0.1 * n(dim), w_post=1 + 0.1 * n(dim), gate=0.5 + 0.2 * n(seqs, dim), w1=n(hid, dim) * dim ** -0.5, b1=0.1 * n(hid),
             w2=n(64, hid) * hid ** -0.5, b2=0.1 * n(64))
    h, z = n(rows, dim), n(rows, dim)
    taken = torch.randint(0, 64, (rows,), generator=g, device='cuda')
    mask = torch.rand(rows, generator=g, device='cuda') > 0.1
    adv = n(seqs)
    d = {k: v.double().requires_grad_(True) for k, v in dict(p, h=h, z=z).items()}
    _, y = block64(d, d['h'], d['z'], ptr)
    logits = torch.nn.functional.silu(y @ d['w1'].t() + d['b1']) @ d['w2'].t() + d['b2']
    lp = torch.log_softmax(logits, 1).gather(1, taken[:, None])[:, 0]
    drift = (0.2 * n(rows)).double()
    old = (lp.detach() - drift).float()
    rho = torch.exp(lp - old.double())
    own = torch.repeat_interleave(torch.arange(seqs, device='cuda'), ptr[1:] - ptr[:-1])
    A = adv.double()[own]
    each = -torch.minimum(rho * A, rho.clamp(0.8, 1.2) * A) * mask
    total = torch.zeros(seqs, dtype=torch.float64, device='cuda').index_add(0, own, each)
    count = torch.zeros(seqs, dtype=torch.float64, device='cuda').index_add(0, own, mask.double()).clamp_min(1)
    want_loss = total / count
    want = torch.autograd.grad(want_loss.mean(), list(d.values()))

    leaves = {k: v.clone().requires_grad_(True) for k, v in dict(p, h=h, z=z).items()}
    _, y = edgehip.gate_norm(leaves['h'], leaves['z'], w_pre=leaves['w_pre'], w_post=leaves['w_post'], gate=leaves['gate'],
                             row_ptr=ptr.to(torch.int32), res_scale=0.9)
    x = edgehip.linear8(edgehip.act8(edgehip.linear8(y, leaves['w1'], leaves['b1'])), leaves['w2'], leaves['b2'])
    out = edgehip.policy_loss(x, taken, old, adv, ptr, mask=mask)
    got = torch.autograd.grad(out.loss.mean(), list(leaves.values()), retain_graph=True)
    assert bool(((out.loss.double() - want_loss).abs() <= 1e-4 * (1 + want_loss.abs())).all())
    for k, a, b in zip(leaves, got, want):
        assert float((a.double() - b).norm()) <= 0.03 * float(b.norm()), k
    # the gradient made with the loss, handed on, is the same step
    r = edgehip.policy_loss_grad(x.detach(), taken, old, adv, ptr, mask=mask)
    more = torch.autograd.grad(x, list(leaves.values()), r.dlogits)
    for k, a, b in zip(leaves, got, more):
        assert float((a - b).norm()) <= 1e-5 * float(a.norm()), k


def _step(form, graphs, T, params, seed=2):
    model = H.build_model(params, T, cases.max_degree_of(graphs))
    model.train()
    model.train_form = form
    b = H.graph_batch(graphs, degree_dtype=np.int64)
    gen = torch.Generator().manual_seed(seed)
    t = torch.full((len(graphs),), T // 3)
    pairs = sum(q['n'] * (q['n'] - 1) // 2 for q in graphs)
    u1, u3 = torch.rand(pairs, 2, generator=gen).cuda(), torch.rand(pairs, 2, generator=gen).cuda()
    nv = model.log_prob(b, t, torch.full((len(graphs),), 1.0 / T), u1, u3)
    (-nv.sum() / (np.log(2) * b.num_entries)).backward()
    return model, b, nv.detach(), {k: v.grad.detach().clone() for k, v in model._denoise_fn.named_parameters() if v.grad is not None}


def kept(x):
    """What an 8-bit checkpoint of x stands for, in plain torch (tests/test_gpu_ckpt8.py holds the kernels to it)."""
    m, k = x.shape
    v = torch.nn.functional.pad(x, (0, -k % 64)).view(m, -1, 64)
    f, e = torch.frexp(v.abs().amax(2, keepdim=True))
    e = torch.where(f <= 127 / 128, e - 7, e - 6).clamp(-120, 121)
    up, down = (((127 + s) << 23).view(torch.float32) for s in (e, -e))
    return (torch.round(v * down) * up).view(m, -1)[:, :k]


class PlainLinear8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b):
        from edgehip import train
        ctx.save_for_backward(kept(x).double(), w)
        return train._Linear.apply(x, w, b)

    @staticmethod
    def backward(ctx, dy):
        q, w = ctx.saved_tensors
        dy = dy.double()
        return (dy @ w.double()).float(), (dy.t().contiguous() @ q).float(), dy.sum(0).float()


class PlainAct8(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, kind):
        from edgehip import ckpt8
        ctx.kind, q = kind, kept(x).double()
        ctx.save_for_backward(q)
        return ckpt8.act8_fwd(x, 'silu' if kind == 1 else 'mish')[0]

    @staticmethod
    def backward(ctx, dy):
        (q,) = ctx.saved_tensors
        with torch.enable_grad():
            q = q.detach().requires_grad_(True)
            f = torch.nn.functional.silu if ctx.kind == 1 else torch.nn.functional.mish
            (d,) = torch.autograd.grad(f(q), q, dy.double())
        return d.float(), None


class PlainOps8:
    """The layers' ops with 8-bit checkpoints in plain torch: the same forward values to the bit, so the same kept values."""
    linear = staticmethod(lambda x, w, b, kept=None: PlainLinear8.apply(x, w, b))
    act = staticmethod(lambda x, kind=1: PlainAct8.apply(x, kind))
    keep = staticmethod(lambda x: None)


def near(got, want):
    """The bound the training ops are held to everywhere (2e-4 of a gradient's size; gradients that cancel, of 1e-3 of the
    largest)."""
    assert set(got) == set(want) and len(got) > 80
    gmax = max(float(g.norm()) for g in want.values())
    for k, g in want.items():
        assert float((got[k] - g).norm()) <= 2e-4 * max(float(g.norm()), 1e-3 * gmax), k


def test_the_training_form_with_8_bit_checkpoints(monkeypatch):
    """train_form 'ops8' computes the loss of 'ops' (the same kernels on the same inputs); its gradients are those of the same
    network with plain 8-bit checkpoints."""
    from edgehip import train
    graphs = cases.ragged_graphs(5) + cases.ragged_graphs(6)
    params = orc.random_tgnn_params(4)
    _, _, nv, exact = _step('ops', graphs, 48, params)
    _, _, nv8, got = _step('ops8', graphs, 48, params)
    assert torch.allclose(nv, nv8, rtol=1e-6, atol=1e-9)
    monkeypatch.setattr(train, '_Ops8', PlainOps8)
    _, _, _, want = _step('ops8', graphs, 48, params)
    near(got, want)
    assert any(float((got[k] - exact[k]).norm()) > 2e-4 * float(exact[k].norm()) for k in exact)      # (they really are kept in 8 bits)


def test_tuning_the_graph_sampler_on_its_own_decisions(monkeypatch):
    """The active pairs of a batch, what was taken there and `aptr` go into the policy loss: the network's gradient is that
    of the formula in fp64 on the same logits, with whole and with 8-bit checkpoints."""
    import edgehip
    from edgehip import train
    from edgehip.model import _state
    graphs = cases.ragged_graphs(5)
    model, b, _, _ = _step('ops', graphs, 48, orc.random_tgnn_params(4))
    net, st = model._denoise_fn, _state(b)
    t_graph = torch.full((b.num_graphs,), 16, dtype=torch.int32, device='cuda')
    row, col = b.active_row, b.active_col
    assert row.numel() > 50
    gen = torch.Generator(device='cuda').manual_seed(8)
    adv = torch.randn(b.num_graphs, generator=gen, device='cuda')
    taken = torch.randint(0, 2, (row.numel(),), generator=gen, device='cuda')
    n = st['aptr'][1:] - st['aptr'][:-1]
    own = torch.repeat_interleave(torch.arange(b.num_graphs, device='cuda'), n)
    old = None

    def gradients(keep8, formula):
        nonlocal old
        net.zero_grad()
        logits = train.tgnn_pair_logits(net, b, b.adj, st['deg_t'], st['flags'], t_graph, row, col, keep8=keep8)
        if old is None:
            old = edgehip.row_logp(logits.detach(), taken) - 0.1
        if formula:
            lp = torch.log_softmax(logits.double(), 1).gather(1, taken[:, None])[:, 0]
            rho = torch.exp(lp - old.double())
            each = -torch.minimum(rho * adv.double()[own], rho.clamp(0.8, 1.2) * adv.double()[own]) / n[own]
            loss = torch.zeros(b.num_graphs, dtype=torch.float64, device='cuda').index_add(0, own, each)
        else:
            loss = edgehip.policy_loss(logits, taken, old, adv, st['aptr']).loss
        loss.sum().backward()
        return loss.detach().double(), {k: p.grad.clone() for k, p in net.named_parameters() if p.grad is not None}
    got, want, got8 = gradients(False, False), gradients(False, True), gradients(True, False)
    assert bool(((got[0] - want[0]).abs() <= 1e-6 * (1 + want[0].abs())).all())
    near(got[1], want[1])
    monkeypatch.setattr(train, '_Ops8', PlainOps8)
    near(got8[1], gradients(True, True)[1])


def test_a_gate_per_graph_of_a_batch():
    """`node_ptr` of a batch is a row_ptr: every graph's nodes see its own row, as graph by graph with one vector."""
    import edgehip
    b = H.graph_batch(cases.ragged_graphs(7))
    p = b.node_ptr.tolist()
    h, z = torch.randn(b.num_nodes, 64, device='cuda'), torch.randn(b.num_nodes, 64, device='cuda')
    g, w = torch.randn(b.num_graphs, 64, device='cuda'), torch.ones(64, device='cuda')
    got = edgehip.gate_norm(h, z, w_pre=w, w_post=w, gate=g, row_ptr=b.node_ptr)
    for i, (a, c) in enumerate(zip(p, p[1:])):
        one = edgehip.gate_norm(h[a:c], z[a:c], w_pre=w, w_post=w, gate=g[i])
        assert torch.equal(one[0], got[0][a:c]) and torch.equal(one[1], got[1][a:c])


def _whole(v):
    """Forward and backward of all operators, through their differentiable forms."""
    import edgehip
    leaves = {k: t.detach().requires_grad_(True) for k, t in v.items() if t.is_floating_point() and k not in ('old', 'adv')}
    h, y = edgehip.gate_norm(leaves['h'], leaves['z'], w_pre=leaves['w'], gate=leaves['g'], kind='rms')
    x = edgehip.linear8(edgehip.act8(edgehip.linear8(y, leaves['a'])), leaves['b'])
    a = edgehip.policy_loss(x, v['taken'], v['old'], v['adv'], v['ptr']).loss.sum()
    b = edgehip.preference_loss(x, v['taken'], v['ptr']).loss.sum()
    return [a.detach(), b.detach(), h.detach()] + list(torch.autograd.grad(a + b + h.sum(), list(leaves.values())))


def _inputs(seed):
    g = torch.Generator(device='cuda').manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g, device='cuda')
    return dict(h=n(300, 128), z=n(300, 128), w=n(128), g=n(128), a=n(256, 128) * 0.1, b=n(64, 256) * 0.1,
                taken=torch.randint(0, 64, (300,), generator=g, device='cuda'), old=n(300) * 0.1 - 4, adv=n(4),
                ptr=torch.tensor([0, 50, 180, 180, 300], device='cuda'))


def test_two_steps_at_once_on_two_streams():
    v = [_inputs(1), _inputs(2)]
    want = [_whole(x) for x in v]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    out = [[], []]
    for k in range(6):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                out[i].append(_whole(v[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for r in out[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


def test_a_whole_step_captured_and_replayed():
    v = _inputs(3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                          # what a first call sets up is set up outside the graph
        _whole(v)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _whole(v)
    for k in range(4):
        new = _inputs(10 + k)
        for name in v:
            v[name].copy_(new[name])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        assert all(torch.equal(a, b) for a, b in zip(got, _whole(v))), k


def test_a_second_backward_of_one_forward():
    import edgehip
    v = _inputs(4)
    x = torch.randn(300, 64, device='cuda', requires_grad=True)
    for loss in (edgehip.policy_loss(x, v['taken'], v['old'], v['adv'], v['ptr']).loss, edgehip.preference_loss(x, v['taken'], v['ptr']).loss):
        w = torch.arange(1.0, 1 + loss.numel(), device='cuda')
        (one,) = torch.autograd.grad(loss, x, w, retain_graph=True)
        (two,) = torch.autograd.grad(loss, x, 2 * w, retain_graph=True)
        (three,) = torch.autograd.grad(loss, x, w)
        assert torch.equal(one, three) and bool(((two - 2 * one).abs() <= 1e-6 * one.abs() + 1e-12).all())


def test_second_derivatives_are_refused():
    """The backward passes are kernels without a graph of their own: a gradient of a gradient is an error, not a wrong value."""
    import edgehip
    v = lambda *s: torch.randn(*s, device='cuda').requires_grad_(True)
    ptr = torch.tensor([0, 3, 8], device='cuda')
    taken = torch.zeros(8, dtype=torch.int64, device='cuda')
    x, z, w = v(8, 64), v(8, 64), v(64, 64)
    for out in (edgehip.gate_norm(x, z)[1], edgehip.act8(x), edgehip.linear8(x, w),
                edgehip.policy_loss(x, taken, torch.zeros(8, device='cuda'), torch.ones(2, device='cuda'), ptr).loss,
                edgehip.preference_loss(x, taken, ptr).loss):
        first, = torch.autograd.grad(out.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match='once_differentiable'):
            first.sum().backward()


def test_offsets_past_32_bits():
    """More than 2^31 values in a tensor: the last rows come out as they do in a tensor of their own, bit for bit."""
    import edgehip
    rows, dim, last = (1 << 20) + 5003, 2048, 300
    g = torch.Generator(device='cuda').manual_seed(11)
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device='cuda')
    for a in range(0, rows, 1 << 17):
        x[a:a + (1 << 17)] = torch.randn(min(1 << 17, rows - a), dim, generator=g, device='cuda')
    tail = x[-last:].clone()
    w = torch.rand(dim, generator=g, device='cuda') + 0.5
    ho, y, st = edgehip.block.gate_norm_fwd(x, x, w_pre=w, gate=w, want_stats=True)
    ho1, y1, st1 = edgehip.block.gate_norm_fwd(tail, tail, w_pre=w, gate=w, want_stats=True)
    assert torch.equal(ho[-last:], ho1) and torch.equal(y[-last:], y1) and torch.equal(st[-last:], st1)
    del ho
    b = edgehip.block.gate_norm_bwd(y, x, x, x, st, w_pre=w, gate=w)
    b1 = edgehip.block.gate_norm_bwd(y1, tail, tail, tail, st1, w_pre=w, gate=w)
    assert torch.equal(b['dh'][-last:], b1['dh']) and torch.equal(b['dz'][-last:], b1['dz'])
    del b, y
    a, p = edgehip.ckpt8.act8_fwd(x)
    a1, p1 = edgehip.ckpt8.act8_fwd(tail)
    assert torch.equal(a[-last:], a1) and torch.equal(p.codes[-last:], p1.codes) and torch.equal(p.exps[-last:], p1.exps)
    assert torch.equal(edgehip.ckpt8.act8_bwd(x, p)[-last:], edgehip.ckpt8.act8_bwd(tail, p1))
    # the weight's gradient: dY is zero but for the last rows, so only they can show
    a.zero_()
    a[-last:] = tail
    dw, db = edgehip.ckpt8.linear8_bwd_weight(a, p)
    dw1, db1 = edgehip.ckpt8.linear8_bwd_weight(tail, p1)
    # fp32 sums of 300 exact products in another order: 300 half steps of their sizes' sum
    size = tail.float().abs().t() @ p1.unpack(torch.float32).abs()
    assert bool(((dw - dw1).abs() <= 600 * 2.0 ** -24 * size).all()) and bool(((db - db1).abs() <= 600 * 2.0 ** -24 * tail.float().abs().sum(0)).all())
    del a, p, dw
    taken = torch.randint(0, dim, (rows,), generator=g, device='cuda')
    lp = edgehip.row_logp(x, taken)
    assert torch.equal(lp[-last:], edgehip.row_logp(tail, taken[-last:]))
    ptr = torch.tensor([0, rows - last, rows], device='cuda')
    adv = torch.tensor([0.0, 1.5], device='cuda')
    r = edgehip.policy_loss_grad(x, taken, lp, adv, ptr, reduce='sum')
    r1 = edgehip.policy_loss_grad(tail, taken[-last:].contiguous(), lp[-last:].contiguous(), adv[1:], torch.tensor([0, last], device='cuda'),
                                  reduce='sum', weight=torch.tensor([0.5], device='cuda'))
    assert torch.equal(r.dlogits[-last:], r1.dlogits) and not bool(r.dlogits[:last].any())

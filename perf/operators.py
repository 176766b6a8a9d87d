"""What is timed of the operators for training and tuning deep blocks: a gated residual step with the norms on either
side of it (edgehip.block), activation checkpoints in 8 bits with the backward passes that read them (edgehip.ckpt8),
and the clipped policy and paired preference losses over rows of logits (edgehip.tune).

`run` with own = False is each operator in elementary torch operations, in 32 bits; with own = True it is the calls a
user makes of this package.  `exact` is the definition in 64 bits, written apart from both."""
import math
import os
import sys

import torch

own = False

DEV = 'cuda'
T = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
BYTES = {'f32': 4, 'bf16': 2, 'f16': 2}
EPS = 1e-6
GROUP = 64                 # values of a row that share one exponent in a checkpoint
CLIP_LO, CLIP_HI = 0.2, 0.28


# ---- the cases ------------------------------------------------------------------------------------------------
def _norm(name, rows, dim, stream, branch, norm, gate, groups, train):
    return dict(name=name, op='norm', rows=rows, dim=dim, stream=stream, branch=branch, norm=norm, gate=gate, groups=groups,
                train=train)


def _act(name, rows, dim, dtype, kind):
    return dict(name=name, op='act', rows=rows, dim=dim, dtype=dtype, kind=kind)


def _linear(name, rows, out, inp, dtype):
    return dict(name=name, op='linear', rows=rows, out=out, inp=inp, dtype=dtype)


def _policy(name, rows, classes, dtype, seqs, per_row, kl, masked):
    return dict(name=name, op='policy', rows=rows, classes=classes, dtype=dtype, seqs=seqs, per_row=per_row, kl=kl, masked=masked)


def _pref(name, rows, classes, dtype, pairs, kind, masked):
    return dict(name=name, op='pref', rows=rows, classes=classes, dtype=dtype, pairs=pairs, kind=kind, masked=masked)


def listed():
    return [
        # one token through one block while serving: launch latency
        _norm('norm token', 1, 4096, 'bf16', 'bf16', 'rms', 'vector', 0, False),
        # the nodes of a 64-graph polblogs batch at this package's width, one gate row per graph: a training step
        _norm('norm nodes', 78208, 64, 'f32', 'f32', 'layer', 'group', 64, True),
        # a training step's tokens at a wide model's width
        _norm('norm tokens', 16384, 4096, 'bf16', 'bf16', 'rms', 'vector', 0, True),
        # a width no vector divides, residual stream kept in 32 bits, a gate of its own for every row
        _norm('norm odd', 5003, 1101, 'f32', 'bf16', 'layer', 'row', 0, True),
        # the hidden activations of this package's two-layer networks (64 -> 256 -> 64) over the same batch
        _act('act8 nodes', 78208, 256, 'f32', 'silu'),
        # the weight gradient of the query projection (128 -> 8 x 64) over the same batch
        _linear('linear8 nodes', 78208, 512, 128, 'f32'),
        # a small layer with sizes no tile divides
        _linear('linear8 odd', 777, 99, 130, 'f16'),
        # a wide model's square projection over a training step's tokens
        _linear('linear8 wide', 16384, 4096, 4096, 'bf16'),
        # the active pairs of 64 generated graphs, two classes each: tuning the graph sampler on a score of its graphs
        _policy('policy pairs', 1000003, 2, 'f32', 64, False, True, False),
        # generated answers of a model with a word-piece vocabulary, padding masked
        _policy('policy tokens', 8192, 32003, 'bf16', 32, True, True, True),
        # a handful of short answers over a small alphabet: latency
        _pref('preference small', 150, 1000, 'f32', 3, 'sigmoid', True),
        # chosen and rejected answers over a large vocabulary
        _pref('preference tokens', 4096, 131072, 'bf16', 8, 'sigmoid', True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(['norm', 'norm', 'act', 'linear', 'linear', 'policy', 'policy', 'pref'])
    if op == 'norm':
        dim = _log_int(rng, 8, 8192)
        rows = _log_int(rng, 1, min(131072, 16384 * 4096 // dim))
        stream, branch = rng.choice([('f32', 'f32'), ('bf16', 'bf16'), ('f16', 'f16'), ('f32', 'bf16')])
        gate = rng.choice(['none', 'vector', 'group', 'row'])
        groups = _log_int(rng, 1, min(rows, 512)) if gate == 'group' else 0
        c = _norm('', rows, dim, stream, branch, rng.choice(['rms', 'layer']), gate, groups, rng.random() < 0.75)
    elif op == 'act':
        dim = _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(131072, 16384 * 4096 // dim))
        c = _act('', rows, dim, rng.choice(['f32', 'bf16', 'f16']), rng.choice(['silu', 'mish']))
    elif op == 'linear':
        out, inp = _log_int(rng, 16, 4096), _log_int(rng, 16, 4096)
        dtype = rng.choice(['f32', 'bf16', 'f16'])
        rows = _log_int(rng, 1, 16384 if dtype == 'bf16' or out * inp < 1 << 20 else 8192)
        c = _linear('', rows, out, inp, dtype)
    else:
        classes = _log_int(rng, 2, 131072)
        rows = _log_int(rng, 8, min(1000000, 4096 * 131072 // 2 // classes))
        dtype = rng.choice(['f32', 'bf16', 'f16'])
        if op == 'policy':
            c = _policy('', rows, classes, dtype, _log_int(rng, 1, max(1, min(512, rows // 4))), rng.random() < 0.5,
                        rng.random() < 0.6, rng.random() < 0.6)
        else:
            c = _pref('', rows, classes, dtype, _log_int(rng, 1, max(1, min(128, rows // 8))), rng.choice(['sigmoid', 'square']),
                      rng.random() < 0.6)
    del c['name']
    return c


# ---- inputs -----------------------------------------------------------------------------------------------------
def _cuts(n, parts, gen, dtype):
    """[parts + 1] offsets of ragged pieces of n rows; the pieces may be empty."""
    cut = torch.randint(0, n + 1, (parts - 1,), generator=gen, device=DEV).sort().values
    return torch.cat([cut.new_zeros(1), cut, cut.new_full((1,), n)]).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed) * 7919 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEV)

    s = dict(case)
    if case['op'] == 'norm':
        n, d = case['rows'], case['dim']
        th, tz = T[case['stream']], T[case['branch']]
        loud = 1.0 + 9.0 * (torch.rand(d, generator=gen, device=DEV) < 0.01)          # a few channels far above the rest
        s['h'], s['z'] = (normal(n, d) * loud * 2).to(th), (normal(n, d) * 0.7 + 0.1).to(tz)
        s['w_pre'], s['w_post'] = 1 + 0.1 * normal(d), 1 + 0.1 * normal(d)
        layer = case['norm'] == 'layer'
        s['b_pre'], s['b_post'] = (0.1 * normal(d), 0.1 * normal(d)) if layer else (None, None)
        s['gate'], s['row_ptr'] = None, None
        if case['gate'] == 'vector':
            s['gate'] = 0.5 + 0.2 * normal(d)
        elif case['gate'] == 'group':
            s['gate'] = 0.5 + 0.2 * normal(case['groups'], d)
            s['row_ptr'] = _cuts(n, case['groups'], gen, torch.int32)
        elif case['gate'] == 'row':
            s['gate'] = (0.5 + 0.2 * normal(n, d)).to(tz)
        if case['train']:
            s['dh_out'], s['dy'] = (normal(n, d) * 0.01).to(th), (normal(n, d) * 0.01).to(tz)
        s['res_scale'] = 0.875
    elif case['op'] == 'act':
        x = normal(case['rows'], case['dim']) * 1.5
        x[torch.rand(case['rows'], generator=gen, device=DEV) < 0.02] = 0              # padded rows
        s['x'], s['dy'] = x.to(T[case['dtype']]), (normal(case['rows'], case['dim']) * 0.01).to(T[case['dtype']])
    elif case['op'] == 'linear':
        m, k = case['rows'], case['inp']
        x = normal(m, k) * (1.0 + 9.0 * (torch.rand(k, generator=gen, device=DEV) < 0.01))
        s['x'] = x.to(T[case['dtype']])
        s['dy'] = (normal(m, case['out']) * 0.01).to(T[case['dtype']])
    else:
        r, c = case['rows'], case['classes']
        logits = torch.empty(r, c, dtype=T[case['dtype']], device=DEV)
        taken = torch.empty(r, dtype=torch.int64, device=DEV)
        logp = torch.empty(r, dtype=torch.float64, device=DEV)
        step = max(1, (1 << 27) // c)
        for a in range(0, r, step):                                # in pieces: few copies of a large input at once
            x = normal(min(step, r - a), c) * 2.5
            if c >= 64:
                x[:, ::97] = float('-inf')                         # classes that may not be taken
            x = x.to(T[case['dtype']])
            logits[a:a + step] = x
            x = x.float()
            u = torch.rand(x.shape, generator=gen, device=DEV).clamp_(1e-9, 1 - 1e-7)
            t = (x - (-u.log()).log()).argmax(1)                    # drawn from the policy itself
            taken[a:a + step] = t
            x = x.double()
            logp[a:a + step] = x.gather(1, t[:, None])[:, 0] - torch.logsumexp(x, 1)
            del x, u
        s['logits'], s['taken'], s['mask'] = logits, taken, None
        seqs = case['seqs'] if case['op'] == 'policy' else 2 * case['pairs']
        s['seq_ptr'] = _cuts(r, seqs, gen, torch.int64)
        if case['masked']:
            s['mask'] = torch.rand(r, generator=gen, device=DEV) > 0.15
            logits[~s['mask'], 0] = float('nan')                   # what stands in padding must not matter
        drift = 0.2 * torch.randn(r, generator=gen, device=DEV, dtype=torch.float64)
        if case['op'] == 'policy':
            for edge in (math.log(1 - CLIP_LO), math.log(1 + CLIP_HI)):
                # a ratio on the very edge of the clip has two derivatives: none of them lies there
                drift = torch.where((drift - edge).abs() < 1e-4, drift + 3e-4, drift)
            s['old_logp'] = (logp - drift).float()
            s['advantage'] = normal(r if case['per_row'] else seqs)
        s['ref_logp'] = None
        if case['op'] == 'pref' or case['kl']:
            s['ref_logp'] = (logp + 0.1 * torch.randn(r, generator=gen, device=DEV, dtype=torch.float64)).float()
        s['kl_coef'] = 0.05 if case['op'] == 'policy' and case['kl'] else 0.0
        # 16-bit floats lose gradients as small as 1 / (sequences x their rows): their losses are summed and scaled up
        s['reduce'] = 'sum' if case['dtype'] == 'f16' and case['op'] == 'policy' else 'mean'
        s['weight'] = torch.full((case['seqs'] if case['op'] == 'policy' else case['pairs'],), 64.0, device=DEV) if case['dtype'] == 'f16' else None
        s['beta'] = 0.1
    return s


# ---- the framework's calls ---------------------------------------------------------------------------------------
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'graph-generation-edge_amd')
if PACKAGE not in sys.path:
    sys.path.append(PACKAGE)                                       # imported by the calls below only


def _own_norm(s):
    import edgehip.block as block
    kw = {k: s[k] for k in ('w_pre', 'b_pre', 'w_post', 'b_post', 'gate', 'row_ptr', 'res_scale')}
    h_out, y, stats = block.gate_norm_fwd(s['h'], s['z'], kind=s['norm'], eps=EPS, want_stats=s['train'], **kw)
    if not s['train']:
        return dict(h=h_out, y=y)
    g = block.gate_norm_bwd(s['dh_out'], s['dy'], s['h'], s['z'], stats, kind=s['norm'], eps=EPS, **kw)
    return dict(h=h_out, y=y, **g)


def _own_act(s):
    import edgehip.ckpt8 as ckpt8
    y, kept = ckpt8.act8_fwd(s['x'], s['kind'])
    return dict(y=y, dx=ckpt8.act8_bwd(s['dy'], kept, s['kind']))


def _own_linear(s):
    import edgehip.ckpt8 as ckpt8
    kept = ckpt8.pack8(s['x'])
    dw, db = ckpt8.linear8_bwd_weight(s['dy'], kept)
    return dict(dw=dw, db=db)


def _own_policy(s):
    import edgehip.tune as tune
    r = tune.policy_loss_grad(s['logits'], s['taken'], s['old_logp'], s['advantage'], s['seq_ptr'], ref_logp=s['ref_logp'],
                              mask=s['mask'], weight=s['weight'], clip=(CLIP_LO, CLIP_HI), kl_coef=s['kl_coef'],
                              reduce=s['reduce'])
    return dict(loss=r.loss, kl=r.kl, clipped=r.clipped, dlogits=r.dlogits)


def _own_pref(s):
    import edgehip.tune as tune
    r = tune.preference_loss_grad(s['logits'], s['taken'], s['seq_ptr'], ref_logp=s['ref_logp'], mask=s['mask'], beta=s['beta'],
                                  label_smoothing=0.05 if s['kind'] == 'sigmoid' else 0.0, kind=s['kind'], weight=s['weight'])
    return dict(loss=r.loss, margin=r.margin, dlogits=r.dlogits)


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _stats(x, layer):
    """(x - mean) and 1 / its size, over the last axis."""
    c = x - x.mean(1, keepdim=True) if layer else x
    return c, torch.rsqrt((c * c).mean(1, keepdim=True) + EPS)


def _owner(ptr, n):
    """The piece each row lies in."""
    return torch.searchsorted(ptr[1:].contiguous(), torch.arange(n, device=ptr.device, dtype=ptr.dtype), right=True)


def _plain_norm(s):
    layer = s['norm'] == 'layer'
    h, z = s['h'].float(), s['z'].float()
    c, r = _stats(z, layer)
    zh = c * r
    u = zh * s['w_post']
    if s['b_post'] is not None:
        u = u + s['b_post']
    gate, own_of = s['gate'], None
    if gate is None:
        g = 1.0
    elif s['row_ptr'] is not None:
        own_of = _owner(s['row_ptr'], h.shape[0])
        g = gate[own_of]
    else:
        g = gate.float()
    ho = s['res_scale'] * h + g * u
    c, rh = _stats(ho, layer)
    hh = c * rh
    y = hh * s['w_pre']
    if s['b_pre'] is not None:
        y = y + s['b_pre']
    out = dict(h=ho.to(s['h'].dtype), y=y.to(s['z'].dtype))
    if not s['train']:
        return out
    dy, dho = s['dy'].float(), s['dh_out'].float()
    t = dy * s['w_pre']
    back = t - hh * (t * hh).mean(1, keepdim=True)
    if layer:
        back = back - t.mean(1, keepdim=True)
    dho = dho + rh * back
    du = dho * g
    t = du * s['w_post']
    back = t - zh * (t * zh).mean(1, keepdim=True)
    if layer:
        back = back - t.mean(1, keepdim=True)
    out |= dict(dh=(s['res_scale'] * dho).to(s['h'].dtype), dz=(r * back).to(s['z'].dtype), dw_pre=(dy * hh).sum(0),
                dw_post=(du * zh).sum(0))
    if layer:
        out |= dict(db_pre=dy.sum(0), db_post=du.sum(0))
    if gate is not None:
        dg = dho * u
        if own_of is not None:
            dg = torch.zeros_like(gate).index_add_(0, own_of, dg)
        elif gate.dim() == 1:
            dg = dg.sum(0)
        out['dgate'] = dg.to(gate.dtype)
    return out


def _plain_pack(x):
    """What a checkpoint of x stands for: whole multiples, at most 127, of a power of two for each GROUP values of a row."""
    m, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % GROUP)).view(m, -1, GROUP)
    f, e = torch.frexp(x.abs().amax(2, keepdim=True))
    e = torch.where(f <= 127 / 128, e - 7, e - 6).clamp_min(-120)
    up, down = (((127 + v) << 23).view(torch.float32) for v in (e, -e))           # 2^e and 2^-e to the bit
    return (torch.round(x * down) * up).view(m, -1)[:, :k]


def _plain_act(s):
    x, dy = s['x'].float(), s['dy'].float()
    q = _plain_pack(s['x'])
    if s['kind'] == 'silu':
        y = x * torch.sigmoid(x)
        p = torch.sigmoid(q)
        d = p * (1 + q * (1 - p))
    else:
        y = x * torch.tanh(torch.log1p(torch.exp(-x.abs())) + x.clamp_min(0))
        t = torch.tanh(torch.log1p(torch.exp(-q.abs())) + q.clamp_min(0))
        d = t + q * (1 - t * t) * torch.sigmoid(q)
    return dict(y=y.to(s['x'].dtype), dx=(dy * d).to(s['dy'].dtype))


def _plain_linear(s):
    dy = s['dy'].float()
    return dict(dw=dy.t() @ _plain_pack(s['x']), db=dy.sum(0))


def _plain_rows(s):
    """log-probability of what each row took, its softmax, and the rows that count."""
    x = s['logits'].float()
    m = x.amax(1, keepdim=True)
    p = torch.exp(x - m)
    total = p.sum(1, keepdim=True)
    taken = s['taken'][:, None]
    logp = (x.gather(1, taken) - m).double() - total.double().log()
    p = p / total
    valid = torch.ones_like(s['taken'], dtype=torch.bool) if s['mask'] is None else s['mask']
    return logp[:, 0], p, valid


def _plain_dlogits(s, p, valid, coef):
    """coef (1 at what was taken - softmax), nothing where the row does not count."""
    coef = torch.where(valid, coef, 0.0).float()
    d = -coef[:, None] * p
    d.scatter_add_(1, s['taken'][:, None], coef[:, None])
    return torch.where(valid[:, None], d, 0.0).to(s['logits'].dtype)


def _per_seq(s, v, valid):
    run_sum = torch.cumsum(torch.where(valid, v.double(), 0.0), 0)
    upto = torch.where(s['seq_ptr'] > 0, run_sum[(s['seq_ptr'] - 1).clamp_min(0)], 0.0)
    return upto[1:] - upto[:-1]


def _plain_policy(s):
    logp, p, valid = _plain_rows(s)
    own_of = _owner(s['seq_ptr'], logp.shape[0])
    seqs = s['seq_ptr'].numel() - 1
    adv = (s['advantage'] if s['per_row'] else s['advantage'][own_of]).double()
    ratio = torch.exp(logp - s['old_logp'])
    cut = torch.where(adv > 0, ratio > 1 + CLIP_HI, (adv < 0) & (ratio < 1 - CLIP_LO))
    gain = adv * torch.where(cut, ratio.clamp(1 - CLIP_LO, 1 + CLIP_HI), ratio)
    d = torch.where(cut, 0.0, -adv * ratio)
    kl = torch.zeros_like(logp)
    if s['ref_logp'] is not None:
        gap = s['ref_logp'].double() - logp
        kl = torch.expm1(gap) - gap
        d = d - s['kl_coef'] * torch.expm1(gap)
    count = _per_seq(s, torch.ones_like(logp), valid).clamp_min(1) if s['reduce'] == 'mean' else logp.new_ones(seqs)
    weight = 1 / seqs if s['weight'] is None else s['weight'].double()
    loss = _per_seq(s, s['kl_coef'] * kl - gain, valid) / count
    return dict(loss=loss.float(), kl=(_per_seq(s, kl, valid) / count).float(),
                clipped=_per_seq(s, cut, valid).round().to(torch.int32),
                dlogits=_plain_dlogits(s, p, valid, d * (weight / count)[own_of]))


def _plain_pref(s):
    logp, p, valid = _plain_rows(s)
    own_of = _owner(s['seq_ptr'], logp.shape[0])
    pairs = s['pairs']
    total = _per_seq(s, logp - s['ref_logp'], valid)
    margin = total[:pairs] - total[pairs:]
    if s['kind'] == 'sigmoid':
        x = s['beta'] * margin
        loss = torch.log1p(torch.exp(-x.abs())) + (-x).clamp_min(0) + 0.05 * x
        d = s['beta'] * (0.05 - torch.sigmoid(-x))
    else:
        off = margin - 0.5 / s['beta']
        loss, d = off * off, 2 * off
    d = d / pairs if s['weight'] is None else d * s['weight'].double()
    d = torch.cat([d, -d])
    return dict(loss=loss.float(), margin=margin.float(), dlogits=_plain_dlogits(s, p, valid, d[own_of]))


PLAIN = dict(norm=_plain_norm, act=_plain_act, linear=_plain_linear, policy=_plain_policy, pref=_plain_pref)
OWN = dict(norm=_own_norm, act=_own_act, linear=_own_linear, policy=_own_policy, pref=_own_pref)


def run(state):
    return (OWN if own else PLAIN)[state['op']](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def work(case):
    if case['op'] == 'norm':
        n, d = case['rows'], case['dim']
        bh, bz = BYTES[case['stream']], BYTES[case['branch']]
        passes = 2 if case['train'] else 1
        params = d * 4 * (4 if case['norm'] == 'layer' else 2)
        gate = {'none': 0, 'vector': 4 * d, 'group': 4 * d * case['groups'], 'row': bz * n * d}[case['gate']]
        # in: h, z (and the gradients of both outputs); out: both outputs (and the gradients of both inputs)
        return dict(bytes=passes * (2 * n * d * (bh + bz) + params + gate), flops=(40 if case['train'] else 14) * n * d)
    if case['op'] == 'act':
        n = case['rows'] * case['dim']
        return dict(bytes=4 * n * BYTES[case['dtype']], flops=30 * n)
    if case['op'] == 'linear':
        m, n, k, b = case['rows'], case['out'], case['inp'], BYTES[case['dtype']]
        return dict(bytes=m * (n + k) * b + 4 * n * (k + 1), flops=2 * m * n * k)
    r, c, b = case['rows'], case['classes'], BYTES[case['dtype']]
    return dict(bytes=2 * r * c * b + r * 20, flops=8 * r * c)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _norm64(x, w, b, layer):
    if layer:
        mean = x.mean(1, keepdim=True)
        hat = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + EPS)
    else:
        hat = x / torch.sqrt((x ** 2).mean(1, keepdim=True) + EPS)
    return hat * w + b if b is not None else hat * w


def _exact_norm(s):
    """The step's own formula under automatic differentiation in 64 bits."""
    names = [k for k in ('h', 'z', 'w_pre', 'w_post', 'b_pre', 'b_post', 'gate') if s[k] is not None]
    with torch.enable_grad():
        v = {k: s[k].double().requires_grad_(s['train']) for k in names}
        gate = v.get('gate', torch.ones((), dtype=torch.float64, device=DEV))
        if s['row_ptr'] is not None:
            gate = torch.repeat_interleave(gate, (s['row_ptr'][1:] - s['row_ptr'][:-1]).long(), dim=0)
        layer = s['norm'] == 'layer'
        ho = s['res_scale'] * v['h'] + gate * _norm64(v['z'], v['w_post'], v.get('b_post'), layer)
        y = _norm64(ho, v['w_pre'], v.get('b_pre'), layer)
        if not s['train']:
            return dict(h=ho, y=y)
        grads = torch.autograd.grad([ho, y], [v[k] for k in names], [s['dh_out'].double(), s['dy'].double()])
    return dict(h=ho.detach(), y=y.detach(), **{'d' + k: g for k, g in zip(names, grads)})


def _pack64(x):
    m, k = x.shape
    out = torch.zeros(m, -(-k // GROUP) * GROUP, dtype=torch.float64, device=DEV)
    out[:, :k] = x.double()
    out = out.view(m, -1, GROUP)
    top = out.abs().amax(2, keepdim=True)
    steps = torch.tensor([math.ldexp(1.0, i) for i in range(-120, 123)], dtype=torch.float64, device=DEV)
    step = steps[torch.searchsorted(127 * steps, top.contiguous())]              # the smallest with top <= 127 steps
    return (torch.round(out / step) * step).view(m, -1)[:, :k]


def _exact_act(s):
    f = torch.nn.functional.silu if s['kind'] == 'silu' else torch.nn.functional.mish
    with torch.enable_grad():
        q = _pack64(s['x']).requires_grad_(True)
        (dx,) = torch.autograd.grad(f(q), q, s['dy'].double())
    return dict(y=f(s['x'].double()), dx=dx)


def _exact_linear(s):
    dy = s['dy'].double()
    return dict(dw=torch.matmul(dy.t().contiguous(), _pack64(s['x'])), db=dy.sum(0))


def _exact_rows(s, per_row_loss):
    """Sequence by sequence: the loss of its rows from their log-probabilities, and the gradient by hand of the softmax."""
    ptr = s['seq_ptr'].tolist()
    keep = torch.ones_like(s['taken'], dtype=torch.bool) if s['mask'] is None else s['mask']
    logp = torch.zeros(s['rows'], dtype=torch.float64, device=DEV)
    step = max(1, (1 << 26) // s['classes'])
    for a in range(0, s['rows'], step):
        x = s['logits'][a:a + step].double()
        logp[a:a + step] = x.gather(1, s['taken'][a:a + step, None])[:, 0] - torch.logsumexp(x, 1)
    logp = torch.where(keep, logp, 0.0)
    with torch.enable_grad():
        leaf = logp.requires_grad_(True)
        out, total = per_row_loss(leaf, keep, ptr)
        (g,) = torch.autograd.grad(total, leaf)
    if s['rows'] * s['classes'] > 1 << 28:
        out['dlogits'] = torch.empty(s['rows'], s['classes'], dtype=torch.float32, device=DEV)
    else:
        out['dlogits'] = torch.empty(s['rows'], s['classes'], dtype=torch.float64, device=DEV)
    for a in range(0, s['rows'], step):
        x = s['logits'][a:a + step].double()
        d = torch.softmax(x, 1).neg_()
        t = s['taken'][a:a + step, None]
        d.scatter_add_(1, t, torch.ones_like(t, dtype=torch.float64))
        d *= g[a:a + step, None]
        d[~keep[a:a + step]] = 0
        out['dlogits'][a:a + step] = d
    return out


def _weighed(s, each):
    return each.mean() if s['weight'] is None else (each * s['weight'].double()).sum()


def _exact_policy(s):
    def loss(logp, keep, ptr):
        seqs = len(ptr) - 1
        owner = torch.repeat_interleave(torch.arange(seqs, device=DEV), s['seq_ptr'][1:] - s['seq_ptr'][:-1])
        adv = (s['advantage'] if s['per_row'] else s['advantage'][owner]).double()
        ratio = torch.exp(logp - s['old_logp'].double())
        bounded = torch.clamp(ratio, 1 - CLIP_LO, 1 + CLIP_HI)
        gain = torch.minimum(ratio * adv, bounded * adv)
        kl = torch.zeros_like(gain)
        if s['ref_logp'] is not None:
            gap = s['ref_logp'].double() - logp
            kl = torch.exp(gap) - gap - 1
        w = keep.double()
        n = torch.zeros(seqs, dtype=torch.float64, device=DEV).index_add(0, owner, w).clamp_min(1)
        if s['reduce'] == 'sum':
            n = torch.ones_like(n)
        sums = [torch.zeros(seqs, dtype=torch.float64, device=DEV).index_add(0, owner, torch.where(keep, v, 0.0)) / n
                for v in (s['kl_coef'] * kl - gain, kl)]
        return dict(loss=sums[0].detach(), kl=sums[1].detach(), clipped=None), _weighed(s, sums[0])
    return _exact_rows(s, loss)


def _exact_pref(s):
    def loss(logp, keep, ptr):
        v = torch.where(keep, logp - s['ref_logp'].double(), 0.0)
        sums = torch.stack([v[a:b].sum() for a, b in zip(ptr[:-1], ptr[1:])])
        margin = sums[:s['pairs']] - sums[s['pairs']:]
        if s['kind'] == 'sigmoid':
            f = torch.nn.functional.logsigmoid
            each = -0.95 * f(s['beta'] * margin) - 0.05 * f(-s['beta'] * margin)
        else:
            each = (margin - 1 / (2 * s['beta'])) ** 2
        return dict(loss=each.detach(), margin=margin.detach()), _weighed(s, each)
    return _exact_rows(s, loss)


EXACT = dict(norm=_exact_norm, act=_exact_act, linear=_exact_linear, policy=_exact_policy, pref=_exact_pref)


def exact(case, seed):
    with torch.no_grad():
        return EXACT[case['op']](prepare(case, seed))

"""What is measured of the sequence layer with a selective state and of the losses that train a generator from rewards.

The two belong to one loop: a generator of token sequences samples with the single-token forms, and is trained with the
forms for whole packed batches, through the log-probabilities of the tokens that it took.

  causal_conv       y_t = act(b + sum_k w_k x_{t-K+1+k}), a channel at a time, over packed or rectangular batches
  selective_scan    h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t,  y_t = (C_t . h_t + D x_t) silu(z_t)
  token_log_probs   log softmax(logits / temperature) at the token that was taken
  policy_loss       clipped ratio times advantage, with a KL term towards a reference

`run` computes the plain forms in elementary torch operations, or, with `own`, calls the framework's operators.
"""
import math

import torch

own = False

DEVICE = 'cuda'
TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases
def _conv(name, mode, dtype, layout, B, lo, hi, D, K):
    return dict(name=name, op='conv', mode=mode, dtype=dtype, layout=layout, B=B, lo=lo, hi=hi, D=D, K=K)


def _scan(name, mode, dtype, layout, B, lo, hi, D, N, G, gate):
    return dict(name=name, op='scan', mode=mode, dtype=dtype, layout=layout, B=B, lo=lo, hi=hi, D=D, N=N, G=G, gate=gate)


def _loss(name, op, mode, dtype, rows, V):
    return dict(name=name, op=op, mode=mode, dtype=dtype, rows=rows, V=V)


def listed():
    return [
        # the training batch of this repository's benchmark: 2048 token sequences of 20 to 100, 512 units
        _conv('conv_train_packed', 'train', 'f32', 'packed', 2048, 20, 100, 512, 4),
        # one long prompt read by a server, batch first, the last inputs of the chunk before it as the state
        _conv('conv_prompt_long', 'infer', 'bf16', 'rect', 1, 16384, 16384, 4096, 4),
        # one token for each of 64 requests
        _conv('conv_step', 'step', 'bf16', 'step', 64, 1, 1, 1024, 4),
        # the training batch of the benchmark
        _scan('scan_train_packed', 'train', 'f32', 'packed', 2048, 20, 100, 512, 16, 1, True),
        # training on one long document in 16 bits
        _scan('scan_train_long', 'train', 'bf16', 'rect', 1, 16384, 16384, 2048, 16, 1, True),
        # one bundle of at most 21 sequences, as the reference trains on, with sizes that divide nothing
        _scan('scan_train_bundle_odd', 'train', 'f32', 'packed', 21, 1, 100, 333, 11, 3, False),
        # one prompt of ordinary length, one user
        _scan('scan_prompt', 'infer', 'bf16', 'rect', 1, 2048, 2048, 1024, 16, 1, True),
        # one token for each of 256 requests
        _scan('scan_step', 'step', 'bf16', 'step', 256, 1, 1, 2048, 16, 1, True),
        # scores of the benchmark's batch under a frozen model, with the vocabulary of the pretrained language
        _loss('logp_score', 'logp', 'infer', 'f32', 122880, 575),
        # their gradient, with a vocabulary of a general tokenizer
        _loss('logp_train', 'logp', 'train', 'bf16', 4096, 32000),
        # one policy step on the benchmark's batch
        _loss('policy_train', 'policy', 'train', 'f32', 122880, 575),
        # one policy step on one bundle, with the benchmark's vocabulary: what a launch costs counts here
        _loss('policy_train_bundle', 'policy', 'train', 'f32', 1260, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['conv', 'conv', 'scan', 'scan', 'scan', 'logp', 'policy', 'policy'])
    dtype = rng.choice(['f32', 'bf16'])
    while True:
        if kind in ('conv', 'scan'):
            layout = rng.choice(['packed', 'packed', 'rect', 'step'])
            mode = 'step' if layout == 'step' else rng.choice(['train', 'train', 'infer'])
            B = _log(rng, 1, 2048)
            hi = 1 if layout == 'step' else _log(rng, 1, 16384 if B < 8 else 256)
            lo = hi if layout != 'packed' else _log(rng, 1, hi)
            D = _log(rng, 16, 4096)
            cost = B * (lo + hi) / 2 * D
            if kind == 'conv':
                if cost <= 2048 * 60 * 512:
                    return _conv('', mode, dtype, layout, B, lo, hi, D, rng.choice([2, 3, 4, 4, 4]))
            else:
                N = rng.choice([16, 16, 16, rng.randint(1, 32), 64])
                G = rng.choice([g for g in (1, 1, 2, 3, 8) if D % g == 0])
                if cost * N <= 2048 * 60 * 512 * 16 and B * hi * D * N <= 2048 * 100 * 512 * 16:
                    return _scan('', mode, dtype, layout, B, lo, hi, D, N, G, rng.random() < 0.7)
        else:
            rows, V = _log(rng, 1, 200000), _log(rng, 2, 131072)
            if rows * V <= 122880 * 575:
                mode = rng.choice(['train', 'train', 'infer'])
                return _loss('', kind, mode, dtype, rows, V)


# --------------------------------------------------------------------------------------------------------------- inputs
def _lengths(case):
    """The lengths belong to the case, as every other size does."""
    g = torch.Generator().manual_seed(case['B'] * 65537 + case['hi'])
    n = torch.randint(case['lo'], case['hi'] + 1, (case['B'],), generator=g)
    if case['layout'] == 'packed' and case['B'] > 1:
        n[0], n[-1] = case['hi'], case['lo']
    return torch.sort(n, descending=True).values


def _rows(case, s):
    """The shape of the leading dimensions of a batch, and what a program keeps of its packing."""
    if case['layout'] == 'step':
        return (case['B'],)
    if case['layout'] == 'rect':
        return (case['B'], case['hi'])
    n = _lengths(case)
    bs = (n.view(1, -1) > torch.arange(int(n[0])).view(-1, 1)).sum(1)
    s['batch_sizes'] = bs
    off = torch.cumsum(bs, 0) - bs
    live = torch.arange(case['B']).view(1, -1) < bs.view(-1, 1)
    s['live'] = live.to(DEVICE)                                                            # [T, B]: whether sequence b has a step t
    s['row_of'] = torch.where(live, off.view(-1, 1) + torch.arange(case['B']), 0).to(DEVICE)    # ... and which row it is
    s['t_of'], s['b_of'] = (i.to(DEVICE) for i in live.nonzero(as_tuple=True))
    if own:
        from paccmann_polymer_amd import state_space
        s['plan'] = state_space.packed_rows(bs, DEVICE)
    return (int(bs.sum()),)


def _step_view(t, case):
    """Batch-first rectangular tensors are handed over as [T, B, ...] views, as nn.GRU takes them."""
    return t.transpose(0, 1) if case['layout'] == 'rect' else t


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dt_ = TYPES[case['dtype']]
    s = dict(case=case)

    def normal(*shape, scale=1.0, dtype=dt_):
        return (torch.randn(*shape, generator=g, device=DEVICE) * scale).to(dtype)

    if case['op'] == 'conv':
        B, D, K = case['B'], case['D'], case['K']
        lead = _rows(case, s)
        s['x'] = _step_view(normal(*lead, 2 * D)[..., :D], case)            # half of a projection's output, as in use
        s['weight'] = normal(D, K, scale=1 / math.sqrt(K), dtype=torch.float32)
        s['bias'] = normal(D, scale=0.1, dtype=torch.float32)
        s['state'] = normal(B, K - 1, D)
        if case['mode'] == 'train':
            s['dy'] = _step_view(normal(*lead, D), case)
            s['dstate'] = normal(B, K - 1, D)
    elif case['op'] == 'scan':
        B, D, N, G = case['B'], case['D'], case['N'], case['G']
        lead = _rows(case, s)
        xz = normal(*lead, 2 * D)
        s['x'], s['z'] = _step_view(xz[..., :D], case), _step_view(xz[..., D:], case) if case['gate'] else None
        s['dt'] = _step_view(normal(*lead, D, scale=0.5), case)
        bc = normal(*lead, 2, G, N)
        s['B'], s['C'] = _step_view(bc[..., 0, :, :], case), _step_view(bc[..., 1, :, :], case)
        s['A'] = -torch.arange(1, N + 1, device=DEVICE, dtype=torch.float32) * torch.exp(normal(D, N, scale=0.1, dtype=torch.float32))
        s['D'] = 1 + normal(D, scale=0.1, dtype=torch.float32)
        step = torch.exp(torch.rand(D, generator=g, device=DEVICE) * math.log(100.0) + math.log(1e-3))       # 1e-3 to 0.1
        s['dt_bias'] = step + torch.log(-torch.expm1(-step))                                                 # softplus(dt_bias) = step
        s['state'] = normal(B, D, N, dtype=torch.float32)
        if case['mode'] == 'train':
            s['dy'] = _step_view(normal(*lead, D), case)
            s['dstate'] = normal(B, D, N, dtype=torch.float32)
    else:
        rows, V = case['rows'], case['V']
        logits = torch.randn(rows, V, generator=g, device=DEVICE) * 2
        tok = torch.randint(1, V, (rows,), generator=g, device=DEVICE) if V > 1 else torch.zeros(rows, dtype=torch.int64, device=DEVICE)
        logits[torch.arange(rows, device=DEVICE), tok] += 4                                    # a model gives the tokens that it took weight
        s['logits'] = logits.to(dt_)
        tok[torch.rand(rows, generator=g, device=DEVICE) < 1 / 60] = 0                         # a sequence's last target is padding
        tok[0] = 1
        s['targets'] = tok
        s['temperature'] = 1.0
        if case['op'] == 'logp':
            if case['mode'] == 'train':
                s['dlogp'] = normal(rows, dtype=torch.float32)
        else:
            lo, hi, s['kl_coef'] = 0.2, 0.28, 0.05
            s['clip_low'], s['clip_high'] = lo, hi
            lp = _log_probs64(s['logits'], tok)
            ratio = 0.15 * torch.randn(rows, generator=g, device=DEVICE, dtype=torch.float64)
            # a ratio on a border has no gradient to compare: none is within 1e-3 of one
            for edge in (math.log(1 - lo), math.log(1 + hi)):
                ratio = torch.where((ratio - edge).abs() < 1e-3, ratio + 3e-3, ratio)
            s['old'] = (lp - ratio).float()
            s['ref'] = (lp + 0.2 * torch.randn(rows, generator=g, device=DEVICE, dtype=torch.float64)).float()
            seqs = max(1, rows // 60)                                                          # one advantage for all tokens of a sequence
            adv = torch.randn(seqs, generator=g, device=DEVICE)
            s['advantages'] = adv[torch.randint(0, seqs, (rows,), generator=g, device=DEVICE)]
    return s


def _log_probs64(logits, tok):
    out = []
    for part, t in zip(logits.split(8192), tok.split(8192)):
        v = part.double()
        out.append(v.gather(1, t[:, None])[:, 0] - torch.logsumexp(v, 1))
    return torch.cat(out)


# ---------------------------------------------------------------------------------------------------------- plain forms
def _spread(s, t):
    """[T, B, ...] of a tensor of rows, in 32 bits; zeros where a sequence has no such step."""
    t = t.float()
    if s['case']['layout'] == 'packed':
        live = s['live'].view(*s['live'].shape, *([1] * (t.dim() - 1)))
        t = torch.where(live, t[s['row_of']], torch.zeros((), device=t.device))
    return t


def _gather(s, t, dtype):
    if s['case']['layout'] == 'packed':
        t = t[s['t_of'], s['b_of']]
    return t.to(dtype)


def _ends(s, B):
    """How many steps each sequence has."""
    if s['case']['layout'] == 'packed':
        return s['live'].sum(0)
    return torch.full((B,), s['case']['hi'], device=DEVICE)


def _conv_plain(s):
    case, w = s['case'], s['weight']
    K, dtype = case['K'], s['x'].dtype
    if case['mode'] == 'step':
        line = torch.cat([s['state'].float(), s['x'].float()[:, None]], 1)                     # [B, K, D]
        pre = (line * w.t()).sum(1) + s['bias']
        return (pre * torch.sigmoid(pre)).to(dtype), line[:, 1:].to(dtype)
    x = _spread(s, s['x'])                                                                     # [T, B, D]
    T, B, D = x.shape
    line = torch.cat([s['state'].float().transpose(0, 1), x])                                  # [K - 1 + T, B, D]
    pre = s['bias'] + sum(line[k:k + T] * w[:, k] for k in range(K))
    sig = torch.sigmoid(pre)
    y = _gather(s, pre * sig, dtype)
    at = _ends(s, B) + torch.arange(K - 1, device=DEVICE)[:, None]                             # [K - 1, B]: the last K - 1 inputs of each
    b = torch.arange(B, device=DEVICE)
    last = line[at, b].transpose(0, 1).to(dtype)
    if case['mode'] != 'train':
        return y, last
    dpre = _spread(s, s['dy']) * sig * (1 + pre * (1 - sig))
    dline = torch.zeros_like(line)
    for k in range(K):
        dline[k:k + T] += dpre * w[:, k]
    dline[at, b] += s['dstate'].float().transpose(0, 1)
    dw = torch.stack([(dpre * line[k:k + T]).sum((0, 1)) for k in range(K)], 1)
    return y, last, _gather(s, dline[K - 1:], dtype), dw, dpre.sum((0, 1)), dline[:K - 1].transpose(0, 1).to(dtype)


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t along the first dimension, by doubling."""
    k = 1
    while k < a.shape[0]:
        b = torch.cat([b[:k], b[k:] + a[k:] * b[:-k]])
        a = torch.cat([a[:k], a[k:] * a[:-k]])
        k *= 2
    return b


def _scan_plain(s):
    case, dtype = s['case'], s['x'].dtype
    D, N, G = case['D'], case['N'], case['G']
    A, per = s['A'], D // case['G']

    def heads(t):                                      # [..., G, N] -> [..., D, N]: the channels of a group share its vectors
        return t.repeat_interleave(per, -2)

    if case['mode'] == 'step':
        x, raw = s['x'].float(), s['dt'].float() + s['dt_bias']
        dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw)))
        h = torch.exp(dt[..., None] * A) * s['state'] + (dt * x)[..., None] * heads(s['B'].float())
        y = (h * heads(s['C'].float())).sum(-1) + s['D'] * x
        if case['gate']:
            z = s['z'].float()
            y = y * z * torch.sigmoid(z)
        return y.to(dtype), h
    x, raw = _spread(s, s['x']), _spread(s, s['dt']) + s['dt_bias']
    dt = torch.where(raw > 20, raw, torch.log1p(torch.exp(raw)))
    if case['layout'] == 'packed':
        dt = dt * s['live'][..., None]                 # a step that a sequence does not have leaves its state alone
    Bm, Cm = heads(_spread(s, s['B'])), heads(_spread(s, s['C']))
    a = torch.exp(dt[..., None] * A)
    b = (dt * x)[..., None] * Bm
    b[0] += a[0] * s['state']
    h = _recur(a, b)
    del b
    y = (h * Cm).sum(-1) + s['D'] * x
    if case['gate']:
        z = _spread(s, s['z'])
        sig = torch.sigmoid(z)
        out = y * z * sig
    else:
        out = y
    if case['mode'] != 'train':
        return _gather(s, out, dtype), h[-1].clone()
    last = h[-1].clone()
    dout = _spread(s, s['dy'])
    dy = dout * z * sig if case['gate'] else dout
    b = dy[..., None] * Cm
    b[-1] += s['dstate']
    dh = _recur(torch.cat([torch.ones_like(a[:1]), a[1:].flip(0)]), b.flip(0)).flip(0)
    del b
    T, B = x.shape[:2]
    dCm = _gather(s, (dy[..., None] * h).view(T, B, G, per, N).sum(3), dtype)
    dBm = _gather(s, (dh * (dt * x)[..., None]).view(T, B, G, per, N).sum(3), dtype)
    through = (dh * Bm).sum(-1)
    dstate = a[0] * dh[0]
    da = dh * a * torch.cat([s['state'][None], h[:-1]])
    dA = (da * dt[..., None]).sum((0, 1))
    ddt = (da * A).sum(-1) + through * x
    draw = ddt * torch.sigmoid(raw)
    if case['layout'] == 'packed':
        draw = draw * s['live'][..., None]
    dx = through * dt + s['D'] * dy
    grads = [_gather(s, dx, dtype), _gather(s, draw, dtype), dA, dBm, dCm, (dy * x).sum((0, 1)), draw.sum((0, 1)), dstate]
    if case['gate']:
        grads.append(_gather(s, dout * y * sig * (1 + z * (1 - sig)), dtype))
    return (_gather(s, out, dtype), last, *grads)


def _softmax_plain(s):
    v = s['logits'].float() / s['temperature']
    v = v - v.max(1, keepdim=True).values
    e = torch.exp(v)
    total = e.sum(1, keepdim=True)
    taken = v.gather(1, s['targets'][:, None])[:, 0].double() - torch.log(total[:, 0].double())
    return e / total, taken, s['targets'] != 0


def _logits_grad(s, p, g, use):
    """g (onehot - p) / temperature, and zeros for the rows that do not count."""
    g = (torch.where(use, g, torch.zeros_like(g)) / s['temperature'])[:, None]
    d = -p * g
    d.scatter_add_(1, s['targets'][:, None], g)
    return d.to(s['logits'].dtype)


def _logp_plain(s):
    p, taken, use = _softmax_plain(s)
    logp = torch.where(use, taken, 0.0).float()
    if s['case']['mode'] != 'train':
        return logp
    return logp, _logits_grad(s, p, s['dlogp'], use)


def _policy_plain(s):
    """The terms of a row in 64 bits: exp(d) - d - 1 loses all of a small d in 32."""
    p, lp, use = _softmax_plain(s)
    zero = torch.zeros_like(lp)
    adv = s['advantages'].double()
    ratio = torch.exp(torch.where(use, lp - s['old'].double(), zero))
    low, high = 1 - s['clip_low'], 1 + s['clip_high']
    free, held = ratio * adv, ratio.clamp(low, high) * adv
    d = torch.where(use, s['ref'].double() - lp, zero)
    kl = torch.exp(d) - d - 1
    n = use.sum().clamp(min=1)
    pg = torch.where(use, -torch.minimum(free, held), zero)
    stats = torch.stack([pg.sum() / n, kl.sum() / n, (use & (held < free)).sum() / n]).float()
    loss = ((pg + s['kl_coef'] * kl).sum() / n).float()
    if s['case']['mode'] != 'train':
        return loss, stats
    g = torch.where(free <= held, -free, zero) + s['kl_coef'] * (1 - torch.exp(d))
    return loss, stats, _logits_grad(s, p, (g / n).float(), use)


# ------------------------------------------------------------------------------------------------------------------ run
def _leaf(t):
    return None if t is None else t.detach().requires_grad_()


def _conv_own(s):
    from paccmann_polymer_amd import state_space as S
    case = s['case']
    if case['mode'] == 'step':
        return S.causal_conv_step(s['x'], s['state'], s['weight'], s['bias'], activation='silu')
    if case['mode'] == 'infer':
        return S.causal_conv(s['x'], s['weight'], s['bias'], plan=s.get('plan'), state=s['state'], activation='silu')
    leaves = [_leaf(s[k]) for k in ('x', 'weight', 'bias', 'state')]
    x, w, b, st = leaves
    y, last = S.causal_conv(x, w, b, plan=s.get('plan'), state=st, activation='silu')
    return (y, last, *torch.autograd.grad((y, last), leaves, (s['dy'], s['dstate'])))


def _scan_own(s):
    from paccmann_polymer_amd import state_space as S
    case = s['case']
    if case['mode'] == 'step':
        return S.selective_scan_step(s['x'], s['dt'], s['A'], s['B'], s['C'], s['state'], D=s['D'], z=s['z'], dt_bias=s['dt_bias'])
    if case['mode'] == 'infer':
        return S.selective_scan(s['x'], s['dt'], s['A'], s['B'], s['C'], D=s['D'], z=s['z'], dt_bias=s['dt_bias'], plan=s.get('plan'), state=s['state'])
    x, dt, A, B, C, D, bias, st, z = leaves = [_leaf(s[k]) for k in ('x', 'dt', 'A', 'B', 'C', 'D', 'dt_bias', 'state', 'z')]
    y, last = S.selective_scan(x, dt, A, B, C, D=D, z=z, dt_bias=bias, plan=s.get('plan'), state=st)
    return (y, last, *torch.autograd.grad((y, last), [t for t in leaves if t is not None], (s['dy'], s['dstate'])))


def _logp_own(s):
    from paccmann_polymer_amd import policy_loss as P
    if s['case']['mode'] == 'infer':
        return P.token_log_probs(s['logits'], s['targets'], ignore_index=0, temperature=s['temperature'])
    logits = _leaf(s['logits'])
    logp = P.token_log_probs(logits, s['targets'], ignore_index=0, temperature=s['temperature'])
    return (logp, *torch.autograd.grad(logp, logits, s['dlogp']))


def _policy_own(s):
    from paccmann_polymer_amd import policy_loss as P
    train = s['case']['mode'] == 'train'
    logits = _leaf(s['logits']) if train else s['logits']
    loss, stats = P.policy_loss(logits, s['targets'], s['old'], s['advantages'], ref_log_probs=s['ref'], clip_low=s['clip_low'],
                                clip_high=s['clip_high'], kl_coef=s['kl_coef'], ignore_index=0, temperature=s['temperature'])
    return (loss, stats, *torch.autograd.grad(loss, logits)) if train else (loss, stats)


def run(state):
    op = state['case']['op']
    if own:
        return {'conv': _conv_own, 'scan': _scan_own, 'logp': _logp_own, 'policy': _policy_own}[op](state)
    return {'conv': _conv_plain, 'scan': _scan_plain, 'logp': _logp_plain, 'policy': _policy_plain}[op](state)


# ----------------------------------------------------------------------------------------------------------------- work
def work(case):
    e = 2 if case['dtype'] == 'bf16' else 4
    train = case['mode'] == 'train'
    if case['op'] in ('conv', 'scan'):
        if case['layout'] == 'packed':
            rows = case['B'] * (case['lo'] + case['hi']) / 2
        else:
            rows = case['B'] * case['hi']
        cells = rows * case['D']
        if case['op'] == 'conv':
            held = case['B'] * (case['K'] - 1) * case['D'] * e
            # x and y; dy and dx; the states before and after, and their gradients
            return dict(bytes=cells * e * (4 if train else 2) + held * (4 if train else 2) + case['D'] * (case['K'] + 1) * 4 * (2 if train else 1),
                        flops=cells * (2 * case['K'] + 6) * (3 if train else 1))
        N, G = case['N'], case['G']
        held, fixed = case['B'] * case['D'] * N * 4, case['D'] * (N + 2) * 4
        wide = 3 + case['gate']                              # x, dt, y and z
        # training: those, dy, and the gradients of x, dt and z; B and C, and their gradients
        return dict(bytes=cells * e * ((2 * wide) if train else wide) + rows * 2 * G * N * e * (2 if train else 1) + (held * 2 + fixed) * (2 if train else 1),
                    flops=cells * N * (24 if train else 8))
    cells = case['rows'] * case['V']
    small = case['rows'] * (8 + 4 * (3 if case['op'] == 'policy' else 2 if train else 1))
    return dict(bytes=cells * e * (2 if train else 1) + small, flops=cells * (6 if train else 4))


# ---------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'conv': _conv_exact, 'scan': _scan_exact, 'logp': _logp_exact, 'policy': _policy_exact}[case['op']](case, s)


def _walk(case, s):
    """The rows of each time step, and how a tensor of rows is read and written, in 64 bits: the definitions go step by step."""
    if case['layout'] == 'packed':
        bs = s['batch_sizes'].tolist()
        off = [0]
        for n in bs:
            off.append(off[-1] + n)
        return bs, lambda t, i: t[off[i]:off[i + 1]], lambda parts: torch.cat(parts)
    if case['layout'] == 'step':
        return [case['B']], lambda t, i: t, lambda parts: parts[0]
    return [case['B']] * case['hi'], lambda t, i: t[i], lambda parts: torch.stack(parts)


def _conv_exact(case, s):
    bs, at, join = _walk(case, s)
    K, w, bias = case['K'], s['weight'].double(), s['bias'].double()
    x = s['x'].double()
    line = s['state'].double()                                  # [B, K - 1, D], the oldest first
    lines, pres, ys = [], [], []
    for t, n in enumerate(bs):
        full = torch.cat([line[:n], at(x, t).unsqueeze(1)], 1)
        line = torch.cat([full[:, 1:], line[n:]])
        pre = torch.einsum('bkd,dk->bd', full, w) + bias
        lines.append(full)
        pres.append(pre)
        ys.append(pre / (1 + torch.exp(-pre)))
    if case['mode'] != 'train':
        return join(ys), line
    dline = s['dstate'].double()
    dw, db = torch.zeros_like(w), torch.zeros_like(bias)
    dxs, dy = [None] * len(bs), s['dy'].double()
    for t in reversed(range(len(bs))):
        n, sig = bs[t], 1 / (1 + torch.exp(-pres[t]))
        dpre = at(dy, t) * (sig + pres[t] * sig * (1 - sig))
        dfull = torch.einsum('bd,dk->bkd', dpre, w)
        dfull[:, 1:] += dline[:n]
        dw += torch.einsum('bd,bkd->dk', dpre, lines[t])
        db += dpre.sum(0)
        dxs[t] = dfull[:, -1]
        dline = torch.cat([dfull[:, :-1], dline[n:]])
    return join(ys), line, join(dxs), dw, db, dline


def _scan_exact(case, s):
    bs, at, join = _walk(case, s)
    D, N, G = case['D'], case['N'], case['G']
    A, skip, bias = s['A'].double(), s['D'].double(), s['dt_bias'].double()
    group = torch.arange(D, device=DEVICE) // (D // G)
    x, raw, z = s['x'], s['dt'], s['z']
    h = s['state'].double().clone()
    seen, ys = [], []
    for t, n in enumerate(bs):
        xt, rt = at(x, t).double(), at(raw, t).double() + bias
        dt = torch.logaddexp(rt, torch.zeros((), dtype=torch.float64, device=DEVICE))
        if case['mode'] == 'train':
            seen.append(h[:n].clone())
        h[:n] = torch.exp(dt[:, :, None] * A) * h[:n] + (dt * xt)[:, :, None] * at(s['B'], t).double()[:, group]
        y = torch.einsum('bdn,bdn->bd', h[:n], at(s['C'], t).double()[:, group]) + skip * xt
        if case['gate']:
            zt = at(z, t).double()
            y = y * zt / (1 + torch.exp(-zt))
        ys.append(y)
    if case['mode'] != 'train':
        return join(ys), h
    last, dh = h, s['dstate'].double().clone()
    T = len(bs)
    dxs, draws, dBs, dCs, dzs = ([None] * T for _ in range(5))
    dA, dD, dbias = torch.zeros_like(A), torch.zeros_like(skip), torch.zeros_like(bias)
    for t in reversed(range(T)):
        n, xt, rt = bs[t], at(x, t).double(), at(raw, t).double() + bias
        dt = torch.logaddexp(rt, torch.zeros((), dtype=torch.float64, device=DEVICE))
        Bt, Ct = at(s['B'], t).double()[:, group], at(s['C'], t).double()[:, group]
        a = torch.exp(dt[:, :, None] * A)
        now = a * seen[t] + (dt * xt)[:, :, None] * Bt
        dy = at(s['dy'], t).double()
        if case['gate']:
            zt = at(z, t).double()
            sig = 1 / (1 + torch.exp(-zt))
            pre = torch.einsum('bdn,bdn->bd', now, Ct) + skip * xt
            dzs[t] = dy * pre * (sig + zt * sig * (1 - sig))
            dy = dy * zt * sig
        dht = dh[:n] + dy[:, :, None] * Ct
        zero = torch.zeros(n, G, N, dtype=torch.float64, device=DEVICE)
        dCs[t] = zero.index_add(1, group, dy[:, :, None] * now)
        dBs[t] = zero.index_add(1, group, dht * (dt * xt)[:, :, None])
        through = torch.einsum('bdn,bdn->bd', dht, Bt)
        da = dht * seen[t] * a
        dA += (da * dt[:, :, None]).sum(0)
        ddt = torch.einsum('bdn,dn->bd', da, A) + through * xt
        draws[t] = ddt / (1 + torch.exp(-rt))
        dbias += draws[t].sum(0)
        dD += (dy * xt).sum(0)
        dxs[t] = through * dt + skip * dy
        dh[:n] = a * dht
    grads = [join(dxs), join(draws), dA, join(dBs), join(dCs), dD, dbias, dh]
    if case['gate']:
        grads.append(join(dzs))
    return (join(ys), last, *grads)


def _logp_exact(case, s):
    use = s['targets'] != 0
    logp = torch.where(use, _log_probs64(s['logits'], s['targets']), 0.0)
    if case['mode'] != 'train':
        return logp
    return logp, _grad64(s, torch.where(use, s['dlogp'].double(), 0.0))


def _grad64(s, g):
    parts = []
    for v, t, w in zip(s['logits'].split(8192), s['targets'].split(8192), g.split(8192)):
        d = -torch.softmax(v.double(), 1) * w[:, None]
        d[torch.arange(len(t), device=DEVICE), t] += w
        parts.append(d)
    return torch.cat(parts)


def _policy_exact(case, s):
    use = s['targets'] != 0
    lp = _log_probs64(s['logits'], s['targets'])[use]
    old, ref, adv = s['old'][use].double(), s['ref'][use].double(), s['advantages'][use].double()
    n = max(1, lp.numel())
    ratio = torch.exp(lp - old)
    cut = torch.where(adv >= 0, ratio > 1 + s['clip_high'], ratio < 1 - s['clip_low'])       # where the clipped side is the smaller one
    edge = torch.where(adv >= 0, 1 + s['clip_high'], 1 - s['clip_low']).double()
    pg = -adv * torch.where(cut, edge, ratio)
    d = ref - lp
    kl = torch.expm1(d) - d
    loss = (pg.sum() + s['kl_coef'] * kl.sum()) / n
    stats = torch.stack([pg.sum() / n, kl.sum() / n, (cut & (adv != 0)).sum() / n])
    if case['mode'] != 'train':
        return loss, stats
    g = torch.zeros(len(use), dtype=torch.float64, device=DEVICE)
    g[use] = (torch.where(cut, torch.zeros_like(adv), -adv * ratio) - s['kl_coef'] * torch.expm1(d)) / n
    return loss, stats, _grad64(s, g)

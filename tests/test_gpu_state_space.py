"""`causal_conv` and `selective_scan` against their definitions, step by step in 64 bits with autograd's gradients.

Tolerances, in half-steps of fp32 (H = 2^-24), relative to a companion: the same formula on absolute values, with the two ways in
which dt acts (through exp(dt A) and through dt x B) kept apart so that nothing cancels.  Every value that the kernels sum is one of
the companion's terms, so an error relative to terms is one relative to the companion.
  convolution: K products and sums, an exponential, a reciprocal: below 24 H; its gradients have one more product: 32 H, and
    those of weights and bias sum up to L steps: (32 + L) H, at worst.
  scan: a step multiplies by exp(dt A), whose exponent |dt A| <= 2 here has three roundings beside softplus' own eight (26 H at
    most), adds a product (12 H) and rounds once: below 40 H a step, over at most T steps, and N more for the sum over the states.
    Gradients pass through two such chains: 80 (T + 2) H + N H; sums over channels, sequences or steps one half more a term.
  bf16 results add one half-step of theirs, 2^-8 relative."""
import pytest
import torch
from torch.nn.utils.rnn import PackedSequence, pack_sequence

pytestmark = pytest.mark.gpu
H = 2.0 ** -24
DEV = 'cuda'
TYPES = [torch.float32, torch.bfloat16]


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def close(got, want, tol, what=''):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8
    bad = (got.double() - want).abs() - tol
    bad = bad[~(bad <= 0)]
    assert bad.numel() == 0, (what, bad.numel(), float(bad.max()), float(want.abs().max()))


class Layout:
    """Sequences of the given lengths as packed rows, or (all of one length) rectangular, time- or batch-first."""

    def __init__(self, lengths, kind):
        from paccmann_polymer_amd.state_space import packed_rows
        self.lengths, self.kind, self.B, self.T = lengths, kind, len(lengths), max(lengths)
        self.plan = None
        if kind == 'packed':
            self.bs = [sum(n > t for n in lengths) for t in range(self.T)]
            self.plan = packed_rows(torch.tensor(self.bs, dtype=torch.int64), DEV, sequences=self.B)
            self.off = [0]
            for n in self.bs:
                self.off.append(self.off[-1] + n)
        else:
            assert len(set(lengths)) == 1
            self.bs = [self.B] * self.T
        self.rows = sum(lengths)

    def tensor(self, g, *tail, dtype, wide=0, scale=1.0):
        """Random values; `wide` more columns beside them in memory (rows are strided then)."""
        n = tail[-1]
        tail = (*tail[:-1], n + wide)
        if self.kind == 'packed':
            t = randn(g, self.rows, *tail, dtype=dtype, scale=scale)
        elif self.kind == 'time':
            t = randn(g, self.T, self.B, *tail, dtype=dtype, scale=scale)
        else:
            t = randn(g, self.B, self.T, *tail, dtype=dtype, scale=scale).transpose(0, 1)
        return t[..., wide // 2:wide // 2 + n]

    def at(self, t, i):
        return t[self.off[i]:self.off[i + 1]] if self.kind == 'packed' else t[i]

    def join(self, parts, like):
        if not parts:
            return like.new_zeros(like.shape, dtype=torch.float64)
        return torch.cat(parts) if self.kind == 'packed' else torch.stack(parts)


def conv_definition(lay, x, w, bias, state, silu):
    K, line, ys = w.shape[1], state, []
    for t, n in enumerate(lay.bs):
        full = torch.cat([line[:n], lay.at(x, t).unsqueeze(1)], 1)
        line = torch.cat([full[:, 1:], line[n:]])
        pre = (full * w.t()).sum(1) + bias
        ys.append(pre * torch.sigmoid(pre) if silu else pre)
    return lay.join(ys, x), line


LAYOUTS = [([1], 'packed'), ([1], 'time'), ([2, 2, 2], 'batch'), ([16], 'batch'), ([17, 16, 15, 3, 1, 1], 'packed'), ([33, 32, 2, 1, 0, 0], 'packed'),
           ([40] * 3, 'time'), ([70] * 2, 'batch'), ([5] * 37, 'packed')]


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lengths,kind', LAYOUTS)
@pytest.mark.parametrize('D,K,wide,silu,biased,stateful', [
    (64, 4, 64, True, True, True), (5, 4, 3, True, True, True), (130, 3, 0, False, False, True), (16, 2, 0, True, True, False), (24, 1, 0, True, True, True),
    (72, 8, 0, True, True, True), (3, 6, 0, True, False, True), (1, 4, 0, True, True, True)])
def test_causal_conv(D, K, wide, silu, biased, stateful, lengths, kind, dtype):
    from paccmann_polymer_amd.state_space import causal_conv
    lay = Layout(lengths, kind)
    g = torch.Generator(device=DEV).manual_seed(D * 100 + K + lay.rows)
    x, dy = lay.tensor(g, D, dtype=dtype, wide=wide), lay.tensor(g, D, dtype=dtype, wide=wide)
    w, bias = randn(g, D, K, scale=0.5), randn(g, D, scale=0.3) if biased else None
    state, dlast = randn(g, lay.B, K - 1, D, dtype=dtype) if stateful else None, randn(g, lay.B, K - 1, D, dtype=dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, bias, state) if t is not None]
    names = [n for n, t in zip(('x', 'w', 'bias', 'state'), (x, w, bias, state)) if t is not None]
    a = dict(zip(names, leaves))
    y, last = causal_conv(a['x'], a['w'], a.get('bias'), plan=lay.plan, state=a.get('state'), activation='silu' if silu else None)
    grads = dict(zip(names, torch.autograd.grad((y, last), leaves, (dy, dlast))))

    def run(absolute):
        f = (lambda t: t.detach().double().abs()) if absolute else (lambda t: t.detach().double())
        xd, wd, bd, sd = (None if t is None else f(t).requires_grad_() for t in (x, w, bias, state))
        yd, ld = conv_definition(lay, xd, wd, 0.0 if bd is None else bd, torch.zeros(lay.B, K - 1, D, dtype=torch.float64, device=DEV) if sd is None else sd, silu)
        used = [t for t in (xd, wd, bd, sd) if t is not None]
        gr = torch.autograd.grad((yd, ld), used, (f(dy), f(dlast)), allow_unused=True)
        return yd.detach(), ld.detach(), {n: torch.zeros_like(t) if v is None else v for n, t, v in zip(names, used, gr)}

    yw, lw, gw = run(False)
    yc, _, gc = run(True)
    close(y.detach(), yw, 24 * H * (yc + 1e-30) + 1e-37, 'y')
    assert torch.equal(last.detach().double(), lw)
    # silu'(|pre|) is at least 0.5 and |silu'| at most 1.1 everywhere, so twice the companion's gradients bound the terms
    for n in names:
        close(grads[n], gw[n], (32 + (lay.rows if n in ('w', 'bias') else 0)) * H * 3 * gc[n] + 1e-37, n)
    with torch.no_grad():
        again, _ = causal_conv(x, w, bias, plan=lay.plan, state=state, activation='silu' if silu else None)
    assert torch.equal(again, y.detach())


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,D,K', [(1, 1, 4), (3, 65, 3), (7, 130, 8), (64, 256, 4), (5, 33, 1), (0, 8, 4)])
def test_causal_conv_step_continues_the_sequence(B, D, K, dtype):
    from paccmann_polymer_amd.state_space import causal_conv, causal_conv_step
    g = torch.Generator(device=DEV).manual_seed(B + D + K)
    T = 6
    x, w, bias = randn(g, T, B, 2 * D, dtype=dtype)[..., :D], randn(g, D, K, scale=0.5), randn(g, D)
    state = randn(g, B, K - 1, D, dtype=dtype)
    y, last = causal_conv(x, w, bias, state=state)
    kept, s = state.clone(), state
    inplace = state.clone()
    for t in range(T):
        out, s = causal_conv_step(x[t], s, w, bias)
        out2, same = causal_conv_step(x[t], inplace, w, bias, out=inplace)
        assert same is inplace and torch.equal(out, out2)
        # a tap is below 4 and an input below 4 in magnitude or nearly so
        close(out, y[t].double(), 24 * H * (16 * K + 4) * torch.ones_like(y[t], dtype=torch.float64))
    assert torch.equal(s, last) and torch.equal(inplace, last) and torch.equal(state, kept)


def scan_definition(lay, G, x, raw, raw_b, A, B, C, D, z, bias, bias_b, state, softplus):
    """raw, bias and raw_b, bias_b are the same numbers: dt as it acts through the decay, and through the input."""
    width = x.shape[-1]
    group = torch.arange(width, device=DEV) // (width // G)
    h, ys = state, []
    for t, n in enumerate(lay.bs):
        xt = lay.at(x, t)
        da, db = lay.at(raw, t) + bias, lay.at(raw_b, t) + bias_b
        if softplus:
            da, db = (torch.logaddexp(v, torch.zeros((), dtype=v.dtype, device=DEV)) for v in (da, db))
        hn = torch.exp(da[:, :, None] * A) * h[:n] + (db * xt)[:, :, None] * lay.at(B, t)[:, group]
        y = (hn * lay.at(C, t)[:, group]).sum(-1) + (0.0 if D is None else D * xt)
        if z is not None:
            zt = lay.at(z, t)
            y = y * zt * torch.sigmoid(zt)
        ys.append(y)
        h = torch.cat([hn, h[n:]])
    return lay.join(ys, x), h


def scan_case(lengths, kind, D, N, G, dtype, gate, skip, biased, stateful, softplus, wide=0, seed=0):
    lay = Layout(lengths, kind)
    g = torch.Generator(device=DEV).manual_seed(seed + D * 1000 + N * 10 + lay.rows)
    t = dict(x=lay.tensor(g, D, dtype=dtype, wide=wide), dt=lay.tensor(g, D, dtype=dtype, wide=wide, scale=0.5),
             A=-torch.rand(D, N, generator=g, device=DEV) * 2 - 0.05, B=lay.tensor(g, G, N, dtype=dtype, wide=wide), C=lay.tensor(g, G, N, dtype=dtype, wide=wide),
             D=randn(g, D) if skip else None, z=lay.tensor(g, D, dtype=dtype, wide=wide) if gate else None,
             dt_bias=torch.rand(D, generator=g, device=DEV) * 2 - 3 if biased else None, state=randn(g, lay.B, D, N) if stateful else None)
    if not softplus:
        t['dt'] = t['dt'].abs() * 0.5
        t['dt_bias'] = None if t['dt_bias'] is None else t['dt_bias'].abs() * 0.1
    return lay, t, lay.tensor(g, D, dtype=dtype), randn(g, lay.B, D, N)


def scan_reference(lay, t, dy, dlast, softplus, absolute):
    """y, last state and gradients in 64 bits; `absolute`: the companion."""
    width, N, G = t['x'].shape[-1], t['A'].shape[1], t['B'].shape[-2]
    mag = (lambda v: v.detach().double().abs()) if absolute else (lambda v: v.detach().double())
    plain = lambda v: v.detach().double()           # noqa: E731
    p = {k: None if v is None else (plain if k in ('dt', 'A', 'dt_bias') else mag)(v).requires_grad_() for k, v in t.items()}
    raw_b = p['dt'].detach().clone().requires_grad_()
    bias_b = None if p['dt_bias'] is None else p['dt_bias'].detach().clone().requires_grad_()
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    state = torch.zeros(lay.B, width, N, dtype=torch.float64, device=DEV) if p['state'] is None else p['state']
    y, last = scan_definition(lay, G, p['x'], p['dt'], raw_b, p['A'], p['B'], p['C'], p['D'], p['z'], zero if p['dt_bias'] is None else p['dt_bias'],
                              zero if bias_b is None else bias_b, state, softplus)
    names = [k for k, v in p.items() if v is not None]
    leaves = [p[k] for k in names] + [raw_b] + ([] if bias_b is None else [bias_b])
    gr = torch.autograd.grad((y, last), leaves, (mag(dy), mag(dlast)), allow_unused=True)
    gr = [torch.zeros_like(v) if d is None else d for v, d in zip(leaves, gr)]
    out = dict(zip(names, gr[:len(names)]))
    two = (lambda a, b: a.abs() + b.abs()) if absolute else (lambda a, b: a + b)
    out['dt'] = two(out['dt'], gr[len(names)])
    if bias_b is not None:
        out['dt_bias'] = two(out['dt_bias'], gr[-1])
        if absolute:                                # sums of what can have either sign: of the rows' magnitudes, times their number at most
            out['dt_bias'] = out['dt'].reshape(-1, width).sum(0)
    if absolute:
        out['A'] = out['A'].abs()
    return y.detach(), last.detach(), out


def check_scan(lengths, kind, D, N, G, dtype, gate=True, skip=True, biased=True, stateful=True, softplus=True, wide=0, grad=True):
    from paccmann_polymer_amd.state_space import selective_scan
    lay, t, dy, dlast = scan_case(lengths, kind, D, N, G, dtype, gate, skip, biased, stateful, softplus, wide)
    names = [k for k, v in t.items() if v is not None]
    a = {k: None if v is None else v.detach().requires_grad_(grad) for k, v in t.items()}
    y, last = selective_scan(**a, plan=lay.plan, dt_softplus=softplus)
    yw, lw, gw = scan_reference(lay, t, dy, dlast, softplus, False)
    yc, lc, gc = scan_reference(lay, t, dy, dlast, softplus, True)
    steps = lay.T + 2
    assert last.dtype == torch.float32 and y.dtype == dtype
    close(y.detach(), yw, (40 * steps + N) * H * yc + 1e-37, 'y')
    close(last.detach(), lw, 40 * steps * H * lc + 1e-37, 'last')
    if not grad:
        return
    grads = dict(zip(names, torch.autograd.grad((y, last), [a[k] for k in names], (dy, dlast))))
    many = {'A': lay.rows, 'D': lay.rows, 'dt_bias': lay.rows, 'B': D, 'C': D}
    for k in names:
        assert grads[k].dtype == t[k].dtype
        # silu' is at most 1.1 and at least 0.5 of the companion's: a factor of 3 covers dz and what passes the gate
        close(grads[k], gw[k], (80 * steps + N + many.get(k, 0)) * H * 3 * gc[k] + 1e-37, k)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('lengths,kind', LAYOUTS)
@pytest.mark.parametrize('D,N,G,wide', [(64, 16, 1, 64), (130, 16, 2, 0), (5, 11, 1, 3), (66, 4, 3, 0), (1, 1, 1, 0)])
def test_selective_scan(D, N, G, wide, lengths, kind, dtype):
    check_scan(lengths, kind, D, N, G, dtype, wide=wide)


@pytest.mark.parametrize('N', [1, 2, 3, 5, 8, 9, 15, 17, 24, 32, 33, 50, 64])
def test_selective_scan_state_counts(N):
    check_scan([21, 17, 16, 4], 'packed', 70, N, 1, torch.float32)
    check_scan([19, 19], 'batch', 12, N, 4, torch.bfloat16)


@pytest.mark.parametrize('gate', [False, True])
@pytest.mark.parametrize('skip,biased,stateful,softplus', [(False, False, False, False), (True, False, True, False), (False, True, False, True), (True, True, False, True), (False, False, True, True)])
def test_selective_scan_optional_inputs(gate, skip, biased, stateful, softplus):
    check_scan([18, 9, 1], 'packed', 40, 16, 2, torch.float32, gate, skip, biased, stateful, softplus)
    check_scan([33, 33], 'time', 40, 7, 1, torch.float32, gate, skip, biased, stateful, softplus)


@pytest.mark.parametrize('lengths,kind,D,N,G', [([1500], 'batch', 48, 16, 1), ([700, 650, 33], 'packed', 33, 16, 3), ([2049], 'time', 20, 6, 2), ([400], 'time', 200, 33, 1)])
@pytest.mark.parametrize('dtype', TYPES)
def test_selective_scan_long(lengths, kind, D, N, G, dtype):
    """Long enough for the time axis to be split."""
    check_scan(lengths, kind, D, N, G, dtype)


def test_selective_scan_of_no_steps():
    from paccmann_polymer_amd.state_space import causal_conv, packed_rows, selective_scan
    plan = packed_rows(torch.zeros(0, dtype=torch.int64), DEV, sequences=3)
    state = torch.randn(3, 8, 4, device=DEV, requires_grad=True)
    A = torch.full((8, 4), -1.0, device=DEV, requires_grad=True)
    x, b = torch.zeros(0, 8, device=DEV, requires_grad=True), torch.zeros(0, 4, device=DEV)
    for kw, data, bc in ((dict(plan=plan), x, b), (dict(), torch.zeros(0, 3, 8, device=DEV, requires_grad=True), torch.zeros(0, 3, 4, device=DEV))):
        y, last = selective_scan(data, data, A, bc, bc, state=state, **kw)
        assert y.numel() == 0 and torch.equal(last, state)
        up = torch.randn(3, 8, 4, device=DEV)
        dA, ds = torch.autograd.grad(last, (A, state), up)
        assert torch.equal(ds, up) and not bool(dA.any())
    cs = torch.randn(3, 3, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, 4, device=DEV, requires_grad=True)
    y, last = causal_conv(x, w, plan=plan, state=cs)
    up = torch.randn(3, 3, 8, device=DEV)
    dw, ds = torch.autograd.grad(last, (w, cs), up)
    assert torch.equal(last, cs) and torch.equal(ds, up) and not bool(dw.any())


def test_packed_sequence_in_and_out():
    from paccmann_polymer_amd.state_space import causal_conv, selective_scan
    g = torch.Generator(device=DEV).manual_seed(3)
    seqs = [randn(g, n, 24) for n in (3, 9, 20, 9)]
    packed = pack_sequence(seqs, enforce_sorted=False)
    w = randn(g, 24, 4)
    y, _ = causal_conv(packed, w)
    assert isinstance(y, PackedSequence) and torch.equal(y.batch_sizes, packed.batch_sizes) and torch.equal(y.sorted_indices, packed.sorted_indices)
    A = -torch.rand(24, 16, generator=g, device=DEV)
    dt, bc = PackedSequence(y.data, *packed[1:]), randn(g, packed.data.shape[0], 16)
    out, last = selective_scan(y, dt, A, bc, bc)
    assert isinstance(out, PackedSequence)
    lengths = [int((packed.batch_sizes > b).sum()) for b in range(4)]
    for b, n in enumerate(lengths):                                     # each sequence alone gives the same
        rows = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(packed.batch_sizes, 0)])[:n] + b
        one, end = selective_scan(y.data[rows][:, None], y.data[rows][:, None], A, bc[rows][:, None], bc[rows][:, None])
        close(one[:, 0], out.data[rows].double(), 40 * (n + 2) * H * 50 * torch.ones(n, 24, dtype=torch.float64, device=DEV))
        close(end[0], last[b].double(), 40 * (n + 2) * H * 50 * torch.ones(24, 16, dtype=torch.float64, device=DEV))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('B,D,N,G', [(1, 1, 1, 1), (3, 65, 16, 1), (7, 66, 11, 3), (64, 256, 16, 2), (5, 33, 64, 1), (2, 40, 30, 5), (0, 8, 4, 1)])
def test_selective_scan_step_continues_the_sequence(B, D, N, G, dtype):
    from paccmann_polymer_amd.state_space import selective_scan_step
    T = 5
    if B == 0:
        e = torch.zeros(0, D, device=DEV, dtype=dtype)
        y, s = selective_scan_step(e, e, torch.zeros(D, N, device=DEV), torch.zeros(0, N, device=DEV, dtype=dtype), torch.zeros(0, N, device=DEV, dtype=dtype), torch.zeros(0, D, N, device=DEV))
        assert y.shape == (0, D) and s.shape == (0, D, N)
        return
    lay, t, dy, dlast = scan_case([T] * B, 'time', D, N, G, dtype, True, True, True, True, True, wide=5)
    yw, lw, _ = scan_reference(lay, t, dy, dlast, True, False)
    yc, lc, _ = scan_reference(lay, t, dy, dlast, True, True)
    s, inplace = t['state'], t['state'].clone()
    keep = s.clone()
    for i in range(T):
        args = (t['x'][i], t['dt'][i], t['A'], t['B'][i], t['C'][i])
        more = dict(D=t['D'], z=t['z'][i], dt_bias=t['dt_bias'])
        y, s = selective_scan_step(*args, s, **more)
        y2, same = selective_scan_step(*args, inplace, out=inplace, **more)
        assert same is inplace and torch.equal(y, y2) and torch.equal(s, inplace)
        close(y, yw[i], (40 * (T + 2) + N) * H * yc[i])
    close(s, lw, 40 * (T + 2) * H * lc)
    assert torch.equal(t['state'], keep)


def test_offsets_beyond_32_bits():
    """Rows further than 2^31 elements apart."""
    from paccmann_polymer_amd.state_space import causal_conv, selective_scan
    g = torch.Generator(device=DEV).manual_seed(11)
    far, T, D, N = 2 ** 31 + 128, 3, 64, 16
    base = torch.empty((T - 1) * far + 4 * D, dtype=torch.bfloat16, device=DEV)
    def view(k, *tail):
        n = 1
        for v in tail:
            n *= v
        t = torch.as_strided(base, (T, 1, *tail), (far, n, *([tail[1], 1] if len(tail) == 2 else [1])), k * D)
        t.copy_(randn(g, T, 1, *tail, dtype=torch.bfloat16))
        return t
    x, dt, B, C = view(0, D), view(1, D), view(2, 1, N), view(3, 1, N)
    near = [t.contiguous() for t in (x, dt, B, C)]
    A, w = -torch.rand(D, N, generator=g, device=DEV), randn(g, D, 4)

    def both(x, dt, B, C):
        leaves = [t.detach().requires_grad_() for t in (x, dt, B, C)]
        y, last = selective_scan(leaves[0], leaves[1], A, leaves[2], leaves[3])
        c, _ = causal_conv(leaves[0], w)
        return (y, last, c, *torch.autograd.grad((y.float().sum(), c.float().sum()), leaves))

    for a, b in zip(both(x, dt, B, C), both(*near)):
        assert torch.equal(a, b)


def test_results_repeat_bit_for_bit():
    from paccmann_polymer_amd.state_space import causal_conv, selective_scan
    lay, t, dy, dlast = scan_case([90, 70, 70, 31, 2] * 1 + [1] * 40, 'packed', 200, 16, 2, torch.float32, True, True, True, True, True)

    def once():
        a = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, last = selective_scan(**a, plan=lay.plan)
        w = torch.ones(200, 4, device=DEV, requires_grad=True)
        c, cl = causal_conv(a['x'], w, plan=lay.plan)
        return (y, last, c, cl, *torch.autograd.grad((y, last, c), [*a.values(), w], (dy, dlast, dy)))

    first = once()
    for _ in range(3):
        for a, b in zip(once(), first):
            assert torch.equal(a, b)


def test_broadcast_inputs_and_partial_upstream():
    """B and C expanded over the sequences, a gradient that arrives for one output only, and expanded gradients."""
    from paccmann_polymer_amd.state_space import selective_scan
    g = torch.Generator(device=DEV).manual_seed(4)
    x, dt = randn(g, 20, 3, 32), randn(g, 20, 3, 32, scale=0.5)
    A, bc = -torch.rand(32, 16, generator=g, device=DEV), randn(g, 20, 1, 16, scale=0.5)
    # gradients at the expanded tensors themselves: beyond them autograd adds dB and dC and the sequences in an order of its own
    b, c = (bc.expand(20, 3, 16).detach().requires_grad_() for _ in range(2))
    assert b.stride(1) == 0
    y, last = selective_scan(x, dt, A, b, c)
    d = torch.autograd.grad(y.sum(), (b, c), retain_graph=True)
    b2, c2 = (bc.expand(20, 3, 16).contiguous().requires_grad_() for _ in range(2))
    y2, _ = selective_scan(x, dt, A, b2, c2)
    d2 = torch.autograd.grad(y2, (b2, c2), torch.ones_like(y2))
    assert torch.equal(y, y2) and torch.equal(d[0], d2[0]) and torch.equal(d[1], d2[1])
    (e,) = torch.autograd.grad(last.sum(), b)
    assert bool(torch.isfinite(e).all()) and bool(e.any())


def test_other_stream_and_graph_replays():
    from paccmann_polymer_amd.state_space import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    lay, t, dy, dlast = scan_case([40, 33, 20, 1], 'packed', 96, 16, 1, torch.float32, True, True, True, True, True)
    w = randn(torch.Generator(device=DEV).manual_seed(1), 96, 4)
    cstate = torch.zeros(4, 3, 96, device=DEV)
    sstate = torch.zeros(4, 96, 16, device=DEV)

    def step():
        a = {k: v.detach().requires_grad_() for k, v in t.items()}
        wl = w.detach().requires_grad_()
        c, _ = causal_conv(a['x'], wl, plan=lay.plan)
        y, last = selective_scan(**{**a, 'x': c}, plan=lay.plan)
        names = [k for k in a]
        one, _ = causal_conv_step(t['x'][:4], cstate, w)
        tok, _ = selective_scan_step(one, t['dt'][:4], t['A'], t['B'][:4], t['C'][:4], sstate)
        return (c.detach(), y.detach(), last.detach(), one, tok, *torch.autograd.grad((y, last), [a[k] for k in names] + [wl], (dy, dlast)))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(side, step()):
        assert torch.equal(a, b)
    del side
    graphs, outs = [], []
    for _ in range(2):                                                          # two captured graphs, each with workspaces of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    base = t['x'].clone()
    for k in range(3):
        t['x'].copy_(base * (1 + 0.25 * k))
        for graph in graphs:
            graph.replay()
        want = step()
        torch.cuda.synchronize()
        for out in outs:
            for a, b in zip(out, want):
                assert torch.equal(a, b), k


def test_no_sequences():
    from paccmann_polymer_amd.state_space import causal_conv, selective_scan
    x = torch.zeros(5, 0, 8, device=DEV, requires_grad=True)
    bc = torch.zeros(5, 0, 4, device=DEV)
    A, w = torch.full((8, 4), -1.0, device=DEV, requires_grad=True), torch.ones(8, 4, device=DEV, requires_grad=True)
    y, last = selective_scan(x, x, A, bc, bc)
    c, cl = causal_conv(x, w)
    assert y.shape == x.shape and last.shape == (0, 8, 4) and c.shape == x.shape and cl.shape == (0, 3, 8)
    dA, dw = torch.autograd.grad(y.sum() + c.sum(), (A, w))
    assert not bool(dA.any()) and not bool(dw.any())


@pytest.mark.parametrize('T', [3, 5, 200])
def test_infinities_stay_where_the_formula_has_them(T):
    """States that forget at once (A = -inf), an infinite input in a last step and beside it other sequences and channels that are not
    touched by it; lengths that end inside a tile and inside a split."""
    from paccmann_polymer_amd.state_space import causal_conv, selective_scan
    lay, t, dy, dlast = scan_case([T, T, T - 1], 'packed', 20, 16, 1, torch.float32, True, True, True, True, True)
    a = {k: v.clone() for k, v in t.items()}
    a['A'][:, 3] = float('-inf')
    leaves = {k: v.detach().requires_grad_() for k, v in a.items()}
    y, last = selective_scan(**leaves, plan=lay.plan)
    g = dict(zip(a, torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))))
    assert all(bool(torch.isfinite(v).all()) for v in (y, last, *g.values()))
    b = {k: v.clone() for k, v in t.items()}
    b['A'][:, 3] = -1e30                                                # forgets as completely
    y2, last2 = selective_scan(**b, plan=lay.plan)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    row = int(lay.off[T - 1] + 1)                                       # the last step of sequence 1
    c = {k: v.clone() for k, v in t.items()}
    c['x'][row, 7] = float('inf')
    clean, clean_last = selective_scan(**t, plan=lay.plan)
    y3, last3 = selective_scan(**c, plan=lay.plan)
    assert bool(torch.isinf(last3[1, 7]).all())
    keep = torch.ones_like(y3, dtype=torch.bool)
    keep[row, 7] = False
    assert torch.equal(y3[keep], clean[keep]) and torch.equal(last3[[0, 2]], clean_last[[0, 2]])
    w = torch.randn(20, 4, device=DEV)
    y4, y5 = causal_conv(c['x'], w, plan=lay.plan)[0], causal_conv(t['x'], w, plan=lay.plan)[0]
    assert torch.equal(y4[keep], y5[keep])


@pytest.mark.parametrize('shape', [(1, 3), (4, 1), (1, 1)])
def test_the_only_step_or_sequence_may_have_any_stride(shape):
    """What a slice of one step (sequence) of a far larger tensor hands over; only the strides that are walked count."""
    from paccmann_polymer_amd.state_space import causal_conv, selective_scan
    g = torch.Generator(device=DEV).manual_seed(11)
    T, B, D, N = *shape, 12, 8

    def far(t):
        s = list(t.stride())
        for i in range(2):
            if t.shape[i] == 1:
                s[i] = 2 ** 33
        return t.as_strided(t.shape, s)
    x, dt, Bm, C, z = (randn(g, T, B, n, scale=0.5) for n in (D, D, N, N, D))
    w, A = randn(g, D, 4), -randn(g, D, N).abs()
    for near, away in zip(causal_conv(x, w), causal_conv(far(x), w)):
        assert torch.equal(near, away)
    near, away = [], []
    for got, f in ((near, lambda t: t), (away, far)):
        leaves = [v.detach().requires_grad_() for v in (x, dt, Bm, C, z)]
        y, last = selective_scan(f(leaves[0]), f(leaves[1]), A, f(leaves[2]), f(leaves[3]), z=f(leaves[4]))
        got += [y, last, *torch.autograd.grad(y.square().sum() + last.sum(), leaves)]
    for a, b in zip(near, away):
        assert torch.equal(a, b)
    # rows of a packed batch of one row
    from paccmann_polymer_amd.state_space import packed_rows
    row = x[:1, 0]
    plan = packed_rows(torch.ones(1, dtype=torch.int64), DEV)
    assert torch.equal(causal_conv(row, w, plan=plan)[0], causal_conv(row.as_strided((1, D), (2 ** 33, 1)), w, plan=plan)[0])


def test_more_sequences_than_a_grid_has_rows():
    """4.3 million sequences of a step each: their sums take more chunks than 65535."""
    from paccmann_polymer_amd.state_space import selective_scan
    g = torch.Generator(device=DEV).manual_seed(12)
    B = 4_300_000
    x, dt, Bm, C = (randn(g, 1, B, 1, scale=0.5) for _ in range(4))
    A = torch.full((1, 1), -1.0, device=DEV, requires_grad=True)
    D = torch.ones(1, device=DEV, requires_grad=True)
    y, last = selective_scan(x, dt, A, Bm, C, D=D)
    s = torch.nn.functional.softplus(dt.double())
    h = s * x.double() * Bm.double()
    close(y, C.double() * h + x.double(), 40 * H * (C.double() * h).abs() + 3 * H * x.double().abs())
    dA, dD = torch.autograd.grad(y.sum(), (A, D))
    assert float(dA) == 0.0                        # no state before the first step
    xs = x.double()
    assert abs(float(dD) - float(xs.sum())) <= 2 * H * float(xs.abs().sum())


@pytest.mark.parametrize('N', [8, 16, 32])
@pytest.mark.parametrize('T', [5, 100])
def test_states_and_parameters_anywhere_in_memory(T, N):
    """A, the state and its gradient from an address that is no multiple of 16 bytes: other accesses, the same sums."""
    from paccmann_polymer_amd.state_space import selective_scan, selective_scan_step
    g = torch.Generator(device=DEV).manual_seed(13)
    B, D = 3, 20

    def shifted(t):
        room = t.new_empty(t.numel() + 1)
        return room[1:].view(t.shape).copy_(t)
    x, dt, Bm, C = (randn(g, T, B, n, scale=0.5) for n in (D, D, N, N))
    A, state, dlast = -randn(g, D, N).abs(), randn(g, B, D, N), randn(g, B, D, N)
    results = []
    for f in (torch.clone, shifted):
        leaves = [x.clone().requires_grad_(), f(A).detach().requires_grad_(), f(state).detach().requires_grad_()]
        y, last = selective_scan(leaves[0], dt, leaves[1], Bm, C, state=leaves[2])
        step = selective_scan_step(x[0], dt[0], f(A), Bm[0], C[0], f(state))
        results.append([y, last, *torch.autograd.grad((y, last), leaves, (x, f(dlast))), *step])
    for a, b in zip(*results):
        assert torch.equal(a, b)


def same_kind(got, want, what=''):
    """NaN and infinities (with their signs) stand where the 64-bit definition has them."""
    want = want.to(got.dtype)
    for kind in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(kind(got), kind(want)), (what, kind.__name__, int((kind(got) != kind(want)).sum()))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('silu', [False, True])
@pytest.mark.parametrize('D', [8, 5, 72, 70])                    # rows of 16 lanes and whole waves, four channels a lane and one
@pytest.mark.parametrize('K', range(1, 9))
def test_causal_conv_infinite_inputs_reach_k_steps(K, D, silu, dtype):
    """An infinite input and a NaN in the middle of two sequences, and an infinite upstream gradient: what a tap does not reach is as without."""
    from paccmann_polymer_amd.state_space import causal_conv, causal_conv_step
    lay = Layout([40, 40, 40, 21], 'packed')
    g = torch.Generator(device=DEV).manual_seed(K * 100 + D)
    x, dy = lay.tensor(g, D, dtype=dtype), lay.tensor(g, D, dtype=dtype)
    w, bias = torch.rand(D, K, generator=g, device=DEV) + 0.1, randn(g, D, scale=0.3)
    state, dlast = randn(g, lay.B, K - 1, D, dtype=dtype), randn(g, lay.B, K - 1, D, dtype=dtype)

    def run(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w, bias, state)]
        y, last = causal_conv(leaves[0], leaves[1], leaves[2], plan=lay.plan, state=leaves[3], activation='silu' if silu else None)
        return (y.detach(), last.detach(), *torch.autograd.grad((y, last), leaves, (dy, dlast)))

    def want(x, dy):
        leaves = [t.detach().double().requires_grad_() for t in (x, w, bias, state)]
        y, last = conv_definition(lay, *leaves, False)
        y = torch.nn.functional.silu(y) if silu else y          # its derivative as one factor: as a sum of two, an infinite dy makes inf - inf of it
        used = [y, last] if K > 1 else [y]
        gr = torch.autograd.grad(used, leaves, (dy.double(), dlast.double())[:len(used)], allow_unused=True)
        return (y.detach(), last.detach(), *(torch.zeros_like(t) if d is None else d for t, d in zip(leaves, gr)))

    clean = run(x, dy)
    inf, at = float('inf'), 13
    rows = torch.stack([lay.off[t] + torch.arange(lay.B) if n == lay.B else torch.cat([lay.off[t] + torch.arange(n), torch.full((lay.B - n,), lay.rows)])
                        for t, n in enumerate(lay.bs)])                                       # [T, B]: a sequence's rows; behind its last, none
    for field, values in (('x', ((1, 2, inf), (2, 4, float('nan')))), ('dy', ((1, 2, inf), (0, 3, -inf)))):
        xs, ds = x.clone(), dy.clone()
        hit_y, hit_dx = (torch.zeros(lay.rows + 1, D, dtype=torch.bool, device=DEV) for _ in range(2))
        for b, c, value in values:
            (xs if field == 'x' else ds)[rows[at, b], c] = value
            if field == 'x':
                hit_y[rows[at:at + K, b], c] = True
                if silu:
                    hit_dx[rows[at - K + 1:at + K, b], c] = True
            else:
                hit_dx[rows[at - K + 1:at + 1, b], c] = True
        got, expected = run(xs, ds), want(xs, ds)
        for name, a, b in zip(('y', 'last', 'dx', 'dw', 'dbias', 'dstate'), got, expected):
            same_kind(a, b, (field, name))
        assert torch.equal(got[0][~hit_y[:-1]], clean[0][~hit_y[:-1]])
        assert torch.equal(got[2][~hit_dx[:-1]], clean[2][~hit_dx[:-1]])
        assert torch.equal(got[5], clean[5])                                                  # nothing reaches the state before the first step
        if field == 'x':
            s = state
            for t in range(40):
                n = lay.bs[t]
                out, s = causal_conv_step(xs[lay.off[t]:lay.off[t + 1]], s[:n], w, bias, 'silu' if silu else None)
                same_kind(out, got[0][lay.off[t]:lay.off[t + 1]].double(), ('step', t))


@pytest.mark.parametrize('T', [1, 3, 5, 7, 16, 23, 200])
@pytest.mark.parametrize('N', [16, 11, 32])
def test_gradients_of_an_infinite_last_input(N, T):
    """The state that it makes is read by no step: gradients of A, x and the first state are those of any other input there."""
    from paccmann_polymer_amd.state_space import selective_scan
    lay, t, dy, dlast = scan_case([T, T, max(T - 1, 1)], 'packed', 20, N, 1, torch.float32, True, True, True, True, True)
    row = int(lay.off[T - 1] + 1)                                       # the last step of sequence 1

    def grads(t):
        leaves = {k: v.detach().requires_grad_() for k, v in t.items()}
        y, last = selective_scan(**leaves, plan=lay.plan)
        return dict(zip(t, torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast))))

    clean = grads(t)
    bad = {k: v.clone() for k, v in t.items()}
    bad['x'][row, 7] = float('inf')
    got = grads(bad)
    for k in ('A', 'x', 'state'):
        assert torch.equal(got[k], clean[k]), k
    want = scan_reference(lay, bad, dy, dlast, True, False)[2]
    for k in ('dt', 'B', 'C', 'D', 'dt_bias'):
        same_kind(got[k], want[k], k)


def positive(t):
    """The same case without cancelling infinities: what is not a decay is positive."""
    return {k: v if v is None or k in ('A', 'dt', 'dt_bias') else v.abs() + 0.1 for k, v in t.items()}


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('skip,gate', [(False, False), (False, True), (True, True)])
@pytest.mark.parametrize('T', [4, 21, 70])
@pytest.mark.parametrize('N', [1, 3, 5, 8, 11, 16, 17, 33, 50, 64])
def test_selective_scan_infinities_are_the_definitions(N, T, skip, gate, dtype):
    """An infinity in x, dt, B, C or the upstream gradient: states, channels and steps that do not exist turn no infinite result into NaN, and no finite
    one into anything else."""
    from paccmann_polymer_amd.state_space import selective_scan
    D, inf, at = 20, float('inf'), T // 2
    lay, t, dy, dlast = scan_case([T, T], 'time', D, N, 2, dtype, gate, skip, True, True, True)
    t, dy, dlast = positive(t), dy.abs() + 0.1, dlast.abs() + 0.1
    names = [k for k, v in t.items() if v is not None]
    for field in ('x', 'dt', 'B', 'C', 'dy'):
        p, up = {k: None if v is None else v.clone() for k, v in t.items()}, dy.clone()
        if field in ('B', 'C'):
            p[field][at, 1, 0, N // 2] = inf
        else:
            (up if field == 'dy' else p['x'])[at, 1, 7] = inf
        leaves = {k: None if v is None else v.detach().requires_grad_() for k, v in p.items()}
        y, last = selective_scan(**leaves)
        got = dict(zip(names, torch.autograd.grad((y, last), [leaves[k] for k in names], (up, dlast))))
        yw, lw, want = scan_reference(lay, p, up, dlast, True, False)
        same_kind(y.detach(), yw, (field, 'y'))
        same_kind(last.detach(), lw, (field, 'last'))
        for k in names:
            same_kind(got[k], want[k], (field, k))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('skip', [False, True])
@pytest.mark.parametrize('N', [1, 3, 4, 11, 16, 30, 33, 64])
def test_selective_scan_step_infinities_are_the_definitions(N, skip, dtype):
    from paccmann_polymer_amd.state_space import selective_scan_step
    lay, t, _, _ = scan_case([1, 1], 'time', 20, N, 2, dtype, True, skip, True, True, True)
    t = positive(t)
    for field in ('x', 'dt', 'B', 'C'):
        p = {k: None if v is None else v.clone() for k, v in t.items()}
        p[field].view(2, -1)[1, 0] = float('inf')
        y, s = selective_scan_step(p['x'][0], p['dt'][0], p['A'], p['B'][0], p['C'][0], p['state'], D=p['D'], z=p['z'][0], dt_bias=p['dt_bias'])
        yw, sw = scan_definition(lay, 2, *(None if p[k] is None else p[k].double() for k in ('x', 'dt', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'dt_bias', 'state')), True)
        same_kind(y, yw[0], (field, 'y'))
        same_kind(s, sw, (field, 'state'))


@pytest.mark.parametrize('shape,batch_first', [((6, 3), True), ((6, 3), False), ((1, 3), False), ((1, 3), True), ((6, 1), True)])
def test_results_may_be_changed_in_place(shape, batch_first):
    """A residual added to y where it lies, in every layout, before the backward pass."""
    from paccmann_polymer_amd.state_space import causal_conv, selective_scan
    g = torch.Generator(device=DEV).manual_seed(21)
    T, B, D, N = *shape, 12, 8
    x = randn(g, B, T, D).transpose(0, 1) if batch_first else randn(g, T, B, D)
    bc, A, w = randn(g, T, B, N), -randn(g, D, N).abs(), randn(g, D, 4)

    def run(inplace):
        leaf = x.detach().requires_grad_()
        y, last = selective_scan(leaf, x, A, bc, bc)
        c, cl = causal_conv(leaf, w)
        for i, t in enumerate((y, c)):
            assert t.stride() == x.stride() or 1 in shape                # laid out as x is
        if inplace:
            y += x
            c.mul_(2.0)
            last.add_(1.0)
            cl.zero_()
        else:
            y, c, last = y + x, c * 2.0, last + 1.0
        return y.detach(), c.detach(), torch.autograd.grad((y.square().sum() + c.square().sum() + last.square().sum()), leaf)[0]

    for a, b in zip(run(True), run(False)):
        assert torch.equal(a, b)


@pytest.mark.parametrize('T,A,dt', [(2048, 1.0, 1.0), (2048, -1.0, -1.0), (700, 4.0, 1.0)])
def test_states_that_grow_from_zero(T, A, dt):
    """Decays above one over more steps than fp32 holds the product of, with nothing to multiply: a state (a gradient) of zero stays zero, in one
    piece and in splits."""
    from paccmann_polymer_amd.state_space import selective_scan
    D, N, few = 8, 16, 10
    g = torch.Generator(device=DEV).manual_seed(T)
    lay = Layout([T], 'time')
    t = dict(x=torch.zeros(T, 1, D, device=DEV), dt=torch.full((T, 1, D), dt, device=DEV), A=torch.full((D, N), A, device=DEV),
             B=randn(g, T, 1, 1, N), C=randn(g, T, 1, 1, N), D=None, z=None, dt_bias=None, state=torch.zeros(1, D, N, device=DEV))
    t['x'][T - few:] = randn(g, few, 1, D)
    dy, dlast = torch.zeros(T, 1, D, device=DEV), torch.zeros(1, D, N, device=DEV)
    dy[:few] = randn(g, few, 1, D)
    names = [k for k, v in t.items() if v is not None]
    leaves = {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}
    y, last = selective_scan(**leaves, dt_softplus=False)
    got = dict(zip(names, torch.autograd.grad((y, last), [leaves[k] for k in names], (dy, dlast))))
    yw, lw, want = scan_reference(lay, t, dy, dlast, False, False)
    yc, lc, comp = scan_reference(lay, t, dy, dlast, False, True)
    # dt has one sign here, which the companion keeps: all of its terms have the same one, and their magnitude is what bounds an error
    yc, lc, comp = yc.abs(), lc.abs(), {k: v.abs() for k, v in comp.items()}
    # |dt A| <= 4 here: twice what a step of the other tests loses
    close(y.detach(), yw, (80 * (few + 2) + N) * H * yc + 1e-37, 'y')
    close(last.detach(), lw, 80 * (few + 2) * H * lc + 1e-37, 'last')
    for k in names:
        close(got[k], want[k], (160 * (few + 2) + N + (D if k in ('B', 'C') else 0)) * H * 3 * comp[k] + 1e-37, k)


def test_an_infinite_state_stays_infinite_across_splits():
    """Its decay over thousands of steps is below what fp32 holds; no step's is."""
    from paccmann_polymer_amd.state_space import selective_scan
    T, D, N = 4096, 8, 16
    lay = Layout([T], 'time')
    g = torch.Generator(device=DEV).manual_seed(1)
    x, dt, bc = randn(g, T, 1, D), torch.full((T, 1, D), 0.5, device=DEV), randn(g, T, 1, 1, N).abs()
    A, state = torch.full((D, N), -1.0, device=DEV), torch.zeros(1, D, N, device=DEV)
    state[0, 3] = float('inf')
    y, last = selective_scan(x, dt, A, bc, bc, state=state, dt_softplus=False)
    assert bool(torch.isposinf(y[:, 0, 3]).all()) and bool(torch.isposinf(last[0, 3]).all())
    keep = [i for i in range(D) if i != 3]
    assert bool(torch.isfinite(y[:, :, keep]).all())


MANY = [100 - b * 80 // 2047 for b in range(2048)]                      # 2048 sequences of 100 to 20 steps


@pytest.mark.parametrize('lengths,kind,D,K,wide', [
    (MANY, 'packed', 32, 4, 0),                  # more items than a backward launch has room for: its blocks take several, one after the other
    (MANY, 'packed', 256, 3, 8),                 # runs of 32 steps
    (MANY, 'packed', 512, 4, 0),                 # runs of 64
    (MANY[::8], 'packed', 512, 4, 1),            # runs of 16, a channel a lane
    ([100] * 40, 'batch', 4100, 4, 0)])          # at most 64 blocks for each of 17 blocks of channels
@pytest.mark.parametrize('dtype', TYPES)
def test_causal_conv_of_many_runs(lengths, kind, D, K, wide, dtype):
    test_causal_conv(D, K, wide, True, True, True, lengths, kind, dtype)


@pytest.mark.parametrize('walk', ['steps', 'sequences'])
def test_offsets_beyond_32_bits_reach_the_kernels(walk):
    """Steps (sequences) just under 2^30 elements apart: taken as they lie, and their offsets pass 2^32 bytes."""
    from paccmann_polymer_amd import state_space as S
    g = torch.Generator(device=DEV).manual_seed(12)
    far, D, N = 2 ** 30 - 64, 64, 16
    T, B = (5, 2) if walk == 'steps' else (2, 5)
    base = torch.empty(4 * far + 16 * D, dtype=torch.bfloat16, device=DEV)

    def view(k, *tail):
        n = (1 if len(tail) == 1 else tail[1])
        near = 8 * D
        t = torch.as_strided(base, (T, B, *tail), (*((far, near) if walk == 'steps' else (near, far)), *([n, 1] if len(tail) == 2 else [1])), k * D)
        t.copy_(randn(g, T, B, *tail, dtype=torch.bfloat16))
        return t
    x, dt, z, dy, dc = (view(k, D) for k in range(5))
    B_, C_ = view(5, 1, N), view(6, 1, N)
    for name, t in (('x', x), ('dt', dt), ('z', z), ('dy', dy), ('dc', dc), ('B', B_), ('C', C_)):
        batch = S._Batch('test', x, None)
        assert batch.take(name, t, tuple(t.shape[2:]), t.dtype).data_ptr() == t.data_ptr()
    A, w = -torch.rand(D, N, generator=g, device=DEV), randn(g, D, 4)

    def both(x, dt, z, B, C, dy, dc):
        leaves = [t.detach().requires_grad_() for t in (x, dt, z, B, C)]
        y, last = S.selective_scan(leaves[0], leaves[1], A, leaves[3], leaves[4], z=leaves[2])
        c, cl = S.causal_conv(leaves[0], w)
        return (y, last, c, cl, *torch.autograd.grad((y, c), leaves, (dy, dc)))

    for a, b in zip(both(x, dt, z, B_, C_, dy, dc), both(*(t.contiguous() for t in (x, dt, z, B_, C_, dy, dc)))):
        assert torch.equal(a, b)


def test_captured_steps_in_place_and_captured_splits():
    """A captured token step whose states are updated where they lie: every replay is one step further; and a captured training pass over sequences
    long enough for splits in both directions."""
    from paccmann_polymer_amd.state_space import causal_conv, causal_conv_step, selective_scan, selective_scan_step
    g = torch.Generator(device=DEV).manual_seed(31)
    B, D, N, K, T = 3, 40, 16, 3, 4
    xs, dts, bs, cs = randn(g, T, B, D), randn(g, T, B, D, scale=0.5), randn(g, T, B, N), randn(g, T, B, N)
    A, w = -torch.rand(D, N, generator=g, device=DEV), randn(g, D, K)
    x, dt, b, c = (t[0].clone() for t in (xs, dts, bs, cs))
    conv, state = torch.zeros(B, K - 1, D, device=DEV), torch.zeros(B, D, N, device=DEV)

    def token(x, dt, b, c, conv, state):
        h, _ = causal_conv_step(x, conv, w, out=conv)
        return selective_scan_step(h, dt, A, b, c, state, out=state)[0]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = token(x, dt, b, c, conv, state)
    eager_conv, eager_state = torch.zeros_like(conv), torch.zeros_like(state)
    conv.zero_(), state.zero_()
    for t in range(T):
        for held, new in ((x, xs), (dt, dts), (b, bs), (c, cs)):
            held.copy_(new[t])
        graph.replay()
        want = token(xs[t], dts[t], bs[t], cs[t], eager_conv, eager_state)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(conv, eager_conv) and torch.equal(state, eager_state)

    lay, p, dy, dlast = scan_case([700, 650, 33], 'packed', 48, 16, 1, torch.float32, True, True, True, True, True)

    def train():
        leaves = {k: v.detach().requires_grad_() for k, v in p.items()}
        h, _ = causal_conv(leaves['x'], torch.ones(48, 5, device=DEV), plan=lay.plan)
        y, last = selective_scan(**{**leaves, 'x': h}, plan=lay.plan)
        return (y.detach(), last.detach(), *torch.autograd.grad((y, last), list(leaves.values()), (dy, dlast)))

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = train()
    base = p['x'].clone()
    for k in range(3):
        p['x'].copy_(base * (1 + 0.25 * k))
        graph.replay()
        want = train()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k

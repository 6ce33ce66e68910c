"""`token_log_probs` and `policy_loss` against their definitions in 64 bits.

Tolerances, in half-steps of fp32 (H = 2^-24).  The exponent of a term is (v - m) times a rounded constant: three roundings, so a
term e^-u is off by at most 3u + 2 (the exponential itself) halves relative, and since sum e^-u u <= log(V) sum e^-u the sum s by
3 log V + 2, plus one half for each addition on a value's way (at most 64 in a thread, 6 across lanes, 16 across waves).  With
V <= 2^18 that is below 130 H: lp is off by at most 130 H, and by one rounding of itself when it is stored.  A gradient
g (onehot - p) has p off by that and by its own exponent's error 3u + 2, where p u <= u e^-u <= 0.37: below |g| (p 140 + 8) H.  bf16
results add one half-step of theirs, 2^-8 relative."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
H = 2.0 ** -24


def make(rows, V, dtype, seed, scale=2.0, ignored=0.2, ld=None, offset=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    ld = V if ld is None else ld
    store = torch.randn(rows * ld + offset, generator=g, device='cuda') * scale
    logits = store.to(dtype)[offset:].view(rows, ld)[:, :V]
    tgt = torch.randint(1 if V > 1 else 0, V, (rows,), generator=g, device='cuda')
    tgt[torch.rand(rows, generator=g, device='cuda') < ignored] = 0
    return logits, tgt, g


def definition(logits, tgt, temperature):
    v = logits.double() / temperature
    lp = torch.log_softmax(v, 1)
    return lp.gather(1, tgt.clamp(0, logits.shape[1] - 1)[:, None])[:, 0], lp.exp()


def close(got, want, tol, dtype):
    if dtype == torch.bfloat16:
        tol = tol * (1 + 2.0 ** -8) + want.abs() * 2.0 ** -8
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float((got.double() - want).abs().max()))


CASES = [(1, 1), (1, 2), (3, 5), (7, 64), (33, 65), (130, 257), (5, 575), (9, 1025), (4, 2050), (3, 8199), (3, 16391), (2, 33001), (2, 70001), (1, 131073)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,V', CASES)
def test_token_log_probs(rows, V, dtype):
    from paccmann_polymer_amd.policy_loss import token_log_probs
    for temperature, ld, offset in ((1.0, V, 0), (0.7, V + 3, 1)):
        logits, tgt, g = make(rows, V, dtype, rows + V, ld=ld, offset=offset)
        use = tgt != 0
        want, p = definition(logits, tgt, temperature)
        x = logits.detach().requires_grad_()
        lp = token_log_probs(x, tgt, temperature=temperature)
        want = torch.where(use, want, 0.0)
        close(lp.detach(), want, 130 * H + H * want.abs(), torch.float32)
        assert torch.equal(lp.detach(), token_log_probs(logits, tgt, temperature=temperature))        # the same with and without a backward
        up = torch.randn(rows, generator=g, device='cuda')
        (d,) = torch.autograd.grad(lp, x, up)
        gr = (torch.where(use, up, 0.0) / temperature).double()[:, None]
        dwant = -p * gr
        dwant.scatter_add_(1, tgt[:, None], gr)
        assert d.dtype == dtype and d.shape == logits.shape
        close(d, dwant, gr.abs() * (140 * p + 8) * H, dtype)


def policy_definition(logits, tgt, old, adv, ref, lo, hi, beta, temperature):
    x = logits.double().requires_grad_()
    use = tgt != 0
    lp = torch.log_softmax(x / temperature, 1).gather(1, tgt[:, None])[:, 0][use]
    A = adv.double()[use]
    ratio = torch.exp(lp - old.double()[use])
    free, held = ratio * A, ratio.clamp(1 - lo, 1 + hi) * A
    pg = -torch.minimum(free, held)
    kl = torch.zeros_like(pg)
    if ref is not None:
        d = ref.double()[use] - lp
        kl = torch.expm1(d) - d
    n = max(1, int(use.sum()))
    loss = (pg.sum() + beta * kl.sum()) / n
    (grad,) = torch.autograd.grad(loss, x) if x.numel() else (x,)
    return loss.detach(), torch.stack([pg.sum() / n, kl.sum() / n, (held < free).sum() / n]).detach(), grad, (pg.abs().sum() / n).detach()


def policy_inputs(logits, tgt, g, lo, hi):
    """Ratios on both sides of the clip's borders, none within 1e-3 of one (a ratio on a border has no gradient to compare)."""
    rows = logits.shape[0]
    lp, _ = definition(logits, tgt, 1.0)
    u = 0.3 * torch.randn(rows, generator=g, device='cuda', dtype=torch.float64)
    for edge in (math.log(1 - lo), math.log(1 + hi)):
        u = torch.where((u - edge).abs() < 1e-3, u + 3e-3, u)
    return (lp - u).float(), torch.randn(rows, generator=g, device='cuda'), (lp + 0.3 * torch.randn(rows, generator=g, device='cuda', dtype=torch.float64)).float()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,V', CASES + [(5000, 40), (20011, 3)])
def test_policy_loss(rows, V, dtype):
    from paccmann_polymer_amd.policy_loss import policy_loss
    lo, hi, beta = 0.2, 0.28, 0.05
    logits, tgt, g = make(rows, V, dtype, rows * 3 + V)
    old, adv, ref = policy_inputs(logits, tgt, g, lo, hi)
    use = (tgt != 0)[:, None]
    for r, b in ((ref, beta), (None, 0.0)):
        loss_w, stats_w, grad_w, size = policy_definition(logits, tgt, old, adv, r, lo, hi, b, 1.0)
        x = logits.detach().requires_grad_()
        loss, stats = policy_loss(x, tgt, old, adv, r, clip_low=lo, clip_high=hi, kl_coef=b)
        # a ratio is off by 130 H relative, a KL term by |e^d - 1| 130 H; each mean is rounded once
        tol = 130 * H * (size + 0.5 + 2 * b) + H
        assert abs(float(loss.detach() - loss_w)) <= float(tol) + H * abs(float(loss_w))
        assert bool(((stats.double() - stats_w).abs() <= tol + H * stats_w.abs()).all()), (stats, stats_w)
        with torch.no_grad():
            again, st2 = policy_loss(logits, tgt, old, adv, r, clip_low=lo, clip_high=hi, kl_coef=b)
        assert torch.equal(again, loss.detach()) and torch.equal(st2, stats)
        (d,) = torch.autograd.grad(loss, x)
        assert d.dtype == dtype and d.shape == logits.shape
        # the row's factor: |ratio A| + b |e^d - 1| over n, off by 130 H of each and two roundings
        n = max(1, int(use.sum()))
        lp, p = definition(logits, tgt, 1.0)
        gmax = torch.exp(lp - old.double()) * adv.double().abs() + (b * torch.exp(ref.double() - lp) if r is not None else 0.0)
        close(d, grad_w, torch.where(use, gmax[:, None] / n * (p * 272 + 140) * H, 0.0), dtype)


def test_policy_loss_upstream_gradient_and_second_backward():
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(50, 70, torch.float32, 1)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    x = logits.detach().requires_grad_()
    loss, _ = policy_loss(x, tgt, old, adv, ref, kl_coef=0.1)
    (d1,) = torch.autograd.grad(loss, x, retain_graph=True)
    keep = d1.clone()
    (d3,) = torch.autograd.grad(loss * -3.0, x, retain_graph=True)
    assert torch.equal(d1, keep)                                    # what was handed out is not touched again
    assert torch.equal(d3, keep * -3.0)
    (d0,) = torch.autograd.grad(loss * 0.0, x)
    assert not bool(d0.any())


def test_rows_that_do_not_count_leak_nothing():
    """NaN and infinities in every input of an ignored row, and infinite logits in a row that counts."""
    from paccmann_polymer_amd.policy_loss import policy_loss, token_log_probs
    inf, nan = float('inf'), float('nan')
    logits, tgt, g = make(12, 33, torch.float32, 2, ignored=0.0)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    tgt[3] = tgt[7] = 0
    logits, old, adv, ref = logits.clone(), old.clone(), adv.clone(), ref.clone()
    logits[5, :20] = -inf                                           # tokens that may not be taken
    tgt[5] = 30
    lp5 = torch.log_softmax(logits[5].double(), 0)[30]
    old[5] = ref[5] = float(lp5)
    want = policy_definition(logits, tgt, old, adv, ref, 0.2, 0.2, 0.1, 1.0)
    logits[3] = nan
    logits[7] = inf
    for t in (old, adv, ref):
        t[3], t[7] = nan, -inf
    x = logits.detach().requires_grad_()
    loss, stats = policy_loss(x, tgt, old, adv, ref, kl_coef=0.1)
    (d,) = torch.autograd.grad(loss, x)
    assert abs(float(loss.detach() - want[0])) <= 130 * H * float(want[3] + 1) + H
    keep = torch.tensor([i for i in range(12) if i not in (3, 7)], device='cuda')
    assert not bool(d[3].any()) and not bool(d[7].any()) and bool(torch.isfinite(d).all())
    assert float((d[keep].double() - want[2][keep]).abs().max()) <= 1e-6
    assert not bool(d[5, :20].any())
    y = logits.detach().requires_grad_()
    lp = token_log_probs(y, tgt)
    assert float(lp[3].detach()) == 0.0 and float(lp[7].detach()) == 0.0
    up = torch.ones(12, device='cuda')
    up[3], up[7] = nan, inf
    (dl,) = torch.autograd.grad(lp, y, up)
    assert not bool(dl[3].any()) and not bool(dl[7].any()) and bool(torch.isfinite(dl).all())


def test_no_row_counts_and_no_rows():
    from paccmann_polymer_amd.policy_loss import policy_loss, token_log_probs
    for rows in (0, 4):
        x = torch.randn(rows, 9, device='cuda', requires_grad=True)
        tgt = torch.zeros(rows, dtype=torch.int64, device='cuda')
        z = torch.zeros(rows, device='cuda')
        loss, stats = policy_loss(x, tgt, z, z, z, kl_coef=0.1)
        assert float(loss.detach()) == 0.0 and not bool(stats.any())
        (d,) = torch.autograd.grad(loss, x)
        assert d.shape == x.shape and not bool(d.any())
        assert not bool(token_log_probs(x, tgt).any())


def test_target_outside_the_vocabulary_is_nan():
    from paccmann_polymer_amd.policy_loss import policy_loss, token_log_probs
    x = torch.randn(4, 9, device='cuda')
    z = torch.zeros(4, device='cuda')
    for bad in (9, -1, 1 << 40):
        tgt = torch.tensor([1, bad, 2, 0], device='cuda')
        lp = token_log_probs(x, tgt)
        assert torch.isnan(lp).tolist() == [False, True, False, False]
        assert bool(torch.isnan(policy_loss(x, tgt, z, z)[0]))
    assert not bool(torch.isnan(token_log_probs(x, torch.tensor([1, -100, 2, 3], device='cuda'), ignore_index=-100)).any())


def test_gradient_against_differences():
    """Central differences of the 64-bit definition at fp32 logits: the gradient is the derivative of this loss and no other's."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(6, 11, torch.float32, 5)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    x = logits.detach().requires_grad_()
    (d,) = torch.autograd.grad(policy_loss(x, tgt, old, adv, ref, kl_coef=0.3)[0], x)
    step = 1e-4
    for i in range(6):
        for j in range(0, 11, 3):
            e = torch.zeros(6, 11, device='cuda', dtype=torch.float64)
            e[i, j] = step
            up = policy_definition(logits.double() + e, tgt, old, adv, ref, 0.2, 0.2, 0.3, 1.0)[0]
            dn = policy_definition(logits.double() - e, tgt, old, adv, ref, 0.2, 0.2, 0.3, 1.0)[0]
            assert abs(float((up - dn) / (2 * step)) - float(d[i, j])) <= 1e-6      # third derivatives below 10, times step^2 / 6; and fp32


def test_other_stream_and_graph_replays():
    """On a side stream, and captured: every replay sees the inputs of its time; eager work runs between the replays."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(300, 575, torch.float32, 8)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    x = logits.clone().requires_grad_()

    def step():
        loss, stats = policy_loss(x, tgt, old, adv, ref, kl_coef=0.1)
        return loss.detach(), stats, torch.autograd.grad(loss, x)[0]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        side = step()
    torch.cuda.current_stream().wait_stream(s)
    eager = step()
    for a, b in zip(side, eager):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        with torch.no_grad():
            x.copy_(logits * (1.0 + 0.1 * k))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), k


def test_reference_without_a_kl_term_cannot_spoil_it():
    """kl_coef 0: a reference score so far off that e^d overflows is in the statistics, not in the loss or its gradient."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(9, 21, torch.float32, 3, ignored=0.0)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    ref[4] = 200.0
    x = logits.detach().requires_grad_()
    loss, stats = policy_loss(x, tgt, old, adv, ref)
    bare, _ = policy_loss(x, tgt, old, adv)
    assert torch.equal(loss, bare) and float(stats[1]) == float('inf')
    (d,) = torch.autograd.grad(loss, x)
    assert bool(torch.isfinite(d).all())


@pytest.mark.parametrize('seed', range(3))
def test_small_kl_terms_keep_their_digits(seed):
    """d of 1e-2 to 1e-5: d^2 / 2 is far below what e^d rounds to in 32 bits."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(64, 50, torch.float32, 20 + seed, ignored=0.0)
    lp, _ = definition(logits, tgt, 1.0)
    ref = (lp + 10.0 ** (-2 - seed)).float()
    d = ref.double() - lp
    want = (torch.expm1(d) - d).mean()
    _, stats = policy_loss(logits, tgt, lp.float(), torch.zeros(64, device='cuda'), ref, kl_coef=1.0)
    # d is off by what lp is, 130 H; the term by d times that, and eight roundings of its series
    assert abs(float(stats[1]) - float(want)) <= float(d.abs().max()) * 130 * H + 8 * H * float(want)


def test_loss_may_be_changed_in_place():
    """`loss /= n` of accumulated steps; and the statistics are memory of their own."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(30, 20, torch.float32, 4)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    x = logits.detach().requires_grad_()
    loss, stats = policy_loss(x, tgt, old, adv, ref, kl_coef=0.1)
    keep = stats.clone()
    (want,) = torch.autograd.grad(loss / 4, x, retain_graph=True)
    loss /= 4
    loss += 1.0
    (d,) = torch.autograd.grad(loss, x)
    assert torch.equal(d, want) and torch.equal(stats, keep) and loss.dim() == 0
    stats.zero_()


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('off', [-float('inf'), -1e9, -200.0, -20.0, -3.0, -0.26, -0.24, 0.24, 0.26, 3.0, 20.0])
def test_kl_gradient_far_from_the_reference(off, dtype):
    """1 - e^d of a reference that all but forbids the taken token, and on both sides of where its series ends."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(12, 33, dtype, 6, ignored=0.0)
    lp, p = definition(logits, tgt, 1.0)
    old, adv = lp.float(), torch.zeros(12, device='cuda')
    ref = (lp + 0.05).float()
    ref[4] = float(lp[4]) + off
    x = logits.detach().requires_grad_()
    loss, _ = policy_loss(x, tgt, old, adv, ref, kl_coef=0.5)
    (d,) = torch.autograd.grad(loss, x)
    grad_w = policy_definition(logits, tgt, old, adv, ref, 0.2, 0.2, 0.5, 1.0)[2]
    e = torch.exp(ref.double() - lp)
    # the row's factor 0.5 (1 - e^d) / n: e^d is off by 130 H of itself (d is off by what lp is) and by H d, and the difference is rounded once
    size = 0.5 / 12 * (e * (130 + (ref.double() - lp).abs().clamp(max=100)) + (e - 1).abs() * (140 * p.amax(1) + 12))
    close(d, grad_w, (size * H)[:, None].expand_as(grad_w), dtype)
    assert bool(torch.isfinite(d).all()) and bool(d[4].any())


def test_no_advantage_and_a_ratio_beyond_fp32():
    """e^(lp - old) overflows; times an advantage of zero it is zero, in the loss and in the gradient."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(9, 21, torch.float32, 3, ignored=0.0)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    old[2], adv[2] = -120.0, 0.0
    old[5], adv[5] = -120.0, -0.0
    x = logits.detach().requires_grad_()
    loss, stats = policy_loss(x, tgt, old, adv, ref, kl_coef=0.1)
    (d,) = torch.autograd.grad(loss, x)
    want = policy_definition(logits, tgt, old, adv, ref, 0.2, 0.2, 0.1, 1.0)
    assert abs(float(loss.detach() - want[0])) <= 130 * H * float(want[3] + 1) + H
    assert bool(((stats.double() - want[1]).abs() <= 130 * H * (want[3] + 1) + H).all())
    assert float((d.double() - want[2]).abs().max()) <= 1e-6


def test_backward_captured_behind_an_eager_forward_pass(monkeypatch):
    """A graph replays its multiplication by the upstream gradient: what the eager forward pass wrote once must not be its operand."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(30, 20, torch.float32, 4)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    x = logits.detach().requires_grad_()
    loss, _ = policy_loss(x, tgt, old, adv, ref, kl_coef=0.1)
    held = loss.grad_fn.grad
    keep = held.clone()
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    (d,) = torch.autograd.grad(loss * 4.0, x)
    assert torch.equal(held, keep) and torch.equal(d, keep * 4.0)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,V', [(12001, 300), (45003, 9), (4201, 3001), (6001, 700)])
def test_more_rows_than_a_launch_holds_at_once(rows, V, dtype):
    """Blocks that go from row to row: what is loaded ahead, a last round that not every group has a row of, sums carried across rows, and
    rows of 256 threads that use their LDS again."""
    test_token_log_probs(rows, V, dtype)
    test_policy_loss(rows, V, dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,V,ld,offset', [(40, 575, 577, 1), (6, 2050, 2053, 3), (1500, 33, 35, 1), (3, 9001, 9003, 5), (1, 140001, 140001, 1)])
def test_policy_gradient_of_a_slice(rows, V, ld, offset, dtype):
    """Logits whose rows begin at other offsets from 16 bytes than the gradient's: the same results as of a copy that lies as the gradient does."""
    from paccmann_polymer_amd.policy_loss import policy_loss
    logits, tgt, g = make(rows, V, dtype, rows + V, ld=ld, offset=offset)
    old, adv, ref = policy_inputs(logits, tgt, g, 0.2, 0.2)
    lp, p = definition(logits, tgt, 1.0)
    loss_w, stats_w, grad_w, size = policy_definition(logits, tgt, old, adv, ref, 0.2, 0.2, 0.05, 1.0)
    x = logits.detach().requires_grad_()
    assert x.data_ptr() % 16 == offset * x.element_size() % 16
    loss, stats = policy_loss(x, tgt, old, adv, ref, kl_coef=0.05)
    (d,) = torch.autograd.grad(loss, x)
    tol = 130 * H * (size + 0.5 + 0.1) + H                              # as in test_policy_loss
    assert abs(float(loss.detach() - loss_w)) <= float(tol) + H * abs(float(loss_w))
    use = (tgt != 0)[:, None]
    gmax = torch.exp(lp - old.double()) * adv.double().abs() + 0.05 * torch.exp(ref.double() - lp)
    close(d, grad_w, torch.where(use, gmax[:, None] / max(1, int(use.sum())) * (p * 272 + 140) * H, 0.0), dtype)


def test_rows_beyond_32_bits():
    """Rows of logits further than 2^32 bytes apart in all: read where they lie, with the results of rows that begin as far from 16 bytes."""
    from paccmann_polymer_amd.policy_loss import policy_loss, token_log_probs
    rows, V, far = 5, 70, 2 ** 30 + 3
    values, tgt, g = make(rows, V, torch.bfloat16, 9, ignored=0.0)
    logits, near = (torch.empty((rows - 1) * ld + V, dtype=torch.bfloat16, device='cuda').as_strided((rows, V), (ld, 1)).copy_(values) for ld in (far, 72 + 3))
    old, adv, ref = policy_inputs(near, tgt, g, 0.2, 0.2)
    out = []
    for t in (logits, near):
        x, y = t.detach().requires_grad_(), t.detach().requires_grad_()
        lp = token_log_probs(x, tgt)
        loss, stats = policy_loss(y, tgt, old, adv, ref, kl_coef=0.1)
        out.append((lp.detach(), loss.detach(), stats, *torch.autograd.grad((lp, loss), (x, y), (adv, torch.ones_like(loss)))))
    for a, b in zip(*out):
        assert torch.equal(a, b)

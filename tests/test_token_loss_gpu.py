"""Token loss kernels against 64-bit arithmetic on the same logits.

Tolerances, with u = 2^-24 (half a step of float32). A term e^(x-m) is off by
the rounding of x-m (u |x-m|), of its product with log2 e (u |x-m| log2 e, in
the exponent, so times ln 2: u |x-m|) and of exp2 (2u): with |x-m| <= R on
the terms that matter, (2R + 2) u relative. Rescaling to a new maximum
repeats that for each of at most log-many rises and each merge; runs of n
values in float32 add n u at the very worst and sqrt(n) u in practice, where
n, a thread's share, is V / 256 or V / 1024. R: terms below e^-16 of the
largest are under 2^-23 of the sum. So s is within
S = (2 * 16 * 4 + V / 256 + 64) u of itself, relative: 192 u for small V,
below 2^-16 throughout these tests (V <= 70001 gives 465 u = 2^-15.1, so
REL = 2^-15 is used for s). log s is then off by REL at most, absolutely,
plus u |log s|, and x_t - m by u |x_t - m|.
"""
import pytest
import torch

from mgwfbp_amd.kernels import token_loss as tl

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
REL = 2.0 ** -15
NEG = float('-inf')
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one class, less than a vector, around vectors and blocks, odd, split rows
SIZES = [(1, 1), (3, 2), (5, 7), (2, 255), (3, 256), (4, 1023), (2, 4096),
         (3, 4097), (700, 1000), (1, 10000), (20, 10001), (2, 50001),
         (1, 70001), (600, 2049)]


def _make(rows, vocab, kind, seed=0, scale=3.0):
    g = torch.Generator().manual_seed(seed * 1000003 + rows * 131 + vocab)
    x = (torch.randn(rows, vocab, generator=g) * scale).to(kind).cuda()
    t = torch.randint(0, vocab, (rows,), generator=g).cuda()
    return x, t


def _exact(x):
    x = x.detach().double()
    # the maximum goes first: beside a row of lowest values log V would be
    # lost in 64 bits too
    x = x - x.amax(1, keepdim=True)
    log = x - x.exp().sum(1, keepdim=True).log()
    p = log.exp()
    h = -(p * log.masked_fill(log == NEG, 0.0)).sum(1)
    return log, p, h


def _near_log(got, want, x):
    """Log probabilities and entropies: REL, and u of what is subtracted."""
    assert got.dtype == torch.float32
    size = x.detach().double().masked_fill(x == NEG, 0.0).abs().amax()
    far = REL + 4 * U * (2 * float(size) + 16)
    off = (got.double() - want).abs()
    worst = float(off.detach().max())
    assert worst <= far, (worst, far)


def _near_grad(got, want, p, coef, kind):
    """A gradient's entry is p (a + b log p) + c: relative 2 REL of the
    magnitudes that go in, and half a step of the type, or half its least
    subnormal."""
    assert got.dtype == kind
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126,
            torch.float16: 2.0 ** -24}[kind]
    far = torch.finfo(kind).eps / 2 * want.abs() + 2 * REL * coef * p + \
        4 * U * coef + tiny
    off = (got.double() - want).abs()
    assert bool((off <= far).all()), float((off - far).max())


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('rows,vocab', SIZES)
def test_log_probs_entropy_and_best(rows, vocab, kind):
    x, t = _make(rows, vocab, kind)
    log, p, h = _exact(x)
    for k in {0, 1, min(5, vocab), min(64, vocab)}:
        r = tl.token_log_probs(x, t, top_k=k)
        _near_log(r.log_probs, log.gather(1, t[:, None])[:, 0], x)
        _near_log(r.entropy, h, x)
        ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
        assert r.top_ids.dtype == torch.int64
        assert torch.equal(r.top_ids, ids)
        if k:
            _near_log(r.top_log_probs, log.gather(1, ids), x)
        assert r.top_log_probs.shape == (rows, k)


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('rows,vocab', SIZES)
def test_log_probs_gradient(rows, vocab, kind):
    x, t = _make(rows, vocab, kind, seed=1)
    x.requires_grad_(True)
    log, p, h = _exact(x)
    g = torch.Generator().manual_seed(9)
    gl = torch.randn(rows, generator=g).cuda()
    ge = torch.randn(rows, generator=g).cuda()
    for use_l, use_e in ((1, 1), (1, 0), (0, 1)):
        r = tl.token_log_probs(x, t)
        outs = [o for o, u in ((r.log_probs, use_l), (r.entropy, use_e))
                if u]
        got, = torch.autograd.grad(
            outs, x, [g for g, u in ((gl, use_l), (ge, use_e)) if u])
        a, b = gl.double()[:, None] * use_l, ge.double()[:, None] * use_e
        want = -p * (a + b * (log + h[:, None]))
        want[torch.arange(rows), t] += a[:, 0]
        coef = a.abs() + b.abs() * (log.abs() + h[:, None].abs() + 1)
        _near_grad(got, want, p, coef, kind)


@pytest.mark.parametrize('wide', [torch.int64, torch.int32])
@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('rows,vocab', SIZES)
def test_cross_entropy(rows, vocab, kind, wide):
    x, t = _make(rows, vocab, kind, seed=2)
    x.requires_grad_(True)
    log, p, _ = _exact(x)
    t[::3] = -100
    if rows == 1:
        t[0] = vocab - 1
    keep = t != -100
    at = torch.where(keep, t, torch.zeros_like(t))
    nll = torch.where(keep, -log.gather(1, at[:, None])[:, 0],
                      torch.zeros((), dtype=torch.float64, device='cuda'))
    n = int(keep.sum())
    hot = torch.zeros_like(p)
    hot[torch.arange(rows), at] = 1.0
    t = t.to(wide)
    each = tl.cross_entropy(x, t, reduction='none')
    _near_log(each, nll, x)
    assert bool((each[~keep] == 0).all())
    w = torch.rand(rows, generator=torch.Generator().manual_seed(3)).cuda()
    for red, coef in (('none', w.double()), ('sum', torch.ones_like(nll)),
                      ('mean', torch.full_like(nll, 1.0 / max(n, 1)))):
        loss = tl.cross_entropy(x, t, reduction=red)
        if red == 'none':
            got, = torch.autograd.grad(loss, x, w)
        else:
            want = nll.sum() / (n if red == 'mean' else 1)
            if n:
                _near_log(loss / (1 if red == 'mean' else n),
                          want / (1 if red == 'mean' else n), x)
            got, = torch.autograd.grad(loss, x)
        if n == 0 and red == 'mean':
            assert torch.isnan(loss)
        c = (coef * keep)[:, None]
        _near_grad(got, (p - hot) * c, p, c, kind)
        assert bool((got[~keep] == 0).all())


@pytest.mark.parametrize('scale', [0.25, 3.0, 65536.0])
@pytest.mark.parametrize('kind', TYPES)
def test_loss_scaled_afterwards(kind, scale):
    """The gradient that comes in is not one: it is rounded once all the
    same."""
    x, t = _make(37, 1003, kind, seed=4)
    x.requires_grad_(True)
    log, p, _ = _exact(x)
    hot = torch.zeros_like(p)
    hot[torch.arange(37), t] = 1.0
    for told in (False, True):
        loss = tl.cross_entropy(x, t, scaled=told) * scale
        got, = torch.autograd.grad(loss, x)
        _near_grad(got, (p - hot) * scale / 37, p,
                   torch.full_like(p, scale / 37), kind)


def test_backward_twice_and_after():
    x, t = _make(33, 515, torch.float32, seed=5)
    x.requires_grad_(True)
    loss = tl.cross_entropy(x, t)
    a, = torch.autograd.grad(loss, x, retain_graph=True)
    b, = torch.autograd.grad(loss, x, torch.tensor(2.0, device='cuda'),
                             retain_graph=True)
    c, = torch.autograd.grad(loss, x, retain_graph=True)
    keep = a.clone()
    a.mul_(7.0)                          # the caller's own by now
    d, = torch.autograd.grad(loss, x)
    assert torch.allclose(b, 2 * keep, rtol=4 * U, atol=0)
    assert torch.allclose(c, keep, rtol=4 * U, atol=0)
    assert torch.allclose(d, keep, rtol=4 * U, atol=0)
    loss = tl.cross_entropy(x, t)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, x, create_graph=True)


def test_logits_changed_before_the_backward():
    x, t = _make(8, 100, torch.float32, seed=6)
    w = torch.ones((), device='cuda', requires_grad=True)
    y = x * w
    loss = tl.cross_entropy(y, t)
    y.detach().add_(1.0)
    with pytest.raises(RuntimeError):
        loss.backward()


def test_gradient_against_differences():
    """One entry at a time, by the plain formula in 64 bits on either
    side."""
    x, t = _make(2, 6, torch.float32, seed=7)
    x.requires_grad_(True)
    r = tl.token_log_probs(x, t)
    got, = torch.autograd.grad((r.log_probs * 2 + r.entropy).sum(), x)
    step = 1e-4
    for i in range(2):
        for j in range(6):
            v = []
            for s in (step, -step):
                y = x.detach().double().clone()
                y[i, j] += s
                log, _, h = _exact(y)
                v.append(float(2 * log[torch.arange(2), t].sum() + h.sum()))
            # third derivatives are below 10, REL is what the kernel may lose
            assert abs((v[0] - v[1]) / (2 * step) - float(got[i, j])) < \
                4 * REL + 10 * step * step


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('vocab', [9, 1000, 40001])
def test_masks(vocab, kind):
    """-inf, the type's lowest value, and rows with nothing left."""
    low = torch.finfo(kind).min
    x, t = _make(6, vocab, kind, seed=8)
    x[0, 3:] = NEG                       # three classes left
    x[1, : vocab - 1] = NEG              # one, the last
    x[2] = low                           # nothing but the lowest value
    x[3, 1:] = low
    x[4] = NEG                           # nothing at all
    t[:] = torch.tensor([1, vocab - 1, 5, 0, 2, 4])
    k = min(5, vocab)
    x.requires_grad_(True)
    r = tl.token_log_probs(x, t, top_k=k)
    keep = [0, 1, 2, 3, 5]
    y = x.detach().double()
    # in the rows that differ from a constant by one value, float32 and
    # 64 bits agree that e^(low - x) is 0
    log, p, h = _exact(y)
    for i in keep:
        assert abs(float(r.log_probs[i].detach()) - float(log[i, t[i]])) < 2 * REL
        assert abs(float(r.entropy[i].detach()) - float(h[i])) < 4 * REL
    ids = torch.sort(x.detach(), dim=1, descending=True, stable=True)[1]
    assert torch.equal(r.top_ids, ids[:, :k])
    assert torch.isnan(r.log_probs[4]) and torch.isnan(r.entropy[4])
    assert r.top_log_probs[0, 3:].tolist() == [NEG] * (k - 3)
    got, = torch.autograd.grad((r.log_probs + r.entropy)[keep].sum(), x)
    assert torch.isfinite(got[keep]).all()
    assert bool((got[0, 3:] == 0).all()) and bool((got[1, :-1] == 0).all())
    # the only class: p = s * fl(1 / s) is 1 within two roundings, u each, and
    # its gradient 1 - p within 2 u, which float16 rounds to u or 2 u
    assert abs(float(got[1, -1])) <= 2 * U
    loss = tl.cross_entropy(x, t, reduction='none')
    got, = torch.autograd.grad(loss[keep].sum(), x)
    assert torch.isfinite(got[keep]).all()
    # the empty row is no fault of its neighbours, and may be ignored
    t[4] = -100
    loss = tl.cross_entropy(x, t)
    assert torch.isfinite(loss)
    got, = torch.autograd.grad(loss, x)
    assert torch.isfinite(got).all() and bool((got[4] == 0).all())


@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('vocab', [2500, 10001, 50001])
def test_peaks_and_offsets(vocab, kind):
    """One logit far above the rest, rows far from zero, and rows whose
    beginning is far below their end. A peaked row's entropy is small, and
    right to a part of itself: H is at least what the peak's own term says."""
    ups = [5.0, 15.0, 20.0, 30.0, 40.0, 42.0, 60.0, 88.0, 90.0, 120.0, 1e4]
    offs = [-1e4, -300.0, -65.0, 65.0, 1e4, 3e6, -3e6, 1e30, -1e30]
    x, t = _make(len(ups) + len(offs) + 3, vocab, kind, seed=18, scale=1.0)
    for i, u in enumerate(ups):
        x[i, vocab // 2 + i] += u
        if i % 2:
            t[i] = vocab // 2 + i
    for i, o in enumerate(offs):
        x[len(ups) + i] += o
    x[-3, : vocab - 100] -= 1e4          # the usual finite masks
    x[-2, : vocab // 2] -= 80.0
    x[-1, ::2] -= 50.0
    x.requires_grad_(True)
    log, p, h = _exact(x)
    r = tl.token_log_probs(x, t)
    lp = log.gather(1, t[:, None])[:, 0]
    # t is off by u |t| and log s by REL, and a product follows
    far = REL + 4 * U * lp.abs()
    assert bool(((r.log_probs.double() - lp).abs() <= far).all())
    # u / s and log2 s are both near 0 in a peaked row: REL is of s - 1
    assert bool(((r.entropy.double() - h).abs()
                 <= 4 * REL * h + 16 * U).all()), \
        ((r.entropy.double() - h).abs() / (4 * REL * h + 16 * U)).max()
    rows = x.size(0)
    hot = torch.zeros_like(p)
    hot[torch.arange(rows), t] = 1.0
    loss = tl.cross_entropy(x, t, reduction='sum')
    want = -lp.sum()
    assert abs(float(loss.detach()) - float(want)) <= \
        rows * REL + 4 * U * float(lp.abs().sum())
    got, = torch.autograd.grad(loss, x)
    one = torch.ones_like(p)
    _near_grad(got, p - hot, p, one, kind)
    got, = torch.autograd.grad(
        tl.cross_entropy(x, t, reduction='none').sum(), x)
    _near_grad(got, p - hot, p, one, kind)


@pytest.mark.parametrize('value', [float('nan'), float('inf')])
def test_rows_that_are_not_finite(value):
    x, t = _make(3, 5000, torch.float32, seed=9)
    x[1, 4321] = value
    r = tl.token_log_probs(x, t, top_k=3)
    ref = torch.log_softmax(x, 1)[torch.arange(3), t]
    assert torch.equal(torch.isnan(r.log_probs), torch.isnan(ref))
    assert torch.isnan(r.entropy).tolist() == [False, True, False]
    assert int(r.top_ids[1, 0]) == 4321
    x.requires_grad_(True)
    got, = torch.autograd.grad(
        tl.cross_entropy(x, t, reduction='none').sum(), x)
    assert torch.isnan(got[1]).all()
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all()


@pytest.mark.parametrize('vocab', [64, 600, 5000, 60001])
@pytest.mark.parametrize('k', [1, 20, 64])
def test_equal_values(vocab, k):
    """Ties, more of them than the search holds: the lowest index first."""
    x = torch.zeros(3, vocab, device='cuda')
    x[1, ::2] = -0.0                     # both zeros are the same value
    x[2] = (torch.arange(vocab, device='cuda') % 3).float()
    r = tl.token_log_probs(x, torch.zeros(3, dtype=torch.long,
                                          device='cuda'), top_k=k)
    ids = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(r.top_ids, ids)
    assert torch.isfinite(r.top_log_probs).all()


def test_targets_outside_the_classes():
    """Nothing is read for them; they are NaN, and their neighbours are
    not."""
    x, t = _make(5, 300, torch.float32, seed=10)
    t[1], t[3] = 300, -7
    x.requires_grad_(True)
    r = tl.token_log_probs(x, t)
    assert torch.isnan(r.log_probs).tolist() == [False, True, False, True,
                                                 False]
    assert torch.isfinite(r.entropy).all()
    each = tl.cross_entropy(x, t, reduction='none')
    assert torch.isnan(each).tolist() == [False, True, False, True, False]
    got, = torch.autograd.grad(each.sum(), x)
    assert torch.isnan(got[1]).all() and torch.isfinite(got[0]).all()
    loss = tl.cross_entropy(x, t)
    assert torch.isnan(loss)
    got, = torch.autograd.grad(loss, x)
    assert torch.isnan(got[3]).all() and torch.isfinite(got[4]).all()


@pytest.mark.parametrize('kind', TYPES)
def test_strides_shapes_and_neighbours(kind):
    big, _ = _make(12, 777, kind, seed=11)
    t = torch.randint(0, 500, (2, 3), device='cuda')
    for x in (big[:6, 5:705].reshape(2, 3, 700),
              big.view(2, 6, 777)[:, ::2, 3:603],
              big.t()[:600].t()[:6].view(2, 3, 600),
              big[:1, :600].expand(6, 600).reshape(2, 3, 600),
              big[:1, :600].expand(2, 3, 600)):
        y = x.detach().clone().contiguous().view(6, -1)
        a = tl.token_log_probs(x, t, top_k=3)
        b = tl.token_log_probs(y, t.view(-1), top_k=3)
        # the order of a row's sums goes by where it begins in memory, so
        # that both are as near to the truth as any other row, not the same
        log, _, h = _exact(y)
        for r in (a, b):
            _near_log(r.log_probs.view(-1), log.gather(
                1, t.view(-1, 1))[:, 0], y)
            _near_log(r.entropy.view(-1), h, y)
            _near_log(r.top_log_probs.view(6, 3),
                      log.gather(1, b.top_ids), y)
        assert torch.equal(a.top_ids.view(6, 3), b.top_ids)
        z = x.detach().requires_grad_(True)
        w = y.detach().requires_grad_(True)
        gz, = torch.autograd.grad(tl.cross_entropy(z, t), z)
        gw, = torch.autograd.grad(tl.cross_entropy(w, t.view(-1)), w)
        assert gz.shape == x.shape
        p = _exact(y)[1]
        hot = torch.zeros_like(p)
        hot[torch.arange(6), t.view(-1)] = 1.0
        for got in (gz.reshape(6, -1), gw):
            _near_grad(got, (p - hot) / 6, p, torch.full_like(p, 1 / 6),
                       kind)


@pytest.mark.parametrize('kind', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('rows,vocab,k', [
    (2, 300001, 64), (1, 1100003, 0), (3, 600007, 64), (600, 131073, 3),
    (2, 2100001, 20)])
def test_long_rows(rows, vocab, k, kind):
    """Rows that no block holds: split, and streamed where the slices are
    still too long."""
    x, t = _make(rows, vocab, kind, seed=17)
    x[0, ::7] = NEG
    t[0] = 1
    x.requires_grad_(True)
    r = tl.token_log_probs(x, t, top_k=k)
    far = 4 * REL                        # a thread's share is V / 4096 here
    for i in range(0, rows, 97):
        log, p, h = _exact(x[i:i + 1])
        assert abs(float(r.log_probs[i].detach())
                   - float(log[0, t[i]])) <= far
        assert abs(float(r.entropy[i].detach()) - float(h[0])) <= far
        ids = torch.sort(x[i].detach(), descending=True,
                         stable=True)[1][:k]
        assert torch.equal(r.top_ids[i], ids)
    loss = tl.cross_entropy(x, t)
    assert abs(float(loss.detach())
               + float(r.log_probs.detach().mean())) <= far
    got, = torch.autograd.grad(loss, x)
    for i in range(0, rows, 97):
        log, p, _ = _exact(x[i:i + 1])
        p[0, t[i]] -= 1.0
        want = p / rows
        off = (got[i].double() - want[0]).abs()
        most = torch.finfo(kind).eps / 2 * want[0].abs() + \
            2 * far * want[0].abs() + 4 * U / rows
        assert bool((off <= most).all())


def test_more_rows_than_a_launch_takes():
    """Refused, not cut short: 2^24 blocks of 256 threads are one thread too
    many."""
    x = torch.zeros(1, 2, dtype=torch.bfloat16, device='cuda')
    x = x.expand(1 << 24, 2)
    t = torch.zeros(1 << 24, dtype=torch.int32, device='cuda')
    with pytest.raises(ValueError):
        tl.token_log_probs(x, t)
    r = tl.token_log_probs(x[:-1], t[:-1])
    assert abs(float(r.entropy[-1]) - 0.6931472) < 1e-6
    assert bool((r.log_probs == r.log_probs[0]).all())


def test_one_row_and_none():
    x, _ = _make(1, 50, torch.float32)
    v = x[0]
    t = torch.tensor(3, device='cuda')
    r = tl.token_log_probs(v, t, top_k=2)
    assert r.log_probs.shape == () and r.top_ids.shape == (2,)
    assert tl.cross_entropy(v, t, reduction='none').shape == ()
    e = torch.zeros(0, 50, device='cuda', requires_grad=True)
    none = torch.zeros(0, dtype=torch.long, device='cuda')
    assert torch.isnan(tl.cross_entropy(e, none))
    assert tl.cross_entropy(e, none, reduction='sum') == 0
    assert tl.cross_entropy(e, none, reduction='none').shape == (0,)
    assert tl.token_log_probs(e, none, top_k=2).top_ids.shape == (0, 2)
    g, = torch.autograd.grad(tl.cross_entropy(e, none, reduction='sum'), e)
    assert g.shape == (0, 50)


def test_expanded_gradient_and_other_type():
    x, t = _make(9, 400, torch.float32, seed=12)
    x.requires_grad_(True)
    a, = torch.autograd.grad(
        tl.cross_entropy(x, t, reduction='none').sum(), x)
    b, = torch.autograd.grad(tl.cross_entropy(x, t, reduction='sum'), x)
    assert torch.allclose(a, b, rtol=8 * U, atol=0)
    r = tl.token_log_probs(x, t)
    c, = torch.autograd.grad(r.log_probs.double().sum(), x)
    assert torch.allclose(c, -b, rtol=8 * U, atol=0)


def test_far_rows():
    """Row offsets past 2^31 elements."""
    rows, vocab = 40000, 60000
    x = torch.zeros(rows, vocab, dtype=torch.bfloat16, device='cuda')
    x[-1], _ = _make(1, vocab, torch.bfloat16, seed=13)
    t = torch.zeros(rows, dtype=torch.long, device='cuda')
    t[-1] = vocab - 3
    t[1:-1] = -100
    last = x[-1:].clone().requires_grad_(True)
    x.requires_grad_(True)
    loss = tl.cross_entropy(x, t, reduction='sum')
    g, = torch.autograd.grad(loss, x)
    l2 = tl.cross_entropy(last, t[-1:], reduction='sum')
    g2, = torch.autograd.grad(l2, last)
    assert torch.allclose(g[-1:].float(), g2.float(),
                          rtol=torch.finfo(torch.bfloat16).eps, atol=0)
    assert bool((g[5] == 0).all()) and bool((g[rows - 2] == 0).all())
    assert tl.token_log_probs(x.detach()[-2:], t[-2:],
                              top_k=1).top_ids[1, 0] == x[-1].argmax()


def test_refusals():
    x, t = _make(4, 30, torch.float32)
    for bad, error in ((dict(top_k=65), ValueError),
                       (dict(top_k=31), ValueError),
                       (dict(top_k=-1), ValueError)):
        with pytest.raises(error):
            tl.token_log_probs(x, t, **bad)
    with pytest.raises(TypeError):
        tl.cross_entropy(x.double(), t)
    with pytest.raises(TypeError):
        tl.cross_entropy(x, t.float())
    with pytest.raises(ValueError):
        tl.cross_entropy(x, t.cpu())
    with pytest.raises(ValueError):
        tl.cross_entropy(x, t[:3])
    with pytest.raises(ValueError):
        tl.cross_entropy(x, t, reduction='max')
    with pytest.raises(ValueError):
        tl.cross_entropy(x[:, :0], t)


def test_module():
    x, t = _make(40, 333, torch.float32, seed=14)
    t[:4] = -100
    for kw in ({}, dict(reduction='sum'), dict(reduction='none'),
               dict(ignore_index=7), dict(label_smoothing=0.1),
               dict(weight=torch.rand(333, device='cuda'))):
        if kw.get('ignore_index') == 7:
            t = t.clamp(min=0)
        a, b = (x.clone().requires_grad_(True) for _ in range(2))
        u = tl.MgxCrossEntropyLoss(**kw)(a, t)
        v = torch.nn.CrossEntropyLoss(**kw)(b, t)
        assert torch.allclose(u, v, rtol=1e-5, atol=1e-5)
        u.sum().backward()
        v.sum().backward()
        assert torch.allclose(a.grad, b.grad, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize('rows,vocab', [(2, 50001), (300, 1001)])
def test_captured(rows, vocab):
    """Forward and backward in one graph, replayed between eager calls."""
    x, t = _make(rows, vocab, torch.bfloat16, seed=15)
    x.requires_grad_(True)

    def call():
        r = tl.token_log_probs(x, t, top_k=4)
        g1, = torch.autograd.grad([r.log_probs, r.entropy], x,
                                  [torch.ones_like(r.log_probs)] * 2)
        loss = tl.cross_entropy(x, t)
        g2, = torch.autograd.grad(loss * 3, x)
        g3, = torch.autograd.grad(tl.cross_entropy(x, t), x)
        return [r.log_probs, r.entropy, r.top_ids, g1, loss, g2, g3]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    for k in range(4):
        y, u = _make(rows, vocab, torch.bfloat16, seed=20 + k)
        with torch.no_grad():
            x.copy_(y)
        t.copy_(u)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


def test_same_bits_every_time():
    x, t = _make(64, 5003, torch.float32, seed=16)
    x.requires_grad_(True)
    first = None
    for _ in range(3):
        loss = tl.cross_entropy(x, t)
        g, = torch.autograd.grad(loss, x)
        if first is None:
            first = (loss, g)
        assert torch.equal(loss, first[0]) and torch.equal(g, first[1])


def _bounds(log):
    """How far a row's sum s may be off, relative, and M, the mean distance
    from the maximum. Each term of s is off by 4 u and by 2 u of its distance
    from the maximum, and on its way into s it is rounded at most A times: a
    thread adds up at most 256 elements here, and twelve steps of the merges
    take four roundings each. Roundings of a sum with the largest term in it
    are no larger than what is added to it, so for a row with all but q of
    its mass in one class they come to q at most."""
    a = 320
    p = log.exp()
    best = log.amax(1)
    q = (1.0 - best.exp()).clamp(min=0.0)
    far = torch.minimum(a * U * torch.ones_like(q), q) + a * U * q + 8 * U
    m = -(p * (log - best[:, None]).masked_fill(log == NEG, 0.0)).sum(1)
    return far, m, a


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('vocab', [2, 5, 9, 15, 16, 300, 2500, 10001, 50001,
                                   100003, 400003, 2100001])
def test_statistics_of_peaked_rows(vocab, kind):
    """A class far above the rest, wherever it stands, as the target and not:
    the log probability is 0 at most, the entropy 0 at least, and both, the
    loss and its gradient, are right to a few roundings of their own size,
    which they are only if the sums are taken against a reference near the
    row's maximum (beside one that is 20 below it, 30 u of a loss near 0 are
    lost). t is within 2 u of itself and log2 s within 2, and a difference
    follows: 6 u of the log probability."""
    ups = [0.0, 0.5, 3.0, 9.0, 16.3, 21.0, 26.0, 30.0, 39.0, 50.0, 88.0]
    places = [vocab - 1, vocab // 2, vocab // 3]
    if vocab > 200000:
        ups, places = ups[4:8], places[:2]
    x, t = _make(len(ups) * len(places), vocab, kind, seed=30, scale=0.5)
    for i, u in enumerate(ups):
        for j, at in enumerate(places):
            row = i * len(places) + j
            x[row, at] = u + 1.0
            t[row] = at if (i + j) % 3 else 1
    x.requires_grad_(True)
    r = tl.token_log_probs(x.detach(), t, top_k=1)
    each = tl.cross_entropy(x, t, reduction='none').detach()
    for i in range(x.size(0)):
        log, p, h = _exact(x[i:i + 1])
        far, m, a = _bounds(log)
        far, m, h = float(far), float(m), float(h)
        lp = float(log[0, t[i]])
        near = far + 6 * U * abs(lp)
        assert float(r.log_probs[i]) <= 0.0
        assert abs(float(r.log_probs[i]) - lp) <= near, (i, lp)
        assert float(r.top_log_probs[i, 0]) <= 0.0
        top = float(log.max())
        assert abs(float(r.top_log_probs[i, 0]) - top) <= \
            far + 6 * U * abs(top)
        assert float(r.entropy[i]) >= 0.0
        assert abs(float(r.entropy[i]) - h) <= \
            far + 8 * U * h + (a + 16) * U * m, (i, h)
        y = x.detach()[i:i + 1].requires_grad_(True)
        loss = tl.cross_entropy(y, t[i:i + 1])
        for got in (float(loss.detach()), float(each[i])):
            assert got >= 0.0
            assert abs(got + lp) <= near, (i, got, -lp)
        got, = torch.autograd.grad(loss, y)
        # p is off as s is, and by 2 u of its exponent: its distance from the
        # maximum, or from a reference up to 18 binary orders below that
        want = p.clone()
        want[0, t[i]] -= 1.0
        off = (far + (16 + 2 * 18) * U) * p + 2 * U * p * log.abs().clamp(
            max=1e4) + (torch.finfo(kind).eps / 2 + 2 * U) * want.abs() + \
            {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126,
             torch.float16: 2.0 ** -24}[kind]
        assert bool(((got.double() - want).abs() <= off).all()), i


# The module stands where nn.CrossEntropyLoss stood: what could be done with
# it has to go on. REL covers the sums of float32 on either side.

@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('vocab', [7, 2500])
def test_module_has_higher_derivatives(vocab, reduction):
    x, t = _make(6, vocab, torch.float32, seed=40, scale=1.0)
    t[2] = -100
    w = torch.rand(6, device='cuda') + 0.5
    v = torch.randn(6, vocab, device='cuda')
    out = []
    for loss, kind in ((tl.MgxCrossEntropyLoss(reduction=reduction), x.dtype),
                       (torch.nn.CrossEntropyLoss(reduction=reduction),
                        torch.float64)):
        y = x.to(kind).requires_grad_(True)
        k = w.to(kind).requires_grad_(True)
        l = loss(y, t)
        l = (l * (k if reduction == 'none' else k.sum())).sum()
        g, = torch.autograd.grad(l, y, create_graph=True)
        hx, hk = torch.autograd.grad((g * v).sum(), (y, k),
                                     create_graph=True)
        i, = torch.autograd.grad((hx * v).sum(), y)
        out.append([z.detach().double() for z in (g, hx, hk, i)])
    for a, b in zip(*out):
        assert torch.allclose(a, b, rtol=4 * REL,
                              atol=4 * REL * float(b.abs().max()))
    assert bool((out[0][0][2] == 0).all()) and bool((out[0][1][2] == 0).all())


def test_module_first_derivative_with_a_graph():
    """create_graph=True changes nothing in the gradient itself, masked
    classes and ignored rows that are not finite among it."""
    x, t = _make(5, 1003, torch.bfloat16, seed=41)
    x[0, 5:] = NEG
    t[0] = 2
    x[3] = float('nan')
    t[3] = -100
    x.requires_grad_(True)
    loss = tl.MgxCrossEntropyLoss()(x, t)
    a, = torch.autograd.grad(loss, x, create_graph=True)
    b, = torch.autograd.grad(tl.MgxCrossEntropyLoss()(x, t), x)
    assert torch.allclose(a.detach().float(), b.float(),
                          rtol=torch.finfo(torch.bfloat16).eps, atol=0)
    v = torch.randn(5, 1003, device='cuda').bfloat16()
    h, = torch.autograd.grad((a * v).sum(), x)
    assert torch.isfinite(h).all()
    assert bool((h[3] == 0).all()) and bool((h[0, 5:] == 0).all())


def test_module_under_transforms():
    x, t = _make(12, 50, torch.float32, seed=42)
    a, b = tl.MgxCrossEntropyLoss(), torch.nn.CrossEntropyLoss()
    v = torch.randn_like(x)
    close = dict(rtol=1e-5, atol=1e-6)
    assert torch.allclose(torch.func.grad(lambda y: a(y, t))(x),
                          torch.func.grad(lambda y: b(y, t))(x), **close)
    assert torch.allclose(
        torch.func.vmap(a)(x.view(3, 4, 50), t.view(3, 4)),
        torch.func.vmap(b)(x.view(3, 4, 50), t.view(3, 4)), **close)
    for p, q in zip(torch.func.jvp(lambda y: a(y, t), (x,), (v,)),
                    torch.func.jvp(lambda y: b(y, t), (x,), (v,))):
        assert torch.allclose(p, q, **close)
    y, u = _make(12, 50, torch.float32, seed=43)
    traced = torch.jit.trace(a, (x, t))
    assert torch.allclose(traced(y, u), b(y, u), **close)
    compiled = torch.compile(a, fullgraph=True, backend='eager')
    assert torch.allclose(compiled(y, u), b(y, u), **close)
    assert torch.allclose(a(y, u), b(y, u), **close)


def test_functions_refuse_to_be_traced():
    """A trace would not see the kernels, and its outputs would not be
    computed."""
    x, t = _make(3, 20, torch.float32)
    for call in (lambda x, t: tl.cross_entropy(x, t),
                 lambda x, t: tl.token_log_probs(x, t).log_probs):
        with pytest.raises(RuntimeError):
            torch.jit.trace(call, (x, t))


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('rows,vocab', [(512, 3), (512, 17), (512, 256),
                                        (700, 2500), (700, 10000),
                                        (256, 32771), (64, 50001)])
def test_to_a_few_roundings(rows, vocab, kind):
    """Ordinary rows, closer than REL. An element passes at most the adds of
    its thread's 65 elements and 24 more in the merges, 2 u for its own
    exponential, and 2 u of its distance from the maximum, 2 M in the mean:
    s is within (min(vocab, 65) + 28 + 3 M) u. A log probability and an
    entropy add the roundings of 6 u of their size. That is the worst: errors
    of both signs add up like the root of their number, 10 u for 89 of them,
    and what always has the same sign, of log2 e and of the exponential, is
    2 u + M u / 4, so over all rows the root mean square is held to half of
    that worst or less."""
    x, t = _make(rows, vocab, kind, seed=50, scale=2.0)
    x.requires_grad_(True)
    log, p, h = _exact(x)
    best = log.amax(1, keepdim=True)
    m = -(p * (log - best)).sum(1).detach()
    lp = log.gather(1, t[:, None])[:, 0].detach()
    h = h.detach()
    adds = min(vocab, 65) + 28
    r = tl.token_log_probs(x.detach(), t)
    each = tl.cross_entropy(x.detach(), t, reduction='none')
    for got, want, terms in ((r.log_probs, lp, 0.0), (each, -lp, 0.0),
                             (r.entropy, h, m * adds)):
        off = (got.double() - want).abs()
        worst = (adds + 3 * m + 6 * want.abs() + terms) * U
        assert bool((off <= worst).all()), float((off / worst).max())
        mean = (12 + adds ** 0.5 + m + 3 * want.abs() + terms / 4) * U
        assert float((off / mean).square().mean()) <= 1.0


def test_module_refuses_an_unknown_reduction():
    x, t = _make(3, 20, torch.float32)
    loss = tl.MgxCrossEntropyLoss()
    loss.reduction = 'max'
    with pytest.raises(ValueError):
        loss(x, t)

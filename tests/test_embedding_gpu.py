"""Embedding kernels against 64-bit arithmetic.

Tolerances, with u = 2^-24. The output is one product in float32 (u) rounded
to the weight's type (eps / 2), of a scale rounded to float32 (u). A row of
the gradient adds up c rows in float32, in any grouping: off by at most
c u times the sum of the magnitudes; then the scale (2u) and the type's
rounding (eps / 2); where the type has subnormals, half the least of them.
"""
import math

import pytest
import torch

from mgwfbp_amd.kernels import embedding as em

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF, FH]
TINY = {F32: 2.0 ** -149, BF: 2.0 ** -133, FH: 2.0 ** -24}


def _tokens(n, vocab, how, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + n * 31 + vocab)
    if how == 'even':
        t = torch.randint(0, vocab, (n,), generator=g)
    elif how == 'text':
        u = torch.rand(n, generator=g, dtype=torch.float64)
        t = (torch.exp(u * math.log(vocab)).long() - 1).clamp(0, vocab - 1)
    elif how == 'same':
        t = torch.full((n,), vocab - 1)
    else:                                # runs that end at and around chunks
        t = torch.arange(n) // 32 % vocab
    return t.cuda()


def _weight(vocab, dim, kind, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(vocab, dim, generator=g).to(kind).cuda()


def _check_out(y, t, w, scale):
    assert y.dtype == w.dtype and y.shape == t.shape + w.shape[1:]
    want = w.detach().double()[t] * scale
    far = (torch.finfo(w.dtype).eps / 2 + 2 * U) * want.abs() + TINY[w.dtype]
    if scale == 1.0:
        assert torch.equal(y, w[t])
    assert y.numel() == 0 or bool(((y.double() - want).abs() <= far).all())


def _check_grad(got, t, dout, vocab, scale, pad=None):
    kind, dim = dout.dtype, dout.shape[-1]
    assert got.dtype == kind and got.shape == (vocab, dim)
    t = t.reshape(-1)
    d = dout.reshape(-1, dim).double()
    if vocab * dim < 1 << 23:            # one after another, on the CPU
        t, d, got = t.cpu(), d.cpu(), got.cpu()
    keep = torch.ones_like(t, dtype=torch.bool) if pad is None \
        else t != pad % vocab
    want = torch.zeros(vocab, dim, dtype=torch.float64, device=t.device)
    size = torch.zeros_like(want)
    want.index_add_(0, t[keep], d[keep])
    size.index_add_(0, t[keep], d[keep].abs())
    count = torch.bincount(t[keep], minlength=vocab).double()[:, None]
    far = abs(scale) * ((count + 3) * U * size
                        + torch.finfo(kind).eps / 2 * want.abs()) \
        * (1 + 2 ** -7) + TINY[kind]
    off = (got.double() - want * scale).abs()
    assert bool((off <= far).all()), float((off - far).max())
    gone = count[:, 0] == 0
    assert bool((got[gone] == 0).all())


def _both(t, w, scale, pad=None, seed=5, dout=None):
    w = w.detach().requires_grad_(True)
    y = em.embedding(t, w, scale=scale, padding_idx=pad)
    _check_out(y.detach(), t, w.detach(), scale)
    if dout is None:
        g = torch.Generator().manual_seed(seed)
        dout = torch.randn(y.shape, generator=g).to(w.dtype).cuda()
    got, = torch.autograd.grad(y, w, dout)
    _check_grad(got, t, dout, w.size(0), scale, pad)
    return got


@pytest.mark.parametrize('kind', TYPES)
@pytest.mark.parametrize('n,vocab,dim', [
    (1, 1, 1), (1, 10, 3), (2, 5, 8), (7, 3, 33), (64, 100, 64),
    (65, 100, 255), (700, 10000, 150), (1000, 17, 512), (1024, 65535, 4),
    (1025, 65536, 5), (4096, 300, 7), (4097, 1000, 12)])
@pytest.mark.parametrize('how', ['even', 'text', 'same', 'runs'])
def test_sizes(n, vocab, dim, how, kind):
    _both(_tokens(n, vocab, how), _weight(vocab, dim, kind),
          math.sqrt(dim) if n % 2 else 1.0)


@pytest.mark.parametrize('n,vocab,dim', [
    (16384, 70000, 24), (16385, 70000, 24), (16384, 1 << 19, 2),
    (300, 1 << 25, 1), (20000, (1 << 24) + 3, 1), (50001, 1000, 9),
    (140000, 257, 3), (16381, 5001, 513)])
@pytest.mark.parametrize('how', ['even', 'text', 'same', 'runs'])
def test_large(n, vocab, dim, how):
    _both(_tokens(n, vocab, how), _weight(vocab, dim, F32), 0.5)


def test_very_many_tokens():
    n = 1 << 21
    _both(_tokens(n, 3000, 'text'), _weight(3000, 4, BF), 1.0)


@pytest.mark.parametrize('pad', [0, 4, -1])
def test_padding(pad):
    t = _tokens(999, 50, 'text')
    t[900:] = pad % 50
    got = _both(t, _weight(50, 40, F32), 2.0, pad=pad % 50)
    assert bool((got[pad] == 0).all())
    t[:] = pad % 50                      # nothing but padding
    got = _both(t, _weight(50, 40, F32), 2.0, pad=pad)
    assert bool((got == 0).all())


@pytest.mark.parametrize('wide', [torch.int64, torch.int32])
def test_shapes_types_and_strides(wide):
    w = _weight(37, 20, F32)
    base = _tokens(240, 37, 'even').to(wide)
    for t in (base.view(4, 60), base.view(4, 60).t(), base[::3],
              base.view(2, 3, 40), base[0], base[:0], base.view(4, 60)[:, :0]):
        y = em.embedding(t, w)
        assert torch.equal(y, w[t.long()]) and y.shape == t.shape + (20,)
        v = w.clone().requires_grad_(True)
        y = em.embedding(t, v, scale=3.0)
        d = torch.randn(y.shape, device='cuda')
        got, = torch.autograd.grad(y, v, d)
        _check_grad(got, t.long(), d, 37, 3.0)


@pytest.mark.parametrize('kind', TYPES)
def test_weight_and_gradient_layouts(kind):
    """Rows with gaps, a transposed table, odd offsets; expanded and
    transposed gradients."""
    big = _weight(60, 71, kind, seed=3)
    t = _tokens(130, 50, 'text')
    for w in (big[:50, 3:36], big[5:55, 1:], big.t()[:50, :33]):
        w = w.detach()
        v = w.requires_grad_(True)
        y = em.embedding(t, v, scale=1.5)
        _check_out(y.detach(), t, v.detach(), 1.5)
        n, d = y.shape
        for dout in (torch.ones(1, 1, dtype=kind, device='cuda')
                     .expand(n, d),
                     torch.randn(d, n, device='cuda').to(kind).t(),
                     torch.randn(n, d + 9, device='cuda').to(kind)[:, 4:4 + d]
                     ):
            got, = torch.autograd.grad(y, v, dout, retain_graph=True)
            _check_grad(got, t, dout, 50, 1.5)


def test_tokens_outside_the_table():
    """Nothing is read for them: NaN out, no gradient, neighbours as they
    were."""
    w = _weight(30, 19, F32).requires_grad_(True)
    t = torch.tensor([3, 30, -1, 29, 1 << 40, -(1 << 62), 0], device='cuda')
    y = em.embedding(t, w)
    bad = torch.tensor([False, True, True, False, True, True, False],
                       device='cuda')
    assert torch.isnan(y[bad]).all()
    assert torch.equal(y[~bad], w.detach()[t[~bad]])
    d = torch.randn(7, 19, device='cuda')
    got, = torch.autograd.grad(y, w, d)
    _check_grad(got, t[~bad], d[~bad], 30, 1.0)


def test_far_rows():
    """Offsets past 2^31 elements, in the table and in its gradient."""
    vocab, dim = 1100000, 2048
    w = torch.zeros(vocab, dim, dtype=BF, device='cuda')
    t = torch.tensor([vocab - 1, 5, vocab - 2, vocab - 1], device='cuda')
    w[t] = torch.randn(4, dim, device='cuda').to(BF)
    w.requires_grad_(True)
    y = em.embedding(t, w)
    assert torch.equal(y, w.detach()[t])
    d = torch.randn(4, dim, device='cuda').to(BF)
    got, = torch.autograd.grad(y, w, d)
    assert torch.equal(got[vocab - 2], d[2]) and torch.equal(got[5], d[1])
    both = d[0].double() + d[3].double()
    assert bool(((got[vocab - 1].double() - both).abs()
                 <= 2.0 ** -8 * both.abs() + 2 * U).all())
    assert float(got[1 << 20].abs().sum()) == 0


def test_gradient_against_differences():
    w = _weight(6, 5, F32).requires_grad_(True)
    t = torch.tensor([1, 4, 1, 0], device='cuda')
    c = torch.randn(4, 5, device='cuda')
    got, = torch.autograd.grad((em.embedding(t, w, scale=1.7) * c).sum(), w)
    for i in range(6):
        for j in range(5):
            v = []
            for s in (1.0, -1.0):        # linear: any step is exact
                y = w.detach().double().clone()
                y[i, j] += s
                v.append(float((y[t] * 1.7 * c.double()).sum()))
            assert abs((v[0] - v[1]) / 2 - float(got[i, j])) < 1e-5


def test_same_bits_every_time():
    t = _tokens(5000, 40, 'text')
    w = _weight(40, 130, F32).requires_grad_(True)
    d = torch.randn(5000, 130, device='cuda')
    first, = torch.autograd.grad(em.embedding(t, w), w, d)
    for _ in range(3):
        again, = torch.autograd.grad(em.embedding(t, w), w, d)
        assert torch.equal(first, again)


@pytest.mark.parametrize('n', [50, 5000, 20000])
def test_captured(n):
    t = _tokens(n, 500, 'text')
    w = _weight(500, 36, F32).requires_grad_(True)
    d = torch.randn(n, 36, device='cuda')

    def call():
        y = em.embedding(t, w, scale=2.0)
        return y.detach(), torch.autograd.grad(y, w, d)[0]

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
        t.copy_(_tokens(n, 500, ['even', 'text', 'same', 'runs'][k], seed=k))
        d.copy_(torch.randn(n, 36, device='cuda'))
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, call()):
            assert torch.equal(a, b)


def test_refusals():
    w = _weight(9, 4, F32)
    t = torch.tensor([1, 2], device='cuda')
    for error, call in (
            (TypeError, lambda: em.embedding(t, w.double())),
            (TypeError, lambda: em.embedding(t.float(), w)),
            (ValueError, lambda: em.embedding(t.cpu(), w)),
            (ValueError, lambda: em.embedding(t, w[0])),
            (ValueError, lambda: em.embedding(t, w, padding_idx=9)),
            (ValueError, lambda: em.embedding(t, w, padding_idx=-10))):
        with pytest.raises(error):
            call()
    w.requires_grad_(True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(em.embedding(t, w).sum(), w, create_graph=True)


def test_module():
    t = _tokens(77, 31, 'text').view(7, 11)
    for kw in ({}, dict(padding_idx=2), dict(scale_grad_by_freq=True),
               dict(max_norm=0.5)):
        torch.manual_seed(1)
        a = em.MgxEmbedding(31, 12, **kw).cuda()
        torch.manual_seed(1)
        b = torch.nn.Embedding(31, 12, **kw).cuda()
        d = torch.randn(7, 11, 12, device='cuda')
        ya, yb = a(t), b(t)
        assert torch.equal(ya, yb)
        ya.backward(d)
        yb.backward(d)
        assert torch.allclose(a.weight.grad, b.weight.grad, rtol=1e-5,
                              atol=1e-5)
    c = em.MgxEmbedding(31, 12, scale=3.0).cuda()
    _check_out(c(t).detach(), t, c.weight.detach(), 3.0)


def test_together_a_language_model_step():
    """Embedding, loss and clipped update of the word-level model, as
    DLTrainer and the single-process entry run them, against torch's own
    pieces on the same weights."""
    from mgwfbp_amd.distributed_optimizer import DistributedOptimizer
    from mgwfbp_amd.kernels.token_loss import MgxCrossEntropyLoss
    from mgwfbp_amd.models import lstm
    sides = []
    for own in (True, False):
        torch.manual_seed(2)
        net = lstm(vocab_size=501, embedding_dim=40, hidden_dim=40,
                   batch_size=3, dropout=0.0)
        if not own:
            plain = torch.nn.Embedding(501, 40)
            plain.load_state_dict(net.embedding.state_dict())
            net.embedding = plain
        net = net.cuda()
        sides.append([net, MgxCrossEntropyLoss() if own
                      else torch.nn.CrossEntropyLoss(), None])
    for i, side in enumerate(sides):
        net = side[0]
        opt = torch.optim.SGD(net.parameters(), lr=2.0)
        side[2] = DistributedOptimizer(
            opt, named_parameters=list(net.named_parameters())) \
            if i == 0 else opt
    g = torch.Generator().manual_seed(4)
    losses = []
    for step in range(3):
        x = torch.randint(0, 501, (3, 9), generator=g).cuda()
        y = torch.randint(0, 501, (3, 9), generator=g).cuda()
        got = []
        for i, (net, crit, opt) in enumerate(sides):
            opt.zero_grad()
            out, _ = net(x, net.init_hidden())
            loss = crit(out.view(-1, 501), y.view(-1))
            loss.backward()
            if i == 0:
                opt.step(max_grad_norm=0.25)
            else:
                torch.nn.utils.clip_grad_norm_(net.parameters(), 0.25)
                opt.step()
            got.append(loss.detach())
        losses.append(got)
    for a, b in losses:
        assert torch.allclose(a, b, rtol=1e-4)
    for p, q in zip(sides[0][0].parameters(), sides[1][0].parameters()):
        assert torch.allclose(p, q, rtol=1e-3, atol=1e-5)


@pytest.mark.skip(reason='a run of all GPU tests with this one in it ended '
                  'in a GPU memory fault or a hung queue, and its cause is '
                  'not known; alone it had passed. It stays off the GPU '
                  'until the cause is shown.')
def test_together_the_trainer():
    """DLTrainer on the word-level model: the embedding, the loss and the
    clipped update in training, the log probabilities in test()."""
    from mgwfbp_amd.distributed_optimizer import DistributedOptimizer
    from mgwfbp_amd.dl_trainer import DLTrainer
    from mgwfbp_amd.kernels.token_loss import MgxCrossEntropyLoss
    torch.manual_seed(0)
    t = DLTrainer(0, 1, dist=False, batch_size=4, is_weak_scaling=True,
                  ngpus=1, data_dir='', dataset='ptb', dnn='lstm', lr=1.0,
                  nworkers=1, prefix='t', synthetic=True)
    assert isinstance(t.net.embedding, em.MgxEmbedding)
    assert isinstance(t.criterion, MgxCrossEntropyLoss)
    opt = DistributedOptimizer(
        t.optimizer, named_parameters=list(t.net.named_parameters()))
    t.update_optimizer(opt)
    before = [p.detach().clone() for p in t.net.parameters()]
    hidden = t.net.init_hidden()
    for _ in range(2):
        opt.zero_grad()
        _, hidden = t.train(1, hidden=hidden)
        t.update_model(max_grad_norm=0.25)
    moved = [p.detach() - b for p, b in zip(t.net.parameters(), before)]
    assert all(torch.isfinite(m).all() for m in moved)
    # two updates with lr 1 and gradients of norm at most 0.25 each
    norm = sum(float(m.double().square().sum()) for m in moved) ** 0.5
    assert 0.0 < norm <= 0.5 * (1 + 1e-4)
    t.testloader = [b for b, _ in zip(t.testloader, range(2))]
    ppl = t.test(0)
    t.net.eval()
    total = 0.0
    with torch.no_grad():
        for x, y in t.testloader:
            out, _ = t.net(x.cuda(), t.net.init_hidden())
            total += torch.nn.functional.cross_entropy(
                out.view(-1, 10000), y.cuda().view(-1)).item()
    assert abs(math.log(ppl) - total / 2) < 1e-4
    assert 0.0 <= t.top5_accuracy <= 1.0 and t.mean_entropy > 0.0


# The module is in a model, in the place of nn.Embedding: what could be done
# with that model has to go on. Products and sums of a few terms in float32,
# on either side: U for each.

def _pair(**kw):
    """An MgxEmbedding and torch's with the same weights, and tokens."""
    torch.manual_seed(6)
    a = em.MgxEmbedding(13, 5, **kw).cuda()
    b = torch.nn.Embedding(13, 5, **kw).cuda()
    b.load_state_dict(a.state_dict())
    return a, b, _tokens(40, 13, 'text').view(4, 10)


@pytest.mark.parametrize('pad', [None, 1])
@pytest.mark.parametrize('scale', [1.0, 2.0])
def test_module_has_higher_derivatives(pad, scale):
    a, b, t = _pair(padding_idx=pad)
    a.scale = scale
    c = torch.randn(4, 10, 5, device='cuda')
    v = torch.randn(13, 5, device='cuda')
    out = []
    for m, k in ((a, 1.0), (b, scale)):
        y = ((m(t) * k) ** 3 * c).sum()
        g, = torch.autograd.grad(y, m.weight, create_graph=True)
        h, = torch.autograd.grad((g * v).sum(), m.weight, create_graph=True)
        i, = torch.autograd.grad((h * v).sum(), m.weight)
        out.append((g.detach(), h.detach(), i))
    for x, y in zip(*out):
        assert torch.allclose(x, y, rtol=1e-5, atol=1e-4)
        if pad is not None:
            assert bool((x[pad] == 0).all())


def test_module_under_transforms():
    """torch.func, forward-mode differentiation, tracing, compiling and
    tensors without data see torch's own embedding."""
    a, b, t = _pair()
    w = a.weight.detach()

    def total(m):
        return lambda w: (torch.func.functional_call(
            m, {'weight': w}, (t,)) ** 2).sum()

    assert torch.allclose(torch.func.grad(total(a))(w),
                          torch.func.grad(total(b))(w), rtol=1e-5)
    ws = torch.randn(3, 13, 5, device='cuda')
    assert torch.allclose(torch.func.vmap(total(a))(ws),
                          torch.func.vmap(total(b))(ws), rtol=1e-5)
    v = torch.randn(13, 5, device='cuda')
    for x, y in zip(torch.func.jvp(total(a), (w,), (v,)),
                    torch.func.jvp(total(b), (w,), (v,))):
        assert torch.allclose(x, y, rtol=1e-5)
    traced = torch.jit.trace(a, (t,))
    u = (t + 1) % 13
    assert torch.equal(traced(u), b(u))
    compiled = torch.compile(a, fullgraph=True, backend='eager')
    assert torch.equal(compiled(u), b(u))
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(allow_non_fake_inputs=True) as mode:
        y = a(mode.from_tensor(t))
    assert y.shape == (4, 10, 5)
    assert torch.equal(a(t), b(t))


def test_function_refuses_to_be_traced():
    """A trace would not see the kernel, and its outputs would not be
    computed."""
    w, t = _weight(9, 4, F32), torch.tensor([1, 2], device='cuda')
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda t: em.embedding(t, w), (t,))


@pytest.mark.parametrize('n,vocab', [
    (1024, 511), (1024, 512), (1000, 40),       # sorted, and not, in one block
    (2000, (1 << 21) + 5), (4096, 1 << 20),     # words of 64 bits, four each
    (4097, (1 << 19) - 1), (1025, 1 << 31 >> 9)])
@pytest.mark.parametrize('how', ['even', 'text', 'same'])
def test_at_the_sorts_borders(n, vocab, how):
    _both(_tokens(n, vocab, how), _weight(vocab, 3, BF), 1.0)

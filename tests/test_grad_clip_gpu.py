"""Global-norm clipping kernels against 64-bit arithmetic.

Tolerances. The norm is a sum of at most n squares in 64 bits, off by less
than n * 2^-53, rounded once to float32: half a step, 2^-24, and a little. A
clipped value is g * f with f rounded to float32 (2^-24), the product rounded
to float32 (2^-24), and to the gradient's type (eps / 2); where that type
has subnormals, half the least of them.
"""
import pytest
import torch

from mgwfbp_amd import kernels as K
from mgwfbp_amd.kernels import grad_clip as gc

pytestmark = pytest.mark.gpu

F32, BF, FH = torch.float32, torch.bfloat16, torch.float16
HALF = 2.0 ** -24


def _grads(shapes, types, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=g) * scale).to(t).cuda()
            for s, t in zip(shapes, types)]


def _exact(grads, max_norm, eps=1e-6):
    norm = sum(float(g.double().square().sum()) for g in grads) ** 0.5
    f = min(1.0, max_norm / (norm + eps))
    return [g.double() * f for g in grads], norm


def _check(got, want, like):
    for g, w, t in zip(got, want, like):
        assert g.dtype == t.dtype and g.shape == t.shape
        tiny = {F32: 2.0 ** -149, BF: 2.0 ** -133, FH: 2.0 ** -24}[g.dtype]
        far = torch.finfo(g.dtype).eps / 2 + 2.1 * HALF
        off = (g.double() - w).abs() - far * w.abs() - tiny
        assert g.numel() == 0 or float(off.max()) <= 0, float(off.max())


def _check_norm(norm, want):
    assert norm.dtype == F32 and norm.shape == ()
    assert abs(float(norm) - want) <= 1.01 * HALF * want + 2.0 ** -149


LISTS = [
    ([(1,)], [F32]),
    ([(3,), (5, 7), (1,)], [F32, BF, FH]),
    ([(16384,), (16385,), (16383,)], [F32, F32, F32]),
    ([(129, 1023), (0,), (7, 11, 13)], [BF, F32, FH]),
    ([(1000003,)], [BF]),
    ([(i * 37 + 1,) for i in range(121)], [F32, BF, FH] * 40 + [F32]),
    ([(17,)] * 250, [FH] * 250),
]


@pytest.mark.parametrize('shapes,types', LISTS)
@pytest.mark.parametrize('max_norm', [0.0, 0.3, 1e9])
def test_new_and_in_place(shapes, types, max_norm):
    grads = _grads(shapes, types)
    want, norm = _exact(grads, max_norm)
    before = [g.clone() for g in grads]
    new, n = gc.clip_grads(grads, max_norm)
    _check(new, want, grads)
    _check_norm(n, norm)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    _check_norm(gc.grad_norm(grads), norm)
    params = [torch.nn.Parameter(torch.empty_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    n = gc.clip_grad_norm_(params, max_norm)
    _check_norm(n, norm)
    for g, w in zip(grads, new):
        assert torch.equal(g, w)


def test_same_bits_every_time():
    grads = _grads([(300001,), (77, 513)], [F32, BF])
    a, na = gc.clip_grads(grads, 0.1)
    for _ in range(3):
        b, nb = gc.clip_grads(grads, 0.1)
        assert torch.equal(na, nb)
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('kind', [F32, BF])
def test_offsets_into_a_buffer(kind):
    """Views that begin at any element."""
    flat = _grads([(5000,)], [kind])[0]
    for k in range(1, 9):
        views = [flat[k:k + 1001], flat[1100 + k:1100 + k + 2048],
                 flat[4000 + k:4000 + k]]
        rest = flat.clone()
        want, norm = _exact(views, 0.5)
        new, n = gc.clip_grads(views, 0.5)
        _check(new, want, views)
        _check_norm(n, norm)
        p = [torch.nn.Parameter(torch.empty_like(v)) for v in views]
        for q, v in zip(p, views):
            q.grad = v
        gc.clip_grad_norm_(p, 0.5)
        _check(views, want, views)
        keep = torch.ones(5000, dtype=torch.bool, device='cuda')
        keep[k:k + 1001] = False
        keep[1100 + k:1100 + k + 2048] = False
        assert torch.equal(flat[keep], rest[keep])
        flat.copy_(rest)


def test_orders_and_gaps():
    """channels_last gradients are dense; a slice of columns is not, and
    its neighbours stay as they are."""
    a = torch.randn(6, 5, 3, 3, device='cuda').to(
        memory_format=torch.channels_last)
    b = torch.randn(40, 30, device='cuda')
    whole = b.clone()
    views = [a, b[:, 3:17], b.t()[20:25]]
    want, norm = _exact(views, 1.0)
    new, n = gc.clip_grads(views, 1.0)
    _check(new, want, views)
    _check_norm(n, norm)
    p = [torch.nn.Parameter(torch.empty(v.shape, device='cuda'))
         for v in views]
    for q, v in zip(p, views):
        q.grad = v
    gc.clip_grad_norm_(p, 1.0)
    _check(views, want, views)
    assert torch.equal(b[:, :3], whole[:, :3])
    assert torch.equal(b[:, 25:], whole[:, 25:])


@pytest.mark.parametrize('value', [1e-30, 1e30])
def test_squares_outside_float32(value):
    grads = [torch.full((1000,), value, device='cuda')]
    want, norm = _exact(grads, 0.5, eps=0.0)
    new, n = gc.clip_grads(grads, 0.5, eps=0.0)
    _check_norm(n, norm)
    _check(new, want, grads)


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_not_finite_is_torch(bad):
    g = torch.tensor([1.0, bad, -2.0], device='cuda')
    p = torch.nn.Parameter(torch.zeros(3, device='cuda'))
    q = torch.nn.Parameter(torch.zeros(3, device='cuda'))
    p.grad, q.grad = g.clone(), g.clone()
    n = gc.clip_grad_norm_(p, 1.0)
    m = torch.nn.utils.clip_grad_norm_(q, 1.0)
    assert torch.equal(torch.isnan(n), torch.isnan(m))
    assert torch.equal(torch.isinf(n), torch.isinf(m))
    assert torch.allclose(p.grad, q.grad, equal_nan=True)


def test_refusals():
    one = torch.ones(4, device='cuda')
    with pytest.raises(ValueError):
        gc.clip_grads([one, torch.ones(4)], 1.0)
    with pytest.raises(TypeError):
        gc.clip_grads([one.double()], 1.0)
    with pytest.raises(TypeError):
        gc.clip_grads([one.to_sparse()], 1.0)
    p = torch.nn.Parameter(one.clone())
    q = torch.nn.Parameter(one.clone())
    flat = torch.ones(6, device='cuda')
    p.grad, q.grad = flat[:4], flat[2:]
    with pytest.raises(ValueError):
        gc.clip_grad_norm_([p, q], 1.0)
    with pytest.raises(ValueError):
        gc.clip_grad_norm_([p, p], 1.0)
    p.grad = torch.ones(1, device='cuda').expand(4)
    with pytest.raises(ValueError):
        gc.clip_grad_norm_([p], 1.0)
    assert torch.equal(flat, torch.ones(6, device='cuda'))


def test_on_another_stream_and_captured():
    grads = _grads([(70001,), (33, 65)], [F32, BF], seed=3)
    src = [g.clone() for g in grads]
    want, norm = _exact(src, 0.7)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        new, n = gc.clip_grads(src, 0.7)
        g = torch.cuda.CUDAGraph()
    torch.cuda.current_stream().wait_stream(s)
    _check(new, want, src)
    _check_norm(n, norm)
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        out, m = gc.clip_grads(src, 0.7)
    for k in range(4):
        for t, u in zip(src, grads):
            t.copy_(u * (k + 1))
        want, norm = _exact(src, 0.7)
        g.replay()
        torch.cuda.synchronize()
        _check(out, want, src)
        _check_norm(m, norm)
        e, en = gc.clip_grads(src, 0.7)     # eager work between replays
        assert torch.equal(m, en)
        assert all(torch.equal(x, y) for x, y in zip(out, e))


class TestClippedStep:
    """FusedSGD.step(max_norm=). An update's terms, each rounded once: the
    factor and its product with the gradient, decay times parameter, their
    sum, the momentum's product and sum, lr times the step, and the last
    difference. Each is at most half a step of the sum of the magnitudes
    that go in, so eight of those bound the difference."""

    @pytest.mark.parametrize('shapes', [
        [(1,)], [(64, 3, 7, 7), (1000,), (512, 512), (7,), (129, 33)],
        [(70000,), (3, 65536)]])
    @pytest.mark.parametrize('momentum,nesterov,wd', [
        (0.0, False, 0.0), (0.9, False, 1e-2), (0.9, True, 1e-2)])
    @pytest.mark.parametrize('max_norm', [0.0, 0.25, 1e9])
    def test_against_64_bits(self, shapes, momentum, nesterov, wd, max_norm):
        params = _grads(shapes, [F32] * len(shapes), seed=1)
        grads = _grads(shapes, [F32] * len(shapes), seed=2)
        moms = _grads(shapes, [F32] * len(shapes), seed=4) \
            if momentum else []
        kept = [g.clone() for g in grads]
        scale, lr = 0.5, 0.3
        scaled = [g.double() * scale for g in grads]
        norm = sum(float(g.square().sum()) for g in scaled) ** 0.5
        f = min(1.0, max_norm / (norm + 1e-6))
        want_p, want_m, most = [], [], []
        for i, (p, g) in enumerate(zip(params, scaled)):
            p = p.double()
            d = g * f + wd * p
            size = (g * f).abs() + (wd * p).abs()
            if momentum:
                m = momentum * moms[i].double() + d
                size = size + (momentum * moms[i].double()).abs()
                d = d + momentum * m if nesterov else m
                size = 2 * size
                want_m.append((m, size))
            want_p.append(p - lr * d)
            most.append(p.abs() + lr * size)
        sgd = K.FusedSGD(params, grads, moms, [wd] * len(shapes),
                         momentum=momentum, nesterov=nesterov)
        got = sgd.step(lr, grad_scale=scale, max_norm=max_norm)
        assert abs(float(got) - norm) <= 1.01 * HALF * norm
        for p, w, s in zip(params, want_p, most):
            assert bool(((p.double() - w).abs() <= 8 * HALF * s).all())
        for m, (w, s) in zip(moms, want_m):
            assert bool(((m.double() - w).abs() <= 8 * HALF * s).all())
        assert all(torch.equal(g, k) for g, k in zip(grads, kept))

    def test_without_a_limit_is_the_plain_step(self):
        shapes = [(1000,), (33, 7)]
        a = _grads(shapes, [F32] * 2, seed=1)
        b = [t.clone() for t in a]
        grads = _grads(shapes, [F32] * 2, seed=2)
        sa = K.FusedSGD(a, grads, [], [0.1, 0.0])
        sb = K.FusedSGD(b, grads, [], [0.1, 0.0])
        assert sa.step(0.1) is None
        sb.step(0.1, max_norm=1e9)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        with pytest.raises(ValueError):
            sb.step(0.1, max_norm=-1.0)

    def test_captured(self):
        shapes = [(70001,), (33, 7)]
        p = _grads(shapes, [F32] * 2, seed=1)
        grads = _grads(shapes, [F32] * 2, seed=2)
        eager = [t.clone() for t in p]
        sg = K.FusedSGD(p, grads, [], [0.0, 0.0])
        se = K.FusedSGD(eager, grads, [], [0.0, 0.0])
        sg.enable_lr_buffer()
        sg.set_lr(0.0)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            norm = sg.step(0.1, max_norm=0.5)
        for k in range(4):
            for t in grads:
                t.mul_(1.5)
            sg.set_lr(0.1 / (k + 1))
            g.replay()
            torch.cuda.synchronize()
            n = se.step(0.1 / (k + 1), max_norm=0.5)
            assert torch.equal(n, norm)
            assert all(torch.equal(x, y) for x, y in zip(p, eager))

    def test_trainer_step(self):
        """The word-level model's single-process step: norm, clip and
        update in one, against torch's clip and the plain fused step."""
        from mgwfbp_amd.distributed_optimizer import DistributedOptimizer
        nets = []
        for _ in range(2):
            torch.manual_seed(5)
            net = torch.nn.Sequential(torch.nn.Linear(40, 30),
                                      torch.nn.Linear(30, 7)).cuda()
            opt = DistributedOptimizer(
                torch.optim.SGD(net.parameters(), lr=0.5),
                named_parameters=list(net.named_parameters()))
            assert opt._fused_sgd is not None
            opt.zero_grad()
            (net(torch.ones(4, 40, device='cuda')).square().sum()
             * 10).backward()
            nets.append((net, opt))
        (a, oa), (b, ob) = nets
        oa.step(max_grad_norm=0.25)
        torch.nn.utils.clip_grad_norm_(b.parameters(), 0.25)
        ob.step()
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.allclose(p, q, rtol=1e-6, atol=1e-7)


def test_step_of_many_small_tensors_uses_the_cache():
    """What goes past the cache is decided by the parameters' size, not by
    their number."""
    n = 700
    shapes = [(i % 37 + 1,) for i in range(n)]
    params = _grads(shapes, [F32] * n, seed=1)
    grads = _grads(shapes, [F32] * n, seed=2)
    want = [p.double() for p in params]
    norm = sum(float(g.double().square().sum()) for g in grads) ** 0.5
    sgd = K.FusedSGD(params, grads, [], [0.0] * n)
    assert not sgd._past
    got = sgd.step(0.5, max_norm=0.25)
    assert abs(float(got) - norm) <= 1.01 * HALF * norm
    f = min(1.0, 0.25 / (norm + 1e-6))
    for p, w, g in zip(params, want, grads):
        step = 0.5 * f * g.double()
        most = w.abs() + step.abs()
        assert bool(((p.double() - (w - step)).abs()
                     <= 8 * HALF * most).all())


class TestPastTheCache:
    """From 128 MB on the gradients go past the cache, by other variants of
    the kernels, compared here on the GPU in 64 bits."""

    SHAPES = [(5000, 4001), (16385,), (7,), (3, 65537), (14345679,), (0,),
              (1,)]
    TYPES = [F32, BF, FH, F32, F32, F32, BF]

    @pytest.mark.parametrize('max_norm', [0.3, 1e9])
    def test_new_and_in_place(self, max_norm):
        g = torch.Generator(device='cuda').manual_seed(11)
        grads = [torch.randn(s, generator=g, device='cuda').to(t)
                 for s, t in zip(self.SHAPES, self.TYPES)]
        assert sum(t.numel() * t.element_size() for t in grads) >= 128 << 20
        want, norm = _exact(grads, max_norm)
        before = [t.clone() for t in grads]
        new, n = gc.clip_grads(grads, max_norm)
        _check(new, want, grads)
        _check_norm(n, norm)
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
        params = [torch.nn.Parameter(torch.empty_like(t)) for t in grads]
        for p, t in zip(params, grads):
            p.grad = t
        _check_norm(gc.clip_grad_norm_(params, max_norm), norm)
        assert all(torch.equal(a, b) for a, b in zip(grads, new))

    @pytest.mark.parametrize('momentum,nesterov', [(0.0, False),
                                                   (0.9, True)])
    @pytest.mark.parametrize('max_norm', [0.25, 1e9])
    def test_update(self, momentum, nesterov, max_norm):
        g = torch.Generator(device='cuda').manual_seed(12)
        shapes = self.SHAPES

        def new():
            return [torch.randn(s, generator=g, device='cuda')
                    for s in shapes]
        params, grads = new(), new()
        moms = new() if momentum else []
        wd, lr = 1e-2, 0.3
        norm = sum(float(t.double().square().sum()) for t in grads) ** 0.5
        f = min(1.0, max_norm / (norm + 1e-6))
        old_p = [t.clone() for t in params]
        old_m = [t.clone() for t in moms]
        sgd = K.FusedSGD(params, grads, moms, [wd] * len(shapes),
                         momentum=momentum, nesterov=nesterov)
        assert sgd._past
        got = sgd.step(lr, max_norm=max_norm)
        assert abs(float(got) - norm) <= 1.01 * HALF * norm
        for i, p in enumerate(params):   # as in TestClippedStep
            q, d = old_p[i].double(), grads[i].double() * f
            size = d.abs() + (wd * q).abs()
            d = d + wd * q
            if momentum:
                b = momentum * old_m[i].double()
                m = b + d
                size = 2 * (size + b.abs())
                d = d + momentum * m if nesterov else m
                assert bool(((moms[i].double() - m).abs()
                             <= 8 * HALF * size).all())
            most = q.abs() + lr * size
            assert bool(((p.double() - (q - lr * d)).abs()
                         <= 8 * HALF * most).all())


def test_flat_clip_captured():
    """The clip of one merged buffer, replayed between eager calls. Its sum
    of squares is in float32 and in any order: n u at the worst, of which the
    root halves, beside a few roundings."""
    n = 70001
    buf = torch.zeros(n, device='cuda')
    src = _grads([(n,)], [F32], seed=7)[0]
    buf.copy_(src)
    K.l2norm_clip_(buf, 0.5)             # makes its scratch
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.l2norm_clip_(buf, 0.5)
    for k in range(5):
        buf.copy_(src * (k + 1))
        want = src.double() * (k + 1)
        want *= min(1.0, 0.5 / (float(want.square().sum()) ** 0.5 + 1e-6))
        g.replay()
        torch.cuda.synchronize()
        far = (n / 2 + 8) * HALF
        assert bool(((buf.double() - want).abs() <= far * want.abs()).all())
        other = src * (k + 2)
        K.l2norm_clip_(other, 0.5)
        assert abs(float(other.double().norm()) - 0.5) <= far * 0.5 + 1e-6


def test_flat_clips_at_once():
    """Two captured clips replayed on two streams at once: each has its own
    sum of squares, of which one is 10^4 times the other."""
    n = 1 << 20
    src = [torch.full((n,), s, device='cuda') for s in (0.01, 1.0)]
    bufs = [s.clone() for s in src]
    graphs = [torch.cuda.CUDAGraph() for _ in src]
    torch.cuda.synchronize()
    for buf, graph in zip(bufs, graphs):
        with torch.cuda.graph(graph):
            buf.copy_(src[0] if buf is bufs[0] else src[1])
            K.l2norm_clip_(buf, 0.5)
    streams = [torch.cuda.Stream() for _ in src]
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for buf in bufs:                 # all elements are 0.5 / 2^10
            assert torch.allclose(buf, torch.full_like(buf, 0.5 / 1024),
                                  rtol=1e-3, atol=0)

"""Global-norm clipping on the CPU: the plain forms, the refusals, and the
paths that call them."""
import math

import pytest
import torch

from mgwfbp_amd import kernels as K
from mgwfbp_amd.kernels import grad_clip as gc


def _params(shapes, types=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for i, s in enumerate(shapes):
        t = types[i] if types else torch.float32
        p = torch.nn.Parameter(torch.zeros(s, dtype=t))
        p.grad = torch.randn(s, generator=g).to(t)
        out.append(p)
    return out


@pytest.mark.parametrize('max_norm', [0.0, 0.25, 1e6])
def test_in_place_matches_torch(max_norm):
    shapes = [(7, 5), (33,), (2, 3, 4, 5)]
    a, b = _params(shapes), _params(shapes)
    norm = gc.clip_grad_norm_(a, max_norm)
    ref = torch.nn.utils.clip_grad_norm_(b, max_norm)
    # both round a norm and a product: a few half steps of float32
    assert torch.allclose(norm, ref, rtol=4 * 2.0 ** -24, atol=0)
    for p, q in zip(a, b):
        assert torch.allclose(p.grad, q.grad, rtol=8 * 2.0 ** -24, atol=0)


def test_new_tensors_leave_the_gradients():
    grads = [p.grad for p in _params([(5,), (6, 7)])]
    before = [g.clone() for g in grads]
    new, norm = gc.clip_grads(grads, 0.5)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    assert float(norm) == pytest.approx(float(gc.grad_norm(grads)))
    assert float(gc.grad_norm(new)) == pytest.approx(0.5, rel=1e-5)


def test_none_and_empty():
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(gc.clip_grad_norm_([p], 1.0)) == 0.0
    assert float(gc.clip_grad_norm_([], 1.0)) == 0.0
    assert gc.clip_grads([], 1.0)[0] == []
    assert float(gc.grad_norm([])) == 0.0
    p.grad = torch.ones(3)
    assert float(gc.clip_grad_norm_(p, 10.0)) == pytest.approx(math.sqrt(3))


@pytest.mark.parametrize('call', [
    lambda: gc.clip_grads([torch.ones(2)], -1.0),
    lambda: gc.clip_grads([torch.ones(2)], float('nan')),
    lambda: gc.clip_grads([torch.ones(2)], 1.0, eps=-1e-3),
    lambda: gc.clip_grad_norm_(_params([(2,)]), -0.5),
])
def test_refuses_limits(call):
    with pytest.raises(ValueError):
        call()


def test_native_entry_refuses_host_tensors():
    ext = gc.load_lm()
    with pytest.raises(ValueError):
        ext.grad_norm([torch.ones(3)])
    with pytest.raises(ValueError):
        ext.clip_grads_([torch.ones(3)], 1.0, 0.0)
    with pytest.raises(RuntimeError):
        ext.grad_norm([])
    with pytest.raises(TypeError):
        ext.clip_grads([1.0], 1.0, 0.0)


def test_optimizer_step_clips_on_the_cpu():
    """DistributedOptimizer.step(max_grad_norm=) without the fused update
    equals clipping first and stepping then."""
    from mgwfbp_amd.distributed_optimizer import DistributedOptimizer

    def build():
        torch.manual_seed(3)
        net = torch.nn.Sequential(torch.nn.Linear(6, 5),
                                  torch.nn.Linear(5, 2))
        opt = DistributedOptimizer(
            torch.optim.SGD(net.parameters(), lr=0.5, momentum=0.9),
            named_parameters=list(net.named_parameters()))
        opt.zero_grad()
        (net(torch.ones(4, 6)).square().sum() * 10).backward()
        return net, opt

    a, oa = build()
    b, ob = build()
    oa.step(max_grad_norm=0.1)
    torch.nn.utils.clip_grad_norm_(b.parameters(), 0.1)
    ob.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-7)
    with pytest.raises(ValueError):
        oa.step(max_grad_norm=-1.0)


def test_single_process_entry_uses_the_clipped_step():
    import inspect
    from mgwfbp_amd import dist_trainer
    assert 'max_grad_norm' in inspect.getsource(dist_trainer.mgwfbp)
    assert K.FusedSGD.step.__doc__


class _NoKernels:
    """Stands for the extension where tables are built: on the host."""

    def build_sgd_table(self, *args):
        return torch.zeros(1), torch.zeros(1), torch.ones(1)

    build_pack_table = build_sgd_table


def test_tables_keep_their_tensors(monkeypatch):
    """A table holds addresses, which have to stay the tensors' own for as
    long as it is used, whatever the caller lets go of."""
    import gc
    import weakref
    monkeypatch.setattr(K, 'load_kernels', lambda required=None: _NoKernels())

    def new():
        return [torch.zeros(3), torch.zeros(2)]

    p, g, m, s = new(), new(), new(), new()
    alive = [weakref.ref(t) for t in p + g + m + s]
    tables = (K.FusedSGD(p, g, m, [0.0, 0.0], momentum=0.9),
              K.PackTable(s, [0, 64]))
    del p, g, m, s
    gc.collect()
    assert all(r() is not None for r in alive)
    del tables
    gc.collect()
    assert all(r() is None for r in alive)


@pytest.mark.parametrize('p,g,m,wd', [
    ([3, 2], [3], [], 2), ([3], [2], [], 1), ([3], [3], [2], 1),
    ([3, 2], [3, 2], [3], 2), ([3], [3], [], 0), ([3], [3], [], 1)])
def test_update_table_refuses_lists_that_do_not_fit(p, g, m, wd):
    """The kernels go by the parameters' sizes; the last list fits, but lies
    on the host."""
    def new(sizes):
        return [torch.zeros(n) for n in sizes]
    with pytest.raises((ValueError, RuntimeError), match='fused SGD'):
        K.FusedSGD(new(p), new(g), new(m), [0.0] * wd, momentum=0.5 if m
                   else 0.0)


def test_update_table_refuses_other_types():
    half = [torch.zeros(3, dtype=torch.bfloat16)]
    full = [torch.zeros(3)]
    for p, g, m in ((half, full, full), (full, half, full),
                    (full, full, half)):
        with pytest.raises((ValueError, RuntimeError), match='fused SGD'):
            K.FusedSGD(p, g, m, [0.0], momentum=0.5)


@pytest.mark.parametrize('dnn,dataset,limit', [('lstm', 'ptb', 0.25),
                                               ('lstman4', 'an4', 400)])
def test_single_process_entry_clips(monkeypatch, dnn, dataset, limit):
    """The entry as it runs, with smaller networks: each update is given the
    model's limit, and the word-level model's is plain SGD with the
    gradients scaled to it. A parameter's update has four roundings, of the
    rate, two products and the difference: of the parameter's size for the
    last, and of the step's for the others; a product below the smallest
    normal number is off by half of 2^-149 instead, and a word of next to no
    probability has such a gradient, for a bias that is 0."""
    from mgwfbp_amd import dist_trainer, dl_trainer, models, settings
    monkeypatch.setattr(settings, 'ADAPTIVE_MERGE', False)
    torch.manual_seed(0)
    create = dl_trainer.create_net

    def small(num_classes, name, **kw):
        if name == 'lstm':
            net = models.lstm(vocab_size=kw['vocab_size'], embedding_dim=6,
                              hidden_dim=6, batch_size=kw['batch_size'])
            with torch.no_grad():        # gradients well above the limit
                net.fc.weight.mul_(300.0)
                net.rnn.bias_ih_l1.fill_(2.0)
            return net, None
        return create(num_classes, name, **kw)

    monkeypatch.setattr(dl_trainer, 'create_net', small)
    seen = []

    class Trainer(dl_trainer.DLTrainer):
        def update_model(self, max_grad_norm=None):
            params = [p for p in self.net.parameters()]
            before = [p.detach().clone() for p in params]
            grads = [p.grad.double() for p in params]
            norm = sum(float(g.square().sum()) for g in grads) ** 0.5
            super().update_model(max_grad_norm=max_grad_norm)
            seen.append((max_grad_norm, norm))
            if dnn != 'lstm':
                return
            f = min(1.0, max_grad_norm / (norm + 1e-6))
            for p, b, g in zip(params, before, grads):
                step = self.lr * f * g
                off = (p.detach().double() - (b.double() - step)).abs()
                most = 4 * 2.0 ** -24 * (b.double().abs() + step.abs()) \
                    + 2.0 ** -149
                assert bool((off <= most).all())

    monkeypatch.setattr(dist_trainer, 'DLTrainer', Trainer)
    dist_trainer.mgwfbp(dnn, dataset, '', 1, 0.5, 2, 1, max_epochs=1,
                        num_steps=5, max_iters=2)
    assert [m for m, _ in seen] == [limit, limit]
    if dnn == 'lstm':
        assert all(n > limit for _, n in seen)

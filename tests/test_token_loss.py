"""Cross entropy and token log probabilities on the CPU: the plain forms'
formulas and gradients, and the refusals."""
import math

import pytest
import torch

from mgwfbp_amd.kernels import token_loss as tl
from mgwfbp_amd.kernels.grad_clip import load_lm

NEG = float('-inf')


def test_formulas_in_64_bits():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(3, 4, 11, generator=g, dtype=torch.float64)
    x[0, 0, 3:] = NEG
    t = torch.randint(0, 3, (3, 4), generator=g)
    r = tl.token_log_probs(x, t, top_k=4)
    for i in range(3):
        for j in range(4):
            v = x[i, j].tolist()
            s = math.fsum(math.exp(a) for a in v)
            p = [math.exp(a) / s for a in v]
            lp = math.log(p[int(t[i, j])])
            h = -math.fsum(q * math.log(q) for q in p if q > 0)
            order = sorted(range(11), key=lambda k: (-v[k], k))[:4]
            assert float(r.log_probs[i, j]) == pytest.approx(lp, abs=1e-12)
            assert float(r.entropy[i, j]) == pytest.approx(h, abs=1e-12)
            assert r.top_ids[i, j].tolist() == order
    ce = tl.cross_entropy(x, t, reduction='none')
    assert torch.allclose(ce, -r.log_probs, atol=1e-12)
    assert tl.cross_entropy(x, t).item() == pytest.approx(ce.mean().item())
    assert tl.cross_entropy(x, t, reduction='sum').item() == \
        pytest.approx(ce.sum().item())


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 7, generator=g, dtype=torch.float64,
                    requires_grad=True)
    t = torch.tensor([0, 6, -100, 3])
    assert torch.autograd.gradcheck(
        lambda a: tl.token_log_probs(a, t)[:2], (x,))
    assert torch.autograd.gradcheck(
        lambda a: tl.cross_entropy(a, t), (x,))


def test_masked_classes_have_no_gradient():
    x = torch.tensor([[0.5, NEG, -1.0, NEG]], requires_grad=True)
    r = tl.token_log_probs(x, torch.tensor([2]))
    (r.log_probs + r.entropy).sum().backward()
    assert torch.isfinite(x.grad).all()
    assert x.grad[0, 1] == 0 and x.grad[0, 3] == 0


def test_ignored():
    x = torch.randn(3, 5)
    t = torch.tensor([-100, 2, -100])
    assert tl.cross_entropy(x, t).item() == pytest.approx(
        tl.cross_entropy(x[1:2], t[1:2]).item())
    assert torch.isnan(tl.cross_entropy(x, torch.full((3,), -100)))
    assert tl.token_log_probs(x, t).log_probs[0] == 0


@pytest.mark.parametrize('error,call', [
    (ValueError, lambda x, t: tl.cross_entropy(x, t, reduction='max')),
    (ValueError, lambda x, t: tl.cross_entropy(x, t[:2])),
    (TypeError, lambda x, t: tl.cross_entropy(x, t.float())),
    (ValueError, lambda x, t: tl.token_log_probs(x, t, top_k=6)),
    (ValueError, lambda x, t: tl.token_log_probs(x, t, top_k=-1)),
    (ValueError, lambda x, t: tl.token_log_probs(x[:, :0], t)),
    (IndexError, lambda x, t: tl.token_log_probs(x, t + 5)),
    (IndexError, lambda x, t: tl.cross_entropy(x, t + 5)),
])
def test_refusals(error, call):
    with pytest.raises(error):
        call(torch.randn(3, 5), torch.tensor([0, 1, 2]))


def test_native_entries_refuse_host_tensors():
    ext = load_lm()
    x, t = torch.randn(3, 5), torch.tensor([0, 1, 2])
    with pytest.raises(ValueError):
        ext.cross_entropy(x, t, -100, 1, False)
    with pytest.raises(ValueError):
        ext.token_log_probs(x, t, 0, -100)


def test_module_is_torch_on_the_cpu():
    x, t = torch.randn(6, 9), torch.randint(0, 9, (6,))
    for kw in ({}, dict(reduction='sum'), dict(label_smoothing=0.1),
               dict(weight=torch.rand(9))):
        a = tl.MgxCrossEntropyLoss(**kw)(x, t)
        b = torch.nn.CrossEntropyLoss(**kw)(x, t)
        assert torch.equal(a, b)


def test_word_level_evaluation():
    """DLTrainer.test() scores the word-level model through
    token_log_probs: the same perplexity as the mean cross entropy."""
    from mgwfbp_amd.dl_trainer import DLTrainer
    from mgwfbp_amd.models import lstm
    torch.manual_seed(0)
    t = DLTrainer(rank=0, size=1, dist=False, batch_size=4, ngpus=0,
                  data_dir='', dataset='ptb', dnn='lstm', lr=1.0, nworkers=1,
                  prefix='t', synthetic=True)
    t.net = lstm(vocab_size=10000, batch_size=4, embedding_dim=8,
                 hidden_dim=8)
    t.testloader = [b for b, _ in zip(t.testloader, range(3))]
    ppl = t.test(0)
    t.net.eval()
    total = 0.0
    with torch.no_grad():
        for x, y in t.testloader:
            out, _ = t.net(x, t.net.init_hidden())
            total += torch.nn.functional.cross_entropy(
                out.view(-1, 10000), y.view(-1)).item()
    assert ppl == pytest.approx(math.exp(total / 3), rel=1e-5)
    assert 0.0 <= t.top5_accuracy <= 1.0
    # nearly uniform over 10000 words
    assert t.mean_entropy == pytest.approx(math.log(10000), rel=0.05)


def _rows_with_ties(kind):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, 200, generator=g).to(kind)
    x[1] = x[1].round()                  # many equal values
    x[2] = 0.0
    x[3, ::2] = -0.0
    x[3, 1::2] = 0.0                     # both zeros are the same value
    x[4, 7] = float('nan')
    x[5, 3:90] = float('nan')
    x[6, 4:] = NEG
    x[7, 11] = x[7, 150] = float('inf')
    x[8, 100] = x[8].max()               # the best one twice
    return x.view(3, 3, 200)


@pytest.mark.parametrize('kind', [torch.float32, torch.float64,
                                  torch.bfloat16, torch.float16])
@pytest.mark.parametrize('k', [0, 1, 2, 5, 64])
def test_best_of_equal_values(kind, k):
    x = _rows_with_ties(kind)
    r = tl.token_log_probs_reference(
        x, torch.zeros(3, 3, dtype=torch.long), top_k=k)
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][..., :k]
    assert torch.equal(r.top_ids, ids)
    all_of_them = tl.token_log_probs_reference(
        x[..., :64], torch.zeros(3, 3, dtype=torch.long), top_k=64)
    assert torch.equal(all_of_them.top_ids, torch.sort(
        x[..., :64], dim=-1, descending=True, stable=True)[1])


def test_best_without_sorting_the_row():
    """A few of many classes: the rows are never sorted whole."""
    from torch.utils._python_dispatch import TorchDispatchMode
    longest = []

    class Log(TorchDispatchMode):
        def __torch_dispatch__(self, f, types, args=(), kwargs=None):
            if 'sort' in str(f):
                longest.append(args[0].size(-1))
            return f(*args, **(kwargs or {}))

    with Log():
        for kind in (torch.float32, torch.bfloat16):
            tl.token_log_probs(_rows_with_ties(kind),
                               torch.zeros(3, 3, dtype=torch.long), top_k=5)
    assert max(longest, default=0) <= 5


def _word_level(batches, ntokens=40):
    """A DLTrainer whose word-level model gives the logits of ``batches``,
    (logits, targets) of 4 sequences each, in turn."""
    from mgwfbp_amd.dl_trainer import DLTrainer
    t = DLTrainer(rank=0, size=1, dist=False, batch_size=4, ngpus=0,
                  data_dir='', dataset='ptb', dnn='lstm', lr=1.0, nworkers=1,
                  prefix='t', synthetic=True)

    class Net(torch.nn.Module):
        batch_size = 4

        def __init__(self):
            super().__init__()
            self.ntokens = ntokens
            self.given = iter([x for x, _ in batches])

        def init_hidden(self):
            return None

        def forward(self, x, hidden):
            return next(self.given), hidden

    t.net = Net()
    t.testloader = [(y, y) for _, y in batches]
    return t


def test_evaluation_sums_in_64_bits():
    """Many batches with losses near 10: a float32 sum past 2^14 loses 2^-10
    of each, and the perplexity's exponent with it. Each batch's mean is a
    float32, off by half a step of the loss for each of a few roundings."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 3, 40, generator=g) * 4.0
    y = torch.randint(0, 40, (4, 3), generator=g)
    x.scatter_(-1, y.unsqueeze(-1), -12.0)
    n = 4000
    t = _word_level([(x, y)] * n)
    ppl = t.test(0)
    log = torch.log_softmax(x.double(), -1)
    want = -float(log.gather(-1, y.unsqueeze(-1)).mean())
    h = -float((log.exp() * log).sum(-1).mean())
    assert abs(math.log(ppl) - want) <= 8 * 2.0 ** -24 * want
    assert abs(t.mean_entropy - h) <= 64 * 2.0 ** -24 * h


def test_evaluation_leaves_ignored_targets_out():
    """As the mean cross entropy does: neither in the loss nor in what it is
    divided by, nor among the five best."""
    g = torch.Generator().manual_seed(2)
    batches = []
    want = []
    hits = []
    for i in range(3):
        x = torch.randn(4, 5, 40, generator=g)
        y = torch.randint(0, 40, (4, 5), generator=g)
        y[:, 4 - i:] = -100
        batches.append((x, y))
        want.append(float(torch.nn.functional.cross_entropy(
            x.double().view(-1, 40), y.view(-1))))
        kept = y != -100
        hits.append(float((x.topk(5)[1] == y.unsqueeze(-1)).any(-1)[kept]
                          .double().mean()))
    t = _word_level(batches)
    assert math.log(t.test(0)) == pytest.approx(sum(want) / 3, rel=1e-6)
    assert t.top5_accuracy == pytest.approx(sum(hits) / 3, abs=1e-12)


def test_evaluation_of_a_model_in_64_bits(monkeypatch):
    """The kernels take no float64 logits; such a model is scored by the
    plain form, wherever it lies."""
    from mgwfbp_amd import dl_trainer

    def kernels(logits, targets, **kw):
        raise TypeError('logits must be float32, bfloat16 or float16')

    monkeypatch.setattr(dl_trainer, 'token_log_probs', kernels)
    g = torch.Generator().manual_seed(4)
    x = torch.randn(4, 5, 40, generator=g, dtype=torch.float64)
    y = torch.randint(0, 40, (4, 5), generator=g)
    ppl = _word_level([(x, y)]).test(0)
    assert math.log(ppl) == pytest.approx(float(
        torch.nn.functional.cross_entropy(x.view(-1, 40), y.view(-1))),
        rel=1e-12)

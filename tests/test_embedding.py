"""Token embedding on the CPU: formula, module, refusals."""
import pytest
import torch

from mgwfbp_amd.kernels import embedding as em
from mgwfbp_amd.kernels.grad_clip import load_lm


def test_formula_and_gradient():
    w = torch.randn(7, 3, dtype=torch.float64, requires_grad=True)
    t = torch.tensor([[1, 6, 1], [0, 2, 1]])
    y = em.embedding(t, w, scale=2.5)
    assert y.shape == (2, 3, 3)
    assert torch.equal(y, 2.5 * w[t])
    assert torch.autograd.gradcheck(
        lambda a: em.embedding(t, a, scale=2.5), (w,))
    y = em.embedding(t, w, padding_idx=-6)
    g, = torch.autograd.grad(y.sum(), w)
    assert g[:, 0].tolist() == [1, 0, 1, 0, 0, 0, 1]


def test_module_is_torch_on_the_cpu():
    torch.manual_seed(0)
    a = em.MgxEmbedding(11, 5, padding_idx=3)
    torch.manual_seed(0)
    b = torch.nn.Embedding(11, 5, padding_idx=3)
    assert list(a.state_dict()) == list(b.state_dict())
    t = torch.randint(0, 11, (4, 6))
    assert torch.equal(a(t), b(t))
    c = em.MgxEmbedding(11, 5, scale=3.0)
    assert torch.equal(c(t), 3.0 * c.weight[t])
    assert 'scale' in repr(c) and 'scale' not in repr(a)


@pytest.mark.parametrize('error,call', [
    (TypeError, lambda t, w: em.embedding(t.float(), w)),
    (ValueError, lambda t, w: em.embedding(t, w, padding_idx=7)),
    (ValueError, lambda t, w: em.embedding(t, w, padding_idx=-8)),
    (ValueError, lambda t, w: em.embedding(t, w[0])),
    (IndexError, lambda t, w: em.embedding(t + 7, w)),
    (ValueError, lambda t, w: load_lm().embedding(t, w, 1.0, -1)),
])
def test_refusals(error, call):
    with pytest.raises(error):
        call(torch.tensor([0, 1]), torch.randn(7, 3))


def test_word_level_model_has_it():
    from mgwfbp_amd.models import lstm
    net = lstm(vocab_size=20, embedding_dim=6, hidden_dim=6, batch_size=2)
    assert isinstance(net.embedding, em.MgxEmbedding)
    assert 'embedding.weight' in net.state_dict()

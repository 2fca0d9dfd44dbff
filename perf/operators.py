"""The operators at the two ends of a language model's training step, and what one pass through each costs.

Tokens enter through an embedding table, whose gradient is summed by token; the logits leave through the loss, or
through the log probabilities of given tokens; the gradients are clipped by their global norm before the update.
Each operator is here in its plain form, from elementary tensor operations, and as a call of the framework (`own`).
Sizes: the word-level model of exp_configs/lstm.conf (20 sequences of 35 tokens, 10000 words, 1500 wide) and generic
ones around and above it.
"""
import math
import random

import torch

own = False

EPS = 1e-6          # beside the norm in the clipping factor, as torch.nn.utils.clip_grad_norm_ has it
IGNORE = -100       # a target that takes no part
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}


def listed():
    return [
        # one step of a decoder: the next token of each of 20 sequences, nothing to differentiate
        dict(name='embed_step', op='embed', tokens=20, vocab=10000, dim=1500, type='fp32', scale=1.0, pad=-1,
             train=False),
        # the training batch of exp_configs/lstm.conf: 20 x 35 tokens
        dict(name='embed_words', op='embed', tokens=700, vocab=10000, dim=1500, type='fp32', scale=1.0, pad=-1,
             train=True),
        # a large batch into a large 16-bit table, scaled by sqrt(dim), with padding behind short sequences
        dict(name='embed_large', op='embed', tokens=16381, vocab=60001, dim=2048, type='bf16',
             scale=math.sqrt(2048.0), pad=0, train=True),
        # the loss of one time step of the word-level model: few rows, where launches count
        dict(name='loss_step', op='loss', rows=20, vocab=10000, type='fp32', ignored=0.0),
        # the loss of its whole training batch
        dict(name='loss_words', op='loss', rows=700, vocab=10000, type='fp32', ignored=0.0),
        # a large 16-bit batch over an odd vocabulary (no row starts where a wide load would like it), a tenth ignored
        dict(name='loss_large', op='loss', rows=8190, vocab=50001, type='bf16', ignored=0.1),
        # a decoder that answers with the chosen token's log probability and its alternatives: one token, four sequences
        dict(name='logprobs_step', op='logprobs', rows=4, vocab=50001, type='bf16', top=8, train=False),
        # scoring the word-level model's batch: perplexity, entropy and the five best words
        dict(name='logprobs_words', op='logprobs', rows=700, vocab=10000, type='fp32', top=5, train=False),
        # training on log probabilities with an entropy bonus, each token with a weight of its own
        dict(name='logprobs_train', op='logprobs', rows=4095, vocab=32768, type='bf16', top=0, train=True),
        # the gradients of a small network: 48 tensors, few elements
        dict(name='clip_small', op='clip', kind='fp32', tensors=48, elements=270000, max_norm=0.25),
        # the word-level model's clipped step, all its 11 tensors: norm, factor and update
        dict(name='clip_update_words', op='update', kind='words', tensors=11, elements=0, max_norm=0.25, momentum=0.0),
        # a large model's gradients, 16-bit matrices beside 32-bit vectors, odd sizes
        dict(name='clip_large', op='clip', kind='mixed', tensors=60, elements=300000000, max_norm=1.0),
    ]


def _between(rng, low, high):
    """A whole number of the range, even over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(['embed', 'embed', 'loss', 'loss', 'logprobs', 'logprobs', 'clip', 'update'])
    kind = rng.choice(['fp32', 'bf16', 'fp16'])
    wide = 4 if kind == 'fp32' else 2
    if op == 'embed':
        dim = _between(rng, 33, 2048)
        vocab = _between(rng, 100, min(60001, 60001 * 2048 * 2 // (dim * wide)))
        tokens = _between(rng, 1, min(16381, 16381 * 2048 * 2 // (dim * wide)))
        return dict(op=op, tokens=tokens, vocab=vocab, dim=dim, type=kind,
                    scale=rng.choice([1.0, math.sqrt(dim)]), pad=rng.choice([-1, 0]), train=rng.random() < 0.7)
    if op in ('loss', 'logprobs'):
        vocab = _between(rng, 1000, 50001)
        rows = _between(rng, 1, min(8190, 8190 * 50001 * 2 // (vocab * wide)))
        if op == 'loss':
            return dict(op=op, rows=rows, vocab=vocab, type=kind, ignored=rng.choice([0.0, 0.1, 0.5]))
        rows = max(1, rows // 2)
        if rng.random() < 0.4:
            return dict(op=op, rows=rows, vocab=vocab, type=kind, top=0, train=True)
        return dict(op=op, rows=min(rows, 1024), vocab=vocab, type=kind, top=rng.randint(0, 20), train=False)
    tensors = rng.randint(1, 60)
    elements = _between(rng, 1000, 100000000)
    if op == 'clip':
        return dict(op=op, kind=rng.choice(['fp32', 'bf16', 'mixed']), tensors=tensors, elements=elements,
                    max_norm=rng.choice([0.25, 1.0, 1000.0]))
    return dict(op=op, kind='fp32', tensors=min(tensors, 30), elements=elements, max_norm=rng.choice([0.25, 1.0]),
                momentum=rng.choice([0.0, 0.9]))


def _sizes(case):
    """The shapes of a model's tensors: given ones, or matrices that share the elements out, and a vector for each."""
    if case['kind'] == 'words':
        gates = [(6000, 1500), (6000, 1500), (6000,), (6000,)]
        return [(10000, 1500)] + gates + gates + [(10000, 1500), (10000,)]
    rng = random.Random(case['tensors'] * 1000003 + case['elements'])
    n = case['tensors']
    parts = [math.exp(rng.uniform(0.0, 3.0)) for _ in range((n + 1) // 2)]
    shapes = []
    for i in range(n):
        rows = max(1, int(math.sqrt(parts[i // 2] / sum(parts) * case['elements'])))
        shapes.append((rows,) if i % 2 else (rows, rows + 1))
    return shapes


def _types(case):
    if case['kind'] == 'mixed':
        return [torch.float32 if len(s) == 1 else torch.bfloat16 for s in _sizes(case)]
    return [TYPES[case['kind']] if case['kind'] in TYPES else torch.float32] * len(_sizes(case))


def _elements(case):
    return sum(math.prod(s) for s in _sizes(case))


def work(case):
    wide = 4 if case.get('type', case.get('kind')) in ('fp32', 'words') else 2
    if case['op'] == 'embed':
        rows = case['tokens'] * case['dim'] * wide
        n = 8 * case['tokens'] + min(case['tokens'], case['vocab']) * case['dim'] * wide + rows
        if case['train']:
            n += rows + case['vocab'] * case['dim'] * wide
        return {'bytes': n, 'flops': case['tokens'] * case['dim'] * (2 if case['train'] else 1)}
    if case['op'] in ('loss', 'logprobs'):
        n = case['rows'] * case['vocab']
        train = case['op'] == 'loss' or case['train']
        return {'bytes': n * wide * (2 if train else 1) + 24 * case['rows'], 'flops': n * (8 if train else 4)}
    each = sum(math.prod(s) * t.itemsize for s, t in zip(_sizes(case), _types(case)))
    if case['op'] == 'clip':
        return {'bytes': 2 * each, 'flops': 3 * _elements(case)}
    return {'bytes': each * (5 if case['momentum'] else 3), 'flops': _elements(case) * (8 if case['momentum'] else 6)}


def _words(n, vocab, gen):
    """Tokens as text has them: the r-th most frequent about 1/r as often as the first."""
    u = torch.rand(n, generator=gen, device='cuda', dtype=torch.float64)
    return torch.exp(u * math.log(vocab)).long().sub_(1).clamp_(0, vocab - 1)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def randn(*shape, type=torch.float32):
        return torch.randn(*shape, generator=gen, device='cuda', dtype=type)

    if case['op'] == 'embed':
        kind = TYPES[case['type']]
        weight = randn(case['vocab'], case['dim'], type=kind).mul_(case['dim'] ** -0.5)
        weight.requires_grad_(case['train'])
        tokens = _words(case['tokens'], case['vocab'], gen)
        if case['pad'] >= 0:
            tokens[case['tokens'] - case['tokens'] // 8:] = case['pad']
        grad = randn(case['tokens'], case['dim'], type=kind) if case['train'] else None
        return dict(case=case, weight=weight, tokens=tokens, grad=grad)
    if case['op'] in ('loss', 'logprobs'):
        rows, vocab = case['rows'], case['vocab']
        logits = randn(rows, vocab, type=TYPES[case['type']]).mul_(2.5)
        targets = _words(rows, vocab, gen)
        # a trained model has its target well above the rest more often than not
        lift = torch.rand(rows, 1, generator=gen, device='cuda').mul_(12.0).to(logits.dtype)
        logits.scatter_add_(1, targets[:, None], lift)
        state = dict(case=case, logits=logits)
        if case['op'] == 'loss':
            logits.requires_grad_(True)
            keep = torch.rand(rows, generator=gen, device='cuda') >= case['ignored']
            keep[0] = True
            state['targets'] = torch.where(keep, targets, torch.full_like(targets, IGNORE))
        else:
            logits.requires_grad_(case['train'])
            state['targets'] = targets
            state['grads'] = [randn(rows), randn(rows).mul_(0.01)] if case['train'] else None
        return state
    shapes, types = _sizes(case), _types(case)
    grads = [randn(*s, type=t).mul_(0.02) for s, t in zip(shapes, types)]
    state = dict(case=case, grads=grads)
    if case['op'] == 'update':
        state['params'] = [randn(*s).mul_(0.05) for s in shapes]
        state['momenta'] = [randn(*s).mul_(0.01) for s in shapes] if case['momentum'] else []
        state['decay'] = [1e-4 if case['momentum'] and len(s) > 1 else 0.0 for s in shapes]
        state['lr'] = 0.1
        if own:   # the framework's update keeps a table of its tensors, built with the optimizer
            from mgwfbp_amd.kernels import FusedSGD
            state['sgd'] = FusedSGD(state['params'], grads, state['momenta'], state['decay'],
                                    momentum=case['momentum'])
    return state


def _framework(state):
    case = state['case']
    if case['op'] == 'embed':
        from mgwfbp_amd.kernels.embedding import embedding
        pad = case['pad'] if case['pad'] >= 0 else None
        out = embedding(state['tokens'], state['weight'], scale=case['scale'], padding_idx=pad)
        if not case['train']:
            return [out]
        return [out, torch.autograd.grad(out, state['weight'], state['grad'])[0]]
    if case['op'] == 'loss':
        from mgwfbp_amd.kernels.token_loss import cross_entropy
        loss = cross_entropy(state['logits'], state['targets'], ignore_index=IGNORE)
        return [loss, torch.autograd.grad(loss, state['logits'])[0]]
    if case['op'] == 'logprobs':
        from mgwfbp_amd.kernels.token_loss import token_log_probs
        r = token_log_probs(state['logits'], state['targets'], top_k=case['top'], ignore_index=IGNORE)
        out = [r.log_probs, r.entropy]
        if case['top']:
            out += [r.top_log_probs, r.top_ids]
        if case['train']:
            out += torch.autograd.grad([r.log_probs, r.entropy], [state['logits']], state['grads'])
        return out
    if case['op'] == 'clip':
        from mgwfbp_amd.kernels.grad_clip import clip_grads
        clipped, norm = clip_grads(state['grads'], case['max_norm'], eps=EPS)
        return [norm] + list(clipped)
    norm = state['sgd'].step(state['lr'], max_norm=case['max_norm'], eps=EPS)
    return [norm] + state['params'] + state['momenta']


def _plain_embed(state):
    case = state['case']
    weight, tokens = state['weight'].detach(), state['tokens']
    out = (weight[tokens].float() * case['scale']).to(weight.dtype)
    if not case['train']:
        return [out]
    grad = torch.zeros(weight.shape, dtype=torch.float32, device=weight.device)
    grad.index_add_(0, tokens, state['grad'].float())
    grad.mul_(case['scale'])
    if case['pad'] >= 0:
        grad[case['pad']] = 0
    return [out, grad.to(weight.dtype)]


def _plain_loss(state):
    logits, targets = state['logits'].detach(), state['targets']
    x = logits.float()
    keep = targets != IGNORE
    at = torch.where(keep, targets, torch.zeros_like(targets))[:, None]
    x = x - x.amax(1, keepdim=True)
    e = x.exp()
    s = e.sum(1, keepdim=True)
    each = s.log() - x.gather(1, at)
    share = keep[:, None].float() / keep.sum()
    loss = (each * share).sum()
    grad = e / s * share
    grad.scatter_add_(1, at, -share)
    return [loss, grad.to(logits.dtype)]


def _plain_logprobs(state):
    case = state['case']
    logits, targets = state['logits'].detach(), state['targets']
    x = logits.float()
    m = x.amax(1, keepdim=True)
    x = x - m
    e = x.exp()
    s = e.sum(1, keepdim=True)
    log = x - s.log()
    p = e / s
    entropy = -(p * log).sum(1, keepdim=True)
    out = [log.gather(1, targets[:, None])[:, 0], entropy[:, 0]]
    if case['top']:
        ids = torch.sort(logits, dim=1, descending=True, stable=True)[1][:, :case['top']]
        out += [log.gather(1, ids), ids]
    if case['train']:
        gl, ge = (g[:, None] for g in state['grads'])
        grad = p * (-gl - ge * (log + entropy))
        grad.scatter_add_(1, targets[:, None], gl)
        out.append(grad.to(logits.dtype))
    return out


def _plain_norm(grads):
    return torch.stack([g.float().square().sum(dtype=torch.float64) for g in grads]).sum().sqrt()


def _plain_clip(state):
    case, grads = state['case'], state['grads']
    norm = _plain_norm(grads)
    factor = (case['max_norm'] / (norm + EPS)).clamp(max=1.0).float()
    return [norm.float()] + [(g.float() * factor).to(g.dtype) for g in grads]


def _plain_update(state):
    case = state['case']
    params, momenta = state['params'], state['momenta']
    norm = _plain_norm(state['grads'])
    factor = (case['max_norm'] / (norm + EPS)).clamp(max=1.0).float()
    step = [g * factor + p * d for g, p, d in zip(state['grads'], params, state['decay'])]
    if momenta:
        torch._foreach_mul_(momenta, case['momentum'])
        torch._foreach_add_(momenta, step)
        step = momenta
    torch._foreach_add_(params, step, alpha=-state['lr'])
    return [norm.float()] + params + momenta


def run(state):
    if own:
        return _framework(state)
    plain = {'embed': _plain_embed, 'loss': _plain_loss, 'logprobs': _plain_logprobs, 'clip': _plain_clip,
             'update': _plain_update}
    return plain[state['case']['op']](state)


def exact(case, seed):
    """The definitions in 64 bits: log-sum-exp, one-hot rows and sums by token, on the inputs of prepare()."""
    state = prepare(case, seed)
    if case['op'] == 'embed':
        weight, tokens = state['weight'].detach(), state['tokens']
        out = [weight.double().index_select(0, tokens).mul_(case['scale'])]
        if case['train']:
            grad = torch.zeros(weight.shape, dtype=torch.float64, device=weight.device)
            kept = tokens != case['pad']
            grad.index_put_((tokens[kept],), state['grad'][kept].double() * case['scale'], accumulate=True)
            out.append(grad)
        return out
    if case['op'] in ('loss', 'logprobs'):
        x = state['logits'].detach().double()
        targets = state['targets']
        row = torch.arange(x.shape[0], device=x.device)
        lse = torch.logsumexp(x, 1)
        if case['op'] == 'loss':
            kept = (targets != IGNORE).nonzero()[:, 0]
            loss = (lse[kept] - x[kept, targets[kept]]).mean()
            grad = torch.exp(x.sub_(lse[:, None]))
            grad[targets == IGNORE] = 0
            grad[kept, targets[kept]] -= 1
            return [loss, grad.div_(kept.numel())]
        ids = None
        if case['top']:   # distinct ranks: by value, and by the place where values are the same
            ids = torch.argsort(x, dim=1, descending=True, stable=True)[:, :case['top']]
        x.sub_(lse[:, None])
        entropy = -(x.exp() * x).sum(1)
        out = [x[row, targets], entropy]
        if case['top']:
            out += [x.gather(1, ids), ids]
        if case['train']:
            gl, ge = (g.double() for g in state['grads'])
            p = x.exp()
            grad = -gl[:, None] * p - ge[:, None] * p * (x + entropy[:, None])
            grad[row, targets] += gl
            out.append(grad)
        return out
    norm = math.sqrt(math.fsum(float(torch.linalg.vector_norm(g.double())) ** 2 for g in state['grads']))
    factor = min(1.0, case['max_norm'] / (norm + EPS))
    if case['op'] == 'clip':
        return [torch.tensor(norm, dtype=torch.float64)] + [g.double() * factor for g in state['grads']]
    steps = [g.double() * factor + d * p.double() for g, p, d in zip(state['grads'], state['params'], state['decay'])]
    momenta = [case['momentum'] * m.double() + s for m, s in zip(state['momenta'], steps)]
    params = [p.double() - state['lr'] * s for p, s in zip(state['params'], momenta or steps)]
    return [torch.tensor(norm, dtype=torch.float64)] + params + momenta

"""The operators that training and scoring take beyond the attention layers, as a program calls them.

    loss         softmax cross entropy of a linear head over a large vocabulary, without its logits:
                 a training step (loss and the gradients of hidden states and weight) or the
                 scoring of tokens (one loss per token)
    rms_norm     RMSNorm, forward and backward, with the weight's gradient
    gated_norm   RMSNorm of the first half of a row times its weight times SiLU of the second half,
                 forward and backward, with the weight's gradient
    swiglu       first half of a row times SiLU of the second half, forward and backward

`listed` and `draw` give cases, `prepare` the inputs of one, `run` one pass (elementary torch
operations in 32 bits, or the framework's calls where `own` is set), `work` what a pass cannot do
without, and `exact` the results in 64 bits.
"""

import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16, 'fp32': torch.float32}
EPS = 1e-6         # the norms' epsilon
IGNORED = -100     # the label of a token without a loss


# ---------------------------------------------------------------------------------- cases
def listed():
    """The 172M model's shapes (768 features, 12 heads of 64 with values of 128, MLP 2048, vocabulary
    32000, sequences of 4096), the tiny model's (256 features, MLP 688, 512 tokens), and generic ones."""
    return [
        # pretraining: eight sequences of 4096 tokens through the head of the 172M model
        _loss('loss_train_32768', 32768, 768, 32000, 'bf16', 'mean', 0.0),
        # instruction tuning: 60 % of the tokens are prompts and have no loss
        _loss('loss_train_tuning_8192', 8192, 768, 32000, 'bf16', 'sum', 0.6),
        # a small vocabulary of odd size, an odd token count, fp16, weighted tokens
        _loss('loss_train_odd_3001', 3001, 520, 8003, 'fp16', 'none', 0.1),
        # the tiny model in the parity mode's type
        _loss('loss_train_fp32_512', 512, 256, 32000, 'fp32', 'mean', 0.0),
        # the scores of one short answer's tokens
        _loss('loss_score_48', 48, 768, 32000, 'bf16', 'none', 0.0, train=False),
        # the block norms of a prefill-sized training batch
        _rows('rms_131072x768', 'rms_norm', 131072, 768, 'bf16'),
        # the query heads' norm: short rows, many of them
        _rows('rms_heads_393216x64', 'rms_norm', 393216, 64, 'bf16'),
        # the tiny model in the parity mode's type
        _rows('rms_fp32_512x256', 'rms_norm', 512, 256, 'fp32'),
        # the delta rule's output norm: eight sequences, 12 heads of 128
        _rows('gated_heads_393216x128', 'gated_norm', 393216, 128, 'bf16'),
        # an odd row count and length
        _rows('gated_odd_5003x250', 'gated_norm', 5003, 250, 'fp16'),
        # the MLP's activation
        _rows('swiglu_32768x2048', 'swiglu', 32768, 2048, 'bf16'),
        # the tiny model's in the parity mode's type
        _rows('swiglu_fp32_512x688', 'swiglu', 512, 688, 'fp32'),
    ]


def _loss(name, tokens, dim, vocab, dtype, reduction, ignored, train=True):
    return {'name': name, 'op': 'loss', 'tokens': tokens, 'dim': dim, 'vocab': vocab, 'dtype': dtype,
            'reduction': reduction, 'ignored': ignored, 'train': train}


def _rows(name, op, rows, dim, dtype):
    return {'name': name, 'op': op, 'rows': rows, 'dim': dim, 'dtype': dtype}


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """A case of the listed ones' ranges: 1 to 32768 tokens, 32 to 2048 features, vocabularies of 300 to
    131072, rows of 16 to 8192, every type."""
    op = rng.choice(['loss', 'loss', 'rms_norm', 'gated_norm', 'swiglu'])
    dtype = rng.choice(['bf16', 'bf16', 'fp16', 'fp32'])
    if op == 'loss':
        dim = _log_int(rng, 32, 2048)
        if rng.random() < 0.7:
            dim = -(-dim // 8) * 8
        vocab = _log_int(rng, 300, 131072)
        most = 32768 * 768 * 32000 // (16 if dtype == 'fp32' else 1)
        tokens = _log_int(rng, 1, max(1, min(32768, most // (dim * vocab))))
        case = _loss('', tokens, dim, vocab, dtype, rng.choice(['mean', 'sum', 'none']),
                     rng.choice([0.0, 0.0, 0.1, 0.5, 0.9]), rng.random() < 0.7)
    else:
        dim = _log_int(rng, 16, 8192)
        if rng.random() < 0.7:
            dim = -(-dim // 8) * 8
        most = 131072 * 768 // (2 if dtype == 'fp32' else 1) // (1 if op == 'rms_norm' else 2)
        case = _rows('', op, _log_int(rng, 1, max(1, most // dim)), dim, dtype)
    del case['name']
    return case


def _prompt(case):
    """The tokens come in runs (dialogues), and each run's head (the prompt) has no loss: their lengths."""
    run = min(1000, case['tokens'])
    return run, int(run * case['ignored'])


def _live(case):
    """How many tokens have a loss."""
    run, prompt = _prompt(case)
    whole, rest = divmod(case['tokens'], run)
    return whole * (run - prompt) + max(0, rest - prompt)


# ---------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device='cuda')
    g.manual_seed(seed)
    dtype, dim = DTYPES[case['dtype']], case['dim']

    def normal(*shape):
        return torch.randn(shape, device='cuda', generator=g)

    state = {'case': case}
    if case['op'] == 'loss':
        tokens, vocab = case['tokens'], case['vocab']
        # frequent tokens come far more often than rare ones; the hidden states of a partly trained
        # model lean towards their label's row by different amounts, from a guess to near certainty
        label = (vocab * torch.rand(tokens, device='cuda', generator=g) ** 3).long().clamp_max(vocab - 1)
        weight = normal(vocab, dim)
        lean = 0.3 * torch.rand(tokens, 1, device='cuda', generator=g) * (768 / dim) ** 0.5
        x = normal(tokens, dim) + lean * weight[label]
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True))
        weight *= 2.0 * dim ** -0.5      # logits of the other tokens deviate by 2
        run, prompt = _prompt(case)
        label[torch.arange(tokens, device='cuda') % run < prompt] = IGNORED
        state.update(x=x.to(dtype), weight=weight.to(dtype), label=label)
        if case['train']:
            # per-token losses are weighted (a reward's advantage, a curriculum), a single one arrives as it
            # is, but for fp16's loss scale
            one = torch.full((), 1024.0 if case['dtype'] == 'fp16' else 1.0, device='cuda')
            state['up'] = normal(tokens) if case['reduction'] == 'none' else one
            state['x'].requires_grad_()
            state['weight'].requires_grad_()
        return state
    rows, wide = case['rows'], 1 if case['op'] == 'rms_norm' else 2
    # activations with a few large channels, rows of different sizes; gates of both signs
    x = normal(rows, wide * dim) * (0.5 + torch.rand(rows, 1, device='cuda', generator=g))
    x[:, :dim:37] *= 4.0
    state.update(x=x.to(dtype).requires_grad_(), up=normal(rows, dim).to(dtype))
    if case['op'] != 'swiglu':
        state['weight'] = (1.0 + 0.2 * normal(dim)).to(dtype).requires_grad_()
    return state


# ---------------------------------------------------------------------------------- one pass
def run(state):
    case, op = state['case'], state['case']['op']
    if own:
        from motif_b200 import ops
        if op == 'loss':
            loss = ops.linear_cross_entropy(state['x'], state['weight'], state['label'], ignore_index=IGNORED,
                                            reduction=case['reduction'])
            if not case['train']:
                return {'loss': loss}
            dx, dw = torch.autograd.grad(loss, (state['x'], state['weight']), state['up'])
            return {'loss': loss.detach(), 'dx': dx, 'dw': dw}
        if op == 'swiglu':
            y = ops.swiglu(state['x'])
            return {'y': y.detach(), 'dx': torch.autograd.grad(y, state['x'], state['up'])[0]}
        norm = ops.rms_norm if op == 'rms_norm' else ops.gated_rms_norm
        y = norm(state['x'], state['weight'], EPS)
        dx, dw = torch.autograd.grad(y, (state['x'], state['weight']), state['up'])
        return {'y': y.detach(), 'dx': dx, 'dw': dw}
    with torch.no_grad():
        if op == 'loss':
            return _plain_loss(state)
        return _plain_rms(state) if op == 'rms_norm' else _plain_gated(state)


def _plain_loss(state):
    case, label = state['case'], state['label']
    x, w = state['x'].float(), state['weight'].float()
    live = label != IGNORED
    at = torch.where(live, label, 0)[:, None]
    scores = x @ w.t()
    scores -= scores.amax(-1, keepdim=True)
    target = scores.gather(1, at)[:, 0]
    p = scores.exp_()
    total = p.sum(-1)
    loss = torch.where(live, total.log() - target, 0.0)
    count = live.sum()
    if case['reduction'] != 'none':
        loss = loss.double().sum()
        loss = (loss / count if case['reduction'] == 'mean' else loss).float()
    if not case['train']:
        return {'loss': loss}
    up = state['up'] / count if case['reduction'] == 'mean' else state['up']
    up = torch.where(live, up, 0.0)
    p *= (up / total)[:, None]
    p.scatter_add_(1, at, -up[:, None])
    return {'loss': loss, 'dx': (p @ w).to(state['x'].dtype), 'dw': (p.t() @ x).to(state['weight'].dtype)}


def _plain_norm_back(x, w, up, r):
    """dx and dw of x r w for the gradient `up`, in 32 bits."""
    u = up * w
    dx = r * (u - x * (r * r * (u * x).mean(-1, keepdim=True)))
    return dx, (up * x * r).sum(0, dtype=torch.float64)


def _plain_rms(state):
    x, w, up, dtype = state['x'].float(), state['weight'].float(), state['up'].float(), state['x'].dtype
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    dx, dw = _plain_norm_back(x, w, up, r)
    return {'y': (x * r * w).to(dtype), 'dx': dx.to(dtype), 'dw': dw.to(dtype)}


def _plain_gated(state):
    """The gated norm; without a weight and a norm, SwiGLU."""
    both, up, dtype, dim = state['x'].float(), state['up'].float(), state['x'].dtype, state['case']['dim']
    x, gate = both[:, :dim], both[:, dim:]
    sig = torch.sigmoid(gate)
    act = gate * sig
    slope = sig * (1.0 + gate * (1.0 - sig))
    if state['case']['op'] == 'swiglu':
        return {'y': (x * act).to(dtype), 'dx': torch.cat([up * act, up * x * slope], 1).to(dtype)}
    w = state['weight'].float()
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
    dx, dw = _plain_norm_back(x, w, up * act, r)
    n = x * r * w
    return {'y': (n * act).to(dtype), 'dx': torch.cat([dx, up * n * slope], 1).to(dtype), 'dw': dw.to(dtype)}


# ---------------------------------------------------------------------------------- what it needs
def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    dim = case['dim']
    if case['op'] == 'loss':
        live, vocab = _live(case), case['vocab']
        ends = size * dim * (live + vocab) + 8 * case['tokens'] + 4 * (case['tokens'] if case['reduction'] == 'none' else 1)
        if not case['train']:
            return {'bytes': ends, 'flops': 2 * live * vocab * dim}
        # the scores once and a product for each gradient; every token's gradient is written
        return {'bytes': ends + size * dim * (case['tokens'] + vocab), 'flops': 6 * live * vocab * dim}
    one = case['rows'] * dim * size
    if case['op'] == 'rms_norm':
        return {'bytes': 4 * one + 2 * dim * size, 'flops': 14 * case['rows'] * dim}
    return {'bytes': 6 * one + (2 * dim * size if case['op'] == 'gated_norm' else 0), 'flops': 24 * case['rows'] * dim}


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions in float64, differentiated by autograd; the loss token by token in runs of 1024."""
    state = prepare(case, seed)
    x = state['x'].detach().double()
    if case['op'] == 'loss':
        return _exact_loss(case, state, x)
    dim = case['dim']
    x.requires_grad_()
    a = x[:, :dim]
    leaves = [x]
    if case['op'] != 'swiglu':
        w = state['weight'].detach().double().requires_grad_()
        leaves.append(w)
        a = a / torch.sqrt(a.pow(2).sum(-1, keepdim=True) / dim + EPS) * w
    y = a if case['op'] == 'rms_norm' else a * x[:, dim:] / (1.0 + torch.exp(-x[:, dim:]))
    grads = torch.autograd.grad(y, leaves, state['up'].double())
    return dict(zip(('y', 'dx', 'dw'), (y.detach(), *grads)))


def _exact_loss(case, state, x):
    w = state['weight'].detach().double()
    label, tokens = state['label'], case['tokens']
    count = int((label != IGNORED).sum())
    loss = torch.zeros(tokens, dtype=torch.float64, device='cuda')
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    for at in range(0, tokens, 1024):
        rows = torch.nonzero(label[at:at + 1024] != IGNORED)[:, 0] + at
        if not len(rows):
            continue
        logp = torch.log_softmax(x[rows] @ w.t(), -1)
        loss[rows] = -logp[torch.arange(len(rows), device='cuda'), label[rows]]
        if case['train']:
            g = logp.exp()
            g[torch.arange(len(rows), device='cuda'), label[rows]] -= 1.0
            up = state['up'].double()
            g *= up[rows, None] if case['reduction'] == 'none' else up / (count if case['reduction'] == 'mean' else 1)
            dx[rows] = g @ w
            dw += g.t() @ x[rows]
    if case['reduction'] == 'mean':
        loss = loss.sum() / count
    elif case['reduction'] == 'sum':
        loss = loss.sum()
    return {'loss': loss, 'dx': dx, 'dw': dw} if case['train'] else {'loss': loss}

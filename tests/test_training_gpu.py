"""The training operators together: a decoder-sized stack through `motif_b200.ops` against the same stack in
64 bits, the model's loss without logits, tensors past 2^31 elements, and a captured step."""

import pytest
import torch
import torch.nn.functional as F

from motif_b200 import ops
from motif_b200.config import MotifChordConfig
from motif_b200.model import MotifChordModel
from oracle import ops as oo

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return ((a - b).norm() / b.norm().clamp_min(1e-300)).item()


def parameters(seed, d=64, heads=2, hid=96, vocab=301):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g) * shape[-1] ** -0.5

    p = {'embed': torch.randn(vocab, d, generator=g), 'qkv': normal(3 * d, d), 'gate': normal(2 * d, d), 'o': normal(d, d),
         'up': normal(2 * hid, d), 'down': normal(d, hid), 'beta_g': normal(2 * heads, d)}
    for name, n in (('n1', d), ('n2', d), ('n3', d), ('gn', d // heads)):
        p[name] = 1 + 0.2 * torch.randn(n, generator=g)
    ggd = [0.3 + torch.rand(heads, generator=g), 0.5 * torch.rand(heads, generator=g), torch.rand(heads, generator=g),
           0.5 + torch.rand(heads, generator=g)]
    return p, ggd


def stack(p, ggd, ids, labels, o, heads=2):
    """Embedding, Chord attention, gated delta rule with its gated norm, SwiGLU MLP, loss: `o` has the operators."""
    B, T = ids.shape
    d = p['embed'].shape[1]
    x = F.embedding(ids, p['embed'])

    def split(t):
        return t.view(B, T, heads, -1).transpose(1, 2)

    q, k, v = (split(t).contiguous() for t in F.linear(o.rms_norm(x, p['n1']), p['qkv']).chunk(3, -1))
    log_n = torch.log(torch.arange(1, T + 1, device=ids.device, dtype=ggd[0].dtype)).repeat(B, 1)
    x = x + F.linear(o.chord(q, k, v, *ggd, log_n).transpose(1, 2).reshape(B, T, d), p['o'])
    h = o.rms_norm(x, p['n2'])
    bg = F.linear(h, p['beta_g'])
    beta, g = torch.sigmoid(split(bg[..., :heads])[..., 0]), -0.3 * torch.sigmoid(split(bg[..., heads:])[..., 0])
    key = F.normalize(split(F.linear(h, p['gate'][:d])), dim=-1)
    s, _ = o.delta(key, key, split(h).contiguous(), beta, g)
    gate = split(F.linear(h, p['gate'][d:]))
    x = x + o.gated_rms_norm(torch.cat([s, gate], -1), p['gn']).transpose(1, 2).reshape(B, T, d)
    x = x + F.linear(o.swiglu(F.linear(o.rms_norm(x, p['n3']), p['up'])), p['down'])
    return o.loss(x, p['embed'], labels)


class Ours:
    rms_norm, gated_rms_norm, swiglu = staticmethod(ops.rms_norm), staticmethod(ops.gated_rms_norm), staticmethod(ops.swiglu)
    chord, delta = staticmethod(ops.apply_chord_attention), staticmethod(ops.chunk_gated_delta_rule)
    loss = staticmethod(ops.linear_cross_entropy)


class Plain:
    """The same in plain torch (the oracle's attention and delta rule)."""

    @staticmethod
    def rms_norm(x, w, eps=1e-6):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w

    @classmethod
    def gated_rms_norm(cls, x, w):
        v, g = x.chunk(2, -1)
        return cls.rms_norm(v, w) * F.silu(g)

    @staticmethod
    def swiglu(x):
        v, g = x.chunk(2, -1)
        return v * F.silu(g)

    @staticmethod
    def chord(q, k, v, alpha, beta, mu, ssmax, log_n):
        return oo.chord_attention(q, k, v, alpha, beta, mu, ssmax, log_n, q_start=0)

    @staticmethod
    def delta(q, k, v, beta, g):
        return oo.recurrent_gated_delta_rule(q, k, v, beta, g, None)

    @staticmethod
    def loss(x, w, labels):
        return F.cross_entropy(F.linear(x, w).flatten(0, -2), labels.flatten(), ignore_index=-100)


def batch(seed, B=3, T=70, vocab=301):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, vocab, (B, T), generator=g)
    labels = torch.cat([ids[:, 1:], torch.full((B, 1), -100)], 1)
    labels[0, :40] = -100  # a prompt
    labels[2, 50:] = -100  # padding
    return ids, labels


def test_a_training_step_in_fp32():
    """Each operator's gradients are within 1e-5 of 64 bits where its inputs are the same (their own tests); the
    step passes through seven of them, each of which hands on the errors of those before it, and the weights of
    the layers between are of norm 2 at most: 7 x 2 x 1e-5 bounds the whole."""
    p, ggd = parameters(1)
    ids, labels = batch(2)
    ours = {k: v.cuda().requires_grad_() for k, v in p.items()}
    loss = stack(ours, [t.cuda() for t in ggd], ids.cuda(), labels.cuda(), Ours)
    loss.backward()
    want = {k: v.double().requires_grad_() for k, v in p.items()}
    ref = stack(want, [t.double() for t in ggd], ids, labels, Plain)
    ref.backward()
    assert abs(loss.item() - ref.item()) <= 1e-5 * abs(ref.item())
    for k in p:
        assert ours[k].grad.dtype == torch.float32 and rel(ours[k].grad.cpu(), want[k].grad) < 1.4e-4, (
            k, rel(ours[k].grad.cpu(), want[k].grad))


def test_a_captured_training_step():
    """The whole step and its update as a CUDA graph: replays give what eager steps give, bit for bit."""
    p, ggd = parameters(3)
    ggd = [t.cuda() for t in ggd]
    ids, labels = (t.cuda() for t in batch(4))

    def step(params, ids, labels):
        loss = stack(params, ggd, ids, labels, Ours)
        grads = torch.autograd.grad(loss, list(params.values()))
        with torch.no_grad():
            for w, g in zip(params.values(), grads):
                w.sub_(g, alpha=0.1)
        return loss.detach()

    eager = {k: v.cuda().requires_grad_() for k, v in p.items()}
    captured = {k: v.cuda().requires_grad_() for k, v in p.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = {k: v.cuda().requires_grad_() for k, v in p.items()}
        step(warm, ids, labels)
        graph = torch.cuda.CUDAGraph()
        buf, lab = ids.clone(), labels.clone()
        with torch.cuda.graph(graph, stream=side):
            out = step(captured, buf, lab)
    torch.cuda.current_stream().wait_stream(side)
    with torch.no_grad():
        for k, v in p.items():
            captured[k].copy_(v.cuda())
    for i in range(3):
        ids, labels = (t.cuda() for t in batch(10 + i))
        buf.copy_(ids), lab.copy_(labels)
        graph.replay()
        want = step(eager, ids, labels)
        assert torch.equal(out, want)
        for k in p:
            assert torch.equal(eager[k], captured[k]), k


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_model_loss_without_logits(dtype):
    """The logits of the model are of its dtype, so its own loss is off by a rounding of the largest logit (and the
    label's) each; in fp32 the products' sums of 256 terms are off by 256 e of the sums of magnitudes at most."""
    torch.manual_seed(0)
    cfg = MotifChordConfig(vocab_size=1000, model_dim=256, num_heads=4, num_kv_heads=2, head_k_dim=64, block_n=1)
    m = MotifChordModel(cfg).cuda().to(dtype).eval()
    ids = torch.randint(0, 1000, (2, 130), device='cuda')
    labels = ids.roll(-1, 1)
    labels[0, :60] = -100
    with torch.no_grad():
        full, lean = m(ids, labels=labels), m(ids, labels=labels, return_logits=False)
    top = full.logits.abs().max().item()
    bound = 2 * top * torch.finfo(dtype).eps / 2 + 2 * 256 * E * 256
    assert lean.logits is None and lean.last_logits is None and lean.next_token() is None
    assert torch.equal(lean.hidden_states, full.hidden_states)
    assert abs(lean.loss.item() - full.loss.item()) <= bound, (lean.loss.item(), full.loss.item(), bound)
    # and the cache goes on from there
    one = torch.randint(0, 1000, (2, 1), device='cuda')
    with torch.no_grad():
        assert torch.equal(m(one, cache=lean.cache).logits, m(one, cache=full.cache).logits)
    with pytest.raises(ValueError, match='labels'):
        m(ids, labels=labels[:, 1:], return_logits=False)


def test_more_elements_than_32_bits_count():
    rows, dim = (1 << 31) // 768 + 1000, 768
    assert rows * dim > 1 << 31
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(1))
    x.requires_grad_()
    w = torch.ones(dim, device='cuda', dtype=torch.bfloat16).requires_grad_()
    y = ops.rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), x.detach())
    for part in (slice(0, 5), slice(rows - 5, rows)):
        xs = x[part].detach().clone().requires_grad_()
        ys = ops.rms_norm(xs, w)
        assert torch.equal(y[part], ys) and torch.equal(dx[part], torch.autograd.grad(ys, xs, xs.detach())[0])
    # dw = the sum over rows of x^2 r: about one a row; 2^-9 of it for the last rounding, a thread's sum of up to
    # rows / 296 / 8 terms and the 296 x 8 sums in fp32
    mean = (x[:1 << 16].detach().double().pow(2) * torch.rsqrt(x[:1 << 16].detach().double().pow(2).mean(1, keepdim=True))).mean()
    assert ((dw.double() / rows - mean).abs() <= 2.0 ** -8 * mean + 8 * (2 / rows) ** 0.5 + 0.02).all()
    del y, dx, x

    tokens, dim, vocab = (1 << 31) // 1024 + 700, 1024, 100
    x = torch.empty(tokens, dim, dtype=torch.bfloat16, device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(2))
    w = (0.05 * torch.randn(vocab, dim, device='cuda')).to(torch.bfloat16)
    label = torch.randint(0, vocab, (tokens,), device='cuda')
    x.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, label, reduction='sum')
    dx, = torch.autograd.grad(loss, x)
    for part in (slice(0, 600), slice(tokens - 600, tokens)):
        xs = x[part].detach().clone().requires_grad_()
        want, = torch.autograd.grad(ops.linear_cross_entropy(xs, w, label[part], reduction='sum'), xs)
        # sums of 100 terms may be cut differently in a small call: their fp32 errors are 2^-23 (100 / 16 + 8) of sums
        # of |G| |w| (2 max |w| at most) each, then either is rounded by 2^-9
        assert ((dx[part].double() - want.double()).abs() <= 2.0 ** -8 * want.double().abs() + 1e-5 * w.abs().max()).all()
    each = ops.linear_cross_entropy(x.detach(), w, label, reduction='none')
    # one loss in fp32 each, added in 64 bits and rounded: far below 1e-6 of their sum
    assert abs(each.double().sum().item() - loss.item()) <= 1e-6 * loss.item()

"""Edges of the training operators: labels infinitely far away, logits far from zero, long sums, weights of other
types, calls under torch's transforms, tensors past 2^31 elements, and what a launch tracker sees."""

import pytest
import torch

from motif_b200 import _lib, ops
from motif_b200.config import MotifChordConfig
from motif_b200.model import MotifChordModel

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    _lib.wait_timeouts()
    yield
    assert _lib.wait_timeouts() == 0


def gradients(x, w, label, reduction='mean', up=None):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(x, w, label, reduction=reduction)
    up = torch.ones_like(loss) if up is None else up
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), up))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize('N,V', [(40, 300), (40, 257), (9, 300)])
def test_a_label_whose_logit_is_minus_infinity(dtype, N, V):
    """Its loss is infinite and its gradients are those of a label that is only far away: the label's own probability is
    0 in both.  (The last tile's columns behind the words are -inf as well.)"""
    g = torch.Generator(device='cuda').manual_seed(V)
    x = torch.randn(N, 64, device='cuda', generator=g)
    x[:, 0] = 16
    x = x.to(dtype)
    w = torch.randn(V, 64, device='cuda', generator=g) * 0.2
    w[:, 0] = 0
    far, label = V - 1, torch.randint(0, V - 1, (N,), device='cuda', generator=g)
    label[::3] = far
    w = w.to(dtype)
    w[far, 0] = -100
    want = gradients(x, w, label)
    # 16 times the type's lowest number is -inf in fp32; fp16's own infinity
    w[far, 0] = float('-inf') if dtype == torch.float16 else torch.finfo(dtype).min
    assert want[0].isfinite() and want[1].isfinite().all() and want[2].isfinite().all()
    for reduction in ('mean', 'sum', 'none'):
        with torch.no_grad():
            alone = ops.linear_cross_entropy(x, w, label, reduction=reduction)
        got = gradients(x, w, label, reduction)
        assert torch.equal(got[0], alone) and not got[0].isnan().any() and got[0].isinf().any()
        if reduction == 'none':
            assert torch.equal(got[0].isinf(), label == far)
        assert got[2].isfinite().all()
        if reduction == 'mean':
            assert torch.equal(got[2], want[2])
            if dtype != torch.float16:  # (0 times fp16's infinity)
                assert torch.equal(got[1][:, 1:], want[1][:, 1:])


@pytest.mark.parametrize('kind', [torch.float64, torch.int32, torch.bool])
def test_norm_modules_take_weights_of_any_type(kind):
    """As they did before they took gradients: a weight in a type that no kernel reads is converted to the input's."""
    g = torch.Generator(device='cuda').manual_seed(1)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        x = torch.randn(5, 64, device='cuda', generator=g).to(dtype)
        for module, n in ((ops.RMSNorm, 64), (ops.GatedRMSNorm, 32)):
            w = (2 * torch.randn(n, device='cuda', generator=g)).to(kind)
            m, same = module(n, eps='1e-5').cuda(), module(n, eps=1e-5).cuda()  # (what float() reads will do, too)
            m.weight = torch.nn.Parameter(w, requires_grad=kind == torch.float64)
            same.weight = torch.nn.Parameter(w.to(dtype))
            with torch.no_grad():
                assert torch.equal(m(x), same(x))
            xl, xs = x.clone().requires_grad_(), x.clone().requires_grad_()
            y, z = m(xl), same(xs)
            y.sum().backward(), z.sum().backward()
            assert torch.equal(y, z) and torch.equal(xl.grad, xs.grad)
            if kind == torch.float64:
                assert m.weight.grad.dtype == kind and torch.equal(m.weight.grad, same.weight.grad.double())


def test_labels_are_refused_before_the_cache_moves():
    torch.manual_seed(0)
    cfg = MotifChordConfig(vocab_size=500, model_dim=256, num_heads=4, num_kv_heads=2, head_k_dim=64, block_n=1)
    m = MotifChordModel(cfg).cuda().eval()
    ids = torch.randint(0, 500, (2, 20), device='cuda')
    with torch.no_grad():
        want = m(ids).logits
        cache = m.create_cache()
        for bad in (ids.float(), ids.bool(), ids[:, 1:]):
            with pytest.raises(ValueError, match='labels'):
                m(ids, cache=cache, labels=bad, return_logits=False)
        assert torch.equal(m(ids, cache=cache).logits, want)


def test_views_that_are_negated_lazily():
    g = torch.Generator(device='cuda').manual_seed(5)
    x, w = torch.randn(40, 64, device='cuda', generator=g), torch.randn(64, device='cuda', generator=g)
    head = torch.randn(300, 64, device='cuda', generator=g) * 0.2
    label = torch.randint(0, 300, (40,), device='cuda', generator=g)
    up = torch.randn(40, 64, device='cuda', generator=g)
    neg = torch._neg_view
    for f in (lambda x, w: ops.rms_norm(x, w), lambda x, w: ops.gated_rms_norm(x, w[:32]), lambda x, w: ops.swiglu(x)):
        for grad in (False, True):
            a, b = neg(x).requires_grad_(grad), neg(w).requires_grad_(grad)
            c, d = (-x).requires_grad_(grad), (-w).requires_grad_(grad)
            y, z = f(a, b), f(c, d)
            assert torch.equal(y, z)
            if grad:
                dy = up[:, :y.shape[1]].contiguous()
                for p, q in zip(torch.autograd.grad(y, (a, b), neg(dy), allow_unused=True),
                                torch.autograd.grad(z, (c, d), -dy, allow_unused=True)):
                    assert (p is None and q is None) or torch.equal(p, q)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for n in (40, 9):
            for reduction in ('none', 'mean'):
                a, b = x[:n].to(dtype), head.to(dtype)
                u = up[:n, 0].contiguous() if reduction == 'none' else torch.tensor(1.5, device='cuda')
                want = gradients(-a, -b, label[:n], reduction, -u)
                a, b = neg(a).requires_grad_(), neg(b).requires_grad_()
                loss = ops.linear_cross_entropy(a, b, neg(-label[:n]), reduction=reduction)
                got = (loss, *torch.autograd.grad(loss, (a, b), neg(u)))
                assert all(torch.equal(p, q) for p, q in zip(got, want))


def launched(f):
    tr = _lib.Tracker(events=False)
    before = _lib.set_tracker(tr)
    try:
        f()
        torch.cuda.synchronize()
    finally:
        _lib.set_tracker(before)
    count = tr.launches
    f()  # not counted any more
    assert tr.launches == count
    return count


def test_a_tracker_counts_the_kernels_that_ran():
    """bf16 loss: packed rows, scores, join; with gradients scores, settled rows, their second form, and for dx and dW a
    product and a join of split sums each, for every run of rows.  fp16 and `none`: the backward pass computes scores."""
    g = torch.Generator(device='cuda').manual_seed(1)

    def loss(N, V, dtype, reduction, grads, d=64, shift=0):
        x = torch.randn(N, d, device='cuda', generator=g).to(dtype).requires_grad_('x' in grads)
        w = torch.randn(V, d + shift, device='cuda', generator=g).to(dtype)[:, shift:].requires_grad_('w' in grads)
        label = torch.randint(0, V, (N,), device='cuda', generator=g)

        def run():
            out = ops.linear_cross_entropy(x, w, label, reduction=reduction)
            if 'b' in grads:
                out.sum().backward()
        return launched(run)

    bf16, fp32 = torch.bfloat16, torch.float32
    assert loss(300, 1000, bf16, 'none', '') == loss(300, 1000, bf16, 'mean', '') == 3
    assert loss(300, 1000, bf16, 'mean', '', shift=1) == 4    # the weight is packed
    assert loss(9000, 1000, bf16, 'mean', '') == 4            # the labels are counted first
    assert loss(300, 1000, bf16, 'mean', 'xw') == 8
    assert loss(300, 1000, bf16, 'mean', 'x') == loss(300, 1000, bf16, 'mean', 'w') == 6
    assert loss(9000, 33000, bf16, 'mean', 'xw') == 2 + 2 * 7  # two runs of 7936 rows
    assert loss(300, 1000, bf16, 'mean', 'xwb') == 8 + 1       # and the product with what arrives
    assert loss(300, 1000, bf16, 'none', 'xwb') == 3 + 6
    assert loss(300, 1000, fp32, 'mean', 'xwb') == 9 + 1
    assert loss(9, 1000, fp32, 'mean', 'xwb') == 3 + 3 + 1

    x = torch.randn(50, 128, device='cuda', generator=g)
    w = torch.ones(128, device='cuda', requires_grad=True)
    xl = x.clone().requires_grad_()
    assert launched(lambda: ops.rms_norm(x, w.detach())) == 1
    assert launched(lambda: ops.rms_norm(xl, w)) == 1
    assert launched(lambda: ops.rms_norm(xl, w).sum().backward()) == 1 + 2
    assert launched(lambda: ops.rms_norm(xl, w.detach()).sum().backward()) == 1 + 1
    assert launched(lambda: ops.swiglu(xl).sum().backward()) == 1 + 1


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_losses_of_logits_far_from_zero(dtype):
    """Logits z + w_v with z of 500 to 1000 and w_v multiples of 1 / 16 below 8: products and sums are exact in fp32, and z
    cancels.  What is left, in units e of the loss (|z + w - top| < 16, 24 in powers of two): the exponent's rounding 24
    ln 2 e, log2 e's own 4 e, ex2's 4 e, the sum's V / 32 + 64 e, the logarithm's and the last two sums' 16 e each."""
    V, N = 300, 90
    g = torch.Generator(device='cuda').manual_seed(3)
    z = 500 + 4 * torch.randint(0, 126, (N,), device='cuda', generator=g)
    own = torch.randint(-127, 128, (V,), device='cuda', generator=g) / 16
    x, w = torch.zeros(N, 8, device='cuda'), torch.zeros(V, 8, device='cuda')
    x[:, 0], x[:, 1], w[:, 0], w[:, 1] = z, 1, 1, own
    x, w = x.to(dtype), w.to(dtype)
    assert torch.equal(x[:, 0].float(), z.float()) and torch.equal(w[:, 1].float(), own)
    label = torch.randint(0, V, (N,), device='cuda', generator=g)
    want = own.double().logsumexp(0) - own.double()[label]
    bound = (17 + 4 + 4 + V / 32 + 64 + 48) * E
    with torch.no_grad():
        got = ops.linear_cross_entropy(x, w, label, reduction='none')
    assert (got.double() - want).abs().max() <= bound, (got.double() - want).abs().max() / E
    each = torch.stack([gradients(x[i:i + 1], w, label[i:i + 1], 'sum')[0] for i in range(N)])
    assert (each.double() - want).abs().max() <= bound, (each.double() - want).abs().max() / E


@pytest.mark.parametrize('N', [20, 300])
def test_fp32_scores_of_many_features(N):
    """One word's logit is a sum of 16384 positive products, the others' are 0: the loss is that sum.  512 terms at a time
    are cut off at 24 bits (2 e) once for 16 of them, the six products of parts add 4 such ends and lose 4 e; then 32 sums
    are added with a rounding each, and the loss is rounded."""
    d, V = 16384, 300
    g = torch.Generator(device='cuda').manual_seed(N)
    x = 0.5 + torch.rand(N, d, device='cuda', generator=g)
    w = torch.zeros(V, d, device='cuda')
    w[0] = 0.03 + 0.06 * torch.rand(d, device='cuda', generator=g)
    label = torch.randint(1, V, (N,), device='cuda', generator=g)
    want = x.double() @ w[0].double()
    bound = (2 * (512 / 16 + 4) + 4 + 32 + 4) * E * want
    with torch.no_grad():
        got = ops.linear_cross_entropy(x, w, label, reduction='none')
    assert ((got.double() - want).abs() <= bound).all(), ((got.double() - want).abs() / want).max() / E
    loss = gradients(x, w, label, 'sum')[0]
    assert abs(loss.item() - want.sum().item()) <= (bound.sum() + 2 * E * want.sum()).item()
    got = gradients(x, w, label, 'none')  # G is -1 at the label and 1 at word 0: dW's row there is the sum of x
    total = x.double().sum(0)
    assert ((got[2][0].double() - total).abs() <= (2 * (N / 16 + 8) + 8) * E * total).all()


def test_transforms_are_refused():
    """Forward-mode tangents, vmap, torch.func's gradients and batched upstream gradients: an error, never a number."""
    from torch.autograd import forward_ad as fw

    x = torch.randn(6, 64, device='cuda')
    w, half = torch.ones(64, device='cuda'), torch.ones(32, device='cuda')
    head, label = torch.randn(100, 64, device='cuda') * 0.2, torch.arange(6, device='cuda')
    calls = [lambda x: ops.rms_norm(x, w), lambda x: ops.gated_rms_norm(x, half), ops.swiglu,
             lambda x: ops.linear_cross_entropy(x, head, label[:x.shape[0]]),
             lambda x: ops.linear_cross_entropy(x, head, label[:x.shape[0]], reduction='none')]
    for f in calls:
        for grad in (False, True):
            with fw.dual_level(), pytest.raises(NotImplementedError, match='forward-mode'):
                f(fw.make_dual(x.clone().requires_grad_(grad), torch.ones_like(x)))
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(x.expand(3, 6, 64).clone())
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(x)
        xl = x.clone().requires_grad_()
        y = f(xl)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(y, xl, torch.ones(2, *y.shape, device='cuda'), is_grads_batched=True)
    for f, t in ((lambda w: ops.rms_norm(x, w), w), (lambda w: ops.linear_cross_entropy(x, w, label), head)):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(t)
        with fw.dual_level(), pytest.raises(NotImplementedError, match='forward-mode'):
            f(fw.make_dual(t, torch.ones_like(t)))
    assert ops.rms_norm(x, w).isfinite().all()  # and the calls after those are as ever


def test_weight_gradients_past_32_bits():
    """Only the first and the last rows, the latter past 2^31 elements, have a gradient: dW is that of those rows alone,
    but for the order of its sums (a bound of fp32's: terms one after another, on the sum of magnitudes)."""
    rows, dim = (1 << 31) // 768 + 1000, 768
    x = torch.empty(rows, dim, dtype=torch.bfloat16, device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(1))
    w = torch.ones(dim, device='cuda').requires_grad_()
    dy = torch.zeros(rows, dim, dtype=torch.bfloat16, device='cuda')
    some = torch.cat([torch.arange(40), torch.arange(rows - 900, rows)]).cuda()
    assert (rows - 900) * dim > 1 << 31
    dy[some] = torch.randn(940, dim, device='cuda', generator=torch.Generator('cuda').manual_seed(2)).to(dy.dtype)
    dw, = torch.autograd.grad(ops.rms_norm(x, w), w, dy)
    xs, ds = x[some].double(), dy[some].double()
    terms = ds * xs * torch.rsqrt(xs.square().mean(1, keepdim=True) + 1e-6)
    # r and the products (dim / 32 + 40) e each as in the norms' own tests, up to 940 terms in a row
    assert ((dw.double() - terms.sum(0)).abs() <= (dim / 32 + 40 + 940) * E * terms.abs().sum(0)).all()
    del x, dy, dw

    tokens, dim, vocab = (1 << 31) // 1024 + 700, 1024, 100
    x = torch.empty(tokens, dim, dtype=torch.bfloat16, device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(3))
    w = (0.05 * torch.randn(vocab, dim, device='cuda')).to(torch.bfloat16).requires_grad_()
    label = torch.randint(0, vocab, (tokens,), device='cuda')
    up = torch.zeros(tokens, device='cuda')
    some = torch.cat([torch.arange(30), torch.arange(tokens - 600, tokens)]).cuda()
    assert (tokens - 600) * dim > 1 << 31
    up[some] = 1
    # all tokens have a loss: packed rows past 2^31 elements
    dw, = torch.autograd.grad(ops.linear_cross_entropy(x, w, label, reduction='none'), w, up)
    want, = torch.autograd.grad(ops.linear_cross_entropy(x[some], w, label[some], reduction='none'), w, up[some])
    xs = x[some].double()
    G = torch.softmax(xs @ w.double().t(), 1)
    G[torch.arange(630), label[some]] -= 1
    size = G.abs().t() @ xs.abs()
    # the same roundings of the same G (its logits' sums are those of one tile either way); sums cut off once for 16
    # terms; and each of the two results is within half a step of its sum, 2^-8 of that, so they are 2 x 2^-8 apart
    bound = 2.02 * 2.0 ** -8 * want.double().abs() + 4 * E * (630 / 16 + 8 + 2) * size
    assert ((dw.double() - want.double()).abs() <= bound).all()
    # and all others ignored: the last rows are packed to the front
    label[:tokens - 600] = -100
    dw, = torch.autograd.grad(ops.linear_cross_entropy(x, w, label, reduction='sum'), w)
    want, = torch.autograd.grad(ops.linear_cross_entropy(x[-600:], w, label[-600:], reduction='sum'), w)
    assert torch.equal(dw, want)


LOW = [(dtype, low) for dtype in (torch.bfloat16, torch.float16, torch.float32)
       for low in (-2.0e3, -6.0e4, -1e8, -1e10, -1e20, torch.finfo(dtype).min) if low >= torch.finfo(dtype).min]


@pytest.mark.parametrize('dtype,low', LOW)
@pytest.mark.parametrize('N,V', [(40, 300), (40, 257), (9, 300)])
def test_a_label_that_is_masked_with_a_low_value(dtype, N, V, low):
    """Its loss is what it is below the others, to the rounding of that number, with or without gradients; these are those
    of a label 100 below."""
    g = torch.Generator(device='cuda').manual_seed(V)
    x = torch.randn(N, 64, device='cuda', generator=g)
    x[:, 0] = 1
    x = x.to(dtype)
    w = torch.randn(V, 64, device='cuda', generator=g) * 0.2
    w[:, 0] = 0
    far, label = V - 1, torch.randint(0, V - 1, (N,), device='cuda', generator=g)
    label[::3] = far
    w = w.to(dtype)
    w[far, 0] = -1000
    want = gradients(x, w, label)
    w[far, 0] = low
    s = x.double() @ w.double().t()
    exact = s.logsumexp(1) - s[torch.arange(N), label]
    for reduction in ('none', 'sum', 'mean'):
        with torch.no_grad():
            alone = ops.linear_cross_entropy(x, w, label, reduction=reduction)
        got = gradients(x, w, label, reduction)
        there = {'none': exact, 'sum': exact.sum(), 'mean': exact.mean()}[reduction]
        over = there.abs() > torch.finfo(torch.float32).max
        for loss in (alone, got[0]):
            assert torch.equal(loss.isinf(), over) and not loss.isnan().any()
            # sums of 64 products (the one of the label's is as it is) and of V exponentials: far below 1e-5
            assert ((loss.double() - there).abs() <= 1e-5 + 1e-6 * there.abs())[~over].all()
        assert all(t.isfinite().all() for t in got[1:])
        if reduction == 'mean':
            assert torch.equal(got[2], want[2]) and torch.equal(got[1][:, 1:], want[1][:, 1:])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('size', [1e5, 2e6, 1e9, 1e12, 1e30])
def test_logits_of_any_size(dtype, size):
    """One word in eight is far above the others, by the same amount for all of them: their logits are equal, so a loss is
    the logarithm of their number for their own labels."""
    for N in (40, 9):
        x = torch.zeros(N, 64, device='cuda', dtype=dtype)
        w = torch.zeros(304, 64, device='cuda', dtype=dtype)
        x[:, 0], w[::8, 0] = 1, size
        label = torch.arange(N, device='cuda') * 8 % 304
        for reduction in ('none', 'mean'):
            loss, dx, dw = gradients(x, w, label, reduction)
            with torch.no_grad():
                alone = ops.linear_cross_entropy(x, w, label, reduction=reduction)
            want = torch.full_like(loss, 38).log()
            assert ((loss - want).abs() <= 1e-5).all() and ((alone - want).abs() <= 1e-5).all(), (loss, alone)
            assert dx.isfinite().all() and dw.isfinite().all()

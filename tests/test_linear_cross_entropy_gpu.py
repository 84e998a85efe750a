"""`ops.linear_cross_entropy` against its definition in 64 bits and against differences.

Tolerances.  With u the half step of the tensors' type (`eps / 2`) and e = 2^-24:
  logits   sums of d products in fp32: the tensor cores cut every partial sum off at 24 bits (2 e) once for 16 products
           or less, so a logit is off by ds = 2 e (d / 16 + 4) sum |x_i w_i| (fp32 operands: three bf16 parts keep
           24 bits, the products left out are 4 e of sum |x_i w_i| more)
  loss     its largest logit's and its target's ds, and the sum's: V terms' partial sums, of at most 256 + 8 + ...
           one after another (each pair walks its tiles: V / 2 in the worst case, cut off nowhere, e each) and a
           few units of exp and log: (V / 2 + 64) e would be the bound of a plain running sum; the sums of 32 are
           trees of 2 x 16, so V / 32 + 64 holds
  G        exp(s - top) / sum: |p| (3 ds + (V / 32 + 64 + |s - top|) e) plus u (|p| + [target]) of its one rounding
           (in fp16 also its smallest step, 2^-24 / 2^15; in fp32 three parts: 4 e instead of u)
  dx, dW   the errors of G times the other operand, summed as magnitudes; 2 e (terms / 16 + 8) of the sum of
           magnitudes for the summation; u of the result for the last rounding
  in one pass (mean and sum, bf16 and fp32): what is rounded is exp(s - s_t), relative to which G's error is the
           same; dW's other operand is x / sum rounded to the type (u of |G| |x|); and the result is rounded once
           more when it is multiplied with the gradient that arrives (u).  In bf16 a row's divisor takes back the
           rounding of its label's place, so the others carry that one as well (u p), and three roundings in a row
           are (1 + u)^3 - 1 < 3.03 u
  tiny     an exponential below 2^-126 is 0, so G may be off by that and by as much where it is multiplied:
           2^-125 |g|, times the other operand
  16 fp32 tokens or less, without the tensor cores: a lane adds d / 8 + 4 products one after another and the warp
           five times (ds holds); dx adds up to 64 words one after another (e each) where V / 16 is less
"""

import threading

import pytest
import torch

from motif_b200 import _lib, ops

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    _lib.wait_timeouts()
    yield
    assert _lib.wait_timeouts() == 0


def inputs(N, d, V, dtype, seed, ignored=0.0, sharp=2.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(N, d, device='cuda', generator=g)
    w = torch.randn(V, d, device='cuda', generator=g) * sharp * d ** -0.5
    label = torch.randint(0, V, (N,), device='cuda', generator=g)
    if V > 4 and N > 4:
        label[: N // 4] = label[0].item()  # a frequent word
        label[-1], label[-2] = V - 1, 0
    if ignored:
        label[torch.rand(N, device='cuda', generator=g) < ignored] = -100
    return x.to(dtype), w.to(dtype), label


def reference(x, w, label, reduction, up, ignore=-100):
    """Loss and gradients in 64 bits, and bounds of their errors."""
    dtype, (N, d), V = x.dtype, x.shape, w.shape[0]
    u = torch.finfo(dtype).eps / 2
    few = dtype == torch.float32 and N <= 16
    live = label != ignore
    xd, wd = x.double(), w.double()
    xl, tl = xd[live], label[live]
    n = len(tl)
    row = torch.arange(n, device=x.device)
    s = xl @ wd.t()
    top = s.amax(1, keepdim=True)
    total = (s - top).exp().sum(1, keepdim=True)
    one = (top + total.log())[:, 0] - s[row, tl]
    ds = (2 * (d / 16 + 4) + (4 if dtype == torch.float32 else 0)) * E * (xl.abs() @ wd.abs().t())
    dmax = ds.amax(1)
    bound_one = 2 * dmax + ds[row, tl] + (V / 32 + 64) * E + 2 * E * (one.abs() + top[:, 0].abs() + s[row, tl].abs())
    loss, bound = torch.zeros(N, dtype=torch.float64, device=x.device), torch.zeros(N, dtype=torch.float64, device=x.device)
    loss[live], bound[live] = one, bound_one
    if reduction == 'none':
        g = up.double()[live]
    elif reduction == 'sum':
        loss, bound, g = loss.sum(), bound.sum() + 2 * E * one.abs().sum(), up.double().expand(n)
    else:
        loss, bound, g = loss.sum() / n, bound.sum() / n + 2 * E * one.abs().sum() / n, (up.double() / n).expand(n)
    p = (s - top).exp() / total
    G = p.clone()
    G[row, tl] -= 1
    hit = torch.zeros_like(p)
    hit[row, tl] = 1
    ru = 4 * E if dtype == torch.float32 else u
    dG = p * (3 * dmax[:, None] + (V / 32 + 64 + (top - s).abs()) * E) + ru * G.abs() + 4 * E * hit
    if dtype == torch.float16:
        dG = dG + 2.0 ** -40
    once = reduction != 'none' and dtype != torch.float16
    if once and dtype == torch.bfloat16:
        dG = 1.01 * (dG + u * p)
    if dtype != torch.float16:
        dG = dG + 2.0 ** -125
    ga = g.abs()[:, None]
    G, dG = G * g[:, None], dG * ga + 4 * E * G.abs() * ga
    if reduction == 'none' and dtype == torch.float16 and n:  # G is kept relative to the largest gradient
        dG = dG + 2.0 ** -39 * ga.max()
    dx, bdx = torch.zeros_like(xd), torch.zeros_like(xd)
    dx[live] = G @ wd
    bdx[live] = dG @ wd.abs() + 2 * E * (max(V / 16, 32 if few else 0) + 8) * (G.abs() @ wd.abs())
    dw = G.t() @ xl
    bdw = dG.t() @ xl.abs() + 2 * E * (N / 16 + 8) * (G.abs().t() @ xl.abs())
    tiny = TINY[dtype]
    if once:
        bdw = bdw + (u + 4 * E) * (G.abs().t() @ xl.abs())
        u = 2 * u
    return (loss, dx, dw), (bound, bdx + (u + 4 * E) * dx.abs() + tiny, bdw + (u + 4 * E) * dw.abs() + tiny)


def near(name, got, want, bound):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), (name, int(bad.sum()), bad.nonzero()[:4].tolist(),
                           ((got.double() - want).abs() / bound.clamp_min(1e-300)).max().item())


def run(x, w, label, reduction, up, ignore=-100):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = ops.linear_cross_entropy(x, w, label, ignore_index=ignore, reduction=reduction)
    return (loss, *torch.autograd.grad(loss, (x, w), up))


def upstream(N, reduction, seed=1):
    if reduction != 'none':
        return torch.tensor(1.5, device='cuda')
    return torch.randn(N, device='cuda', generator=torch.Generator(device='cuda').manual_seed(seed))


def check(x, w, label, reduction, up=None, ignore=-100):
    up = upstream(len(label), reduction) if up is None else up
    got = run(x, w, label, reduction, up, ignore)
    want, bound = reference(x, w, label, reduction, up, ignore)
    assert got[0].dtype == torch.float32 and got[1].dtype == x.dtype and got[2].dtype == w.dtype
    for name, a, b, c in zip(('loss', 'dx', 'dw'), got, want, bound):
        near(name, a, b, c)
    with torch.no_grad():
        near('loss alone', ops.linear_cross_entropy(x, w, label, ignore, reduction), want[0], bound[0])
    return got


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('N,d,V', [(1, 64, 256), (5, 64, 300), (130, 64, 1000), (256, 128, 512), (300, 72, 257),
                                   (64, 8, 40), (3, 1, 2), (33, 100, 777), (257, 520, 2051), (1, 768, 32000)])
@pytest.mark.parametrize('reduction', ['mean', 'none'])
def test_small(N, d, V, dtype, reduction):
    x, w, label = inputs(N, d, V, dtype, N + d + V)
    check(x, w, label, reduction)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('N,d,V,ignored', [(2049, 768, 4001, 0.3), (9000, 128, 1031, 0.1), (700, 1032, 20000, 0.0),
                                           (5000, 64, 5000, 0.95), (9000, 64, 17000, 0.0)])
def test_larger(N, d, V, ignored, dtype):
    """More than one run of rows and more than one piece of the vocabulary among them."""
    x, w, label = inputs(N, d, V, dtype, N + d + V, ignored)
    check(x, w, label, 'sum')
    check(x, w, label, 'none')


@pytest.mark.parametrize('dtype', DTYPES)
def test_sharp_logits(dtype):
    """Tokens that are nearly certain (1 - p of 1e-2 to 1e-6) keep their gradients' bits, and logits of hundreds
    overflow nothing."""
    x, w, label = inputs(200, 128, 900, dtype, 4, sharp=4.0)
    label = torch.where(torch.arange(200, device='cuda') % 2 == 0, (x.double() @ w.double().t()).argmax(1), label)
    check(x, w, label, 'none')
    check((x.float() * 20).to(dtype), w, label, 'mean')


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('bad', [float('nan'), float('inf'), float('-inf')])
def test_ignored_tokens_touch_nothing(dtype, bad):
    x, w, label = inputs(300, 96, 700, dtype, 9, ignored=0.5)
    want = run(x, w, label, 'mean', upstream(300, 'mean'))
    dirty = x.clone()
    dirty[label == -100] = bad
    got = run(dirty, w, label, 'mean', upstream(300, 'mean'))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not got[1][label == -100].any() and got[2].isfinite().all()
    # the tokens with a loss, alone: the same bits
    keep = label != -100
    only = run(x[keep], w, label[keep], 'mean', upstream(300, 'mean'))
    assert torch.equal(only[0], want[0]) and torch.equal(only[1], want[1][keep]) and torch.equal(only[2], want[2])


@pytest.mark.parametrize('dtype', DTYPES)
def test_no_token_has_a_loss(dtype):
    x, w, label = inputs(70, 64, 300, dtype, 2)
    label[:] = -100
    for reduction, value in (('mean', float('nan')), ('sum', 0.0), ('none', 0.0)):
        loss, dx, dw = run(x, w, label, reduction, upstream(70, reduction))
        assert torch.equal(loss, torch.full_like(loss, value)) or (value != value and loss.isnan())
        assert not dx.any() and not dw.any()
    for reduction in ('mean', 'sum', 'none'):
        loss, dx, dw = run(x[:0], w, label[:0], reduction, upstream(0, reduction))
        assert dx.shape == (0, 64) and not dw.any() and loss.shape == (() if reduction != 'none' else (0,))


def test_labels_that_are_no_word():
    x, w, label = inputs(40, 64, 300, torch.bfloat16, 3)
    want = run(x, w, label, 'none', torch.ones(40, device='cuda'))
    label[5], label[17], label[30] = 300, -1, 1 << 40
    odd = torch.zeros(40, dtype=torch.bool, device='cuda')
    odd[[5, 17, 30]] = True
    loss, dx, dw = run(x, w, label, 'none', torch.ones(40, device='cuda'))
    assert torch.equal(loss.isnan(), odd) and torch.equal(dx.isnan().any(1), odd) and dw.isnan().all()
    assert torch.equal(loss[~odd], want[0][~odd]) and torch.equal(dx[~odd], want[1][~odd])
    assert run(x, w, label, 'mean', torch.tensor(1.0, device='cuda'))[0].isnan()
    # another value may stand for "no loss", a word of the vocabulary too
    for ignore in (0, 299, -1, 1 << 40):
        lab = torch.where(odd, torch.tensor(ignore, device='cuda'), torch.arange(40, device='cuda') + 20)
        check(x, w, lab, 'sum', ignore=ignore)


@pytest.mark.parametrize('dtype', DTYPES)
def test_strides_alignment_shapes_and_label_types(dtype):
    x, w, label = inputs(60, 100, 333, dtype, 6)
    bigx = torch.randn(60, 140, device='cuda').to(dtype)
    bigw = torch.randn(333, 151, device='cuda').to(dtype)
    for off, woff in ((0, 0), (8, 8), (3, 1), (16, 51)):
        bigx[:, off:off + 100] = x
        bigw[:, woff:woff + 100] = w
        check(bigx[:, off:off + 100], bigw[:, woff:woff + 100], label, 'sum')
    check(x.t().contiguous().t(), w.t().contiguous().t(), label, 'none')
    check(x[::2], w, label[::2], 'mean')
    check(x[:1].expand(60, 100), w, label, 'mean')
    want = run(x, w, label, 'none', upstream(60, 'none'))
    for kind in (torch.int32, torch.int16):
        xl = x.view(3, 4, 5, 100)
        loss = ops.linear_cross_entropy(xl, w, label.to(kind).view(3, 4, 5), reduction='none')
        assert loss.shape == (3, 4, 5) and torch.equal(loss.flatten(), want[0])
    lab = label.repeat_interleave(2)[::2]  # labels apart
    assert torch.equal(ops.linear_cross_entropy(x, w, lab, reduction='none'), want[0])
    one = ops.linear_cross_entropy(x[0], w, label[0], reduction='none')
    assert one.shape == ()
    if dtype == torch.float32:  # so few tokens take another order of d's sum, within the same bound
        exact, bound = reference(x[:1], w, label[:1], 'none', upstream(1, 'none'))
        near('one token', one[None], exact[0], bound[0])
    else:
        assert torch.equal(one, want[0][0])


def test_upstream_gradients_of_any_size_and_stride():
    x, w, label = inputs(90, 64, 500, torch.float16, 8)
    g = torch.Generator(device='cuda').manual_seed(3)
    wide = torch.randn(90, 3, device='cuda', generator=g)
    check(x, w, label, 'none', wide[:, 1])
    check(x, w, label, 'none', torch.tensor(0.25, device='cuda').expand(90))
    check(x, w, label, 'none', torch.zeros(90, device='cuda'))
    for size in (1e-4, 1e3):  # the largest sets the scale: the smallest is within its rounding
        check(x, w, label, 'none', wide[:, 0] * size)
        check(x, w, label, 'mean', torch.tensor(size, device='cuda'))
    for dtype in (torch.bfloat16, torch.float32):
        x, w, label = inputs(90, 64, 500, dtype, 8)
        for size in (1e-20, 1e20):
            check(x, w, label, 'none', wide[:, 0] * size)
            check(x, w, label, 'sum', torch.tensor(size, device='cuda'))


def test_differences():
    """<dx, a> + <dw, b> against a central difference of the 64-bit loss along (a, b); its error is about h^2
    of the third derivative, 1e-8 of values of this size."""
    x, w, label = inputs(12, 40, 70, torch.float32, 5, ignored=0.2)
    _, dx, dw = run(x, w, label, 'sum', torch.tensor(1.0, device='cuda'))
    g = torch.Generator(device='cuda').manual_seed(7)
    a = torch.randn(x.shape, dtype=torch.float64, device='cuda', generator=g)
    b = torch.randn(w.shape, dtype=torch.float64, device='cuda', generator=g)
    h = 1e-5

    def f(t):
        s = (x.double() + t * a) @ (w.double() + t * b).t()
        keep = label != -100
        return (s.logsumexp(1)[keep] - s[keep, label[keep]]).sum()

    slope = ((f(h) - f(-h)) / (2 * h)).item()
    terms = [dx.double() * a, dw.double() * b]
    got, size = sum(t.sum().item() for t in terms), sum(t.abs().sum().item() for t in terms)
    assert abs(got - slope) <= 2e-6 * size


def test_gradient_of_some_inputs_only():
    x, w, label = inputs(300, 64, 1000, torch.bfloat16, 1, ignored=0.1)
    up = torch.tensor(1.0, device='cuda')
    _, dx, dw = run(x, w, label, 'mean', up)
    xl = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(xl, w, label), xl)[0], dx)
    wl = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.linear_cross_entropy(x, wl, label), wl)[0], dw)
    assert not ops.linear_cross_entropy(x, w, label).requires_grad


def test_same_bits_every_time():
    x, w, label = inputs(3000, 256, 5000, torch.bfloat16, 8, ignored=0.2)
    first = run(x, w, label, 'mean', upstream(3000, 'mean'))
    for _ in range(3):
        again = run(x, w, label, 'mean', upstream(3000, 'mean'))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_streams_and_graphs():
    """Two calls at once on two streams; a training step captured into a graph and replayed on other tokens, with
    other numbers of them ignored."""
    a, b = inputs(700, 128, 3001, torch.bfloat16, 1, 0.3), inputs(500, 128, 3001, torch.bfloat16, 2)
    want = [run(*a, 'mean', upstream(700, 'mean')), run(*b, 'mean', upstream(500, 'mean'))]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for i, (s, args) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i] = run(*args, 'mean', upstream(len(args[2]), 'mean'))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for g, e in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(g, e))
    x, w, label = (t.clone() for t in a)
    up = upstream(700, 'mean')
    graphs, outs = [], []
    with torch.cuda.stream(streams[0]):
        for reduction in ('mean', 'none'):
            graph = torch.cuda.CUDAGraph()
            ups = up if reduction == 'mean' else upstream(700, 'none')
            with torch.cuda.graph(graph, stream=streams[0]):
                outs.append(run(x, w, label, reduction, ups))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(streams[0])
    for seed, ignored in ((5, 0.0), (6, 0.9), (7, 1.0), (1, 0.3)):
        nx, nw, nl = inputs(700, 128, 3001, torch.bfloat16, seed, ignored)
        x.copy_(nx), w.copy_(nw), label.copy_(nl)
        for graph in graphs:
            graph.replay()
        for out, reduction in zip(outs, ('mean', 'none')):
            fresh = run(nx, nw, nl, reduction, up if reduction == 'mean' else upstream(700, 'none'))
            assert all(torch.equal(p, q) or (p.isnan().all() and q.isnan().all()) for p, q in zip(out, fresh))


def test_a_large_vocabulary_and_what_it_takes():
    """131072 words, more than a piece; the memory of a step is far below the logits'."""
    x, w, label = inputs(4100, 64, 131072, torch.bfloat16, 3)
    check(x[:300], w, label[:300], 'mean')
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    run(x, w, label, 'mean', upstream(4100, 'mean'))
    peak = torch.cuda.max_memory_allocated() - base
    assert peak < 0.75e9 < 4100 * 131072 * 2, peak


def test_refusals():
    x, w, label = inputs(10, 64, 100, torch.bfloat16, 1)
    bad = [((x.cpu(), w, label), {}, 'CUDA'), ((x, w.cpu(), label), {}, 'CUDA'), ((x, w, label.cpu()), {}, 'CUDA'),
           ((x, w[:, :32], label), {}, 'weight'), ((x, w[0], label), {}, 'weight'), ((x, w[:0], label), {}, 'empty'),
           ((x, w, label[:5]), {}, 'labels'), ((x, w, label[:, None]), {}, 'labels'),
           ((x, w, label.float()), {}, 'whole numbers'), ((x.double(), w.double(), label), {}, 'dtype'),
           ((x, w.float(), label), {}, 'share one dtype'), ((x, w, label), {'reduction': 'max'}, 'reduction')]
    for args, kw, match in bad:
        with pytest.raises(ValueError, match=match):
            ops.linear_cross_entropy(*args, **kw)
    xl = x.clone().requires_grad_()
    with pytest.raises(NotImplementedError, match='second derivatives'):
        torch.autograd.grad(ops.linear_cross_entropy(xl, w, label), xl, create_graph=True)
    wl = w.clone().requires_grad_()
    loss, each = ops.linear_cross_entropy(x, wl, label), ops.linear_cross_entropy(x, wl, label, reduction='none')
    want = torch.autograd.grad(ops.linear_cross_entropy(x, wl, label), wl)[0]
    with torch.no_grad():
        wl.mul_(2)
    assert torch.equal(torch.autograd.grad(loss, wl)[0], want)  # computed with the loss
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        each.sum().backward()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_far_logits_in_some_runs_of_rows(dtype):
    """Labels whose logits are more than 66 below the largest one: their run of rows is computed again, with
    the others' results as they are.  (Runs are of 2^28 / 33024 words = 7936 rows, fp32 2560; no token is
    ignored, so that the far rows are the second's, the fourth's.)"""
    x, w, label = inputs(9000, 64, 33000, dtype, 12)
    alone = run(x, w, label, 'mean', upstream(9000, 'mean'))
    x[8500:8600] = (x[8500:8600].float() * 40).to(dtype)
    far = x[8500:8600].double() @ w.double().t()
    assert (far.amax(1) - far[torch.arange(100), label[8500:8600].clamp_min(0)]).max() > 100
    got = check(x, w, label, 'mean')
    assert torch.equal(got[1][:7680], alone[1][:7680])  # whole runs before them in both types


def test_gradients_are_used_twice():
    x, w, label = (t.clone() for t in inputs(300, 64, 500, torch.bfloat16, 4))
    x.requires_grad_(), w.requires_grad_()
    loss = ops.linear_cross_entropy(x, w, label)
    one = torch.autograd.grad(loss, (x, w), retain_graph=True)
    for t in one:
        t.zero_()  # what a caller does with its gradients changes nothing
    two = torch.autograd.grad(loss, (x, w), torch.tensor(2.0, device='cuda'))
    want = run(x, w, label, 'mean', torch.tensor(2.0, device='cuda'))
    assert torch.equal(two[0], want[1]) and torch.equal(two[1], want[2])


def test_first_call_of_a_host_thread():
    """A thread without a CUDA context of its own (an autograd thread's first call): the tensor maps are made all
    the same."""
    x, w, label = inputs(70, 64, 300, torch.bfloat16, 3)
    want = run(x, w, label, 'none', upstream(70, 'none'))
    sizes = _lib.i64_array((0, 0, 0))
    _lib.call('motif_b200_linear_cross_entropy_bytes', w.data_ptr(), 64, 70, 300, 64, _lib.MB_BF16, sizes)
    state, work = (torch.empty(n, dtype=torch.uint8, device='cuda') for n in (sizes[0], sizes[1]))
    loss, st = torch.empty(70, device='cuda'), torch.cuda.current_stream().cuda_stream
    torch.cuda.synchronize()
    errors = []

    def call():
        try:
            _lib.call('motif_b200_linear_cross_entropy', x.data_ptr(), 64, w.data_ptr(), 64, label.data_ptr(), -100, 0,
                      loss.data_ptr(), 70, 300, 64, state.data_ptr(), sizes[0], work.data_ptr(), sizes[1], _lib.MB_BF16, st)
            _lib.call('motif_b200_gemm', x.data_ptr(), 64, w.data_ptr(), 64, out.data_ptr(), 304, 70, 300, 64, _lib.MB_BF16,
                      st)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    out = torch.empty(70, 304, dtype=torch.bfloat16, device='cuda')
    t = threading.Thread(target=call)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert torch.equal(loss, want[0])


def test_entry_points_refuse_short_buffers():
    x, w, label = inputs(10, 64, 100, torch.bfloat16, 1)
    buf, loss = torch.empty(1 << 20, dtype=torch.uint8, device='cuda'), torch.empty((), device='cuda')
    common = (loss.data_ptr(), 10, 100, 64)
    with pytest.raises(ValueError, match='bytes of state and workspace needed'):
        _lib.call('motif_b200_linear_cross_entropy', x.data_ptr(), 64, w.data_ptr(), 64, label.data_ptr(), -100, 1, *common,
                  buf.data_ptr(), 1000, buf.data_ptr(), buf.numel(), _lib.MB_BF16, None)
    with pytest.raises(ValueError, match='256-byte aligned'):
        _lib.call('motif_b200_linear_cross_entropy', x.data_ptr(), 64, w.data_ptr(), 64, label.data_ptr(), -100, 1, *common,
                  buf.data_ptr() + 16, 1 << 19, buf.data_ptr(), buf.numel(), _lib.MB_BF16, None)
    with pytest.raises(ValueError, match='bytes of workspace needed'):
        _lib.call('motif_b200_linear_cross_entropy_train', x.data_ptr(), 64, w.data_ptr(), 64, label.data_ptr(), -100, 1,
                  loss.data_ptr(), None, None, 10, 100, 64, buf.data_ptr(), buf.numel(), _lib.MB_BF16, None)
    with pytest.raises(NotImplementedError, match='fp16'):
        _lib.call('motif_b200_linear_cross_entropy_train', x.data_ptr(), 64, w.data_ptr(), 64, label.data_ptr(), -100, 1,
                  loss.data_ptr(), None, None, 10, 100, 64, buf.data_ptr(), buf.numel(), _lib.MB_F16, None)
    with pytest.raises(ValueError, match='reduction must be 1 or 2'):
        _lib.call('motif_b200_linear_cross_entropy_train', x.data_ptr(), 64, w.data_ptr(), 64, label.data_ptr(), -100, 0,
                  loss.data_ptr(), None, None, 10, 100, 64, buf.data_ptr(), buf.numel(), _lib.MB_BF16, None)
    with pytest.raises(ValueError, match='unknown reduction'):
        _lib.call('motif_b200_linear_cross_entropy_backward', w.data_ptr(), 64, loss.data_ptr(), 0, 3, None, None, 10, 100, 64,
                  buf.data_ptr(), buf.numel(), buf.data_ptr(), buf.numel(), _lib.MB_BF16, None)


@pytest.mark.parametrize('N,d,V', [(1, 1, 1), (1, 3, 2), (2, 5, 63), (7, 36, 65), (8, 1001, 500), (9, 1028, 4099), (16, 2050, 1300),
                                   (16, 3200, 257), (15, 3199, 129), (16, 3201, 200), (17, 100, 900), (12, 768, 40000)])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
def test_few_fp32_tokens(N, d, V, reduction):
    x, w, label = inputs(N, d, V, torch.float32, N + d, ignored=0.2 if N > 4 else 0.0)
    check(x, w, label, reduction, upstream(N, reduction))


def test_few_fp32_tokens_strides_and_labels():
    """Rows that 16-byte loads cannot take, a weight inside a larger one, and labels that are no word."""
    x, w, label = inputs(11, 133, 701, torch.float32, 2, ignored=0.3)
    label[4] = 700
    wide = torch.full((701, 140), float('nan'), device='cuda')
    wide[:, 1:134] = w
    tall = torch.full((11, 150), float('nan'), device='cuda')
    tall[:, 2:135] = x
    for reduction in ('mean', 'none'):
        up = upstream(11, reduction)
        want = run(x, w, label, reduction, up)
        for got, exact in zip(run(tall[:, 2:135], wide[:, 1:134], label, reduction, up), want):
            assert torch.equal(got, exact)
    label[0], label[1] = 701, -5
    loss, dx, dw = run(x, w, label, 'none', upstream(11, 'none'))
    assert loss[:2].isnan().all() and dx[:2].isnan().all() and not loss[2:].isnan().any() and not dx[2:].isnan().any()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_a_captured_backward_pass_runs_twice(dtype):
    """Forward and backward passes in graphs of their own: each run of the second gives the same gradients."""
    x, w, label = inputs(300, 96, 700, dtype, 4, 0.2)
    up = torch.tensor(1.5, device='cuda')
    want = run(x, w, label, 'mean', up)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    ahead, back = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        xl, wl = x.detach().requires_grad_(), w.detach().requires_grad_()
        with torch.cuda.graph(ahead, stream=stream):
            loss = ops.linear_cross_entropy(xl, wl, label)
        with torch.cuda.graph(back, stream=stream, pool=ahead.pool()):
            grads = torch.autograd.grad(loss, (xl, wl), up)
    torch.cuda.current_stream().wait_stream(stream)
    ahead.replay()
    for _ in range(3):
        back.replay()
        assert all(torch.equal(a, b) for a, b in zip((loss, *grads), want))

"""RMSNorm, GatedRMSNorm and SwiGLU where a gradient is needed (`motif_b200.ops`), against the
formulas in 64 bits and against differences.

Tolerances, element by element, with u the half step of a type (`eps / 2`) and e = 2^-24, a rounding
in fp32.  A thread adds at most `seq` of a row's values one after another, the rest are trees of at
most 8 levels; rsqrt, the reciprocal and ex2 are within 2 units (4 e) each, and ex2's argument is
rounded (|g| e).  So r is off by (seq / 2 + 10) e, silu and its slope by (|g| + 14) e of their terms,
and k = seq + |g| + 40 covers a product of all of them.  What is summed (dx, dw) is off by that of
the sum of its terms' magnitudes, and each output is rounded once more by its own type.
"""

import pytest
import torch

from motif_b200 import ops

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(M, N, wide, dtype, seed, w_dtype=None):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x = torch.randn(M, wide * N, device='cuda', generator=g) * (0.2 + 2 * torch.rand(M, 1, device='cuda', generator=g))
    x[:, ::5] *= 3
    w = 1 + 0.3 * torch.randn(N, device='cuda', generator=g)
    dy = torch.randn(M, N, device='cuda', generator=g)
    return x.to(dtype), w.to(w_dtype or dtype), dy.to(dtype)


def formulas(x, w, dy, eps, kind):
    """y, dx, dw, and the magnitudes that their rounding errors are relative to, in 64 bits."""
    x, dy = x.double(), dy.double()
    N = dy.shape[1]
    one = torch.ones(N, dtype=torch.float64, device=x.device)
    w = one if w is None else w.double()
    v = x[:, :N]
    if kind == 'rms':
        act, slope, steep, far = one, None, None, 0.0
    else:
        gate = x[:, N:]
        sig = torch.sigmoid(gate)
        act, slope = gate * sig, sig * (1 + gate * (1 - sig))
        steep, far = sig * (1 + gate.abs()), gate.abs()
    if kind == 'swiglu':
        y, dv, mag_dv, n, mag_y = v * act, dy * act, (dy * act).abs(), v, (v * act).abs()
        dw = mag_dw = None
    else:
        r = (v.pow(2).mean(1, keepdim=True) + eps).pow(-0.5)
        n = v * r * w
        y = n * act
        u = dy * act * w
        mean = (u * v).mean(1, keepdim=True)
        dv = r * (u - v * r * r * mean)
        mag_dv = r * (u.abs() + v.abs() * r * r * (u * v).abs().mean(1, keepdim=True))
        dw, mag_dw, mag_y = (dy * act * v * r).sum(0), (dy * act * v * r).abs().sum(0), y.abs()
    if kind == 'rms':
        return y, dv, dw, mag_y, mag_dv, mag_dw, far
    dx = torch.cat([dv, dy * n * slope], 1)
    return y, dx, dw, mag_y, torch.cat([mag_dv, (dy * n).abs() * steep], 1), mag_dw, torch.cat([far, far], 1)


def near(name, got, want, bound):
    # a result beyond the type's largest number rounds to infinity: with r = 1000 (a row of zeros) and
    # a gate of 60, dx = 60000 dy w leaves fp16's range
    over = (want.abs() + bound >= torch.finfo(got.dtype).max) & got.isinf() & (got.sign() == want.sign())
    bad = ~((got.double() - want).abs() <= bound) & ~over
    assert not bad.any(), (name, int(bad.sum()), (got.double() - want).abs()[bad].max().item(), bound[bad].min().item())


def run(x, w, dy, eps, kind):
    x = x.detach().requires_grad_()
    leaves = [x] if w is None else [x, w.detach().requires_grad_()]
    if kind == 'rms':
        y = ops.rms_norm(x, leaves[1] if w is not None else None, eps)
    elif kind == 'gated':
        y = ops.gated_rms_norm(x, leaves[1] if w is not None else None, eps)
    else:
        y = ops.swiglu(x)
    return y, torch.autograd.grad(y, leaves, dy)


def check(x, w, dy, eps, kind):
    y, grads = run(x, w, dy, eps, kind)
    M, N = dy.shape
    ry, rdx, rdw, my, mdx, mdw, far = formulas(x, w, dy, eps, kind)
    k = max(32, -(-N // 32) if N <= 1024 else -(-N // 256)) + 40
    u = torch.finfo(x.dtype).eps / 2
    near('y', y, ry, my * (u + (k + (far[:, :N] if kind != 'rms' else 0)) * E) + TINY[x.dtype])
    near('dx', grads[0], rdx, rdx.abs() * u + mdx * (k + far) * E + TINY[x.dtype])
    assert y.dtype == x.dtype and grads[0].dtype == x.dtype
    if w is not None:
        # a thread adds M / (its grid's rows) terms, the CTAs' sums follow in runs of up to 148
        rows = -(-M // 148) + 148 + 32
        fars = far.max() if kind != 'rms' else 0
        near('dw', grads[1], rdw, rdw.abs() * torch.finfo(w.dtype).eps / 2 + mdw * (k + rows + fars) * E + TINY[w.dtype])
        assert grads[1].dtype == w.dtype and grads[1].shape == w.shape


SHAPES = [(1, 1), (3, 7), (5, 8), (33, 64), (1025, 64), (70, 96), (17, 100), (260, 128), (50, 250), (9, 256), (31, 300),
          (12, 512), (4801, 768), (7, 1000), (6, 1024), (5, 1032), (3, 2048), (19, 4096), (700, 4104), (4, 8192), (2, 8200),
          (3, 10001), (40, 701), (11, 301), (21, 2501), (9, 5001), (900, 2048)]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('M,N', SHAPES)
@pytest.mark.parametrize('kind', ['rms', 'gated', 'swiglu'])
def test_formulas(kind, M, N, dtype):
    x, w, dy = inputs(M, N, 1 if kind == 'rms' else 2, dtype, M * 31 + N)
    check(x, None if kind == 'swiglu' else w, dy, 1e-6, kind)


@pytest.mark.parametrize('kind', ['rms', 'gated'])
@pytest.mark.parametrize('w_dtype', DTYPES + [None])
def test_weight_dtypes(kind, w_dtype):
    for dtype in DTYPES:
        x, w, dy = inputs(37, 192, 1 if kind == 'rms' else 2, dtype, 5, w_dtype)
        check(x, w if w_dtype else None, dy, 1e-5, kind)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('kind', ['rms', 'gated', 'swiglu'])
def test_strides_and_alignment(kind, dtype):
    wide = 1 if kind == 'rms' else 2
    for N, left, right in ((64, 1, 0), (64, 8, 8), (64, 8, 3), (100, 0, 4), (1032, 3, 0)):
        big, w, dybig = inputs(23, N + 40, wide, dtype, N + left)
        x = torch.cat([big[:, :left], big[:, 40:40 + wide * N], big[:, :right]], 1)[:, left:left + wide * N]
        dy = dybig[:, left:left + N]
        w = w[:N]
        if kind == 'swiglu':
            w = None
        assert not x.is_contiguous() or left + right == 0
        check(x, w, dy, 1e-6, kind)
    # the gradient of a sum: one value for all rows and columns
    x, w, dy = inputs(23, 64, wide, dtype, 1)
    w = None if kind == 'swiglu' else w
    check(x, w, torch.full((1, 1), 0.5, dtype=dtype, device='cuda').expand(23, 64), 1e-6, kind)
    check(x, w, dy[:1].expand(23, 64), 1e-6, kind)
    # columns apart: a transposed input
    xt = x.t().contiguous().t()
    check(xt, w, dy, 1e-6, kind)
    # one row for all
    check(x[:1].expand(23, wide * 64), w, dy, 1e-6, kind)


def test_leading_dimensions_and_modules():
    g = torch.Generator(device='cuda').manual_seed(3)
    x = torch.randn(2, 3, 5, 48, device='cuda', generator=g)
    norm, gated, act = ops.RMSNorm(48).cuda(), ops.GatedRMSNorm(24).cuda(), ops.SwiGLU()
    assert norm(x).shape == x.shape and gated(x).shape == (2, 3, 5, 24) and act(x).shape == (2, 3, 5, 24)
    for m in (norm, gated):
        y = m(x)
        assert y.requires_grad
        y.square().sum().backward()
        xr, wr = x.double().reshape(-1, 48), torch.ones(m.dim, dtype=torch.float64, device='cuda')
        kind = 'rms' if m is norm else 'gated'
        ry = formulas(xr, wr, torch.zeros(30, m.dim, device='cuda'), 1e-6, kind)[0]
        rdw = formulas(xr, wr, 2 * ry, 1e-6, kind)
        near('dw', m.weight.grad, rdw[2], rdw[5] * 400 * E)
        with torch.no_grad():
            assert not m(x).requires_grad
    # the activation along another dimension
    z = torch.randn(4, 10, 6, device='cuda', generator=g).requires_grad_()
    y = ops.swiglu(z, dim=1)
    up = torch.randn(4, 5, 6, device='cuda', generator=g)
    got, = torch.autograd.grad(y, z, up)
    zr = z.detach().double().requires_grad_()
    want, = torch.autograd.grad(zr[:, :5] * torch.nn.functional.silu(zr[:, 5:]), zr, up.double())
    assert y.shape == (4, 5, 6) and (got.double() - want).abs().max() <= 64 * E * want.abs().max()


@pytest.mark.parametrize('kind', ['rms', 'gated', 'swiglu'])
def test_differences(kind):
    """<dx, a> + <dw, b> against a central difference of the 64-bit forward along (a, b): its error
    is about h^2 of the third derivative, 1e-8 of values of this size."""
    wide = 1 if kind == 'rms' else 2
    x, w, dy = inputs(6, 40, wide, torch.float32, 11)
    _, grads = run(x, None if kind == 'swiglu' else w, dy, 1e-6, kind)
    g = torch.Generator(device='cuda').manual_seed(12)
    a = torch.randn(x.shape, dtype=torch.float64, device='cuda', generator=g)
    b = torch.randn(w.shape, dtype=torch.float64, device='cuda', generator=g)
    h = 1e-5

    def f(t):
        y = formulas(x.double() + t * a, None if kind == 'swiglu' else w.double() + t * b, dy, 1e-6, kind)[0]
        return (y * dy.double()).sum()

    slope = ((f(h) - f(-h)) / (2 * h)).item()
    terms = [(grads[0].double() * a)]
    if kind != 'swiglu':
        terms.append(grads[1].double() * b)
    got, size = sum(t.sum().item() for t in terms), sum(t.abs().sum().item() for t in terms)
    assert abs(got - slope) <= 1e-6 * size + 200 * E * size


@pytest.mark.parametrize('dtype', DTYPES)
def test_edge_values(dtype):
    """Zero rows, a row whose squares are as small as eps, large rows; NaN and infinity stay in their rows."""
    x, w, dy = inputs(40, 128, 1, dtype, 2)
    x[3] = 0
    x[4] *= 1e-3
    x[5] *= 100
    check(x, w, dy, 1e-6, 'rms')
    bad = x.clone()
    bad[7, 5], bad[9, 0], bad[30] = float('nan'), float('inf'), float('-inf')
    y, (dx, dw) = run(bad, w, dy, 1e-6, 'rms')
    y0, (dx0, _) = run(x, w, dy, 1e-6, 'rms')
    keep = [i for i in range(40) if i not in (7, 9, 30)]
    assert torch.equal(y[keep], y0[keep]) and torch.equal(dx[keep], dx0[keep])
    assert y[7].isnan().all() and dx[7].isnan().all() and dw.isnan().any()
    # gates far out on both sides: no NaN where the result is finite
    both = torch.cat([x, x], 1)
    both[:, 128:] = torch.linspace(-60, 60, 128, device='cuda').to(dtype)
    check(both, w, dy, 1e-6, 'gated')
    check(both, None, dy, 1e-6, 'swiglu')


def test_no_rows():
    for dtype in DTYPES:
        w = torch.ones(64, dtype=dtype, device='cuda')
        x = torch.empty(0, 64, dtype=dtype, device='cuda')
        y, (dx, dw) = run(x, w, x, 1e-6, 'rms')
        assert y.shape == dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))
        x = torch.empty(2, 0, 128, dtype=dtype, device='cuda').requires_grad_()
        assert torch.autograd.grad(ops.swiglu(x).sum(), x)[0].shape == x.shape


def test_gradient_of_some_inputs_only():
    x, w, dy = inputs(9, 64, 1, torch.bfloat16, 1)
    _, (dx, dw) = run(x, w, dy, 1e-6, 'rms')
    xl = x.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.rms_norm(xl, w), xl, dy)[0], dx)
    wl = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.rms_norm(x, wl), wl, dy)[0], dw)


def test_same_bits_every_time():
    x, w, dy = inputs(3000, 768, 1, torch.bfloat16, 8)
    _, first = run(x, w, dy, 1e-6, 'rms')
    for _ in range(3):
        _, again = run(x, w, dy, 1e-6, 'rms')
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_streams_and_graphs():
    """On a side stream, and a forward and backward captured into a graph and replayed on new values."""
    x, w, dy = inputs(64, 256, 2, torch.bfloat16, 4)
    want = run(x, w, dy, 1e-6, 'gated')
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(x, w, dy, 1e-6, 'gated')
        graph = torch.cuda.CUDAGraph()
        buf = torch.zeros_like(x)
        with torch.cuda.graph(graph, stream=s):
            out = run(buf, w, dy, 1e-6, 'gated')
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    for scale in (1, 2):
        buf.copy_(x * scale)
        graph.replay()
        want = run(x * scale, w, dy, 1e-6, 'gated')
        assert torch.equal(out[0], want[0]) and all(torch.equal(a, b) for a, b in zip(out[1], want[1]))


def test_refusals():
    x = torch.randn(4, 64, device='cuda')
    w = torch.ones(64, device='cuda')
    for bad, match in (((x.cpu(), w), 'CUDA'), ((x, w.cpu()), 'CUDA'), ((x, w[:32]), 'weight'),
                       ((x.double(), w), 'dtype'), ((x, w.double()), 'dtype'), ((x[0, 0], None), 'last dimension')):
        with pytest.raises(ValueError, match=match):
            ops.rms_norm(*bad)
    with pytest.raises(ValueError, match='2 \\* dim'):
        ops.gated_rms_norm(x[:, :63], w)
    with pytest.raises(ValueError, match='even'):
        ops.swiglu(x[:, :63])
    with pytest.raises(ValueError, match='expects last dim'):
        ops.GatedRMSNorm(48).cuda()(x)
    # a gradient of the gradient is refused, not dropped
    xl = x.clone().requires_grad_()
    for y in (ops.rms_norm(xl, w), ops.gated_rms_norm(xl, w[:32]), ops.swiglu(xl)):
        with pytest.raises(NotImplementedError, match='second derivatives'):
            torch.autograd.grad(y.sum(), xl, create_graph=True)
    # values changed between forward and backward are noticed
    xl = x.clone().requires_grad_()
    y = ops.rms_norm(xl * 1, w.requires_grad_())
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()

"""Gradients where saved-tensor hooks hand the backward pass copies that lie elsewhere: with other addresses,
alignments and strides, on the host in between, or as something else altogether."""

import pytest
import torch

from motif_b200 import _lib, ops

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    _lib.wait_timeouts()
    yield
    assert _lib.wait_timeouts() == 0


def odd(t):
    """A copy that begins one element behind a 256-byte boundary."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    return buf[1:].view(t.shape).copy_(t)


def apart(t):
    """A copy whose rows lie apart, at odd elements; bytes and vectors every second element."""
    if t.dim() < 2:
        return torch.empty(2 * t.numel() + 2, dtype=t.dtype, device=t.device)[1:-1:2].view(t.shape).copy_(t)
    buf = torch.empty(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=t.device)
    return buf[..., 1:-2].copy_(t)


def turned(t):
    """A copy with its first dimension running fastest."""
    return t.mT.contiguous().mT if t.dim() > 1 else t.clone()


HOOKS = {
    'dense': lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
    'host': lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    'odd': lambda: torch.autograd.graph.saved_tensors_hooks(odd, lambda t: t),
    'apart': lambda: torch.autograd.graph.saved_tensors_hooks(apart, lambda t: t),
    'turned': lambda: torch.autograd.graph.saved_tensors_hooks(turned, lambda t: t),
}


def weights(V, d, dtype, g):
    """The same values as rows that the tensor maps take, and as rows that they do not."""
    w = (torch.randn(V, d, device='cuda', generator=g) * 2 * d ** -0.5).to(dtype)
    out = [w]
    for width, at in ((d + 2, 1), ((d + 7) // 8 * 8, 0), ((d + 23) // 8 * 8, 8)):
        buf = torch.zeros(V, width, dtype=dtype, device='cuda')
        out.append(buf[:, at:at + d].copy_(w))
    flat = torch.zeros(V * d + 1, dtype=dtype, device='cuda')
    out.append(flat[1:].view(V, d).copy_(w))
    return out


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('hook', HOOKS)
@pytest.mark.parametrize('N,d,V', [(70, 96, 700), (300, 97, 300), (9, 33, 130)])
def test_loss_that_reads_its_weight_again(hook, dtype, N, d, V):
    g = torch.Generator(device='cuda').manual_seed(N)
    x = torch.randn(N, d, device='cuda', generator=g).to(dtype)
    label = torch.randint(0, V, (N,), device='cuda', generator=g)
    label[::5] = -100
    for reduction in ('none', 'mean') if dtype == torch.float16 else ('none',):
        up = torch.randn(N, device='cuda', generator=g) if reduction == 'none' else torch.tensor(1.5, device='cuda')
        for w in weights(V, d, dtype, g):
            xl, wl = x.clone().requires_grad_(), w.detach().requires_grad_()
            loss = ops.linear_cross_entropy(xl, wl, label, reduction=reduction)
            want = torch.autograd.grad(loss, (xl, wl), up)
            with HOOKS[hook]():
                loss = ops.linear_cross_entropy(xl, wl, label, reduction=reduction)
            got = torch.autograd.grad(loss, (xl, wl), up)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (reduction, w.stride())


@pytest.mark.parametrize('dtype', DTYPES)
def test_a_weight_that_moves_between_the_passes(dtype):
    """`.data` exchanged for another layout of the same values (as sharded parameters do), both ways."""
    g = torch.Generator(device='cuda').manual_seed(1)
    x = torch.randn(50, 64, device='cuda', generator=g).to(dtype).requires_grad_()
    label = torch.randint(0, 300, (50,), device='cuda', generator=g)
    up = torch.randn(50, device='cuda', generator=g)
    forms = weights(300, 64, dtype, g)
    for first in forms:
        w = torch.nn.Parameter(first.detach())
        want = torch.autograd.grad(ops.linear_cross_entropy(x, w, label, reduction='none'), (x, w), up)
        for second in forms:
            w = torch.nn.Parameter(first.detach())
            loss = ops.linear_cross_entropy(x, w, label, reduction='none')
            w.data = second
            got = torch.autograd.grad(loss, (x, w), up)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_other_tensors_than_were_saved_are_refused():
    g = torch.Generator(device='cuda').manual_seed(2)
    x = torch.randn(50, 64, device='cuda', generator=g).half().requires_grad_()
    w = (torch.randn(300, 64, device='cuda', generator=g) * 0.2).half().requires_grad_()
    label = torch.randint(0, 300, (50,), device='cuda', generator=g)
    for change in (lambda t: t[:-1], lambda t: t.float(), lambda t: t.cpu(), lambda t: t.flatten()[:256]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            loss = ops.linear_cross_entropy(x, w, label)
        with pytest.raises(RuntimeError, match='came back as others'):
            loss.backward()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('hook', HOOKS)
@pytest.mark.parametrize('N,d,V', [(70, 96, 700), (33, 97, 300), (9, 33, 130)])
def test_gradients_that_were_computed_with_the_loss(hook, dtype, N, d, V):
    g = torch.Generator(device='cuda').manual_seed(N)
    x = torch.randn(N, d, device='cuda', generator=g).to(dtype).requires_grad_()
    w = (torch.randn(V, d, device='cuda', generator=g) * 0.2).to(dtype).requires_grad_()
    label = torch.randint(0, V, (N,), device='cuda', generator=g)
    up = torch.tensor(1.5, device='cuda')
    want = torch.autograd.grad(ops.linear_cross_entropy(x, w, label), (x, w), up)
    with HOOKS[hook]():
        loss = ops.linear_cross_entropy(x, w, label)
    for keep in (True, False):
        got = torch.autograd.grad(loss, (x, w), up, retain_graph=keep)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_what_a_hook_keeps_is_not_written_to(dtype):
    x = torch.randn(40, 64, device='cuda').to(dtype).requires_grad_()
    w = torch.randn(300, 64, device='cuda').to(dtype).requires_grad_()
    kept = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t) or t, lambda t: t):
        loss = ops.linear_cross_entropy(x, w, torch.arange(40, device='cuda'))
    before = [t.clone() for t in kept]
    got = torch.autograd.grad(loss, (x, w), torch.tensor(3.0, device='cuda'))
    assert kept and all(torch.equal(a, b) for a, b in zip(kept, before))
    for t in got:
        t.zero_()
    assert all(torch.equal(a, b) for a, b in zip(kept, before))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('N', [50, 9])
def test_other_gradients_than_were_saved_are_refused(dtype, N):
    x = torch.randn(N, 64, device='cuda').to(dtype).requires_grad_()
    w = (torch.randn(300, 64, device='cuda') * 0.2).to(dtype).requires_grad_()
    for change in (lambda t: t[:-1], lambda t: t.double(), lambda t: t.half(), lambda t: t.cpu(), lambda t: t.flatten()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
            loss = ops.linear_cross_entropy(x, w, torch.arange(N, device='cuda'))
        with pytest.raises(RuntimeError, match='came back as others'):
            loss.backward()


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('hook', HOOKS)
@pytest.mark.parametrize('kind', ['rms', 'gated', 'swiglu'])
def test_norms(kind, hook, dtype):
    """Dense copies give the same bits.  Rows that vectors take and that come back as ones that they do not: the same but
    for the order of the sums, N / 32 + 40 steps of 2^-24 for a row's and 33 more for dW's, of magnitudes below
    |dy w r| (|x r| + 1) (|g| + 1) < 4 x 3 x 1.3 x 5 x 2 = 156 at these sizes."""
    g = torch.Generator(device='cuda').manual_seed(1)
    for N in (64, 250, 1032):
        x = torch.randn(3, 11, N if kind == 'rms' else 2 * N, device='cuda', generator=g).to(dtype)
        w = torch.randn(N, device='cuda', generator=g).to(dtype)
        dy = torch.randn(3, 11, N, device='cuda', generator=g).to(dtype)
        f = {'rms': ops.rms_norm, 'gated': ops.gated_rms_norm, 'swiglu': lambda x, w: ops.swiglu(x)}[kind]
        xl, wl = x.clone().requires_grad_(), w.clone().requires_grad_()
        leaves = (xl, wl)[:1 if kind == 'swiglu' else 2]
        want = torch.autograd.grad(f(xl, wl), leaves, dy)
        with HOOKS[hook]():
            y = f(xl, wl)
        got = torch.autograd.grad(y, leaves, dy)
        for a, b in zip(got, want):
            if hook in ('dense', 'host'):
                assert torch.equal(a, b)
            tol = 2.02 * torch.finfo(dtype).eps / 2 * b.double().abs() + 2 * (N / 32 + 73) * 2.0 ** -24 * 156
            assert ((a.double() - b.double()).abs() <= tol).all()


def test_other_rows_than_were_saved_are_refused():
    x, w = torch.randn(20, 64, device='cuda').requires_grad_(), torch.ones(64, device='cuda').requires_grad_()
    half = torch.ones(32, device='cuda').requires_grad_()
    calls = (lambda: ops.rms_norm(x, w), lambda: ops.gated_rms_norm(x, half), lambda: ops.swiglu(x), lambda: ops.rms_norm(x))
    for f in calls:
        for change in (lambda t: t[:-1], lambda t: t.double(), lambda t: t.half(), lambda t: t.cpu(), lambda t: t[..., :-2],
                       lambda t: torch.cat([t, t])):
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
                y = f()
            with pytest.raises(RuntimeError, match='came back as another'):
                y.sum().backward()
    # the weight alone, exchanged for a shorter one or one of another type
    for other in (torch.ones(32, device='cuda'), torch.ones(64, device='cuda', dtype=torch.float64)):
        p = torch.nn.Parameter(torch.ones(64, device='cuda'))
        y = ops.rms_norm(x, p)
        p.data = other
        with pytest.raises(RuntimeError, match='came back as another'):
            y.sum().backward()

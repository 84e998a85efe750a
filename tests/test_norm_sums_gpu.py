"""The norms' weight gradient: how its sums over the rows are added."""

import pytest
import torch

from motif_b200 import ops

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


@pytest.mark.parametrize('M,N,rows', [(512, 256, 8), (200, 64, 16), (300, 250, 8), (290, 1024, 1), (148, 2048, 1)])
def test_few_rows_add_without_rounding(M, N, rows):
    """Rows of 1 and -1 have a norm of 1, so the terms are dy and -dy as they are.  There are as many groups of threads as
    rows (`rows` of a CTA), so what is rounded is each CTA's sum, by half a step, and the whole."""
    g = torch.Generator(device='cuda').manual_seed(M)
    x = torch.randn(M, N, device='cuda', generator=g).sign().requires_grad_()
    w = torch.ones(N, device='cuda').requires_grad_()
    y = ops.rms_norm(x, w, 0.0)
    assert torch.equal(y, x)
    dy = torch.randn(M, N, device='cuda', generator=g)
    dw, = torch.autograd.grad(y, w, dy)
    terms = dy.double() * x.detach().double()
    whole = M // rows * rows
    ctas = terms[:whole].view(-1, rows, N).sum(1).abs().sum(0) + terms[whole:].sum(0).abs()
    bound = 1.001 * E * (ctas * (rows > 1) + terms.sum(0).abs())
    assert ((dw.double() - terms.sum(0)).abs() <= bound).all(), ((dw.double() - terms.sum(0)).abs() / bound).max()

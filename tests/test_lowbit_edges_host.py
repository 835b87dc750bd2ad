"""Distillation, norm and microscaled products at the edges of what they document, without a GPU."""
import math

import pytest
import torch

import lowbit_ref as R
from test_lowbit_host import _differences


@pytest.mark.parametrize("outside", ["listed", "masked", "one masked", "free"])
def test_distillation_gradient_against_differences_with_nothing_outside_the_list(outside):
    """With the teacher's log-sum-exp: every class listed, or all others at -inf, leaves the loss without the term of the remaining
    mass, and the gradient is that of what is left.  Divergences of q do not see a shift of the logits, so a row's gradient adds up
    to (1 - 1) or (sum p - sum p) times its scale: 0."""
    g = torch.Generator().manual_seed(5)
    classes, top = 7, 7 if outside == "listed" else 4
    logits = torch.randn(3, classes, generator=g, dtype=torch.float64)
    index = torch.stack([torch.randperm(classes, generator=g)[:top] for _ in range(3)])
    teacher = torch.randn(3, top, generator=g, dtype=torch.float64)
    free = torch.ones(3, classes, dtype=torch.bool).scatter_(1, index, False)
    if outside == "masked":
        logits[free] = -math.inf
    if outside == "one masked":
        logits[1][free[1]] = -math.inf
    lse = torch.logsumexp(teacher / 1.5, 1) + 0.4
    w = torch.tensor([1.0, 0.5, 2.0])
    f = lambda v: R.distill(v, teacher, index, 1.5, 0.7, w, lse)[0]
    grad = R.distill(logits, teacher, index, 1.5, 0.7, w, lse)[1]
    assert torch.allclose(grad, _differences(f, logits), atol=1e-8)
    assert torch.allclose(grad.sum(1), torch.zeros(3, dtype=torch.float64), atol=1e-12)


def test_a_bias_that_waits_for_a_gradient_is_refused():
    """The product's weights and bias are frozen: a gradient that never comes is not to be waited for."""
    from gan_amd import ops
    from gan_amd._lib import GanHipError
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    w, x = ops.MxMatrix(u8(4, 10, 16), u8(1, 10, 4), 100, 10), torch.zeros(3, 100)
    bias = torch.zeros(10, requires_grad=True)
    for rows in (x, x.clone().requires_grad_(True), ops.MxTensor(u8(3, 128), u8(3, 4), 100)):
        with pytest.raises(ValueError, match="bias"):
            ops.mx_matmul(rows, w, bias)
        for frozen in (bias.detach(), None):
            with pytest.raises((GanHipError, RuntimeError)) as e:       # (goes on to the library, which has no GPU here)
                ops.mx_matmul(rows, w, frozen)
            assert "bias" not in str(e.value)


def test_rows_are_quantised_in_the_products_launch_up_to_where_a_launch_of_their_own_is_as_fast():
    """A call that quantises in the product's launch asks for no codes beside the product's own workspace."""
    from gan_amd import _lib as L
    one = lambda fmt, rows, k, n: L.lib.gan_mx_linear_workspace_bytes(0, fmt, rows, k, n) == L.lib.gan_mx_matmul_workspace_bytes(0, fmt, rows, k, n)
    e4m3, e2m1 = L.MX_FORMATS['e4m3'], L.MX_FORMATS['e2m1']
    for rows, n in ((64, 256), (17, 1000), (250, 250), (16, 4000)):
        assert [one(e4m3, rows, k, n) for k in (100, 2048, 2400, 2560, 2561)] == [True] * 4 + [False], (rows, n)
        assert [one(e2m1, rows, k, n) for k in (100, 2048, 2049, 2400, 2560)] == [True] * 2 + [False] * 3, (rows, n)

"""Distillation, norm and microscaled products at the edges of what they document (GPU), against the float64 forms of lowbit_ref.py.

Tolerances are those derived at the head of test_gpu_lowbit.py unless a test derives its own.
"""
import math

import pytest
import torch

import lowbit_ref as R
from test_gpu_lowbit import TYPES, _check_distill, _lists, gen, ids, normal, tiny

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ distillation
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("tau", [1.0, 0.1])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,classes,masked", [(3, 1000, (4, 8)), (2, 1001, (2, 61)), (2, 20000, (100, 20000)), (2050, 200, (64, 200)),
                                                 (2, 140000, (512, 139000))])
def test_distillation_of_low_logits_with_masked_runs(rows, classes, masked, dtype, tau, rest):
    """Runs of classes at -inf beside logits near -200 (log-probabilities used as logits): a thread may hold masked classes alone, and
    their gradient is 0.  The logits lie within 4 tau of each other, so |z - max| <= 40 holds at both temperatures."""
    g = gen(rows + classes)
    logits = (-200 + tau * normal(g, rows, classes).clamp(-4, 4)).to(dtype)
    lo, hi = masked
    logits[:, lo:hi] = -math.inf
    top = min(8, classes - (hi - lo))
    free = torch.cat([torch.arange(lo), torch.arange(hi, classes)]).cuda()
    index = torch.stack([free[torch.randperm(free.numel(), generator=g, device='cuda')[:top]] for _ in range(rows)])
    teacher = tau * 2 * normal(g, rows, top)
    lse = torch.logsumexp(teacher / tau, 1) + 0.3 if rest else None
    w = (torch.arange(rows, device='cuda') % max(1, rows // 40) == 0).float()
    _, grad = _check_distill(logits, teacher, index, tau, 1.0, w, lse)
    assert (grad[:, lo:hi] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,classes,top,outside", [(3, 1, 1, "listed"), (2, 10, 10, "listed"), (3, 100, 100, "listed"), (2, 1024, 1024, "listed"),
                                                      (2051, 9, 9, "listed"), (3, 100, 100, "listed twice"), (2, 300, 5, "masked"),
                                                      (3, 4100, 33, "masked"), (2, 70000, 9, "masked"), (2, 140001, 3, "masked"),
                                                      (2050, 130, 7, "masked"), (4, 500, 20, "masked in some rows")])
def test_distillation_with_nothing_outside_the_list(rows, classes, top, outside, dtype):
    """The teacher's remaining mass is left out of the loss, and out of its gradient, where no class outside the list has any: a row's
    gradient adds up to 0.  Allowed: 2^-17 and a half step of the type for each class by its size, q + p <= 2 in all."""
    g = gen(rows + classes + top)
    logits = (2 * normal(g, rows, classes)).to(dtype)
    index, teacher = _lists(g, rows, classes, top, torch.float32)
    if outside == "listed twice":
        index[:, 1] = index[:, 0]
        logits.scatter_(1, torch.stack([(torch.bincount(i, minlength=classes) == 0).nonzero()[0] for i in index]), -math.inf)
    if outside.startswith("masked"):
        keep = logits.gather(1, index)
        some = slice(None) if outside == "masked" else slice(0, None, 2)
        logits[some] = -math.inf
        logits.scatter_(1, index, keep)
    lse = torch.logsumexp(teacher / 1.5, 1) + 0.4
    w = (torch.arange(rows, device='cuda') % max(1, rows // 40) == 0).float()
    _, grad = _check_distill(logits, teacher, index, 1.5, 0.7, w, lse)
    allowed = 2 * (2.0 ** -17 + torch.finfo(dtype).eps / 2) * 0.7 * 1.5 / float(w.sum()) + classes * tiny(dtype)
    assert (grad.double().sum(1).abs() <= allowed).all()


# ------------------------------------------------------------------------------------------------ products
@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_gradients_pass_through_values_quantised_beforehand(dtype, fmt):
    """`mx_quantize` and then the product: the input's gradient is that of the product given floats, to the bit; a second use adds up;
    rows seen through a stride are reached as well."""
    from gan_amd import ops
    g = gen(61)
    w = ops.mx_pack(normal(g, 100, 40))
    x = normal(g, 30, 100).to(dtype).requires_grad_(True)
    dy = normal(g, 30, 40).to(dtype)
    want, = torch.autograd.grad((ops.mx_matmul(x, w, fmt=fmt),), (x,), (dy,))
    q = ops.mx_quantize(x, fmt)
    y = ops.mx_matmul(q, w)
    got, = torch.autograd.grad((y,), (x,), (dy,))
    assert torch.equal(got, want)
    # (two equal gradients add up without a rounding)
    twice, = torch.autograd.grad([ops.mx_matmul(q, w), ops.mx_matmul(q, w)], (x,), (dy, dy))
    assert torch.equal(twice, 2 * want)
    wide = normal(g, 30, 130).to(dtype)
    wide[:, 7:107] = x.detach()
    wide.requires_grad_(True)
    got, = torch.autograd.grad((ops.mx_matmul(ops.mx_quantize(wide[:, 7:107], fmt), w),), (wide,), (dy,))
    assert torch.equal(got[:, 7:107], want) and (got[:, :7] == 0).all() and (got[:, 107:] == 0).all()
    with torch.no_grad():
        assert ops.mx_quantize(x, fmt).ticket is None
    assert ops.mx_quantize(x.detach(), fmt).ticket is None

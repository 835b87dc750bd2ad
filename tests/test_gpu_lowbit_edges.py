"""Distillation, norm and microscaled products at the edges of what they document (GPU), against the float64 forms of lowbit_ref.py.

Tolerances are those derived at the head of test_gpu_lowbit.py unless a test derives its own.
"""
import math

import pytest
import torch

import lowbit_ref as R
from test_gpu_lowbit import TYPES, _check_distill, _lists, gen, ids, normal

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

"""Norm with residual and 8-bit output, microscaled products and distillation on the GPU against their float64 forms (lowbit_ref.py).

Tolerances count roundings.  u(T) = finfo(T).eps / 2 is the half step of the result's type, E = 2^-24 that of fp32.
  norm      a sum of squares over a thread's <= 64 values and a tree of <= 26: relative error <= 90 E, half of it in its root, then
            division, root and two products: y within (u + 50 E) |y|.  Gradient: two such sums over terms |g n|, each of <= 4 roundings:
            dx within u |dx| + 200 E s (|g| + |n| mean |g n|); dgamma: rows * E over the sum of |dy n|.
  product   exact products, fp32 sums: (K + 8) E sum |a w| + u |y|; the scaled pipe (16-bit results of more than 64 rows, e4m3)
            drops what lies far below the largest product of 64: 2^-13 of sum |a w| besides, a quarter of a 16-bit half step or less.
  gradient  as a product, over the parts of dY (their sum is exact): (parts * terms + 8) E sum |.| + u |.|
  distill   probabilities of relative error <= 2 (|z - max| + |log sum| + 32) E <= 2^-17 for the |z| <= 40 used here.
"""
import math

import pytest
import torch

import lowbit_ref as R

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHORT = {torch.float32: 'f32', torch.bfloat16: 'bf16', torch.float16: 'f16'}
ids = lambda v: SHORT.get(v, None) if isinstance(v, torch.dtype) else None


def half_step(t):
    return torch.finfo(t).eps / 2


def gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device='cuda')


def within(got, ref, tol, what=""):
    got, ref = got.detach().double(), ref.double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    both_nan = torch.isnan(got) & torch.isnan(ref)
    bad = ~((got - ref).abs() <= tol) & ~both_nan & ~((got == ref) & torch.isinf(ref))
    if bool(bad.any()):
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError("%s: %d of %d values off, first at %s: got %r, wanted %r, allowed %r"
                             % (what, int(bad.sum()), bad.numel(), i, float(got[i]), float(ref[i]),
                                float((tol + torch.zeros_like(ref))[i])))


def tiny(t):
    """Smallest step of a type (its subnormals)."""
    return {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}[t]


class layer(object):
    """A store whose variables are being trained."""

    def __init__(self, **variables):
        from gan_amd import variables as V
        self.store = V.VariableStore(device='cuda')
        for name, value in variables.items():
            full = name.replace('__', '/')
            scope, leaf = full.rsplit('/', 1)
            with self.store.variable_scope(scope):
                self.store.get_variable(leaf, value.shape, V.constant_initializer(0.0)).data.copy_(value)
        self.group = self.store.pack('all', self.store.trainable_variables())

    def __enter__(self):
        from gan_amd import variables as V
        self.ctx = V.use_store(self.store)
        self.ctx.__enter__()
        self.group.begin_update()
        return self

    def __exit__(self, *exc):
        self.group.end_update()
        self.ctx.__exit__(*exc)

    def grad(self, name):
        return self.store.vars[name].grad


# ------------------------------------------------------------------------------------------------ norm
SHAPES = [(1, 1), (3, 8), (1, 31), (5, 100), (7, 257), (33, 512), (9, 1000), (2, 2048), (3, 2049), (2, 4096), (1, 8200), (2, 16384), (1, 32768)]


def _mx_equal(q, y64, what):
    """Codes and scales of an MxTensor against float64 values rounded by the definition."""
    code, byte = R.quantize(y64, q.fmt)
    got = q.codes.view(torch.uint8)
    if q.fmt == 'e2m1':
        got = torch.stack([got & 15, got >> 4], -1).flatten(-2)
    got = got.long().unflatten(-1, (-1, 32))
    assert torch.equal(q.scales.view(torch.uint8).long(), byte), what + " scales"
    alive = (byte != 255)[..., None].expand_as(code)
    assert torch.equal(got[alive], code[alive]), what + " codes"


@pytest.mark.parametrize("rows,c", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_forward(rows, c, dtype, residual):
    from gan_amd import ops
    g = gen(rows * 7919 + c)
    x = normal(g, rows, c).to(dtype)
    r = (2 * normal(g, rows, c)).to(dtype) if residual else None
    gamma = 1 + 0.1 * normal(g, c)
    with layer(rms_norm__gamma=gamma) as l, torch.no_grad():
        h = x if r is None else (x.float() + r.float()).to(dtype)
        want = R.rms(h, gamma, 1e-6)
        out = ops.rms_norm(x, residual=r)
        y = out if r is None else out[0]
        assert y.dtype == dtype
        within(y, want, (half_step(dtype) + 50 * E) * want.abs() + tiny(dtype), "y")
        if r is not None:
            assert torch.equal(out[1], h)
        out = ops.rms_norm(x, residual=r, mx=True)
        q = out if r is None else out[0]
        if r is not None:
            assert torch.equal(out[1], h)
        assert tuple(q.shape) == (rows, c) and q.dtype == dtype
        # y is rounded once from 64 bits to fp32 on the way
        _mx_equal(q, want.float(), "norm")
    assert l.grad('rms_norm/gamma').abs().max() == 0     # (no gradient reached it)


@pytest.mark.parametrize("rows,c", SHAPES + [(1500, 64), (3000, 33)])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("residual", [False, True])
def test_norm_gradients(rows, c, dtype, residual):
    from gan_amd import ops
    g = gen(rows * 31 + c)
    x = normal(g, rows, c).to(dtype).requires_grad_(True)
    r = (2 * normal(g, rows, c)).to(dtype).requires_grad_(True) if residual else None
    gamma = 1 + 0.1 * normal(g, c)
    dy, dh = normal(g, rows, c).to(dtype), normal(g, rows, c).to(dtype)
    with layer(rms_norm__gamma=gamma) as l:
        if residual:
            y, h = ops.rms_norm(x, residual=r)
            dx, dr = torch.autograd.grad((y, h), (x, r), (dy, dh))
            assert torch.equal(dx, dr)
        else:
            y, h = ops.rms_norm(x), x
            dx, = torch.autograd.grad((y,), (x,), (dy,))
    wdx, wdg = R.rms_grads(h, gamma, 1e-6, dy, dh if residual else None)
    h, gamma, dy = h.detach().double(), gamma.double(), dy.double()
    s = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)
    gr, n = (dy * gamma).abs(), (h * s).abs()
    size = s * (gr + n * (gr * n).mean(1, keepdim=True)) + (dh.double().abs() if residual else 0)
    within(dx, wdx, half_step(dtype) * wdx.abs() + 200 * E * size + tiny(dtype), "dx")
    # a term of dgamma carries the 50 E of n besides its own roundings
    within(l.grad('rms_norm/gamma'), wdg, (rows + 64) * E * (dy.abs() * n).sum(0) + 1e-30, "dgamma")


def test_norm_of_strided_shared_and_leading_dimensions():
    from gan_amd import ops
    g = gen(5)
    wide = normal(g, 6, 400).bfloat16()
    gamma = 1 + 0.1 * normal(g, 130)
    with layer(rms_norm__gamma=gamma) as l:
        for x in (wide[:, 3:133], wide[:, 200:330], wide[::2, 8:138], wide.t()[:130].t(), wide[0, :390].view(3, 1, 130)):
            r = x.flip(0).contiguous()
            want = R.rms(x.float().add(r.float()).bfloat16(), gamma, 1e-6)
            with torch.no_grad():
                y, h = ops.rms_norm(x, residual=r)
                within(y, want, (half_step(torch.bfloat16) + 50 * E) * want.abs(), "y")
                _mx_equal(ops.rms_norm(x, mx=True), R.rms(x, gamma, 1e-6).float(), "strided")
        # one variable used twice in an update: its gradients add up; a strided input and a gradient through h alone
        x = wide[:, 3:133].detach().requires_grad_(True)
        dy = normal(g, 6, 130).bfloat16()
        l.group.begin_update()
        y1, y2 = ops.rms_norm(x), ops.rms_norm(x)
        dx, = torch.autograd.grad((y1, y2), (x,), (dy, dy))
        _, wdg = R.rms_grads(x.detach(), gamma, 1e-6, dy)
        n = R.rms(x.detach(), torch.ones_like(gamma), 1e-6).abs()
        within(l.grad('rms_norm/gamma'), 2 * wdg, 80 * E * 2 * (dy.double().abs() * n).sum(0), "twice")
        l.group.begin_update()
        y, h = ops.rms_norm(x, residual=x.detach())
        dx, = torch.autograd.grad((h,), (x,), (dy,))
        assert torch.equal(dx, dy)
    assert l.grad('rms_norm/gamma').abs().max() == 0


def test_norm_rows_do_not_see_each_other():
    from gan_amd import ops
    g = gen(6)
    x = normal(g, 6, 300)
    clean = x.clone()
    x[1, 5], x[2, 7], x[3] = math.nan, math.inf, 0.0
    gamma = 1 + 0.1 * normal(g, 300)
    with layer(rms_norm__gamma=gamma), torch.no_grad():
        y, want = ops.rms_norm(x), R.rms(clean, gamma, 1e-6)
        good = [0, 4, 5]
        within(y[good], want[good], 51 * E * want[good].abs(), "clean rows")
        assert torch.isnan(y[1]).all() and torch.isnan(y[2, 7]) and (y[3] == 0).all()
        q = ops.rms_norm(x, mx=True)
        s = q.scales.view(torch.uint8)
        assert (s[1, :10] == 255).all() and s[2, 0] == 255 and (s[2, 1:10] == 1).all() and (s[3] == 1).all()
        v = ops.mx_dequantize(q)
        assert torch.isnan(v[1]).all() and torch.isnan(v[2, :32]).all() and (v[2, 32:] == 0).all() and (v[3] == 0).all()
        assert torch.equal(v[good], ops.mx_dequantize(ops.rms_norm(clean, mx=True))[good])
        assert tuple(ops.rms_norm(x[:0]).shape) == (0, 300) and tuple(ops.rms_norm(x[:0], mx=True).shape) == (0, 300)


# ------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 31), (5, 32), (4, 33), (7, 130), (2, 1024), (300, 257)])
def test_quantised_rows_are_the_definition(rows, c, dtype, fmt):
    from gan_amd import ops
    g = gen(rows + c)
    spread = torch.exp2(torch.randint(-20, 14, (rows, c), generator=g, device='cuda').float())
    x = (normal(g, rows, c) * spread).clamp(-60000, 60000).to(dtype)
    q = ops.mx_quantize(x, fmt)
    _mx_equal(q, x, fmt)
    within(ops.mx_dequantize(q, torch.float32), R.rounded(x, fmt), 0.0, "dequantised")
    if dtype != torch.float16:      # (fp16 has no room for every scale)
        within(ops.mx_dequantize(q), R.rounded(x, fmt), tiny(dtype), "dequantised in its type")


@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
def test_quantisation_at_its_borders(fmt):
    """Ties, the largest element, powers of two, zeros, subnormals, infinities and NaN."""
    from gan_amd import ops
    grid = torch.tensor(R.GRID[fmt], dtype=torch.float64)
    middle = (grid[1:] + grid[:-1]) / 2
    pool = torch.cat([grid, middle, middle * (1 + 2.0 ** -20), middle * (1 - 2.0 ** -20), -grid, -middle])
    rows = []
    for e in (-140, -126, -60, 0, 3, 60, 118):
        block = pool[torch.arange(64 * 6) % pool.numel()].clone().view(-1, 32)
        block[:, 0] = grid[-1]
        rows.append((block * 2.0 ** e).flatten())
        block[:, 0] = grid[-1] * (1 + 2.0 ** -22)          # just too large for its scale
        rows.append((block * 2.0 ** e).flatten())
    x = torch.stack(rows).float().cuda()
    x[0, 32:64] = 0
    x[1, 64:96] = 1e-45
    x[2, 0], x[2, 33], x[2, 70] = math.inf, math.nan, -math.inf
    _mx_equal(ops.mx_quantize(x, fmt), x, fmt)
    q = ops.mx_quantize(x, fmt)
    v = ops.mx_dequantize(q)
    assert torch.isnan(v[2, :96]).all() and not torch.isnan(v[2, 96:]).any()
    assert tuple(ops.mx_quantize(x[:0], fmt).shape) == (0, x.shape[1])


@pytest.mark.parametrize("k,n", [(1, 1), (32, 5), (33, 64), (100, 65), (128, 130), (300, 70), (1000, 257)])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_packed_weights_are_the_definition(k, n, dtype):
    from gan_amd import ops
    g = gen(k * 3 + n)
    m = normal(g, k, n + 3).to(dtype)[:, 1:n + 1]           # rows of a wider matrix
    w = ops.mx_pack(m)
    code, byte = R.quantize(m.t(), 'e2m1')                  # [n, blocks, 32]
    got = torch.stack([w.codes & 15, w.codes >> 4], -1).flatten(-2).long()
    assert torch.equal(got.transpose(0, 1), code)
    assert torch.equal(w.scales.transpose(0, 1).reshape(n, -1).long(), byte)
    within(ops.mx_dequantize(w), R.rounded(m.t(), 'e2m1').t(), 0.0, "unpacked")


# ------------------------------------------------------------------------------------------------ product
def _product(rows, k, n, dtype, fmt, bias=True, seed=0):
    from gan_amd import ops
    g = gen(seed + rows * 13 + k * 7 + n)
    x = normal(g, rows, k).to(dtype)
    m = normal(g, k, n) / math.sqrt(k)
    b = normal(g, n) if bias else None
    w = ops.mx_pack(m)
    y = ops.mx_matmul(x, w, b, fmt=fmt)
    a, wv = R.rounded(x, fmt), R.rounded(m.t(), 'e2m1').t()
    want = torch.mm(a, wv) + (0 if b is None else b.double())
    size = torch.mm(a.abs(), wv.abs()) + (0 if b is None else b.double().abs())
    pipe = 2.0 ** -13 if fmt == 'e4m3' and dtype != torch.float32 else 0.0
    assert y.dtype == dtype
    within(y, want, half_step(dtype) * want.abs() + ((k + 8) * E + pipe) * size + tiny(dtype), "%s %s" % ((rows, k, n), fmt))
    # the quantised input gives the same bits
    assert torch.equal(ops.mx_matmul(ops.mx_quantize(x, fmt), w, b), y)
    return y


@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows", [1, 5, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("k,n", [(1, 1), (33, 5), (128, 16), (200, 100), (1000, 257), (2400, 256)])
def test_product(rows, k, n, dtype, fmt):
    _product(rows, k, n, dtype, fmt, bias=(rows + n) % 3 != 0)


@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,k,n", [(1, 8192, 64), (20, 5000, 20), (3300, 300, 4100), (100, 4000, 130), (4096, 130, 4096)])
def test_product_split_and_large(rows, k, n, dtype, fmt):
    _product(rows, k, n, dtype, fmt, seed=1)


@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("rows", [3, 100])
def test_product_keeps_bad_blocks_and_far_scales_apart(rows, fmt):
    """A block with a NaN spoils its row or its output alone; scales from 2^-60 to 2^60 in one product; leading dimensions."""
    from gan_amd import ops
    g = gen(9)
    x, m = normal(g, rows, 300), normal(g, 300, 70)
    clean = ops.mx_matmul(x, ops.mx_pack(m), fmt=fmt)
    x2, m2 = x.clone(), m.clone()
    x2[1, 40], m2[130, 7] = math.inf, math.nan
    for dtype in TYPES:
        base = ops.mx_matmul(x.to(dtype), ops.mx_pack(m), fmt=fmt)
        y = ops.mx_matmul(x2.to(dtype), ops.mx_pack(m2), fmt=fmt)
        keep = torch.ones(rows, 70, dtype=torch.bool, device='cuda')
        keep[1], keep[:, 7] = False, False
        assert torch.equal(y[keep], base[keep]) and torch.isnan(y[~keep]).all(), dtype
    up = torch.exp2(torch.randint(-60, 61, (rows, 1), generator=g, device='cuda').float())
    far = ops.mx_matmul(x * up, ops.mx_pack(m * 2.0 ** -40), fmt=fmt)
    assert torch.equal(far, clean * up * 2.0 ** -40)
    flat = ops.mx_matmul(x[:2].view(2, 1, 300), ops.mx_pack(m), fmt=fmt)
    assert tuple(flat.shape) == (2, 1, 70) and torch.equal(flat[:, 0], ops.mx_matmul(x[:2], ops.mx_pack(m), fmt=fmt))
    assert tuple(ops.mx_matmul(x[:0], ops.mx_pack(m), fmt=fmt).shape) == (0, 70)


@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,k,n", [(1, 1, 1), (5, 33, 17), (16, 128, 64), (64, 100, 130), (130, 257, 65), (300, 1000, 200), (700, 64, 2500)])
def test_layer_gradients(rows, k, n, dtype, fmt):
    from gan_amd import ops
    g = gen(rows + k + n)
    x = normal(g, rows, k).to(dtype).requires_grad_(True)
    m, b = normal(g, k, n) / math.sqrt(k), normal(g, n)
    dy = normal(g, rows, n).to(dtype)
    parts = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}[dtype]
    a, wv, d = R.rounded(x.detach(), fmt), R.rounded(m.t(), 'e2m1').t(), dy.double()
    with layer(Linear__Matrix=m, Linear__bias=b) as l:
        y = ops.linear_mx(x, n, fmt=fmt)
        assert torch.equal(y, ops.mx_matmul(x.detach(), ops.mx_pack(m), b, fmt=fmt))
        dx, = torch.autograd.grad((y,), (x,), (dy,))
        want, size = torch.mm(d, wv.t()), torch.mm(d.abs(), wv.abs().t())
        within(dx, want, half_step(dtype) * want.abs() + (parts * n + 8) * E * size + tiny(dtype), "dx")
        want, size = torch.mm(a.t(), d), torch.mm(a.abs().t(), d.abs())
        within(l.grad('Linear/Matrix'), want, (parts * rows + 8) * E * size, "dmatrix")
        within(l.grad('Linear/bias'), d.sum(0), (rows + 8) * E * d.abs().sum(0), "dbias")
        first = l.grad('Linear/Matrix').clone(), l.grad('Linear/bias').clone()
        # a second use adds up, from the input as an MxTensor without a gradient of its own
        y = ops.linear_mx(ops.mx_quantize(x.detach(), fmt), n)
        torch.autograd.backward((y,), (dy,))
        within(l.grad('Linear/Matrix'), 2 * want, 2 * (parts * rows + 9) * E * size, "dmatrix twice")
    # frozen weights: the input's gradient alone
    y = ops.mx_matmul(x, ops.mx_pack(m), b, fmt=fmt)
    again, = torch.autograd.grad((y,), (x,), (dy,))
    assert torch.equal(again, dx)
    with layer(Linear__Matrix=m, Linear__bias=b) as l:      # the same bits every time
        torch.autograd.backward((ops.linear_mx(x.detach(), n, fmt=fmt),), (dy,))
        assert torch.equal(l.grad('Linear/Matrix'), first[0]) and torch.equal(l.grad('Linear/bias'), first[1])


def test_large_layer_gradients():
    """The 256-wide tiles of the gradient products."""
    from gan_amd import ops
    g = gen(4)
    rows, k, n = 4096, 4000, 3400
    x = normal(g, rows, k).bfloat16().requires_grad_(True)
    m, b, dy = normal(g, k, n) / math.sqrt(k), normal(g, n), normal(g, rows, n).bfloat16()
    a, wv, d = R.rounded(x.detach(), 'e4m3'), R.rounded(m.t(), 'e2m1').t(), dy.double()
    with layer(Linear__Matrix=m, Linear__bias=b) as l:
        dx, = torch.autograd.grad((ops.linear_mx(x, n),), (x,), (dy,))
    want = torch.mm(d, wv.t())
    within(dx, want, half_step(torch.bfloat16) * want.abs() + (n + 8) * E * torch.mm(d.abs(), wv.abs().t()), "dx")
    within(l.grad('Linear/Matrix'), torch.mm(a.t(), d), (rows + 8) * E * torch.mm(a.abs().t(), d.abs()), "dmatrix")


def test_gradient_parts_carry_infinities_and_large_values():
    from gan_amd import ops
    g = gen(8)
    m = normal(g, 40, 70)
    x = normal(g, 5, 40).requires_grad_(True)
    dy = normal(g, 5, 70)
    dy[1] *= 1e37
    dy[2, 3], dy[3, 4] = math.inf, math.nan
    dx, = torch.autograd.grad((ops.mx_matmul(x, ops.mx_pack(m)),), (x,), (dy,))
    wv = R.rounded(m.t(), 'e2m1').t()
    for r in (0, 1, 4):
        d = dy[r:r + 1].double()
        within(dx[r:r + 1], torch.mm(d, wv.t()), 220 * E * torch.mm(d.abs(), wv.abs().t()), "row %d" % r)
    hit = wv[:, 3] != 0
    assert torch.equal(dx[2][hit], torch.where(wv[:, 3] > 0, math.inf, -math.inf).float()[hit]) and torch.isnan(dx[3]).all()


# ------------------------------------------------------------------------------------------------ distillation
def _lists(g, rows, classes, top, dtype):
    index = torch.stack([torch.randperm(classes, generator=g, device='cuda')[:top] for _ in range(rows)])
    return index, (2 * normal(g, rows, top)).to(dtype)


def _check_distill(logits, teacher, index, tau, weight=1.0, row_weight=None, lse=None):
    from gan_amd import ops
    x = logits.detach().requires_grad_(True)
    loss = ops.distill_topk_mean(x, teacher, index, temperature=tau, weight=weight, row_weight=row_weight, teacher_lse=lse)
    ops.backward(loss)
    cpu = lambda t: None if t is None else t.cpu()
    want, grad, size = R.distill(logits.cpu(), teacher.cpu(), index.cpu(), tau, weight, cpu(row_weight), cpu(lse))
    t = logits.dtype
    within(x.grad.cpu(), grad, half_step(t) * grad.abs() + 2.0 ** -17 * size + tiny(t), "dlogits")
    # l is a sum of terms p (log p - log q), each off by the 2^-17 of its p.  Their sizes add up to <= 60 for logits of <= 40; where
    # a listed class has a logit of the type's lowest value the terms of larger size are positive (p log p >= -1 / e, -log q > 0),
    # so together they are no larger than the loss and the other terms: 2^-17 (60 + |loss|)
    assert abs(float(loss.detach()) - want) <= 2.0 ** -17 * (60 * abs(weight) * tau * tau + abs(want)), (float(loss), want)
    return loss.detach(), x.grad


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("rows,classes,top", [(1, 1, 1), (2, 10, 3), (5, 100, 100), (3, 2047, 16), (4, 2500, 64), (3, 4099, 65), (2, 9001, 128),
                                              (2, 20000, 7), (2, 50257, 50), (1, 131072, 64), (1, 140001, 33)])
def test_distillation(rows, classes, top, dtype, rest):
    g = gen(rows + classes + top)
    logits = (2 * normal(g, rows, classes)).to(dtype)
    index, teacher = _lists(g, rows, classes, top, dtype)
    lse = torch.logsumexp(teacher.float() / 1.5, 1) + 0.2 if rest else None
    _check_distill(logits, teacher, index.int() if rows % 2 else index, 1.5, 0.7, None, lse)


@pytest.mark.parametrize("rest", [False, True])
def test_distillation_rows_lists_and_weights(rest):
    """Short, empty and repeated lists, weights of zero over rows of NaN, masked classes, teachers of -inf, other types."""
    g = gen(3)
    rows, classes, top = 9, 1000, 8
    logits = 3 * normal(g, rows, classes)
    index, teacher = _lists(g, rows, classes, top, torch.float32)
    index[1, 3:] = -1
    index[2] = -1
    index[3, 1] = classes
    index[4, 5] = index[4, 2]
    index[4, 6] = index[4, 2]
    index[5] = index[5, 0]
    teacher[6, 2] = -math.inf
    teacher[8] = -math.inf
    logits[7] = math.nan
    logits[0, 500:] = torch.finfo(torch.float32).min
    logits[1, 10:400] = -math.inf
    logits[1, index[1, :3]] = 1.0
    w = torch.tensor([1, 2, 1, 0.5, 1, 1, 0.25, 0, 1.0], device='cuda')
    lse = torch.logsumexp(teacher, 1) + 0.4 if rest else None
    if rest:
        lse[2] = lse[8] = 0.0
    _, grad = _check_distill(logits, teacher, index, 1.0, 1.0, w, lse)
    for r in (2, 7, 8):
        assert (grad[r] == 0).all()
    for t in (torch.bfloat16, torch.float16):
        tt = teacher.to(t)
        _check_distill(logits, tt, index.int(), 2.0, 0.3, w, None if lse is None else torch.logsumexp(tt.float() / 2, 1).clamp(min=-50) + 0.4)
    loss, grad = _check_distill(logits[:3], teacher[:3], index[:3], 1.0, 1.0, torch.zeros(3, device='cuda'), None)
    assert float(loss) == 0 and (grad == 0).all()
    loss, grad = _check_distill(logits[:2], teacher[:2], index[:2], 1.0, 1.0, torch.tensor([1.0, -1.0], device='cuda'), None)
    assert float(loss) == 0 and (grad == 0).all()


def test_distillation_of_a_certain_student():
    """The rest term where almost all of the student's mass is listed (1 - sum q would be 0), and with every class listed."""
    g = gen(11)
    logits = normal(g, 3, 600)
    index, teacher = _lists(g, 3, 600, 4, torch.float32)
    logits.scatter_(1, index, 30.0)
    lse = torch.logsumexp(teacher, 1) + 0.3
    _check_distill(logits, teacher, index, 1.0, 1.0, None, lse)
    index, teacher = _lists(g, 2, 20, 20, torch.float32)
    _check_distill(normal(g, 2, 20), teacher, index, 1.0, 1.0, None, torch.logsumexp(teacher, 1) + 0.3)


def test_distillation_strides_many_rows_and_large_lists():
    from gan_amd import ops
    g = gen(12)
    wide = 2 * normal(g, 6, 3100)
    for dtype, lo in ((torch.float32, 1), (torch.bfloat16, 3), (torch.bfloat16, 8)):
        index, teacher = _lists(g, 6, 2500, 9, torch.float32)
        _check_distill(wide.to(dtype)[:, lo:lo + 2500], teacher, index, 1.0, 1.0, None, torch.logsumexp(teacher, 1) + 0.1)
    index, teacher = _lists(g, 2, 5000, 1024, torch.float32)
    index[1, 700] = index[1, 3]
    _check_distill(normal(g, 2, 5000), teacher, index, 1.0, 1.0, None, torch.logsumexp(teacher, 1) + 0.1)
    # leading dimensions, and more rows than a workgroup adds the weights of by itself
    rows = 5000
    logits = normal(g, 50, 100, 12).requires_grad_(True)
    index, teacher = torch.randint(0, 12, (50, 100, 2), generator=g, device='cuda'), normal(g, 50, 100, 2)
    w = torch.rand(50, 100, generator=g, device='cuda')
    loss = ops.distill_topk_mean(logits, teacher, index, row_weight=w)
    ops.backward(loss)
    want, grad, size = R.distill(logits.detach().view(rows, 12).cpu(), teacher.view(rows, 2).cpu(), index.view(rows, 2).cpu(), 1.0, 1.0,
                                 w.view(-1).cpu())
    within(logits.grad.view(rows, 12).cpu(), grad, 2.0 ** -17 * size, "dlogits")
    assert abs(float(loss) - want) <= 2.0 ** -17 * 20


# ------------------------------------------------------------------------------------------------ together
def _student(g, rows=96, width=200, classes=700):
    x, r = normal(g, rows, width), 2 * normal(g, rows, width)
    gamma, m, b = 1 + 0.1 * normal(g, width), normal(g, width, classes) / 8, normal(g, classes)
    index, teacher = _lists(g, rows, classes, 6, torch.float32)
    lse = torch.logsumexp(teacher, 1) + 0.2
    l = layer(rms_norm__gamma=gamma, head__Matrix=m, head__bias=b)
    return l, x, r, (gamma, m, b), (index, teacher, lse)


def _student_step(l, x, r, index, teacher, lse):
    from gan_amd import ops
    with l:
        xx = x.detach().requires_grad_(True)
        q, h = ops.rms_norm(xx, residual=r, mx=True)
        loss = ops.distill_topk_mean(ops.linear_mx(q, teacher_classes(l), 'head'), teacher, index, teacher_lse=lse)
        dx, = torch.autograd.grad(loss, xx)
    return loss.detach(), h.detach(), dx


def teacher_classes(l):
    return l.store.vars['head/Matrix'].shape[1]


def test_student_step_end_to_end():
    g = gen(21)
    l, x, r, (gamma, m, b), (index, teacher, lse) = _student(g)
    loss, h, dx = _student_step(l, x, r, index, teacher, lse)
    assert torch.equal(h, x + r)
    a, wv = R.rounded(R.rms(h, gamma, 1e-6).float(), 'e4m3'), R.rounded(m.t(), 'e2m1').t()
    logits = torch.mm(a, wv) + b.double()
    want, dl, size = R.distill(logits.cpu(), teacher.cpu(), index.cpu(), lse=lse.cpu())
    dl, size = dl.cuda(), size.cuda()
    # an error d in the logits changes q by at most 2 q d: with d <= (K + 8) E sum |a w| < 2^-14 that is 2^-13 of `size`
    off = 2.0 ** -13 * size
    assert abs(float(loss) - want) <= 2.0 ** -13 * 20
    within(l.grad('head/Matrix'), torch.mm(a.t(), dl), torch.mm(a.abs().t(), off), "dmatrix")
    within(l.grad('head/bias'), dl.sum(0), off.sum(0), "dbias")
    da, da_off = torch.mm(dl, wv.t()), torch.mm(off, wv.abs().t())
    wdx, wdg = R.rms_grads(h, gamma, 1e-6, da)
    s = 1 / torch.sqrt((h.double() ** 2).mean(1, keepdim=True) + 1e-6)
    n, go = (h * s).abs(), da_off * gamma.abs()
    within(dx, wdx, 2 * s * (go + n * (go * n).mean(1, keepdim=True)), "dx")
    within(l.grad('rms_norm/gamma'), wdg, 2 * (da_off * n).sum(0), "dgamma")


def test_student_step_captured_and_replayed():
    """Three replays on new inputs, with eager steps of the same layers between them, against eager results."""
    g = gen(22)
    l, x, r, _, (index, teacher, lse) = _student(g)
    names = ('rms_norm/gamma', 'head/Matrix', 'head/bias')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _student_step(l, x, r, index, teacher, lse)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _student_step(l, x, r, index, teacher, lse)
        grads = [l.grad(n).clone() for n in names]
    for k in range(3):
        x.copy_(normal(g, *x.shape))
        teacher.copy_(normal(g, *teacher.shape))
        lse.copy_(torch.logsumexp(teacher, 1) + 0.2)
        graph.replay()
        got = [t.clone() for t in out] + [t.clone() for t in grads]
        torch.cuda.synchronize()
        want = list(_student_step(l, x, r, index, teacher, lse)) + [l.grad(n) for n in names]
        for a, b in zip(got, want):
            assert torch.equal(a, b), k


def test_two_streams_do_not_share_scratch():
    """Split products, gradients and losses of two streams at once give what they give alone."""
    from gan_amd import ops
    g = gen(23)
    work = []
    for _ in range(2):
        x, m, dy = normal(g, 40, 4000).requires_grad_(True), normal(g, 4000, 48) / 60, normal(g, 40, 48)
        work.append((x, ops.mx_pack(m), dy))

    def once(x, w, dy):
        y = ops.mx_matmul(x, w)
        return y.detach(), torch.autograd.grad((y,), (x,), (dy,))[0]
    alone = [once(*v) for v in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        got = []
        for s, v in zip(streams, work):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(once(*v))
        torch.cuda.synchronize()
        for a, b in zip(got, alone):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_gpu_calls_that_are_refused():
    from gan_amd import ops
    from gan_amd._lib import GanHipError
    w = ops.mx_pack(torch.randn(64, 8, device='cuda'))
    with pytest.raises(GanHipError):
        ops.mx_matmul(torch.zeros(3, 64), w)                # a tensor of another device
    with pytest.raises(GanHipError):
        ops.mx_matmul(torch.zeros(3, 64, device='cuda'), w, bias=torch.zeros(8))
    with pytest.raises(GanHipError):
        ops.distill_topk_mean(torch.zeros(3, 64, device='cuda'), torch.zeros(3, 2), torch.zeros(3, 2, dtype=torch.int64, device='cuda'))
    with layer(rms_norm__gamma=torch.ones(40000)):
        with pytest.raises(GanHipError):
            ops.rms_norm(torch.zeros(1, 40000, device='cuda'))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_distillation_with_everything_outside_the_list_masked(dtype):
    """All other classes at the type's lowest value: their share of the remaining mass is still theirs."""
    g = gen(31)
    logits = normal(g, 2, 300).to(dtype)
    index, teacher = _lists(g, 2, 300, 5, torch.float32)
    keep = logits.gather(1, index)
    logits.fill_(torch.finfo(dtype).min)
    logits.scatter_(1, index, keep)
    _check_distill(logits, teacher, index, 2.0, 1.0, None, torch.logsumexp(teacher / 2, 1) + 0.3)


def test_empty_batches_give_empty_gradients():
    from gan_amd import ops
    x = torch.zeros(0, 64, device='cuda', requires_grad=True)
    with layer(rms_norm__gamma=torch.ones(64), Linear__Matrix=torch.ones(64, 8), Linear__bias=torch.ones(8)) as l:
        y = ops.linear_mx(ops.rms_norm(x), 8)
        assert tuple(y.shape) == (0, 8)
        dx, = torch.autograd.grad((y,), (x,), (torch.zeros(0, 8, device='cuda'),))
        assert tuple(dx.shape) == (0, 64)
    assert all(float(l.grad(n).abs().max()) == 0 for n in ('rms_norm/gamma', 'Linear/Matrix', 'Linear/bias'))
    dx, = torch.autograd.grad((ops.mx_matmul(x, ops.mx_pack(torch.ones(64, 8, device='cuda'))),), (x,), (torch.zeros(0, 8, device='cuda'),))
    assert tuple(dx.shape) == (0, 64)


@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,k,n", [(16, 700, 9000), (24, 1024, 16384), (40, 8200, 600), (128, 300, 1000), (70, 8192, 128), (200, 4224, 2100)])
def test_product_at_the_choices_of_kernel(rows, k, n, dtype, fmt):
    _product(rows, k, n, dtype, fmt, seed=5)


def test_distillation_of_the_largest_vocabulary_and_list():
    g = gen(41)
    classes, top = 1 << 20, 1024
    logits = normal(g, 1, classes)
    index, teacher = _lists(g, 1, classes, top, torch.float32)
    for t in (torch.float32, torch.bfloat16):
        _check_distill(logits.to(t), teacher, index, 1.0, 1.0, None, torch.logsumexp(teacher, 1) + 0.2)


def test_a_loss_backward_twice_and_gradients_of_shared_logits():
    """A retained loss gives its gradient again; two losses on the same logits add theirs."""
    from gan_amd import ops
    g = gen(42)
    x = normal(g, 5, 300).requires_grad_(True)
    index, teacher = _lists(g, 5, 300, 4, torch.float32)
    loss = ops.distill_topk_mean(x, teacher, index)
    first, = torch.autograd.grad(loss, x, retain_graph=True)
    first = first.clone()
    again, = torch.autograd.grad(loss, x)
    assert torch.equal(first, again)
    ops.backward([ops.distill_topk_mean(x, teacher, index), ops.distill_topk_mean(x, teacher, index, weight=0.5)])
    within(x.grad, 1.5 * first.double(), 2.0 ** -23 * 1.5 * first.double().abs() + 1e-12, "sum")


@pytest.mark.parametrize("dtype,size", [(torch.float32, 1e30), (torch.float32, 1e-25), (torch.bfloat16, 1e38), (torch.bfloat16, 1e-30)])
def test_norm_of_values_whose_squares_leave_fp32(dtype, size):
    from gan_amd import ops
    g = gen(51)
    x = (normal(g, 3, 700).clamp(-3, 3) * size).to(dtype)
    gamma = 1 + 0.1 * normal(g, 700)
    with layer(rms_norm__gamma=gamma), torch.no_grad():
        want = R.rms(x, gamma, 0.0)
        # (1 / 1e38 is subnormal in fp32: 2^-23 relative, two E, on top)
        within(ops.rms_norm(x, epsilon=0.0), want, (half_step(dtype) + 52 * E) * want.abs(), "y")
        _mx_equal(ops.rms_norm(x, epsilon=0.0, mx=True), want.float(), "codes")


def test_norm_of_more_rows_than_one_axis_of_a_grid_holds():
    """70 million rows of one value each: y = gamma x / sqrt(x^2 + eps)."""
    from gan_amd import ops
    g = gen(52)
    x = normal(g, 70000000, 1).bfloat16()
    with layer(rms_norm__gamma=torch.full((1,), 1.5)), torch.no_grad():
        y = ops.rms_norm(x)
    for part in (slice(0, 1000), slice(34000000, 34001000), slice(-1000, None)):
        want = R.rms(x[part], torch.full((1,), 1.5, device='cuda'), 1e-6)
        within(y[part], want, (half_step(torch.bfloat16) + 50 * E) * want.abs(), "rows")
    assert bool((y.sign() == x.sign()).all())


def test_distillation_from_a_teacher_whose_list_is_all_masked():
    """Logits of the type's lowest value divided by a temperature below 1 are still logits: p is uniform over them."""
    g = gen(53)
    logits = normal(g, 3, 200)
    index, teacher = _lists(g, 3, 200, 5, torch.float32)
    teacher[0] = torch.finfo(torch.float32).min
    teacher[1, 2:] = torch.finfo(torch.float32).min
    _check_distill(logits, teacher, index, 0.5)
    _check_distill(logits, teacher.bfloat16().clamp(min=torch.finfo(torch.bfloat16).min), index, 0.5)


def test_a_pass_is_captured_while_an_eager_one_lives():
    from gan_amd import ops
    g = gen(54)
    l, x, r, _, (index, teacher, lse) = _student(g)
    names = ('rms_norm/gamma', 'head/Matrix', 'head/bias')

    def loss():
        q, _ = ops.rms_norm(x, residual=r, mx=True)
        return ops.distill_topk_mean(ops.linear_mx(q, teacher_classes(l), 'head'), teacher, index, teacher_lse=lse)

    def step():
        with l:
            ops.backward(loss())
    with l:
        alive = loss()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
        grads = [l.grad(n).clone() for n in names]
    with l:
        ops.backward(alive)
    want = [l.grad(n).clone() for n in names]
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(grads, want):
            assert torch.equal(a, b)
        step()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,k,n", [(1, 40, 8), (63, 130, 24), (64, 100, 64), (128, 384, 72), (65, 30, 7), (192, 257, 320), (2048, 96, 512)])
def test_gradients_apart_are_those_computed_together(rows, k, n, dtype):
    """The three entry points agree to the bit: weights frozen, input without a gradient, both."""
    from gan_amd import ops
    g = gen(rows + k + n)
    x, m, dy = normal(g, rows, k).to(dtype), normal(g, k, n), normal(g, rows, n).to(dtype)
    with layer(Linear__Matrix=m, Linear__bias=torch.zeros(n, device='cuda')) as l:
        xx = x.clone().requires_grad_(True)
        dx, = torch.autograd.grad((ops.linear_mx(xx, n),), (xx,), (dy,))
        both = [l.grad(v).clone() for v in ('Linear/Matrix', 'Linear/bias')]
        l.group.begin_update()
        torch.autograd.backward((ops.linear_mx(x, n),), (dy,))
        alone = [l.grad(v).clone() for v in ('Linear/Matrix', 'Linear/bias')]
    frozen, = torch.autograd.grad((ops.mx_matmul(xx, ops.mx_pack(m)),), (xx,), (dy,))
    assert torch.equal(dx, frozen) and torch.equal(both[0], alone[0]) and torch.equal(both[1], alone[1])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,c", [(9000, 5), (5000, 64), (3001, 128), (2500, 200), (1100, 4096), (1030, 8192), (600, 20000)])
def test_norm_gradients_of_many_rows_a_team(rows, c, dtype):
    """Every width of team with several rows for each, and partial sums of several workgroups."""
    test_norm_gradients(rows, c, dtype, True)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("classes,top", [(5, 2), (130, 9), (1027, 70), (2000, 16)])
def test_distillation_of_many_short_rows(classes, top, dtype):
    """More rows than one sum of weights takes, against the loss of a few of them at a time: the mean is linear in the rows."""
    from gan_amd import ops
    g = gen(classes)
    rows = 4200
    logits = (2 * normal(g, rows, classes)).to(dtype)
    index = torch.randint(0, classes, (rows, top), generator=g, device='cuda')
    teacher, w = 2 * normal(g, rows, top), torch.rand(rows, generator=g, device='cuda')
    w[5] = 0
    lse = torch.logsumexp(teacher, 1) + 0.2
    x = logits.requires_grad_(True)
    loss = ops.distill_topk_mean(x, teacher, index, row_weight=w, teacher_lse=lse)
    ops.backward(loss)
    total = w.double().sum().cpu()
    pick = [0, 5, 2047, 4199]
    want, grad, size = R.distill(logits.detach()[pick].cpu(), teacher[pick].cpu(), index[pick].cpu(), row_weight=w[pick].cpu(), lse=lse[pick].cpu())
    share = (w[pick].double().sum().cpu() / total).item()
    # (the sum of 4200 weights: 64 E more)
    within(x.grad[pick].cpu(), grad * share, half_step(dtype) * share * grad.abs() + (2.0 ** -17 + 64 * E) * share * size + tiny(dtype), "dlogits")
    parts = [ops.distill_topk_mean(logits.detach()[a:a + 1000], teacher[a:a + 1000], index[a:a + 1000], row_weight=w[a:a + 1000],
                                   teacher_lse=lse[a:a + 1000]) for a in range(0, rows, 1000)]
    mean = sum(float(p) * float(w[a:a + 1000].double().sum() / w.double().sum()) for p, a in zip(parts, range(0, rows, 1000)))
    # (both sides have the 2^-17 of a term of size <= 60)
    assert abs(float(loss.detach()) - mean) <= 2 * 2.0 ** -17 * 60


@pytest.mark.parametrize("fmt", ['e4m3', 'e2m1'])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("rows,k,n", [(64, 1024, 1024), (31, 2048, 512), (100, 1000, 500), (200, 600, 100), (16, 2048, 70), (20, 2400, 40), (250, 128, 256)])
def test_product_of_rows_quantised_by_the_product(rows, k, n, dtype, fmt):
    _product(rows, k, n, dtype, fmt, seed=6)


def test_product_of_strided_rows_quantised_by_the_product():
    from gan_amd import ops
    g = gen(61)
    wide, w = normal(g, 70, 900).bfloat16(), ops.mx_pack(normal(g, 333, 48))
    for x in (wide[:, 5:338], wide[:, 8:341], wide[::2, :333], wide.t()[:70, :70].repeat(1, 5)[:, :333]):
        assert torch.equal(ops.mx_matmul(x, w), ops.mx_matmul(ops.mx_quantize(x.contiguous()), w))

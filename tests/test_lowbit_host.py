"""Norm, microscaled product and distillation without a GPU: the float64 forms the GPU tests compare with are themselves checked
against differences, and the calls that have to be refused are refused before any launch."""
import ctypes

import pytest
import torch

import lowbit_ref as R


def _differences(f, x, step=1e-5):
    g = torch.zeros_like(x)
    for i in range(x.numel()):
        d = torch.zeros_like(x)
        d.view(-1)[i] = step
        g.view(-1)[i] = (f(x + d) - f(x - d)) / (2 * step)
    return g


def test_norm_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    h, gamma, dy = (torch.randn(3, 7, generator=g, dtype=torch.float64) for _ in range(3))
    gamma = gamma[0]
    dx, dgamma = R.rms_grads(h, gamma, 1e-3, dy)
    assert torch.allclose(dx, _differences(lambda v: (R.rms(v, gamma, 1e-3) * dy).sum(), h), atol=1e-8)
    assert torch.allclose(dgamma, _differences(lambda v: (R.rms(h, v, 1e-3) * dy).sum(), gamma), atol=1e-8)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("twice", [False, True])
def test_distillation_gradient_against_differences(rest, twice):
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(4, 9, generator=g, dtype=torch.float64)
    teacher = torch.randn(4, 3, generator=g, dtype=torch.float64)
    index = torch.tensor([[0, 4, 8], [1, 2, -1], [3, 3 if twice else 5, 7], [-1, 9, -1]])
    lse = torch.logsumexp(teacher / 1.5, 1) + 0.3 if rest else None
    w = torch.tensor([1.0, 0.5, 2.0, 1.0])
    f = lambda v: R.distill(v, teacher, index, 1.5, 0.7, w, lse)[0]
    assert torch.allclose(R.distill(logits, teacher, index, 1.5, 0.7, w, lse)[1], _differences(f, logits), atol=1e-8)


@pytest.mark.parametrize("fmt", ["e4m3", "e2m1"])
def test_rounding_keeps_every_element_within_half_a_step(fmt):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(50, 96, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-100, 100, (50, 1), generator=g).double())
    v = R.rounded(x, fmt)
    grid = torch.tensor(R.GRID[fmt], dtype=torch.float64)
    top = x.abs().unflatten(1, (-1, 32)).amax(-1, keepdim=True).expand(50, 3, 32).flatten(1)
    # the scale is at most twice the largest element over the format's largest value
    step = (grid[1:] - grid[:-1]).max() * 2 * top / grid[-1]
    assert ((v - x).abs() <= step / 2).all()
    assert torch.equal(R.rounded(v, fmt), v)


FAKE = ctypes.c_void_p(4096)


def _refused(rc, words):
    from gan_amd import _lib as L
    assert rc != 0 and words in L.lib.gan_last_error(), L.lib.gan_last_error()


def test_library_refuses_before_any_launch():
    from gan_amd import _lib as L
    lib, p, odd = L.lib, FAKE, ctypes.c_void_p(4096 + 2)
    _refused(lib.gan_rms_norm_fwd(7, 4, 64, p, 64, None, 0, p, 1e-6, None, p, None, None, None, None), b"element type")
    _refused(lib.gan_rms_norm_fwd(0, 4, 0, p, 64, None, 0, p, 1e-6, None, p, None, None, None, None), b"0 values")
    _refused(lib.gan_rms_norm_fwd(0, 4, 32769, p, 32769, None, 0, p, 1e-6, None, p, None, None, None, None), b"32769 values")
    _refused(lib.gan_rms_norm_fwd(0, 4, 64, p, 63, None, 0, p, 1e-6, None, p, None, None, None, None), b"row stride")
    _refused(lib.gan_rms_norm_fwd(0, 4, 64, p, 64, p, 64, p, 1e-6, None, p, None, None, None, None), b"h exactly with a residual")
    _refused(lib.gan_rms_norm_fwd(0, 4, 64, p, 64, None, 0, p, 1e-6, None, p, p, p, None, None), b"one of y or mx_codes")
    _refused(lib.gan_rms_norm_bwd(0, 4, 64, p, 64, p, p, p, None, p, p, 0, None, 0, None), b"workspace")
    _refused(lib.gan_mx_quantize(0, 2, 4, 64, p, 64, p, p, None), b"format")
    _refused(lib.gan_mx_quantize(0, 0, 4, 64, p, 32, p, p, None), b"stride")
    _refused(lib.gan_mx_quantize(0, 0, 4, 64, p, 64, odd, p, None), b"aligned")
    _refused(lib.gan_mx_pack(0, 1 << 23, 4, p, 4, p, p, None), b"up to")
    _refused(lib.gan_mx_pack(0, 64, 4, p, 3, p, p, None), b"row stride")
    _refused(lib.gan_mx_matmul(1, 0, -1, 64, 64, p, p, p, p, None, p, None, 0, None), b"-1 rows")
    _refused(lib.gan_mx_matmul(1, 0, 4, 64, 64, p, p, odd, p, None, p, None, 0, None), b"aligned")
    need = lib.gan_mx_matmul_workspace_bytes(0, 0, 1000, 64, 2000)
    assert need > 0
    _refused(lib.gan_mx_matmul(0, 0, 1000, 64, 2000, p, p, p, p, None, p, p, need - 1, None), b"workspace")
    need = lib.gan_mx_linear_workspace_bytes(1, 0, 100, 8192, 64)
    assert need > 0 and lib.gan_mx_linear_workspace_bytes(1, 0, 1, 64, 64) == 0      # (one token: nothing to keep between launches)
    _refused(lib.gan_mx_linear(1, 0, 100, 8192, 64, p, 8192, p, p, None, p, p, need - 1, None), b"workspace")
    _refused(lib.gan_mx_linear(1, 0, 1, 64, 64, p, 63, p, p, None, p, None, 0, None), b"stride")
    _refused(lib.gan_mx_linear(1, 0, 1, 64, 64, None, 64, p, p, None, p, None, 0, None), b"null")
    _refused(lib.gan_mx_matmul_dgrad(0, 4, 64, 64, p, p, p, p, None, 0, None), b"workspace")
    _refused(lib.gan_mx_matmul_wgrad(0, 0, 0, 64, 64, p, p, p, p, None, 0, p, 1 << 30, None), b"0 rows")
    ws = lib.gan_distill_topk_workspace_bytes(4)
    args = lambda **k: [{**dict(dtype=0, rows=4, classes=9, logits=p, ld=9, tdt=0, teacher=p, index=p, ib=4, top=3, lse=None, rw=None,
                                tau=1.0, weight=1.0, acc=0, loss=p, grad=p, ws=p, wn=ws, st=None), **k}[n] for n in
                        ("dtype", "rows", "classes", "logits", "ld", "tdt", "teacher", "index", "ib", "top", "lse", "rw", "tau",
                         "weight", "acc", "loss", "grad", "ws", "wn", "st")]
    for words, k in ((b"element type", dict(dtype=5)), (b"0 rows", dict(rows=0)), (b"0 classes", dict(classes=0)),
                     (b"1048577 classes", dict(classes=(1 << 20) + 1, ld=1 << 21)), (b"lists of 0", dict(top=0)),
                     (b"lists of 1025", dict(top=1025)), (b"indices of 2", dict(ib=2)), (b"temperature", dict(tau=0.0)),
                     (b"temperature", dict(tau=float('nan'))), (b"null", dict(loss=None)), (b"row stride", dict(ld=8)),
                     (b"workspace", dict(wn=ws - 1))):
        _refused(lib.gan_distill_topk_mean(*args(**k)), words)


def test_python_layer_refuses_what_does_not_go_together():
    from gan_amd import ops
    from gan_amd import variables as V
    x = torch.zeros(4, 64)
    with V.use_store(V.VariableStore(device='cpu')):
        with pytest.raises(TypeError):
            ops.rms_norm(x.double())
        with pytest.raises(ValueError):
            ops.rms_norm(x, residual=torch.zeros(4, 63))
        with pytest.raises(ValueError):
            ops.rms_norm(x, residual=x.bfloat16())
        with pytest.raises(ValueError):
            ops.rms_norm(torch.zeros(4, 0))
    with pytest.raises(ValueError):
        ops.mx_quantize(x, 'e5m2')
    with pytest.raises(TypeError):
        ops.mx_quantize(x.int())
    with pytest.raises(ValueError):
        ops.mx_pack(x[0])
    u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8)
    for codes, scales, k, n in ((u8(4, 10, 16), u8(1, 10, 4), 129, 10), (u8(4, 10, 16), u8(1, 9, 4), 128, 10), (x, x, 128, 10)):
        with pytest.raises(ValueError):
            ops.MxMatrix(codes, scales, k, n)
    w = ops.MxMatrix(u8(4, 10, 16), u8(1, 10, 4), 100, 10)
    for codes, scales, k, fmt in ((u8(3, 128), u8(3, 4), 129, 'e4m3'), (u8(3, 128), u8(2, 4), 100, 'e4m3'),
                                  (u8(3, 128), u8(3, 4), 100, 'e2m1'), (u8(3, 128), u8(3, 4), 100, 'fp8')):
        with pytest.raises(ValueError):
            ops.MxTensor(codes, scales, k, fmt)
    q = ops.MxTensor(u8(3, 128), u8(3, 4), 100)
    assert tuple(q.shape) == (3, 100) and tuple(w.shape) == (100, 10)
    with pytest.raises(ValueError):
        ops.mx_matmul(x, w)                                 # 64 values a row against 100 inputs
    with pytest.raises(ValueError):
        ops.mx_matmul(torch.zeros(3, 100), w, bias=torch.zeros(9))
    with pytest.raises(ValueError):
        ops.mx_matmul(torch.zeros(3, 100), w, fmt='fp4')
    t, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    for bad in (dict(teacher_index=i[:, :2]), dict(teacher_logits=t[:3]), dict(row_weight=torch.zeros(3)),
                dict(row_weight=torch.zeros(4, dtype=torch.float64)), dict(teacher_lse=torch.zeros(4, 1)), dict(temperature=-1.0)):
        with pytest.raises(ValueError):
            ops.distill_topk_mean(**{**dict(logits=x, teacher_logits=t, teacher_index=i), **bad})
    with pytest.raises(TypeError):
        ops.distill_topk_mean(x, t, i.float())
    with pytest.raises(ValueError):
        ops.distill_topk_mean(x[:0], t[:0], i[:0])


def test_ranges_beyond_the_documented_ones_are_refused():
    from gan_amd import _lib as L
    from gan_amd import ops
    from gan_amd import variables as V
    lib, p, x = L.lib, FAKE, torch.zeros(4, 64)
    _refused(lib.gan_rms_norm_fwd(0, 4, 64, p, 64, None, 0, p, -1e-6, None, p, None, None, None, None), b"epsilon")
    _refused(lib.gan_distill_topk_mean(0, 4000001, 9, p, 9, 0, p, p, 4, 3, None, None, 1.0, 1.0, 0, p, p, p, 1 << 30, None), b"4000001 rows")
    _refused(lib.gan_distill_topk_mean(0, 4, 9, p, 9, 0, p, p, 4, 3, None, None, 1e-20, 1.0, 0, p, p, p, 1 << 30, None), b"temperature")
    with V.use_store(V.VariableStore(device='cpu')):
        for eps in (-1e-6, float('nan'), float('inf')):
            with pytest.raises(ValueError):
                ops.rms_norm(x, epsilon=eps)
    t, i = torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int64)
    for tau in (1e-20, 1e20, float('nan')):
        with pytest.raises(ValueError):
            ops.distill_topk_mean(x, t, i, temperature=tau)
    # counts that a 32-bit argument would wrap around (expanded: nothing of that size is allocated)
    for shape in ((1 << 32, 64), (2, (1 << 32) + 64)):
        with pytest.raises(ValueError):
            ops._rows_of(torch.zeros(1, 1).expand(shape))


def test_a_capture_has_leaves_of_its_own(monkeypatch):
    from gan_amd import _lib, ops
    device = torch.device('cuda', 0)
    eager = ops._token_key(device, True)
    assert eager == ops._token_key(device, True) != ops._token_key(device, False)
    monkeypatch.setattr(_lib, 'capturing', lambda: True)
    monkeypatch.setattr(ops, 'stream', lambda: 7)
    first = ops._token_key(device, True)
    monkeypatch.setattr(ops, 'stream', lambda: 8)
    assert len({eager, first, ops._token_key(device, True)}) == 3


def test_both_gradients_at_once_are_refused_without_their_parts():
    from gan_amd import _lib as L
    lib, p, odd = L.lib, FAKE, ctypes.c_void_p(4096 + 2)
    need = lib.gan_mx_matmul_bwd_workspace_bytes(1, 64, 64, 64)
    assert need > lib.gan_mx_matmul_dgrad_workspace_bytes(1, 64, 64, 64) > 0 and lib.gan_mx_matmul_bwd_workspace_bytes(1, 0, 64, 64) == 0
    call = lambda rows=64, dy=p, dx=p, dm=p, a=p, n=need: lib.gan_mx_matmul_bwd(1, 0, rows, 64, 64, a, p, p, p, dy, dx, dm, None, 0, p, n, None)
    _refused(call(rows=0), b"0 rows")
    _refused(call(dx=None), b"null")
    _refused(call(dm=None), b"null")
    _refused(call(a=None), b"null")
    _refused(call(dy=odd), b"aligned")
    _refused(call(n=need - 1), b"workspace")


def test_linear_mx_shares_linears_variables():
    """By name, shape and reuse, as `linear` does (the products themselves need a GPU)."""
    from gan_amd import ops
    from gan_amd import variables as V
    st = V.VariableStore(device='cpu')
    with V.use_store(st):
        with pytest.raises(ValueError):
            ops.linear_mx(torch.zeros(2, 8), 3, 'head', reuse=True)         # nothing there to share
        with st.variable_scope('net'):
            a = ops._variable(st, 'head', 'Matrix', (8, 3), V.random_normal_initializer(0.02))
        assert list(st.vars) == ['net/head/Matrix'] and a.shape == (8, 3)
        with st.variable_scope('net'):
            assert ops._variable(st, 'head', 'Matrix', (8, 3), V.random_normal_initializer(0.02), True) is a
            with pytest.raises(ValueError):
                ops.linear_mx(torch.zeros(2, 7), 3, 'head')                  # another shape

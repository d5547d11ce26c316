"""GPU parity of layer norm and its gradients against the float64 definition
(oracle/lm_ops.py), and the operator's refusals.

Tolerances, with u = 2^-24 (float32) and uo the rounding of the output type:
a row's mean carries a few u |x| per partial sum, which divided by the row's
deviation is k = 1 + max|x| / sd in units of a normalised value.  So
  y:  uo |y| + 32 u k (|w| (1 + |xh|) + |b|)
  dx: uo |dx| + 64 u k rstd (|g| + mean|g| + |xh| mean|g xh|)
  dw: uo |dw| + (rows / 148 + 600) u sum |dy| (1 + |xh|) k   (serial rows per
      block, plus the blocks), and the same with sum |dy| for db.
"""
import numpy as np
import pytest
import torch

import manifold_b200 as gfn
from oracle import lm_ops as O

DEV = "cuda:0"
U = 2.0 ** -24
UO = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-38, torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24}


def _np(t):
    return t.detach().double().cpu().numpy()


def _check(got, want, tol, what):
    got = _np(got)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), np.abs(got - want).max(), np.max(np.abs(got - want) / tol))


def _compare(x, w, b, dy, eps, y, dx, dw, db):
    xn, wn, dn = _np(x), None if w is None else _np(w), _np(dy)
    D = xn.shape[-1]
    x2, d2 = xn.reshape(-1, D), dn.reshape(-1, D)
    mu = x2.mean(-1, keepdims=True)
    rstd = 1 / np.sqrt(x2.var(-1, keepdims=True) + eps)
    k = 1 + np.abs(x2).max(-1, keepdims=True) * rstd
    xh = (x2 - mu) * rstd
    wa = np.ones(D) if wn is None else wn
    want = O.layer_norm(xn, wn, None if b is None else _np(b), eps).reshape(-1, D)
    bt = 0.0 if b is None else np.abs(_np(b))
    o, t = UO[x.dtype], TINY[x.dtype]
    _check(y.reshape(-1, D), want, t + o * np.abs(want) + 32 * U * k * (np.abs(wa) * (1 + np.abs(xh)) + bt), "y")
    rx, rw, rb = O.layer_norm_backward(xn, dn, wn, eps)
    rx = rx.reshape(-1, D)
    g = d2 * wa
    scale = rstd * (np.abs(g) + np.abs(g).mean(-1, keepdims=True)
                    + np.abs(xh) * np.abs(g * xh).mean(-1, keepdims=True))
    if dx is not None:
        _check(dx.reshape(-1, D), rx, t + o * np.abs(rx) + 64 * U * k * scale, "dx")
    n = (x2.shape[0] / 148 + 600) * U
    if dw is not None:
        ow = UO[w.dtype]
        _check(dw, rw, 1e-37 + ow * np.abs(rw) + n * (np.abs(d2) * (1 + np.abs(xh)) * k).sum(0), "dw")
    if db is not None:
        _check(db, rb, 1e-37 + UO[b.dtype] * np.abs(rb) + n * np.abs(d2).sum(0), "db")


def _run(shape, dtype, wdtype, seed=0, offset=0.0, eps=1e-5, affine="wb"):
    g = torch.Generator().manual_seed(seed)
    D = shape[-1]
    x = (torch.randn(*shape, generator=g) * 1.5 + offset).to(dtype).to(DEV).requires_grad_(True)
    w = (1 + 0.3 * torch.randn(D, generator=g)).to(wdtype).to(DEV).requires_grad_(True) if "w" in affine else None
    b = (0.3 * torch.randn(D, generator=g)).to(wdtype).to(DEV).requires_grad_(True) if "b" in affine else None
    dy = torch.randn(*shape, generator=g).to(dtype).to(DEV)
    y = gfn.layer_norm(x, w, b, eps)
    assert y.dtype == dtype and y.shape == x.shape
    leaves = [t for t in (x, w, b) if t is not None]
    grads = list(torch.autograd.grad(y, leaves, dy))
    dx = grads.pop(0)
    dw = grads.pop(0) if w is not None else None
    db = grads.pop(0) if b is not None else None
    _compare(x, w, b, dy, eps, y, dx, dw, db)
    with torch.no_grad():
        assert torch.equal(gfn.layer_norm(x, w, b, eps), y)
    again = torch.autograd.grad(gfn.layer_norm(x, w, b, eps), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(again, [t for t in (dx, dw, db) if t is not None]))


SHAPES = [(1, 1), (3, 1), (1, 7), (5, 33), (2, 3, 64), (17, 100), (64, 128), (130, 256), (9, 512), (33, 1000),
          (40, 1001), (1, 1024), (700, 130), (12, 1536), (7, 2048), (5, 2056), (11, 4099), (3, 8192), (2, 16384),
          (2, 20001), (3, 40000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,wdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                          (torch.float16, torch.float32)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_layer_norm_matches_definition(shape, dtype, wdtype):
    _run(shape, dtype, wdtype, seed=len(shape) + shape[-1])


@pytest.mark.gpu
@pytest.mark.parametrize("affine", ["", "w", "b"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("dim", [96, 777, 2048])
def test_layer_norm_without_weight_or_bias(dim, dtype, affine):
    _run((37, dim), dtype, torch.float32, seed=dim, affine=affine)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [128, 1001, 4096])
def test_layer_norm_large_offset_keeps_the_variance(dim):
    # mean 1000 deviations away: sums of squares would lose the variance
    _run((20, dim), torch.float32, torch.float32, seed=dim, offset=1500.0)


@pytest.mark.gpu
def test_layer_norm_constant_rows_and_eps():
    x = torch.full((4, 384), 3.25, device=DEV)
    b = torch.randn(384, device=DEV)
    assert torch.equal(gfn.layer_norm(x, torch.ones_like(b), b), b.expand(4, -1))
    _run((6, 320), torch.float32, torch.float32, seed=1, eps=0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2000, 30011])
def test_layer_norm_many_rows_sum_the_weight_gradient(rows):
    _run((rows, 264), torch.float32, torch.float32, seed=rows)
    _run((rows, 261), torch.bfloat16, torch.float32, seed=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layer_norm_strided_rows_transposed_and_expanded(dtype):
    g = torch.Generator().manual_seed(5)
    base = torch.randn(6, 50, 3 * 96 + 2, generator=g).to(dtype).to(DEV)
    w, b = torch.randn(96, generator=g).to(DEV), torch.randn(96, generator=g).to(DEV)
    views = [base[..., 96:192], base[..., 1:97], base[:, ::2, 2:98], base.transpose(0, 1)[..., 5:101],
             base[..., :288].reshape(6, 50, 96, 3)[..., 1], base[:1, :, :96].expand(4, -1, -1),
             base[0, 0, :96].expand(9, 96), base[3, 4, :96]]
    for v in views:
        xv = v.detach().requires_grad_(True)
        wv, bv = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
        y = gfn.layer_norm(xv, wv, bv)
        assert y.is_contiguous()
        dyb = torch.randn(*y.shape, 2, generator=g).to(dtype).to(DEV)
        for dy in (dyb[..., 0], dyb[..., 0].contiguous(), dyb[..., :1, 0].expand(y.shape)):
            dx, dw, db = torch.autograd.grad(y, (xv, wv, bv), dy, retain_graph=True)
            _compare(v, w, b, dy, 1e-5, y, dx, dw, db)


@pytest.mark.gpu
def test_layer_norm_partial_gradients_and_empty_rows():
    x = torch.randn(8, 130, device=DEV)
    dy = torch.randn(8, 130, device=DEV)
    w, b = torch.randn(130, device=DEV), torch.randn(130, device=DEV)
    xg = x.clone().requires_grad_(True)
    dx, = torch.autograd.grad(gfn.layer_norm(xg, w, b), xg, dy)
    _compare(x, w, b, dy, 1e-5, gfn.layer_norm(x, w, b), dx, None, None)
    wg = w.clone().requires_grad_(True)
    dw, = torch.autograd.grad(gfn.layer_norm(x, wg, b), wg, dy)
    _compare(x, w, b, dy, 1e-5, gfn.layer_norm(x, w, b), None, dw, None)
    bg = b.clone().requires_grad_(True)
    db, = torch.autograd.grad(gfn.layer_norm(x, w, bg), bg, dy)
    _compare(x, w, b, dy, 1e-5, gfn.layer_norm(x, w, b), None, None, db)
    for shape in ((0, 130), (3, 0, 130)):
        e = torch.empty(shape, device=DEV, requires_grad=True)
        y = gfn.layer_norm(e, wg, bg)
        assert y.shape == shape
        dx, dw, db = torch.autograd.grad(y, (e, wg, bg), torch.empty(shape, device=DEV))
        assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dim", [64, 1001])
def test_layer_norm_non_finite_rows_stay_in_their_row(dim, bad):
    x = torch.randn(9, dim, device=DEV)
    ref = gfn.layer_norm(x)
    x[4, dim // 2] = bad
    y = gfn.layer_norm(x)
    assert torch.isnan(y[4]).all()
    keep = [r for r in range(9) if r != 4]
    assert torch.equal(y[keep], ref[keep])


@pytest.mark.gpu
def test_layer_norm_module_matches_torch_and_side_stream():
    torch.manual_seed(0)
    ref = torch.nn.LayerNorm(512).to(DEV)
    torch.nn.init.normal_(ref.weight)
    mod = gfn.LayerNorm(512).to(DEV)
    mod.load_state_dict(ref.state_dict())
    x = torch.randn(4, 9, 512, device=DEV)
    torch.testing.assert_close(mod(x), ref(x), rtol=1e-5, atol=1e-5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y = mod(x)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(y, mod(x))


@pytest.mark.gpu
def test_layer_norm_gradient_against_differences():
    g = torch.Generator().manual_seed(8)
    x = torch.randn(3, 40, generator=g).double()
    w, b, dy = (torch.randn(40, generator=g).double(), torch.randn(40, generator=g).double(),
                torch.randn(3, 40, generator=g).double())
    leaves = [t.float().to(DEV).requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(gfn.layer_norm(*leaves), leaves, dy.float().to(DEV))
    f = lambda *a: float((O.layer_norm(*[t.numpy() for t in a]) * dy.numpy()).sum())  # noqa: E731
    for k, (t, gr) in enumerate(zip((x, w, b), grads)):
        for i in range(0, t.numel(), 7):
            hi, lo = [u.clone() for u in (x, w, b)], [u.clone() for u in (x, w, b)]
            hi[k].view(-1)[i] += 1e-6
            lo[k].view(-1)[i] -= 1e-6
            # central difference: 1e-12 truncation, 1e-9 cancellation; the kernel: ~1e-6 of terms of order 3
            assert abs((f(*hi) - f(*lo)) / 2e-6 - float(gr.view(-1)[i])) < 2e-5


@pytest.mark.gpu
def test_layer_norm_second_derivative_and_changed_input_are_refused():
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    y = gfn.layer_norm(x)
    gx, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()
    h = x * 1.0
    y = gfn.layer_norm(h)
    h.add_(1.0)
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.gpu
def test_layer_norm_refusals_on_the_gpu():
    x = torch.randn(4, 32, device=DEV)
    w = torch.ones(32, device=DEV)
    for args in ((x.double(),), (x, torch.ones(31, device=DEV)), (x, w.bfloat16()), (x, w.half(), w),
                 (x, w.cpu()), (x.long(),), (x, torch.ones(1, 32, device=DEV)),
                 (torch.empty(4, 0, device=DEV),), (torch.tensor(1.0, device=DEV),),
                 (x.bfloat16(), w, w.bfloat16())):
        with pytest.raises(gfn.GfnError):
            gfn.layer_norm(*args)
    lib = gfn._lib.load()
    n = lib.gfn_layer_norm_backward_workspace_floats(4, 32)
    st = lib.gfn_layer_norm_backward(x.data_ptr(), 32, x.data_ptr(), 32, None, x.data_ptr(), 0, 0, 4, 32, None,
                                     w.data_ptr(), None, x.data_ptr(), n - 1, None)
    assert st == 1 and b"workspace" in lib.gfn_last_error_message()


def test_layer_norm_refusals():
    with pytest.raises(gfn.GfnError):  # no CPU path
        gfn.layer_norm(torch.zeros(2, 3))
    with pytest.raises(gfn.GfnError):
        gfn.LayerNorm((4, 5))
    lib = gfn._lib.load()
    assert lib.gfn_layer_norm_forward(None, 4, None, None, 0, 0, 2, 4, 1e-5, None, None, None) == 1
    assert lib.gfn_layer_norm_forward(None, 4, None, None, 0, 0, -1, 4, 1e-5, None, None, None) == 1
    assert lib.gfn_layer_norm_forward(None, 4, None, None, 0, 0, 0, 4, 1e-5, None, None, None) == 0
    assert lib.gfn_layer_norm_forward(16, 4, None, None, 7, 7, 1, 4, 1e-5, 16, None, None) == 2
    assert lib.gfn_layer_norm_forward(16, 3, None, None, 0, 0, 2, 4, 1e-5, 16, None, None) == 1
    assert lib.gfn_layer_norm_backward_workspace_floats(5, 0) == -1


def test_layer_norm_definition_gradient_against_differences():
    rng = np.random.default_rng(0)
    x, w, b, dy = rng.standard_normal((3, 7)), rng.standard_normal(7), rng.standard_normal(7), rng.standard_normal((3, 7))
    grads = O.layer_norm_backward(x, dy, w)
    for k, g in enumerate(grads):
        for i in range(g.size):
            args = [[x.copy(), w.copy(), b.copy()] for _ in range(2)]
            args[0][k].reshape(-1)[i] += 1e-6
            args[1][k].reshape(-1)[i] -= 1e-6
            d = ((O.layer_norm(*args[0]) - O.layer_norm(*args[1])) * dy).sum() / 2e-6
            assert abs(d - g.reshape(-1)[i]) < 1e-7

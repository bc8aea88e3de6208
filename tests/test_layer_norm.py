"""Layer norm forward and backward against its definition in 64 bits.  Tolerances are bounds on fp32 arithmetic: U = 2^-24 is half a unit in
the last place of fp32, G = 64 U bounds the relative error of a sum of up to 40000 terms as the kernels form it (at most 40 additions in a
row in one thread, then a tree over at most 1024 threads), and each output adds half a unit of its own type."""
import pytest
import torch

import triton_tenstorrent_b200 as tt
from triton_tenstorrent_b200 import _lib, ops

U = 2.0 ** -24
G = 64 * U
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(t):
    return torch.finfo(t).eps / 2


def reference(x, w, b, dy, eps):
    """y, mean, rstd, dx, dw, db and the elementwise tolerances of y, dx, dw, db, all fp64 (x, dy: [rows, cols])."""
    x, n = x.double(), x.shape[-1]
    wd = torch.ones(n, dtype=torch.float64, device=x.device) if w is None else w.double()
    bd = torch.zeros(n, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1 / (var + eps).sqrt()
    h = (x - mean) * rstd
    # error of h: the mean's (G of the mean magnitude), the difference's rounding, the variance's relative error (half of it reaches rstd; the
    # mean's error enters it squared) and rsqrt's
    tol_mean = G * x.abs().mean(-1, keepdim=True) + U * mean.abs()
    # when the spread is small against the mean's error, the variance is off by the square of that error
    tol_h = rstd * (tol_mean + 2 * U * x.abs()) + h.abs() * (2 * G + 8 * U + (rstd * tol_mean).square())
    y = h * wd + bd
    tol_y = wd.abs() * tol_h + 4 * U * ((h * wd).abs() + bd.abs())
    out = {"y": (y, tol_y), "mean": (mean[:, 0], tol_mean[:, 0]), "rstd": (rstd[:, 0], (rstd * (2 * G + 8 * U + (rstd * tol_mean).square()))[:, 0])}
    if dy is not None:
        dy = dy.double()
        u = dy * wd
        c1, c2 = u.mean(-1, keepdim=True), (u * h).mean(-1, keepdim=True)
        dx = rstd * (u - c1 - h * c2)
        tol_c1 = G * u.abs().mean(-1, keepdim=True)
        tol_c2 = G * (u * h).abs().mean(-1, keepdim=True) + (u.abs() * tol_h).mean(-1, keepdim=True)
        tol_dx = rstd * (4 * U * (u.abs() + c1.abs() + (h * c2).abs()) + tol_c1 + h.abs() * tol_c2 + tol_h * c2.abs())
        tol_dx = tol_dx + dx.abs() * (2 * G + 8 * U + (rstd * tol_mean).square())
        out["dx"] = (dx, tol_dx)
        out["dw"] = ((dy * h).sum(0), G * (dy * h).abs().sum(0) + (dy.abs() * tol_h).sum(0))
        out["db"] = (dy.sum(0), G * dy.abs().sum(0))
    return out


def check(name, got, want):
    ref, tol = want
    assert got.shape == ref.shape, name
    got = got.double()
    least = 0.0 if got.numel() == 0 else torch.finfo(torch.float16).smallest_normal * 2.0 ** -10      # a subnormal step of fp16
    limit = tol + half_of[name] * (ref.abs() + tol) + (least if half_of[name] == half(torch.float16) else 1e-37)
    off = (got - ref).abs() - limit
    assert not bool((off > 0).any()) and not bool(torch.isnan(got).any()), f"{name}: {float((got - ref).abs().max())} off, {float(off.max())} over the bound"


half_of = {}


def run_and_check(x, w, b, dy, eps=1e-5, cols=None):
    cols = x.shape[-1]
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b, eps)
    wt = torch.float32 if w is None else w.dtype
    half_of.update(y=half(x.dtype), dx=half(x.dtype), dw=half(wt), db=half(wt), mean=U, rstd=U)
    ref = reference(x.reshape(-1, cols), w, b, None if dy is None else dy.reshape(-1, cols), eps)
    assert y.shape == x.shape and y.dtype == x.dtype and mean.shape == x.shape[:-1] and y.is_contiguous()
    check("y", y.view(-1, cols), ref["y"])
    check("mean", mean.view(-1), ref["mean"])
    check("rstd", rstd.view(-1), ref["rstd"])
    if dy is not None:
        dx, dw, db = tt.layer_norm_backward(dy, x, w, mean, rstd)
        assert dx.shape == x.shape and dx.dtype == x.dtype and dw.dtype == wt and db.dtype == wt
        check("dx", dx.reshape(-1, cols), ref["dx"])
        check("dw", dw, ref["dw"])
        check("db", db, ref["db"])


def make(rows, cols, dtype, wdtype, seed=0, shift=0.3):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return ((rn(rows, cols) * 1.5 + shift).to(dtype), (rn(cols) * 0.3 + 1).to(wdtype), rn(cols).to(wdtype), rn(rows, cols).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 4096), (5, 7), (2, 31), (130, 33), (64, 128), (67, 257), (9, 1000), (301, 1024), (33, 1537), (20, 2056),
                                       (600, 4096), (7, 5001), (3, 8192), (149, 8200), (2, 16384), (4, 16387), (3, 32768), (2, 40000)])
def test_matches_the_definition(rows, cols, dtype):
    x, w, b, dy = make(rows, cols, dtype, dtype)
    run_and_check(x, w, b, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cols", [96, 515, 2048, 8192])
def test_fp32_weights_and_missing_ones(cols, dtype):
    x, w, b, dy = make(37, cols, dtype, torch.float32)
    run_and_check(x, w, b, dy)
    run_and_check(x, w, None, dy)
    run_and_check(x, None, b, dy)
    run_and_check(x, None, None, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_alignment_and_broadcast(dtype):
    x, w, b, dy = make(40, 520, dtype, dtype)
    run_and_check(x[:, :512], w[:512], b[:512], dy[:, :512])              # row pitch above the row length
    run_and_check(x[:, 1:514], w[1:514], b[1:514], dy[:, 3:516])          # bases off any 16-byte boundary, odd length
    run_and_check(x[:, 8:136], w[8:136], b[8:136], dy[:, 4:132])          # one operand aligned, the other not
    run_and_check(x[::3], w, b, dy[::3])
    run_and_check(x.view(4, 10, 520).transpose(0, 1), w, b, dy.view(4, 10, 520).transpose(0, 1))   # rows not in one pitch
    run_and_check(x.t().contiguous().t(), w, b, dy)                       # inner stride not one
    run_and_check(x[:1].expand(40, 520), w, b, dy[:1].expand(40, 520))    # one row seen forty times
    run_and_check(x[0], w, b, dy[0])                                      # no row dimension at all
    run_and_check(x[:, :1], w[:1], b[:1], dy[:, :1])


@pytest.mark.gpu
def test_many_rows_narrow_and_large_mean():
    x, w, b, dy = make(70001, 40, torch.bfloat16, torch.float32)
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    half_of.update(y=half(x.dtype), dx=half(x.dtype), dw=U, db=U, mean=U, rstd=U)
    ref = reference(x, w, b, dy, 1e-5)
    dx, dw, db = tt.layer_norm_backward(dy, x, w, mean, rstd)
    check("y", y, ref["y"])
    check("dx", dx, ref["dx"])
    # 70001 rows: at most 70001 / 296 additions in a row and 37 + 8 joins
    scale = (70001 / 296 + 45) / 64 + 1
    check("dw", dw, (ref["dw"][0], scale * ref["dw"][1]))
    check("db", db, (ref["db"][0], scale * ref["db"][1]))
    # a mean far above the spread: E[x^2] - mean^2 would lose every digit here
    x, w, b, dy = make(17, 3000, torch.float32, torch.float32, shift=3000.0)
    run_and_check(x, w, b, dy)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_constant_rows_and_non_finite_rows(dtype):
    x, w, b, dy = make(6, 384, dtype, dtype)
    x[1] = 2.0                       # variance zero: y is the bias
    x[4] = 0.0
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b, 1e-5)
    assert torch.equal(y[1], b) and torch.equal(y[4], b)
    assert torch.allclose(rstd[1], torch.full_like(rstd[1], 1e-5 ** -0.5), rtol=1e-6)
    clean, clean_dx = y.clone(), tt.layer_norm_backward(dy, x, w, mean, rstd)[0]
    x[2, 5], x[3, 7] = float("nan"), float("inf")
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b, 1e-5)
    dx = tt.layer_norm_backward(dy, x, w, mean, rstd)[0]
    keep = torch.tensor([0, 1, 4, 5], device="cuda")
    assert torch.equal(y[keep], clean[keep]) and torch.equal(dx[keep], clean_dx[keep])     # other rows untouched
    assert bool(y[2].isnan().all()) and bool(dx[2].isnan().all()) and bool(y[3].isnan().any())


@pytest.mark.gpu
def test_empty_and_partial_gradients():
    x, w, b, dy = make(0, 64, torch.bfloat16, torch.float32)
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    dx, dw, db = tt.layer_norm_backward(dy, x, w, mean, rstd)
    assert y.shape == (0, 64) and dx.shape == (0, 64) and not bool(dw.any()) and not bool(db.any())
    x, w, b, dy = make(50, 640, torch.float32, torch.float32)
    _, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    full = tt.layer_norm_backward(dy, x, w, mean, rstd)
    for need in [(True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, False)]:
        for got, want, wanted in zip(tt.layer_norm_backward(dy, x, w, mean, rstd, *need), full, need):
            assert (got is None) if not wanted else torch.equal(got, want)


@pytest.mark.gpu
def test_autograd_against_the_formula_and_differences():
    x, w, b, dy = make(24, 200, torch.float32, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    tt.layer_norm(leaves[0].view(4, 6, 200), *leaves[1:]).backward(dy.view(4, 6, 200))
    _, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    for leaf, want in zip(leaves, tt.layer_norm_backward(dy, x, w, mean, rstd)):
        assert torch.equal(leaf.grad, want)

    def f(x, w, b):
        c = x - x.mean(-1, keepdim=True)
        return ((c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b) * dy.double()).sum()

    g = torch.Generator(device="cuda").manual_seed(3)
    for leaf, k in zip(leaves, range(3)):
        args = [t.double() for t in (x, w, b)]
        d = torch.randn(leaf.shape, generator=g, device="cuda", dtype=torch.float64)
        step = 1e-5
        hi, lo = ([a + s * step * d if i == k else a for i, a in enumerate(args)] for s in (1, -1))
        slope = float((f(*hi) - f(*lo)) / (2 * step))
        # differences: O(step^2) and 2^-53 |f| / step; the gradient: a few G of its terms
        got = float((leaf.grad.double() * d).sum())
        bound = 1e-6 * float(d.norm() * leaf.grad.double().norm()) + 4 * G * float((leaf.grad.double() * d).abs().sum())
        assert abs(got - slope) <= bound


@pytest.mark.gpu
def test_broadcast_gradient_mixed_types_and_frozen_leaves():
    x, w, b, _ = make(10, 96, torch.bfloat16, torch.float32)
    x.requires_grad_(True)
    b.requires_grad_(True)
    tt.layer_norm(x, None, b).sum().backward()        # an expanded gradient; fp32 bias without a weight
    assert b.grad.dtype == torch.float32 and torch.equal(b.grad, torch.full_like(b, 10.0))
    assert x.grad.dtype == torch.bfloat16 and float(x.grad.abs().max()) < 1e-5
    assert not tt.layer_norm(x.detach(), w).requires_grad


@pytest.mark.gpu
def test_other_stream_graph_and_determinism():
    x, w, b, dy = make(500, 1536, torch.bfloat16, torch.bfloat16)
    want = tt.layer_norm_with_stats(x, w, b)
    want_grads = tt.layer_norm_backward(dy, x, w, *want[1:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = tt.layer_norm_with_stats(x, w, b)
        grads = tt.layer_norm_backward(dy, x, w, *got[1:])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want + want_grads, got + grads))
    graphs, outs = [], []
    for _ in range(2):               # two graphs, replayed in turn: neither may disturb the other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = tt.layer_norm_with_stats(x, w, b)
            outs.append(got + tt.layer_norm_backward(dy, x, w, *got[1:]))
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(p, q) for p, q in zip(want + want_grads, out))


@pytest.mark.gpu
def test_host_tensors():
    x, w, b, dy = (t.cpu() for t in make(12, 72, torch.float32, torch.float32))
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    grads = tt.layer_norm_backward(dy, x, w, mean, rstd)
    assert all(not t.is_cuda for t in (y, mean, rstd, *grads))
    assert torch.allclose(y, torch.nn.functional.layer_norm(x, (72,), w, b), atol=1e-5)


def test_refusals():
    x = torch.zeros(4, 8)
    for bad, error in [(dict(x=x.double()), TypeError), (dict(x=torch.zeros(4, 0)), ValueError), (dict(x=torch.tensor(1.0)), ValueError),
                       (dict(weight=torch.zeros(7)), ValueError), (dict(weight=torch.zeros(8, dtype=torch.bfloat16)), TypeError),
                       (dict(bias=torch.zeros(8, 1)), ValueError), (dict(x=x.bfloat16(), weight=torch.zeros(8), bias=torch.zeros(8).bfloat16()), TypeError),
                       (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError)]:
        with pytest.raises(error):
            tt.layer_norm(**{"x": x, **bad})
    stats = torch.zeros(4)
    for args in [(torch.zeros(4, 7), x, None, stats, stats), (x.bfloat16(), x, None, stats, stats), (x, x, None, stats.double(), stats),
                 (x, x, None, stats, torch.zeros(3))]:
        with pytest.raises(ValueError):
            tt.layer_norm_backward(*args)
    assert ops._DTYPES[torch.float16] == _lib.DTYPE_F16


def test_entry_point_refusals():
    lib = _lib.load()
    fwd = lambda x=16, y=16, rows=4, cols=8, ldx=8, ldy=8, dt=0, wdt=0, eps=1e-5: lib.b200k_layer_norm_fwd(  # noqa: E731
        x, None, None, y, None, None, rows, cols, ldx, ldy, dt, wdt, eps, None)
    for bad in [dict(dt=3), dict(dt=-1), dict(dt=1, wdt=2), dict(rows=-1), dict(cols=0), dict(cols=2 ** 31), dict(rows=2 ** 60, cols=2 ** 20), dict(x=None),
                dict(y=None), dict(x=18), dict(y=17, dt=1, wdt=1), dict(ldx=-8), dict(ldy=7), dict(eps=-1.0), dict(eps=float("nan"))]:
        assert fwd(**bad) == _lib.ERR_INVALID_ARG and "layer_norm" in _lib.last_error(), bad
    assert fwd(rows=0) == _lib.OK
    floats = lib.b200k_layer_norm_bwd_workspace(1000, 64)
    assert floats >= 2 * 64 and lib.b200k_layer_norm_bwd_workspace(-1, 64) == 0
    bwd = lambda dy=16, work=16, floats=floats, lddx=64, dw=16: lib.b200k_layer_norm_bwd(  # noqa: E731
        dy, 16, None, 16, 16, 16, dw, None, work, floats, 1000, 64, 64, 64, lddx, 0, 0, None)
    for bad in [dict(dy=None), dict(work=None), dict(floats=floats - 1), dict(lddx=63)]:
        assert bwd(**bad) == _lib.ERR_INVALID_ARG, bad
    assert "workspace" in _lib.last_error() or "stride" in _lib.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols,pad", [(1, 7), (40, 8), (200, 24), (257, 3), (384, 16), (513, 1), (520, 8), (1000, 24), (1026, 2), (2051, 5), (2056, 8), (4104, 8), (5000, 8), (8200, 56),
                                      (9001, 2), (16384, 8)])
def test_nothing_outside_the_rows_is_written(cols, pad, dtype):
    rows, ld = 5, cols + pad
    x, w, b, dy = make(rows, cols, dtype, dtype)
    lib, code = _lib.load(), ops._DTYPES[dtype]
    y, dx = (torch.full((rows + 2, ld), 777.0, device="cuda", dtype=dtype) for _ in range(2))
    stats = torch.full((2, rows + 8), 777.0, device="cuda")
    grads = torch.full((2, cols + 32), 777.0, device="cuda", dtype=dtype)
    floats = lib.b200k_layer_norm_bwd_workspace(rows, cols)
    work = torch.full((floats + 64,), 777.0, device="cuda")
    size = x.element_size()
    stream = ops._stream()
    _lib.check(lib.b200k_layer_norm_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), y.data_ptr() + ld * size, stats.data_ptr(), stats[1].data_ptr(), rows,
                                        cols, cols, ld, code, code, 1e-5, stream))
    _lib.check(lib.b200k_layer_norm_bwd(dy.data_ptr(), x.data_ptr(), w.data_ptr(), stats.data_ptr(), stats[1].data_ptr(), dx.data_ptr() + ld * size,
                                        grads.data_ptr(), grads[1].data_ptr(), work.data_ptr(), floats, rows, cols, cols, cols, ld, code, code, stream))
    want = tt.layer_norm_with_stats(x, w, b)
    want_grads = tt.layer_norm_backward(dy, x, w, *want[1:])
    half_of.update(y=half(dtype), dx=half(dtype), dw=half(dtype), db=half(dtype), mean=U, rstd=U)
    ref = reference(x, w, b, dy, 1e-5)
    for buf, name in ((y, "y"), (dx, "dx")):
        check(name, buf[1:rows + 1, :cols], ref[name])
        assert bool((buf[0] == 777).all()) and bool((buf[rows + 1] == 777).all()) and bool((buf[1:rows + 1, cols:] == 777).all())
    for buf, names, n in ((stats, ("mean", "rstd"), rows), (grads, ("dw", "db"), cols)):
        for i, name in enumerate(names):
            check(name, buf[i, :n], ref[name])
            assert bool((buf[i, n:] == 777).all())
    assert bool((work[floats:] == 777).all()) and want_grads[0].shape == x.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_of_a_million_elements(dtype):
    """The bound G for sums of any length.  Equal terms are the worst case: their roundings all go one way for as long as the sum stays in one binade."""
    x, w, b, dy = make(3, (1 << 20) + 3, dtype, dtype)
    run_and_check(x, w, b, dy)
    x[1], dy[1] = 0.3, 0.7
    x[2] = x[2].abs() + 1
    run_and_check(x, w, b, dy)


@pytest.mark.gpu
def test_many_long_rows():
    """Column sums over 5000 rows of 16400 elements, terms all of one sign: at most 32 additions in a row in fp32, 888 parts joined by 32 threads of 28 each, and a tree."""
    x, w, b, dy = make(5000, 16400, torch.bfloat16, torch.float32)
    dy.fill_(0.7)
    x, w = x.abs(), None
    _, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    _, _, db = tt.layer_norm_backward(dy, x, w, mean, rstd, need_dx=False, need_dw=False)
    want = 5000 * float(dy[0, 0])
    assert float((db.double() - want).abs().max()) <= (32 + 28 + 5 + 1) * U * want


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [40, 128, 515, 600, 1024, 2051, 4104, 5000, 8192, 8200, 9001, 12000, 16384, 16400])
def test_non_finite_rows_leave_the_others_as_they_are(cols, dtype):
    """At every row shape: rows that share a reduction, a warp or a stage of the ring, rows that are read twice, and rows off any alignment."""
    x, w, b, dy = make(13, cols, dtype, dtype, seed=cols)
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    dx = tt.layer_norm_backward(dy, x, w, mean, rstd)[0]
    bad_x, bad_dy = [2, 5, 12], 8
    x2, dy2 = x.clone(), dy.clone()
    x2[2, cols - 1], x2[5, 0], x2[12, cols // 2] = float("nan"), float("inf"), float("-inf")
    dy2[bad_dy, cols // 3] = float("inf")
    y2, mean2, rstd2 = tt.layer_norm_with_stats(x2, w, b)
    dx2, dw2, db2 = tt.layer_norm_backward(dy2, x2, w, mean2, rstd2)
    keep = torch.ones(13, dtype=torch.bool, device="cuda")
    keep[bad_x] = False
    assert torch.equal(y2[keep], y[keep]) and torch.equal(mean2[keep], mean[keep]) and torch.equal(rstd2[keep], rstd[keep])
    assert bool(y2[bad_x].isnan().all()) and not bool(mean2[bad_x].isfinite().any())
    keep[bad_dy] = False
    assert torch.equal(dx2[keep], dx[keep]) and bool(dx2[bad_x].isnan().all()) and not bool(dx2[bad_dy].isfinite().any())
    assert bool(dw2.isnan().all()) and bool(db2.isfinite().sum() == cols - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols,dtype", [(700, 40, torch.bfloat16), (333, 600, torch.float16), (301, 8192, torch.bfloat16), (150, 16384, torch.float32), (7, 20000, torch.bfloat16),
                                             (200, 2051, torch.bfloat16)])
def test_captured_and_replayed_with_other_inputs(rows, cols, dtype):
    x, w, b, dy = make(rows, cols, dtype, torch.float32)
    call = lambda: (lambda s: s + tt.layer_norm_backward(dy, x, w, *s[1:]))(tt.layer_norm_with_stats(x, w, b))  # noqa: E731
    call()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call())
        graphs.append(graph)
    for seed in (1, 2):
        for t, new in zip((x, w, b, dy), make(rows, cols, dtype, torch.float32, seed)):
            t.copy_(new)
        for graph in graphs:
            graph.replay()
        want = call()
        assert all(torch.equal(p, q) for out in outs for p, q in zip(want, out))

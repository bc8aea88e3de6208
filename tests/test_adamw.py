"""The AdamW step against its definition in 64 bits, the 8-bit moments against their definition (codes, scales, stochastic rounding).

Tolerances: U = 2^-24 is half a unit in the last place of fp32.  m takes three roundings of terms no larger than |b1 m| + |(1 - b1) g|, v four; b1,
1 - b1, b2 and 1 - b2 are themselves rounded once.  p takes the roundings of decay, step size, root, quotient and two sums: with D the size of the
update, 4 U |p| + 24 U D covers them."""
import copy
import pickle

import numpy as np
import pytest
import torch

import triton_tenstorrent_b200 as tt
from triton_tenstorrent_b200 import _lib, ops, optim

U = 2.0 ** -24
BLOCK = 256
SHAPES = [(1,), (7,), (256,), (300, 5), (0,), (1000,), (16384,), (16385,), (33, 1025), (4, 3, 2)]


def half(t):
    return torch.finfo(t).eps / 2


def exact_step(p, g, m, v, t, lr, betas, eps, wd, scale=1.0):
    """(p, m, v, tolerances of p, m, v) in fp64; p, g, m, v as they are held before the step, t the number of this step."""
    b1, b2 = betas
    p, m, v = p.double(), m.double(), v.double()
    g = g.double() * scale
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    d = v1.sqrt() / (1 - b2 ** t) ** 0.5 + eps
    update = lr / (1 - b1 ** t) * m1 / d
    tol_m = 4 * U * ((b1 * m).abs() + ((1 - b1) * g).abs()) + 1e-44
    tol_v = 6 * U * (b2 * v + (1 - b2) * g * g) + 1e-44
    tol_p = 4 * U * p.abs() + 24 * U * update.abs() + lr / (1 - b1 ** t) * tol_m / d
    return p * (1 - lr * wd) - update, m1, v1, tol_p, tol_m, tol_v


def make(shapes, dtype, gdtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    params = [(rn(*s) * 0.1).to(dtype) for s in shapes]
    grads = [(rn(*s) * torch.exp(rn(*s) * 1.5) * 1e-2).to(gdtype) for s in shapes]
    return params, grads


def near(got, ref, tol, dtype=torch.float32):
    limit = tol + half(dtype) * (ref.abs() + tol) + (2.0 ** -25 if dtype == torch.float16 else 1e-44)
    assert got.shape == ref.shape and bool(((got.double() - ref).abs() <= limit).all()), float(((got.double() - ref).abs() - limit).max())


HYPER = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype,master", [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
                                                 (torch.bfloat16, torch.float32, True), (torch.bfloat16, torch.bfloat16, True),
                                                 (torch.float16, torch.float16, False), (torch.float16, torch.float16, True),
                                                 (torch.float16, torch.float32, False), (torch.float16, torch.float32, True),
                                                 (torch.bfloat16, torch.float32, False)])
def test_three_steps_with_fp32_moments(dtype, gdtype, master):
    params, _ = make(SHAPES, dtype, gdtype)
    opt = tt.AdamW(params, master_weights=master, **HYPER)
    for t in range(1, 4):
        grads = make(SHAPES, dtype, gdtype, seed=t)[1]
        work = opt.split(opt.master) if master else params
        before = [x.clone() for x in work], [x.clone() for x in opt.split(opt.moments()[0])], [x.clone() for x in opt.split(opt.moments()[1])]
        opt.step(grads)
        after = (opt.split(opt.master) if master else params), opt.split(opt.moments()[0]), opt.split(opt.moments()[1])
        for i in range(len(params)):
            p, m, v, tol_p, tol_m, tol_v = exact_step(before[0][i], grads[i], before[1][i], before[2][i], t, **{k: HYPER[k] for k in ("lr", "betas", "eps")},
                                                      wd=HYPER["weight_decay"])
            near(after[0][i], p, tol_p, torch.float32 if master else dtype)
            near(after[1][i], m, tol_m)
            near(after[2][i], v, tol_v)
            assert torch.equal(params[i], after[0][i].to(dtype))
    assert opt.step_count() == 3


def mix32(x):
    x = x & 0xFFFFFFFF
    x = x ^ (x >> 16)
    x = (x * 0xDDB3D743) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xB504F335) & 0xFFFFFFFF
    return x ^ (x >> 16)


def values(bits):
    c = np.arange(1 << (4 + bits))
    v = (1 + (c % (1 << bits)) / (1 << bits)) * 2.0 ** (c >> bits)
    v[0], v[-1] = 0.0, np.nan
    return v


def random16(n, index, step, seed):
    salt = mix32(mix32((seed + step * 0x9E3779B9) & 0xFFFFFFFF) + index)
    h = mix32((np.arange(n, dtype=np.int64) + salt) & 0xFFFFFFFF)
    return h & 0xFFFF, h >> 16


def check_codes(x, tol, codes, scales, rnd, bits):
    """codes and scales of x (fp64, what was rounded) by the definition: neighbours chosen by the random bits.  The kernel rounds an fp32 number
    that is within `tol` of x (more than a few U of x where m's two terms cancel): an element whose decision lies that near is only held to
    being a neighbour, and one that near to zero may have either sign."""
    n = x.size
    v = values(bits)
    top = v[-2]
    for b in range(-(-n // BLOCK)):
        s = slice(b * BLOCK, min(n, (b + 1) * BLOCK))
        mag, c, r, t = np.abs(x[s]), codes[s].astype(np.int64), rnd[s], tol[s]
        peak = mag.max()
        if peak == 0:
            assert not c.any()
            continue
        assert np.log2(scales[b]) % 1 == 0 and peak / scales[b] <= top * (1 + 16 * U) and (2 * peak / scales[b] > top * (1 - 16 * U) or scales[b] == 2.0 ** -126)
        k = c & (v.size - 1)
        if bits == 3:
            assert (((c >= 128) == (x[s] < 0)) | (mag <= t)).all()
        y = np.minimum(mag / scales[b], top)
        low = np.searchsorted(v[:-1], y, side="right") - 1          # the code at or below y
        high = np.minimum(low + 1, v.size - 2)
        step = np.where(high > low, v[high] - v[low], 1.0)
        part = (y - v[low]) / step
        below = (2 * r + 1) / 131072 - part if bits == 3 else np.where(y > 0, -1.0, 1.0)
        sure = np.where(low == 0, below, 1 - r / 65536 - part)      # below zero: up
        expect = np.where(sure <= 0, high, low)
        edge = np.abs(sure) < 64 * U * 2 ** (bits + 1) + 2 * t / scales[b] / step
        off = (k != expect) & ~edge
        assert not off.any(), (np.nonzero(off)[0][:5], k[off][:5], expect[off][:5], y[off][:5])
        assert ((k == low) | (k == high) | (np.abs(y - v[k]) <= 64 * U * y + t / scales[b]))[edge].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gdtype,master", [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
                                                 (torch.bfloat16, torch.float32, True), (torch.float16, torch.float16, True),
                                                 (torch.float16, torch.float32, False), (torch.bfloat16, torch.bfloat16, True)])
def test_three_steps_with_8_bit_moments(dtype, gdtype, master):
    params, _ = make(SHAPES, dtype, gdtype)
    opt = tt.AdamW(params, master_weights=master, state_bits=8, seed=5, **HYPER)
    for t in range(1, 4):
        grads = make(SHAPES, dtype, gdtype, seed=t)[1]
        work = opt.split(opt.master) if master else params
        before = [x.clone() for x in work], *([x.clone() for x in opt.split(y)] for y in opt.moments())
        opt.step(grads)
        held = opt.state_dict()
        m_now, v_now = (opt.split(x) for x in opt.moments())
        work = opt.split(opt.master) if master else params
        for i, a in enumerate(opt.offsets):
            n = params[i].numel()
            if n == 0:
                continue
            p, m, v, tol_p, tol_m, _ = exact_step(before[0][i], grads[i], before[1][i], before[2][i], t, **{k: HYPER[k] for k in ("lr", "betas", "eps")},
                                              wd=HYPER["weight_decay"])
            near(work[i], p, tol_p, torch.float32 if master else dtype)
            rm, rr = random16(n, i, t, 5)
            blocks = slice(a // BLOCK, a // BLOCK + -(-n // BLOCK))
            mc, rc = held["exp_avg"][a:a + n].cpu().numpy(), held["exp_avg_sq_root"][a:a + n].cpu().numpy()
            ms, rs = held["exp_avg_scale"][blocks].double().cpu().numpy(), held["exp_avg_sq_root_scale"][blocks].double().cpu().numpy()
            root = v.sqrt().reshape(-1).cpu().numpy()
            check_codes(m.reshape(-1).cpu().numpy(), tol_m.reshape(-1).cpu().numpy(), mc, ms, rm, 3)
            check_codes(root, 8 * U * root, rc, rs, rr, 4)
            # the values that moments() gives
            per = np.arange(n) // BLOCK
            want_m = values(3)[mc & 127] * np.where(mc >= 128, -1, 1) * ms[per]
            want_v = (values(4)[rc] * rs[per]) ** 2
            assert np.abs(m_now[i].reshape(-1).double().cpu().numpy() - want_m).max() <= 2 * U * np.abs(want_m).max() + 1e-44
            assert (np.abs(v_now[i].reshape(-1).double().cpu().numpy() - want_v) <= 4 * U * want_v + 1e-44).all()
    tail = held["exp_avg"][opt.offsets[1] + 7:opt.offsets[2]]
    assert not bool(tail.any())                   # the padding of a block stays zero


def test_hash_is_even():
    # the random bits of 2^16 neighbouring elements: mean and correlation within five standard deviations
    for index, step, seed in [(0, 1, 0), (1, 1, 0), (0, 2, 0), (5, 1000, 7)]:
        lo, hi = (x / 65536 for x in random16(65536, index, step, seed))
        for x in (lo, hi):
            assert abs(x.mean() - 0.5) < 5 * (1 / 12 / 65536) ** 0.5
            assert abs(np.corrcoef(x[:-1], x[1:])[0, 1]) < 5 / 256
        assert abs(np.corrcoef(lo, hi)[0, 1]) < 5 / 256


@pytest.mark.gpu
def test_8_bit_moments_follow_the_fp32_ones():
    """A second moment decays by 0.1 % a step, far below half a step of its code: with stochastic rounding it still follows on average."""
    n = 1 << 16
    p, (g,) = [torch.zeros(n, device="cuda")], make([(n,)], torch.float32, torch.float32, seed=9)[1]
    opts = [tt.AdamW([p[0].clone()], lr=1e-3, betas=(0.9, 0.999), weight_decay=0.0, state_bits=b) for b in (32, 8)]
    for t in range(400):
        for opt in opts:
            opt.step([g if t == 0 else g * 0.1])
    (m0, v0), (m1, v1) = (opt.moments() for opt in opts)
    # The roundings of different elements are independent, so that the means over 2^16 elements agree to well under 1 %.
    assert abs(float(v1.sqrt().mean() / v0.sqrt().mean()) - 1) < 0.01
    assert abs(float(m1.abs().mean() / m0.abs().mean()) - 1) < 0.01
    # One element's r: a step moves it by c = 0.0005 at most, a code's step is d <= 1/16, so it is rounded up or down with variance c d, and
    # after 400 steps it is off by sqrt(400 c d) = 0.112 (r decays, and its error with it).  The mean over the path is off by less than the end,
    # m's roundings (half of d = 1/8, remembered for 10 steps, so 0.0625 / sqrt(0.19) sqrt(20 / 400) = 0.032) add in squares, and E[1/r] is
    # above 1/E[r] by half the variance at most, 0.0063.
    assert float((opts[1].params[0] - opts[0].params[0]).norm() / opts[0].params[0].norm()) < (0.112 ** 2 + 0.032 ** 2) ** 0.5 + 0.0063


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_unaligned_tensors_and_strided_gradients(bits, dtype):
    base, grad = torch.randn(5000, device="cuda").to(dtype), torch.randn(5000, device="cuda").to(dtype)
    params = [base[1:1 + 700].clone(), base[:0], base[2000:2000 + 640].clone()]
    views = [base[1:1 + 700], base[:0], base[2000:2000 + 640]]
    grads = [grad[3:703], grad[:0], grad[1000:1000 + 1280][::2]]
    a, b = tt.AdamW(views, state_bits=bits), tt.AdamW(params, state_bits=bits)
    kept = base.clone()
    for _ in range(2):
        a.step(list(grads))
        b.step([g.clone() for g in grads])
    assert all(torch.equal(x, y) for x, y in zip(views, params)) and all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))
    assert torch.equal(base[:1], kept[:1]) and torch.equal(base[701:2000], kept[701:2000]) and torch.equal(base[2640:], kept[2640:])


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_non_finite_gradients_stay_with_their_element(bits):
    params, grads = make([(1000,)], torch.float32, torch.float32)
    clean = [params[0].clone()]
    a, b = tt.AdamW(params, state_bits=bits), tt.AdamW(clean, state_bits=bits)
    bad = grads[0].clone()
    bad[10], bad[300], bad[999] = float("nan"), float("inf"), float("-inf")
    keep = torch.ones(1000, dtype=torch.bool, device="cuda")
    keep[[10, 300, 999]] = False
    ok = grads[0].clone()
    ok[~keep] = 0.0
    for _ in range(2):
        a.step([bad])
        b.step([ok])
    assert torch.equal(params[0][keep], clean[0][keep])
    assert bool((~params[0][~keep].isfinite()).all())
    for x, y in zip(a.moments(), b.moments()):
        assert torch.equal(a.split(x)[0][keep], b.split(y)[0][keep])


@pytest.mark.gpu
def test_skipped_gradients_mixed_types_and_autograd():
    w = torch.randn(64, 48, device="cuda", requires_grad=True)
    b = torch.randn(48, device="cuda").bfloat16().requires_grad_(True)
    frozen = torch.randn(100, device="cuda")
    opt = tt.AdamW([w, b, frozen], master_weights=True, state_bits=8, lr=0.1)
    was = frozen.clone(), w.detach().clone(), b.detach().clone()
    (w.sum() + b.float().square().sum()).backward()
    opt.step()
    assert torch.equal(frozen, was[0]) and not torch.equal(w, was[1]) and not torch.equal(b, was[2])
    assert opt.step_count() == 1
    opt.zero_grad()
    opt.step()                                     # no gradient at all: no step
    assert opt.step_count() == 1 and w.grad is None


@pytest.mark.gpu
def test_parameters_that_move_between_steps():
    w = torch.nn.Parameter(torch.randn(8, 8, device="cuda"))
    v = torch.nn.Parameter(torch.randn(5, device="cuda"))
    opt, plain = tt.AdamW([w, v]), [w.detach().clone(), v.detach().clone()]
    twin = tt.AdamW(plain)
    g = [torch.randn(8, 8, device="cuda"), torch.randn(5, device="cuda")]
    opt.step(g)
    twin.step(g)
    w.data = w.data.clone()                          # another place, the same shape: followed
    opt.step(g)
    twin.step(g)
    assert torch.equal(w, plain[0]) and torch.equal(v, plain[1])
    kept = w.data
    for moved in (torch.zeros(4, 8, device="cuda"), torch.zeros(8, 8), torch.zeros(8, 8, device="cuda").t()[:, ::2], kept.t()):
        w.data = moved
        with pytest.raises(ValueError, match="no longer"):
            opt.step(g)
    w.data = kept
    opt.step(g)
    twin.step(g)
    assert torch.equal(w, plain[0]) and opt.step_count() == 3
    sparse = torch.zeros(5, device="cuda").to_sparse()
    with pytest.raises((ValueError, RuntimeError)):
        opt.step([g[0], sparse])
    opt.step([None, g[1]])
    assert opt.step_count() == 4


@pytest.mark.gpu
def test_a_parameter_that_shrinks_in_place_is_refused():
    w, v = torch.nn.Parameter(torch.randn(8, 8, device="cuda")), torch.nn.Parameter(torch.randn(5, device="cuda"))
    opt, g = tt.AdamW([w, v]), [torch.randn(8, 8, device="cuda"), torch.randn(5, device="cuda")]
    opt.step(g)
    whole = w.data
    before = whole.clone()
    w.data = whole[:4]                               # the same address
    with pytest.raises(ValueError, match="no longer"):
        opt.step(g)
    assert torch.equal(whole, before) and opt.step_count() == 1


@pytest.mark.gpu
def test_a_backward_pass_that_needs_the_old_values_fails():
    w = torch.randn(32, device="cuda", requires_grad=True)
    opt = tt.AdamW([w])
    loss = (w * w).sum()
    opt.step([torch.ones(32, device="cuda")])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.gpu
@pytest.mark.parametrize("count", [41, 400, 401, 833])
def test_many_tensors(count):
    shapes = [(1 + 37 * i % 500,) for i in range(count)]
    params, grads = make(shapes, torch.float32, torch.float32)
    single = [p.clone() for p in params]
    opt = tt.AdamW(params)
    before = _lib.load().b200k_launch_count()
    opt.step(grads)
    assert _lib.load().b200k_launch_count() - before == -(-count // 400)
    opt.step(grads)
    for p, g in zip(single, grads):
        one = tt.AdamW([p])
        one.step([g])
        one.step([g])
    assert all(torch.equal(x, y) for x, y in zip(params, single)) and opt.step_count() == 2


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_on(bits):
    params, grads = make([(3000,), (17,)], torch.bfloat16, torch.float32)
    eager = [p.clone() for p in params]
    lr = torch.full((1,), 1e-2, device="cuda")
    scale = torch.ones(1, device="cuda")
    a = tt.AdamW(params, lr=lr, state_bits=bits, master_weights=True, seed=3)
    b = tt.AdamW(eager, lr=1e-2, state_bits=bits, master_weights=True, seed=3)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        a.step(grads, grad_scale=scale)
    for t in range(4):
        if t == 2:
            lr.fill_(5e-3)
            scale.fill_(0.5)
            b.lr = 5e-3
        graph.replay()
        b.step(grads, grad_scale=1.0 if t < 2 else 0.5)
    # lr = 1e-2 and 5e-3 as fp32 differ from the doubles by U: the update by 2 U of itself
    assert a.step_count() == b.step_count() == 4
    assert torch.allclose(a.master, b.master, rtol=4 * U, atol=4e-2 * 8 * U)
    if bits == 8:
        assert all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip_and_other_stream(bits):
    params, grads = make(SHAPES, torch.bfloat16, torch.bfloat16)
    copy = [p.clone() for p in params]
    a = tt.AdamW(params, state_bits=bits, master_weights=True)
    a.step(grads)
    b = tt.AdamW(copy, state_bits=bits, master_weights=True)
    held = a.state_dict()
    b.load_state_dict({k: v.cpu() if torch.is_tensor(v) else v for k, v in held.items()})
    for p, q in zip(copy, params):
        p.copy_(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step(grads)
    torch.cuda.current_stream().wait_stream(side)
    a.step(grads)
    assert all(torch.equal(x, y) for x, y in zip(params, copy)) and all(torch.equal(x, y) for x, y in zip(a.moments(), b.moments()))
    with pytest.raises(ValueError):
        b.load_state_dict({"step": 1})
    with pytest.raises(ValueError):
        b.load_state_dict({**held, "exp_avg": held["exp_avg"][:-1]})


@pytest.mark.gpu
def test_refusals_on_the_device():
    p = torch.zeros(8, 4, device="cuda")
    for params, kw, error in [([p, p], {}, ValueError), ([p, p[2:4]], {}, ValueError), ([p.t()], {}, ValueError), ([p, p.cpu()], {}, ValueError),
                              ([p.double()], {}, TypeError), ([p], dict(lr=-1.0), ValueError), ([p], dict(lr=torch.zeros(1)), ValueError),
                              ([p], dict(eps=-1e-9), ValueError), ([p], dict(weight_decay=float("nan")), ValueError)]:
        with pytest.raises(error):
            tt.AdamW(params, **kw)
    opt = tt.AdamW([p])
    for grads, error in [([], ValueError), ([torch.zeros(8, 5, device="cuda")], ValueError), ([torch.zeros(8, 4)], ValueError),
                         ([torch.zeros(8, 4, device="cuda").half()], TypeError)]:
        with pytest.raises(error):
            opt.step(grads)
    with pytest.raises(ValueError):
        opt.step([torch.zeros(8, 4, device="cuda")], grad_scale=torch.ones(2, device="cuda"))
    assert opt.step_count() == 0 and not bool(p.any())


def test_refusals():
    for params, kw, error in [([], {}, ValueError), ([torch.zeros(4)], {}, ValueError), ([torch.zeros(4)], dict(state_bits=4), ValueError),
                              ([torch.zeros(4)], dict(betas=(1.0, 0.9)), ValueError), ([torch.zeros(4, dtype=torch.int32)], {}, TypeError), (["x"], {}, TypeError)]:
        with pytest.raises(error):
            tt.AdamW(params, **kw)


def test_subnormal_eps_is_refused():
    with pytest.raises(ValueError, match="2\\^-126"):
        tt.AdamW([torch.zeros(4)], eps=1e-39)
    rows = np.zeros((1, 9), dtype=np.int64)
    assert _lib.load().b200k_adamw(rows.ctypes.data, 1, 0, 0, 32, 4096, 1e-3, None, 0.9, 0.999, 1e-39, 0.0, 1.0, None, 0, 1, None) == _lib.ERR_INVALID_ARG
    assert "2^-126" in _lib.last_error()


def test_entry_point_refusals():
    lib = _lib.load()
    rows = np.zeros((2, 9), dtype=np.int64)
    rows[:, [optim._P, optim._G, optim._M, optim._V]] = 4096
    rows[:, optim._N] = 10

    def call(rows=rows, n=2, dtype=0, gdtype=0, bits=32, state=4096, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0):
        return lib.b200k_adamw(rows.ctypes.data, n, dtype, gdtype, bits, state, lr, None, b1, b2, eps, wd, 1.0, None, 0, 1, None)

    def changed(column, value):
        r = rows.copy()
        r[1, column] = value
        return dict(rows=r)

    for bad in [dict(n=0), dict(dtype=3), dict(dtype=1, gdtype=2), dict(bits=16), dict(state=None), dict(state=4100), dict(b1=1.0), dict(b2=-0.1),
                dict(b1=float("nan")), dict(eps=-1.0), dict(wd=float("nan")), dict(lr=-1.0), changed(optim._N, 0), changed(optim._P, 0), changed(optim._G, 4097),
                changed(optim._M, 4100), changed(optim._V, 0), changed(optim._MASTER, 4096), dict(bits=8)]:
        assert call(**bad) == _lib.ERR_INVALID_ARG and "adamw" in _lib.last_error(), bad
    assert lib.b200k_adamw_moments(None, None, None, None, None, None, 0, None) == _lib.OK
    for blocks in (-1, 4):
        assert lib.b200k_adamw_moments(None, None, None, None, None, None, blocks, None) == _lib.ERR_INVALID_ARG
    assert ops._DTYPES[torch.bfloat16] == _lib.DTYPE_BF16


def plain_decode(codes, scales, bits):
    mag = (codes & ((1 << (4 + bits)) - 1)).to(torch.int32)
    value = ((mag << (23 - bits)) + (127 << 23)).view(torch.float32)
    value = torch.where(mag == 0, torch.zeros_like(value), value)
    value = torch.where((codes >= 128) & (bits == 3), -value, value)
    return (value.view(-1, BLOCK) * scales[:, None]).view(-1)


def plain_encode(x, random16, bits):
    mag = x.abs().view(-1, BLOCK)
    exponent = ((mag.amax(dim=1).view(torch.int32) + ((1 << (24 - bits)) - 1)) >> 23).clamp(min=16)
    scales, inverse = ((exponent - 15) << 23).view(torch.float32), ((269 - exponent) << 23).view(torch.float32)
    y = (mag * inverse[:, None]).view(-1)
    least = 1 + 2.0 ** -bits
    raw = (y.view(torch.int32) - (127 << 23) + (random16 << (7 - bits)).to(torch.int32)) >> (23 - bits)
    small = ((2 * random16 + 1).to(torch.float32) * (least * 2.0 ** -17) < y) if bits == 3 else y > 0
    code = torch.where(y < least, small.to(torch.int32), raw)
    return (torch.where(x < 0, code + 128, code) if bits == 3 else code).to(torch.uint8), scales


@pytest.mark.gpu
@pytest.mark.parametrize("spread,size", [(0.0, 1.0), (1.5, 1e-3), (3.0, 1e-8), (6.0, 1e8), (12.0, 1.0), (12.0, 1e-18)])
def test_8_bit_moments_equal_the_formula_in_ieee_fp32(spread, size):
    """Every product, sum and root that reaches a moment is one IEEE operation in the order of the formula, so that scales and codes (but for the
    sign of a zero) are equal, not near: nothing may be merged into a multiply-add, and the root is the correctly rounded one over the whole
    range of a squared gradient, subnormal and near-overflowing ones included."""
    n, steps = 1 << 21, 3
    g = torch.Generator(device="cuda").manual_seed(int(spread * 10))
    rn = lambda: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    opt = tt.AdamW([torch.zeros(n, device="cuda")], betas=(0.9, 0.999), state_bits=8, seed=9)
    m8 = r8 = torch.zeros(n, dtype=torch.uint8, device="cuda")
    ms = rs = torch.zeros(n // BLOCK, device="cuda")
    for t in range(1, steps + 1):
        grad = (rn() * torch.exp(rn() * spread) * size).clamp(-1e19, 1e19)
        grad[torch.rand(n, generator=g, device="cuda") < 0.05] = 0.0
        grad[: 4 * BLOCK] = 0.0
        opt.step([grad])
        m = plain_decode(m8, ms, 3) * 0.9 + grad * (1 - 0.9)
        r = plain_decode(r8, rs, 4)
        root = torch.sqrt(r * r * 0.999 + (grad * grad) * (1 - 0.999))
        lo, hi = (torch.from_numpy(x).cuda() for x in random16(n, 0, t, 9))
        m8, ms = plain_encode(m, lo, 3)
        r8, rs = plain_encode(root, hi, 4)
        held = opt.state_dict()
        assert torch.equal(held["exp_avg_scale"], ms) and torch.equal(held["exp_avg_sq_root_scale"], rs)
        assert torch.equal(held["exp_avg_sq_root"], r8)
        got = held["exp_avg"]
        assert bool(((got == m8) | ((got & 127 == 0) & (m8 & 127 == 0))).all())


def peak_encode(x, random16, bits):
    """Codes and scales by the rule scale = a block's peak / the largest code's value, for both moments with the same rounding below code 1."""
    top = (2.0 - 2.0 ** (1 - bits)) * 2.0 ** 15
    mag = x.abs().view(-1, BLOCK)
    peak = mag.amax(dim=1)
    tops = torch.full_like(peak, top)
    scales, inverse = peak / tops, torch.where(peak > 0, tops / peak, torch.zeros_like(peak))
    y = torch.minimum(mag * inverse[:, None], tops[:, None]).view(-1)
    least = 1 + 2.0 ** -bits
    raw = (y.view(torch.int32) - (127 << 23) + (random16 << (7 - bits)).to(torch.int32)) >> (23 - bits)
    small = (2 * random16 + 1).to(torch.float32) * (least * 2.0 ** -17) < y
    code = torch.where(y < least, small.to(torch.int32), raw)
    return (torch.where(x < 0, code + 128, code) if bits == 3 else code).to(torch.uint8), scales


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, False), (torch.float16, True)])
@pytest.mark.parametrize("spread,size", [(0.0, 1.0), (1.5, 1e-3), (6.0, 1e2), (1.5, 1e-18)])
def test_a_state_with_other_scales_goes_on_with_their_rule(spread, size, dtype, master):
    """Codes and scales equal to the formula in IEEE fp32, three steps after load_state_dict took over moments whose scales are the blocks' peaks / the
    largest code's value; then once more through state_dict.  (The sign of a zero is free.)"""
    n = (1 << 19) + 3
    padded = -(-n // BLOCK) * BLOCK
    g = torch.Generator(device="cuda").manual_seed(int(spread * 10))
    rn = lambda: torch.randn(n, generator=g, device="cuda") * torch.exp(torch.randn(n, generator=g, device="cuda") * spread)  # noqa: E731
    pad = lambda x: torch.nn.functional.pad(x, (0, padded - n))  # noqa: E731
    params = [(torch.randn(n, generator=g, device="cuda")).to(dtype)]
    opt = tt.AdamW(params, betas=(0.9, 0.999), state_bits=8, seed=9, master_weights=master)
    half_way = torch.full((padded,), 32768, dtype=torch.int64, device="cuda")
    live = torch.rand(padded, generator=g, device="cuda") < 0.95
    live[: 4 * BLOCK] = False
    m8, ms = peak_encode(pad(rn() * size * 0.1) * live, half_way, 3)
    r8, rs = peak_encode(pad(rn() * size).abs() * live, half_way, 4)
    held = opt.state_dict()
    held.update(step=70, exp_avg=m8, exp_avg_scale=ms, exp_avg_sq_root=r8, exp_avg_sq_root_scale=rs)
    opt.load_state_dict(held)
    for t in range(71, 75):
        if t == 74:
            opt.load_state_dict(opt.state_dict())
        grad = rn() * size
        grad[: 4 * BLOCK] = 0.0
        opt.step([grad.to(dtype) if dtype == torch.bfloat16 else grad])
        grad = pad((grad.to(dtype) if dtype == torch.bfloat16 else grad).float())
        m = plain_decode(m8, ms, 3) * 0.9 + grad * (1 - 0.9)
        r = plain_decode(r8, rs, 4)
        root = torch.sqrt(r * r * 0.999 + (grad * grad) * (1 - 0.999))
        lo, hi = (torch.from_numpy(x).cuda() for x in random16(padded, 0, t, 9))
        m8, ms = peak_encode(m, lo, 3)
        r8, rs = peak_encode(root, hi, 4)
        held = opt.state_dict()
        assert torch.equal(held["exp_avg_scale"], ms) and torch.equal(held["exp_avg_sq_root_scale"], rs)
        assert torch.equal(held["exp_avg_sq_root"], r8)
        got = held["exp_avg"]
        assert bool(((got == m8) | ((got & 127 == 0) & (m8 & 127 == 0))).all())


@pytest.mark.gpu
def test_peak_scales_of_tiny_and_non_finite_blocks():
    """Blocks whose peak has no finite inverse keep finite moments, within a step of their codes (1/8, of at least 2^-126), and a non-finite gradient stays with
    its element."""
    n = 4 * BLOCK
    opt = tt.AdamW([torch.zeros(n, device="cuda")], state_bits=8)
    m = torch.ones(n, device="cuda")
    m[BLOCK:2 * BLOCK] = torch.linspace(1e-36, 1e-34, BLOCK, device="cuda")
    m[2 * BLOCK:3 * BLOCK] = 0.0
    half_way = torch.full((n,), 32768, dtype=torch.int64, device="cuda")
    m8, ms = peak_encode(m, half_way, 3)
    m8[BLOCK:2 * BLOCK], ms[1] = 30, 1e-37
    held = opt.state_dict()
    held.update(exp_avg=m8, exp_avg_scale=ms)
    opt.load_state_dict(held)
    was = opt.moments()[0].clone()
    grad = torch.zeros(n, device="cuda")
    grad[2 * BLOCK + 5], grad[3 * BLOCK + 7] = float("nan"), float("inf")
    opt.step([grad])
    now = opt.moments()[0]
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[[2 * BLOCK + 5, 3 * BLOCK + 7]] = True
    assert bool((now.isnan() == bad).all()) and float(opt._ms[2]) == 0
    want = was * 0.9
    assert bool(((now - want).abs()[~bad] <= (want / 8 * 1.001 + 1.25 * 2.0 ** -126)[~bad]).all())


def test_state_bits_of_the_entry_point():
    rows = np.zeros((1, 9), dtype=np.int64)
    rows[:, [optim._P, optim._G, optim._M, optim._V]] = 4096
    rows[:, optim._N] = 10
    for bits in (256, 32 + _lib.ADAMW_PEAK_SCALES, 8 + 2 * _lib.ADAMW_PEAK_SCALES, 8 + _lib.ADAMW_PEAK_SCALES):      # the last one: null scales
        assert _lib.load().b200k_adamw(rows.ctypes.data, 1, 0, 0, bits, 4096, 1e-3, None, 0.9, 0.999, 1e-8, 0.0, 1.0, None, 0, 1, None) == _lib.ERR_INVALID_ARG
    assert "null pointer" in _lib.last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("bits,dtype,master", [(32, torch.float32, False), (8, torch.bfloat16, True), (8, torch.float32, False), (32, torch.float16, True)])
@pytest.mark.parametrize("how", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
def test_a_copied_optimiser_has_memory_of_its_own(bits, dtype, master, how):
    params, grads = make(SHAPES, dtype, dtype)
    a = tt.AdamW([torch.nn.Parameter(p) for p in params], state_bits=bits, master_weights=master, seed=4)
    a.step(grads)
    b = how(a)
    addresses = lambda o: {t.data_ptr() for t in (*o.params, o._m, o._v, o._ms, o._vs, o.master, o._state) if t is not None and t.numel()}  # noqa: E731
    assert not addresses(a) & addresses(b)
    own = {optim._M: (b._m, 1), optim._V: (b._v, 1), optim._MS: (b._ms, BLOCK), optim._VS: (b._vs, BLOCK), optim._MASTER: (b.master, 1)}
    for column, (t, per) in own.items():           # every address of the table lies in the copy's own buffers
        at = b._table[:, column]
        if t is None:
            assert not at.any()
        else:
            assert (at == t.data_ptr() + np.array(b.offsets) // per * t.element_size()).all()
    state = lambda o: [t.detach().clone() for t in (*o.params, *o.moments(), *([o.master] if master else []))]  # noqa: E731
    before = state(a)
    b.step(grads)
    assert all(torch.equal(x, y) for x, y in zip(before, state(a))) and a.step_count() == 1 and b.step_count() == 2
    after = state(b)
    a.step(grads)
    assert all(torch.equal(x, y) for x, y in zip(after, state(a))) and all(torch.equal(x, y) for x, y in zip(after, state(b)))
    del a
    b.step(grads)
    assert b.step_count() == 3


@pytest.mark.gpu
def test_a_module_copied_with_its_optimiser():
    layer = torch.nn.Linear(16, 8, device="cuda")
    opt = tt.AdamW(layer.parameters())
    layer2, opt2 = copy.deepcopy((layer, opt))
    assert all(p is q for p, q in zip(opt2.params, layer2.parameters()))
    x = torch.randn(4, 16, device="cuda")
    for net, o in ((layer, opt), (layer2, opt2)):
        net(x).square().sum().backward()
        o.step()
    assert all(torch.equal(p, q) for p, q in zip(layer.parameters(), layer2.parameters()))


@pytest.mark.gpu
def test_betas_cannot_be_changed_under_the_step_count():
    p = torch.zeros(8, device="cuda")
    opt = tt.AdamW([p], betas=(0.5, 0.75))
    with pytest.raises(AttributeError):
        opt.betas = (0.9, 0.999)
    assert opt.betas == (0.5, 0.75)
    opt.step([torch.ones(8, device="cuda")])
    m, v = opt.moments()
    assert bool((m[:8] == 0.5).all()) and bool((v[:8] == 0.25).all())


def walk(params, grads, shapes=None, device=0, dtype=0, count=None):
    """fill_rows over `params`; (its answer, the two columns that it fills)."""
    dims = np.array([n for s in (shapes or [p.shape for p in params]) for n in (len(s), *s)], dtype=np.int64)
    count = len(params) if count is None else count
    table = np.zeros((max(1, len(params)), 9), dtype=np.int64)
    return _lib.tensor_list().fill_rows(params, grads, count, dims.ctypes.data, table.ctypes.data, 9, device, dtype), table[:, :2]


def test_the_walk_over_host_tensors_and_wrong_lists_leaves_all_to_the_general_case():
    p = [torch.zeros(3), torch.zeros(2, 2)]
    for params, grads, kw in [(p, p, {}), (p, None, {}), (tuple(p), p, {}), (p, tuple(p), {}), (p, p[:1], {}), (p, [None, p[1]], {}), (["x", p[1]], p, dict(shapes=[(3,), (2, 2)])),
                              (p, p, dict(count=1)), (p, p, dict(count=3)), (p, p, dict(dtype=7)), ([], [], {})]:
        assert walk(params, grads, **kw)[0] == -1
    with pytest.raises(TypeError):
        _lib.tensor_list().fill_rows(p, p)
    with pytest.raises(TypeError):
        walk(p, p, device="cuda")


@pytest.mark.gpu
def test_the_walk_takes_only_what_fits():
    p = [torch.zeros(3, device="cuda"), torch.zeros(2, 2, device="cuda"), torch.zeros((), device="cuda")]
    g = [torch.ones_like(t) for t in p]
    at = p[0].get_device()
    got, columns = walk(p, g, device=at)
    assert got == 1 and columns.tolist() == [[x.data_ptr(), y.data_ptr()] for x, y in zip(p, g)]
    for x, y in zip(p, g):
        x.grad = y
    assert walk(p, None, device=at)[0] == 1 and (walk(p, None, device=at)[1] == columns).all()
    half = [t.bfloat16() for t in p]
    assert walk(half, [t.bfloat16() for t in g], device=at, dtype=1)[0] == 0 and walk(half, g, device=at, dtype=1)[0] == 1
    for i, wrong in [(0, g[0][:2]), (0, g[0].half()), (0, g[0].cpu()), (0, None), (1, g[1].view(4)), (1, torch.zeros(2, 4, device="cuda")[:, ::2]), (1, g[1].to_sparse()),
                     (2, g[2].view(1)), (1, torch.zeros(2, 2, device="meta"))]:
        assert walk(p, [wrong if k == i else t for k, t in enumerate(g)], device=at)[0] == -1, i
        if wrong is not None:
            assert walk([wrong if k == i else t for k, t in enumerate(p)], g, [t.shape for t in p], device=at)[0] == -1, i
    assert walk(half, [g[0], g[1].bfloat16(), g[2]], device=at, dtype=1)[0] == -1          # mixed gradients
    assert walk(p, g, device=at + 1)[0] == -1 and walk(p, g, device=at, dtype=1)[0] == -1
    p[1].grad = None
    assert walk(p, None, device=at)[0] == -1


@pytest.mark.gpu
def test_gradients_as_a_tuple_and_from_the_parameters_give_the_same_step():
    params, grads = make([(40, 3), (7,), (1,)], torch.float32, torch.float32)
    sets = [[torch.nn.Parameter(p.clone()) for p in params] for _ in range(3)]
    for p, g in zip(sets[2], grads):
        p.grad = g.clone()
    for ps, g in zip(sets, (grads, tuple(grads), None)):
        opt = tt.AdamW(ps)
        opt.step(g)
        opt.step(g)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(*sets))


@pytest.mark.gpu
def test_a_step_out_of_range_is_refused_before_anything_is_taken_over():
    opt = tt.AdamW([torch.zeros(8, device="cuda")])
    held = opt.state_dict()
    for step in (-1, 1 << 63):
        with pytest.raises(ValueError, match="step"):
            opt.load_state_dict({**held, "step": step, "exp_avg": torch.ones_like(held["exp_avg"])})
    assert opt.step_count() == 0 and not bool(opt.moments()[0].any())

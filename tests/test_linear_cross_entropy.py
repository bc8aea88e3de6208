"""Linear cross entropy, forward and backward, against its definition in 64 bits.

Tolerances (U = 2^-24).  A product's accumulator takes one partial sum per 16 elements of K and may lose 4 U of the sum of magnitudes with
each.  The logarithm of the sum of exponentials is off by the worst logit's error, 64 U for the sum and 4 U of itself; a probability by the errors
in its exponent.  dlogits are rounded to the operands' type (half a unit, in fp16 also half of the smallest step), dh and dw once more."""
import pytest
import torch

import triton_tenstorrent_b200 as tt
from triton_tenstorrent_b200 import _lib

U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16]


def half(t):
    return torch.finfo(t).eps / 2


def make(T, D, V, dtype, ignored=0.0, seed=0, spread=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn(T, D, generator=g, device="cuda").to(dtype)
    w = (torch.randn(V, D, generator=g, device="cuda") * spread / D ** 0.5).to(dtype)
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    y[torch.rand(T, generator=g, device="cuda") < ignored] = -100
    return h, w, y


def reference(h, w, y, d_losses, ignore=-100):
    """Values and tolerances in fp64: {"losses", "lse", "dh", "dw"}; d_losses: fp64 [T]."""
    dtype = h.dtype
    kept = torch.nonzero(y != ignore)[:, 0]
    hk, wd, yk, g = h[kept].double(), w.double(), y[kept], d_losses[kept][:, None]
    T, D, V = h.shape[0], h.shape[1], w.shape[0]
    rows = torch.arange(len(kept), device=h.device)
    logits = hk @ wd.t()
    tol_l = 4 * U * (D / 16 + 1) * (hk.abs() @ wd.abs().t())
    lse = torch.logsumexp(logits, 1)
    tol_lse = tol_l.amax(1) + 64 * U + 4 * U * lse.abs()
    out = {}

    def put(name, value, tol):
        full, full_tol = (torch.zeros((T, *value.shape[1:]), dtype=torch.float64, device=h.device) for _ in range(2))
        full[kept], full_tol[kept] = value, tol
        out[name] = (full, full_tol)

    put("lse", lse, tol_lse)
    put("losses", lse - logits[rows, yk], tol_lse + tol_l[rows, yk] + 4 * U * logits[rows, yk].abs())
    prob = torch.exp(logits - lse[:, None])
    tol_p = prob * (tol_l + tol_lse[:, None] + 8 * U * (1 + logits.abs() + lse[:, None].abs()))
    prob[rows, yk] -= 1
    dl = g * prob
    tol_dl = g.abs() * tol_p + (half(dtype) + 2 * U) * (dl.abs() + g.abs() * tol_p)
    if dtype == torch.float16:
        tol_dl = tol_dl + (g.abs().amax() if g.numel() else 0.0) * 2.0 ** -39
    del logits, tol_l, tol_p, prob
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-40

    def out_tol(value, tol, magnitude, k, other):
        # a dlogit below 2^-126 is subnormal, in fp32 and in bf16, and may count as zero
        tol = tol + 4 * U * (k / 16 + 40) * magnitude + 2.0 ** -126 * other.abs().sum(0)
        return tol + half(dtype) * (value.abs() + tol) + least

    dh = dl @ wd
    put("dh", dh, out_tol(dh, tol_dl @ wd.abs(), dl.abs() @ wd.abs(), V, wd))
    dw = dl.t() @ hk
    out["dw"] = (dw, out_tol(dw, tol_dl.t() @ hk.abs(), dl.abs().t() @ hk.abs(), T, hk))
    return out


def check(name, got, want):
    ref, tol = want
    assert got.shape == ref.shape and not bool(got.isnan().any()), name
    off = (got.double() - ref).abs() - tol
    assert off.numel() == 0 or float(off.max()) <= 0, f"{name}: {float(off.max())} over the bound, at {float((got.double() - ref).abs().max())}"


def poison():
    """Fills what the allocator will hand out as workspace with NaN."""
    for n in (1 << 10, 1 << 16, 1 << 20, 1 << 26):
        t = [torch.full((n,), float("nan"), device="cuda") for _ in range(3)]
        del t


def run_and_check(h, w, y, ignore=-100, seed=1):
    D = h.shape[-1]
    h2, y1 = h.reshape(-1, D), y.reshape(-1)
    T = h2.shape[0]
    g = torch.randn(T, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    poison()
    losses, lse = tt.linear_cross_entropy_with_lse(h, w, y, ignore)
    dh, dw = tt.linear_cross_entropy_backward(h, w, y, lse, g.view(y.shape), ignore)
    assert losses.shape == y.shape and losses.dtype == torch.float32 and dh.shape == h.shape and dh.dtype == h.dtype and dw.dtype == w.dtype
    want = reference(h2, w, y1, g.double(), ignore)
    check("losses", losses.reshape(-1), want["losses"])
    check("lse", lse.reshape(-1), want["lse"])
    check("dh", dh.reshape(-1, D), want["dh"])
    check("dw", dw, want["dw"])
    # the reduced forms: one gradient for all
    kept = (y1 != ignore)
    count = max(1, int(kept.sum()))
    for reduction, part in (("mean", 1 / count), ("sum", 1.0)):
        loss = tt.linear_cross_entropy(h, w, y, ignore, reduction)
        assert abs(float(loss) - float(want["losses"][0].sum()) * part) <= (float(want["losses"][1].sum()) + 4 * U * float(want["losses"][0].abs().sum())) * part + 1e-30
    if kept.any():
        scale = 0.375
        want = reference(h2, w, y1, torch.full((T,), scale / count, dtype=torch.float64, device="cuda"), ignore)
        dh, dw = tt.linear_cross_entropy_backward(h, w, y, lse, torch.tensor(scale, device="cuda"), ignore, "mean")
        check("dh", dh.reshape(-1, D), want["dh"])
        check("dw", dw, want["dw"])
    assert tt.device_status() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V", [(1, 8, 1), (1, 64, 300), (2, 64, 256), (5, 72, 255), (33, 64, 257), (128, 128, 128), (130, 136, 1000), (257, 520, 777), (700, 96, 5001),
                                   (300, 64, 40003), (2500, 256, 3001), (1, 4096, 20011), (64, 1024, 19000)])
def test_matches_the_definition(T, D, V, dtype):
    run_and_check(*make(T, D, V, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,D,V,ignored", [(1, 64, 100, 1.0), (40, 64, 500, 0.5), (300, 64, 500, 0.97), (1000, 128, 777, 0.3), (515, 64, 300, 1.0), (2048, 64, 1000, 0.9)])
def test_ignored_tokens(T, D, V, ignored, dtype):
    h, w, y = make(T, D, V, dtype, ignored)
    h[y == -100] = float("nan")                    # what stands there does not matter
    run_and_check(h, w, y)


@pytest.mark.gpu
@pytest.mark.parametrize("T,D,V", [(8192, 64, 40001), (70000, 8, 4501)])
def test_several_pieces_of_the_vocabulary(T, D, V):
    assert 2 * T * V > 512 << 20
    h, w, y = make(T, D, V, torch.bfloat16, 0.1)
    run_and_check(h, w, y)


@pytest.mark.gpu
def test_strides_shapes_and_other_ignore_index():
    h, w, y = make(60, 136, 333, torch.bfloat16)
    y[::7] = 5
    run_and_check(h.view(4, 15, 136), w, y.view(4, 15), ignore=5)
    run_and_check(h[:, :128], w[:, 8:], y)                                   # row pitches above D
    run_and_check(h[:, 1:129], w[:, 3:131], y)                               # off 16-byte boundaries: copied
    run_and_check(h.t().contiguous().t(), w.t().contiguous().t(), y)
    run_and_check(h[:1].expand(60, 136), w, y)                               # the same row again and again
    run_and_check(h[::2], w[::3], y[::2] % 111)
    run_and_check(h[0], w, y[0])                                             # a single token without a token dimension
    h, w, y = make(5, 64, 100, torch.float16)
    run_and_check(h[:0], w, y[:0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits_and_confident_tokens(dtype):
    h, w, y = make(200, 64, 600, dtype, spread=100.0)                        # logits of hundreds: exp overflows without the maximum
    y[:100] = (h[:100].double() @ w.double().t()).argmax(1)
    run_and_check(h, w, y)


@pytest.mark.gpu
def test_infinite_weights_and_wrong_targets():
    h, w, y = make(40, 64, 300, torch.bfloat16)
    h = h.abs()
    clean = tt.linear_cross_entropy(h, w[:299], y % 299, reduction="none")
    w[299] = float("-inf")                                                   # an entry that cannot occur
    got = tt.linear_cross_entropy(h, w, y % 299, reduction="none")
    assert torch.allclose(got, clean, rtol=1e-6, atol=1e-5)
    h, w, y = make(40, 64, 300, torch.float16)
    good = tt.linear_cross_entropy(h, w, y, reduction="none")
    for bad in (300, -1, -101, 2 ** 40, -2 ** 62):
        y2 = y.clone()
        y2[7] = bad
        losses = tt.linear_cross_entropy(h, w, y2, reduction="none")
        keep = torch.arange(40, device="cuda") != 7
        assert bool(losses[7].isnan()) and torch.equal(losses[keep], good[keep]) and bool(tt.linear_cross_entropy(h, w, y2).isnan())
        lse = tt.linear_cross_entropy_with_lse(h, w, y2)[1]
        dh, dw = tt.linear_cross_entropy_backward(h, w, y2, lse, torch.ones((), device="cuda"), reduction="mean")
        assert bool(dh[7].isnan().all()) and not bool(dh[keep].isnan().any()) and bool(dw.isnan().all())
    h[3] = float("nan")                                                      # NaN in a token that counts stays in its row
    losses = tt.linear_cross_entropy(h, w, y, reduction="none")
    keep = torch.arange(40, device="cuda") != 3
    assert bool(losses[3].isnan()) and torch.equal(losses[keep], good[keep])


@pytest.mark.gpu
def test_gradients_of_very_different_size():
    h, w, y = make(300, 64, 500, torch.float16)
    g = torch.randn(300, device="cuda") * 10.0 ** torch.linspace(-6, 4, 300, device="cuda")
    lse = tt.linear_cross_entropy_with_lse(h, w, y)[1]
    dh, dw = tt.linear_cross_entropy_backward(h, w, y, lse, g)
    want = reference(h, w, y, g.double())
    fine = want["dh"][0].abs() < 60000
    check("dh", torch.where(fine, dh, torch.zeros_like(dh)), (torch.where(fine, want["dh"][0], 0.0), want["dh"][1]))
    fine = want["dw"][0].abs() < 60000
    check("dw", torch.where(fine, dw, torch.zeros_like(dw)), (torch.where(fine, want["dw"][0], 0.0), want["dw"][1]))
    dh, dw = tt.linear_cross_entropy_backward(h, w, y, lse, torch.zeros(300, device="cuda"))
    assert not bool(dh.any()) and not bool(dw.any())


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_autograd_against_the_formula_and_differences(reduction):
    h, w, y = make(48, 64, 120, torch.bfloat16, 0.2)
    g = torch.randn(48, device="cuda") if reduction == "none" else torch.tensor(1.75, device="cuda")
    hl, wl = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = tt.linear_cross_entropy(hl.view(6, 8, 64), wl, y.view(6, 8), reduction=reduction)
    loss.backward(g.view(6, 8) if reduction == "none" else g)
    lse = tt.linear_cross_entropy_with_lse(h, w, y)[1]
    dh, dw = tt.linear_cross_entropy_backward(h, w, y, lse, g, reduction=reduction)
    assert torch.equal(hl.grad, dh) and torch.equal(wl.grad, dw)
    only_h = tt.linear_cross_entropy_backward(h, w, y, lse, g, reduction=reduction, need_dw=False)
    only_w = tt.linear_cross_entropy_backward(h, w, y, lse, g, reduction=reduction, need_dh=False)
    assert torch.equal(only_h[0], dh) and only_h[1] is None and only_w[0] is None and torch.equal(only_w[1], dw)

    kept = y != -100
    count = int(kept.sum())

    def f(h, w):
        logits = h @ w.t()
        each = (torch.logsumexp(logits, 1) - logits.gather(1, y.clamp(min=0)[:, None])[:, 0]) * kept
        return float((each * g.double()).sum() / (count if reduction == "mean" else 1))

    rnd = torch.Generator(device="cuda").manual_seed(4)
    for k, (leaf, grad) in enumerate(((h, dh), (w, dw))):
        d = torch.randn(leaf.shape, generator=rnd, device="cuda", dtype=torch.float64)
        step = 1e-5
        args = [h.double(), w.double()]
        hi, lo = ([a + s * step * d if i == k else a for i, a in enumerate(args)] for s in (1, -1))
        slope = (f(*hi) - f(*lo)) / (2 * step)
        # every element of the gradient is off by three roundings of bf16 at most (dlogits' of each of its terms, bounded by the norms, and its own)
        bound = 3 * half(torch.bfloat16) * float((grad.double() * d).abs().sum()) + 1e-6 * (1 + abs(slope))
        assert abs(float((grad.double() * d).sum()) - slope) <= bound


@pytest.mark.gpu
def test_broadcast_gradient_and_frozen_leaves():
    h, w, y = make(30, 64, 90, torch.float16)
    h.requires_grad_(True)
    tt.linear_cross_entropy(h, w, y, reduction="none").sum().backward()     # an expanded gradient
    a = h.grad.clone()
    h.grad = None
    tt.linear_cross_entropy(h, w, y, reduction="sum").backward()
    assert torch.equal(a, h.grad) and w.grad is None
    assert not tt.linear_cross_entropy(h.detach(), w, y).requires_grad


@pytest.mark.gpu
def test_other_stream_graphs_and_determinism():
    h, w, y = make(400, 128, 3001, torch.bfloat16, 0.3)
    one = torch.ones((), device="cuda")

    def both():
        losses, lse = tt.linear_cross_entropy_with_lse(h, w, y)
        return (losses, lse, tt.linear_cross_entropy(h, w, y), *tt.linear_cross_entropy_backward(h, w, y, lse, one, reduction="mean"))

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):                                  # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both())
        graphs.append(graph)
    for _ in range(2):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for out in outs for p, q in zip(want, out))
    y.copy_(torch.where(y == -100, 7, torch.where(y % 2 == 0, -100, y)))    # other tokens count now, another number of them
    for graph in graphs:
        graph.replay()
    want = both()
    assert all(torch.equal(p, q) for out in outs for p, q in zip(want, out))


@pytest.mark.gpu
def test_host_tensors():
    h, w, y = (t.cpu() for t in make(20, 64, 50, torch.bfloat16))
    h.requires_grad_(True)
    loss = tt.linear_cross_entropy(h, w, y)
    loss.backward()
    assert not loss.is_cuda and not h.grad.is_cuda
    want = torch.nn.functional.cross_entropy(h.detach().float() @ w.float().t(), y)
    assert abs(float(loss.detach()) - float(want)) < 1e-5


def test_refusals():
    h, w, y = torch.zeros(4, 16).bfloat16(), torch.zeros(10, 16).bfloat16(), torch.zeros(4, dtype=torch.int64)
    for bad, error in [(dict(h=h.float()), TypeError), (dict(weight=w.half()), TypeError), (dict(targets=y.int()), TypeError), (dict(targets=y[:3]), ValueError),
                       (dict(weight=w[:, :8]), ValueError), (dict(weight=w[:0]), ValueError), (dict(h=h[:, :12], weight=w[:, :12]), ValueError),
                       (dict(weight=w[0]), ValueError), (dict(reduction="max"), ValueError), (dict(h=h[:, :0], weight=w[:, :0]), ValueError)]:
        with pytest.raises(error):
            tt.linear_cross_entropy(**{"h": h, "weight": w, "targets": y, **bad})
    lse = torch.zeros(4)
    for args, kw in [((h, w, y, lse.double(), lse), {}), ((h, w, y, lse[:3], lse), {}), ((h, w, y, lse, lse[:2]), {}), ((h, w, y, lse, lse), dict(reduction="mean")),
                     ((h, w, y, lse, lse.bfloat16()), {})]:
        with pytest.raises(ValueError):
            tt.linear_cross_entropy_backward(*args, **kw)


def test_sizes_beyond_the_entry_points_integers_are_refused():
    row, wide, one = torch.zeros(1, 8).bfloat16(), torch.zeros(1, 1).bfloat16(), torch.zeros(1, dtype=torch.int64)
    many = (1 << 32) + 5                                  # 5 in 32 bits
    for bad in [dict(h=row.expand(many, 8), targets=one.expand(many)), dict(weight=row.expand(many, 8)), dict(h=wide.expand(1, 1 << 32), weight=wide.expand(1, 1 << 32)),
                dict(ignore_index=1 << 63)]:
        with pytest.raises(ValueError, match="at most 2|int64"):
            tt.linear_cross_entropy(**{"h": row, "weight": row, "targets": one, **bad})
    assert _lib.load().b200k_lce_fwd(256, 256, 256, 256, 256, 256, 256, 1 << 40, 4, (1 << 30) + 8, 4, (1 << 30) + 8, (1 << 30) + 8, -100, 0, 1, None) == _lib.ERR_INVALID_ARG


def test_entry_point_refusals():
    lib = _lib.load()
    assert lib.b200k_lce_workspace(0, 64, 10, 0) == 0
    size = {b: lib.b200k_lce_workspace(64, 64, 1000, b) for b in (0, 1)}
    # no logits: far below T V values for a large vocabulary, and at most 512 MiB of dlogits in the backward
    assert lib.b200k_lce_workspace(8192, 64, 1 << 20, 1) < (513 << 20) + 8 * 8192 * 64
    for backward in (0, 1):
        def call(h=256, w=256, y=256, lse=256, other=256, work=256, size=size[backward], T=64, D=64, V=1000, ldh=64, ldw=64, red=1, dt=1):
            if backward:
                return lib.b200k_lce_bwd(h, w, y, lse, other, 256, 256, work, size, T, D, V, ldh, ldw, -100, red, dt, None)
            return lib.b200k_lce_fwd(h, w, y, 256, lse, other, work, size, T, D, V, ldh, ldw, -100, red, dt, None)
        for bad in [dict(h=None), dict(w=None), dict(y=None), dict(lse=None), dict(other=None), dict(work=None), dict(work=264), dict(size=size[backward] - 1), dict(T=-1),
                    dict(D=0), dict(D=60), dict(V=0), dict(ldh=56), dict(ldw=68), dict(h=264), dict(red=3), dict(red=-1), dict(dt=0), dict(dt=3), dict(V=2 ** 30 + 1)]:
            assert call(**bad) == _lib.ERR_INVALID_ARG and "linear_cross_entropy" in _lib.last_error(), (backward, bad)


def exactly(h, w, y):
    """(lse, losses) of exactly representable logits in 64 bits, and the tolerance of either: no product or sum of a logit is rounded, so that what is left is the
    sum of exponentials (64 U) and four roundings of lse and of the target's logit (its product with log2 e, that constant, the sum, the way back)."""
    logits = h.double() @ w.double().t()
    lse = torch.logsumexp(logits, 1)
    hit = logits.gather(1, y[:, None])[:, 0]
    return lse, lse - hit, 64 * U + 4 * U * (lse.abs() + hit.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [5, 128, 200, 700])
@pytest.mark.parametrize("D", [512, 4096, 8192])
def test_exactly_representable_logits(T, D, dtype):
    """Sums that are exact at every step must come out exact, whatever D: small whole numbers, a single feature that counts, features that end early,
    large parts that cancel, and a row that is one feature."""
    g = torch.Generator(device="cuda").manual_seed(D)
    V = 777
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    whole = lambda *s: torch.randint(-3, 4, s, generator=g, device="cuda").to(dtype)  # noqa: E731
    cases = [(whole(T, D), whole(V, D))]
    h, w = torch.ones(T, D, device="cuda", dtype=dtype), torch.zeros(V, D, device="cuda", dtype=dtype)
    w[:, 0] = torch.randint(-60, 61, (V,), generator=g, device="cuda").to(dtype)
    cases.append((h, w))                                                     # all at the first step, then zeros
    w = torch.zeros_like(w)
    w[:, :40] = 2 * whole(V, 40)
    cases.append((whole(T, D), w))                                           # padded columns
    w = torch.zeros_like(w)
    w[:, 3], w[:, D // 2 + 1], w[:, D - 1] = 240.0, -240.0, whole(V)         # parts that cancel
    cases.append((h, w))
    one = torch.zeros_like(h)
    one[torch.arange(T), torch.randint(0, D, (T,), generator=g, device="cuda")] = 1.0
    cases.append((one, 32 * whole(V, D)))                                    # a row that is one feature
    for h, w in cases:
        lse, losses = tt.linear_cross_entropy_with_lse(h, w, y)[::-1]
        want_lse, want, tol = exactly(h, w, y)
        assert bool(((lse.double() - want_lse).abs() <= tol).all()), float(((lse.double() - want_lse).abs() - tol).max())
        assert bool(((losses.double() - want).abs() <= tol).all()), float(((losses.double() - want).abs() - tol).max())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [100, 600])
def test_the_error_of_a_logit_does_not_grow_with_its_length(T):
    """Sums of growing size: a part of 512 loses at most 4 U of its own sum with each of its 32 steps of 16, and adding the D / 512 parts rounds to nearest, so that a
    logit is off by (128 + D / 512) U of its sum of magnitudes, whatever D.  A loss of one entry is the logit's difference to lse, both off by that."""
    D = 16384
    g = torch.Generator(device="cuda").manual_seed(2)
    h, w = (torch.rand(T, D, generator=g, device="cuda") / 8).bfloat16(), (torch.rand(300, D, generator=g, device="cuda") / 8).bfloat16()
    y = torch.randint(0, 300, (T,), generator=g, device="cuda")
    losses, lse = tt.linear_cross_entropy_with_lse(h, w, y)
    want_lse, want, tol = exactly(h, w, y)
    tol = tol + (128 + D / 512) * U * (h.double() @ w.double().t()).amax(1)
    assert bool(((lse.double() - want_lse).abs() <= tol).all())
    assert bool(((losses.double() - want).abs() <= 2 * tol).all())

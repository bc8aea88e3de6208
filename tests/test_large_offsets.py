"""Tensors whose element offsets pass 31 and byte offsets 32 bits: norm, linear cross entropy and AdamW give what they give for the same
numbers in a small tensor, bit for bit (their sums' order depends on the sizes of the call alone)."""
import pytest
import torch

import triton_tenstorrent_b200 as tt

pytestmark = pytest.mark.gpu


def far_rows(t, pitch):
    """t's rows, `pitch` elements apart."""
    room = torch.empty((t.shape[0] - 1) * pitch + t.shape[1], device="cuda", dtype=t.dtype)
    view = room.as_strided(t.shape, (pitch, 1))
    view.copy_(t)
    return view


@pytest.mark.parametrize("cols,pitch", [(200, 1 << 30), (1000, (1 << 30) + 1), (1000, 1 << 30), (20001, 1 << 30)])
def test_layer_norm_rows_far_apart(cols, pitch):
    torch.manual_seed(0)
    x, dy, w, b = (torch.randn(*s, device="cuda").bfloat16() for s in [(4, cols), (4, cols), (cols,), (cols,)])
    y, mean, rstd = tt.layer_norm_with_stats(x, w, b)
    dx, dw, db = tt.layer_norm_backward(dy, x, w, mean, rstd)
    far = far_rows(x, pitch)
    y2, mean2, rstd2 = tt.layer_norm_with_stats(far, w, b)
    # an odd pitch takes narrower accesses, whose sums run in another order: each is within a few units of 2^-24 of the other, so that a rounded
    # result differs by one unit (2^-7 of it) where it differs, and sums of 4 rows in fp32 round to values one unit apart too
    same = torch.equal if pitch % 8 == 0 else lambda p, q: torch.allclose(p.float(), q.float(), rtol=2 ** -7, atol=1e-5)
    assert same(y2, y) and same(mean2, mean) and same(rstd2, rstd)
    dx2, dw2, db2 = tt.layer_norm_backward(dy, far, w, mean, rstd)
    assert same(dx2, dx) and same(dw2, dw) and same(db2, db)
    dx2, dw2, db2 = tt.layer_norm_backward(far_rows(dy, pitch), x, w, mean, rstd)
    assert same(dx2, dx) and same(dw2, dw) and same(db2, db)


@pytest.mark.parametrize("T", [9, 300])
def test_linear_cross_entropy_far_rows(T):
    torch.manual_seed(0)
    D, V = 64, 9
    h, w = torch.randn(T, D, device="cuda").bfloat16(), torch.randn(V, D, device="cuda").bfloat16()
    y = torch.randint(0, V, (T,), device="cuda")
    g = torch.rand(T, device="cuda")
    losses, lse = tt.linear_cross_entropy_with_lse(h, w, y)
    dh, dw = tt.linear_cross_entropy_backward(h, w, y, lse, g)
    h2 = far_rows(h, (1 << 32) // T // 8 * 8 + 8)
    w2 = far_rows(w, 1 << 29)
    losses2, lse2 = tt.linear_cross_entropy_with_lse(h2, w2, y)
    assert torch.equal(losses2, losses) and torch.equal(lse2, lse)
    dh2, dw2 = tt.linear_cross_entropy_backward(h2, w2, y, lse, g)
    assert torch.equal(dh2, dh) and torch.equal(dw2, dw)


def test_linear_cross_entropy_large_weight():
    """W of more than 2^31 elements: the last entries' dW, and dh, when all probability lies on the last entries (the others' logits are 0
    beside 60, which leaves e^-60 each)."""
    torch.manual_seed(0)
    T, D, V = 16, 8192, (1 << 18) + 300
    w = torch.zeros(V, D, device="cuda", dtype=torch.bfloat16)
    h = (1 + torch.arange(T * D, device="cuda").view(T, D) % 2).bfloat16()
    w[-64:, 0] = 60
    h[:, 0] = 1
    y = torch.randint(V - 64, V, (T,), device="cuda")
    g = torch.ones(T, device="cuda")
    losses, lse = tt.linear_cross_entropy_with_lse(h, w, y)
    want = 60 + torch.log(torch.tensor(64.0))
    # a sum of 8192 products is truncated 512 times, by up to 2^-25 of it each; lse itself is rounded a few times
    assert torch.allclose(lse.cpu(), want.expand(T), rtol=512 * 2 ** -25 + 2 ** -21, atol=0)
    dh, dw = tt.linear_cross_entropy_backward(h, w, y, lse, g)
    # dlogits = 1 / 64 - [v = y], each rounded to bf16 (2^-8 of it) once, dW and dh rounded once more; the cancelling terms of dh are 64 of 1 / 64
    # against 1, the roundings of which weigh 60 * 2 * 2^-8
    dl = torch.full((T, 64), 1 / 64, dtype=torch.float64)
    dl[torch.arange(T), (y - (V - 64)).cpu()] -= 1
    ref = dl.t() @ h.double().cpu()
    bound = 2 ** -8 * (dl.abs().t() @ h.double().abs().cpu()) + 2 ** -8 * ref.abs() + 1e-4
    assert bool(((dw[-64:].double().cpu() - ref).abs() <= bound).all())
    assert float(dw[:1000].float().abs().max()) < 1e-20 and float(dw[1 << 17:(1 << 17) + 1000].float().abs().max()) < 1e-20
    assert float(dh[:, 0].float().abs().max()) <= 60 * 2 * 2 ** -8 and not bool(dh[:, 1:].any())


def test_adamw_more_than_2_to_31_elements():
    torch.manual_seed(0)
    n, tail = (1 << 31) + 5000, 9096                  # the tail begins on a block of 256 and spans the 2^31st element
    p, g = (torch.zeros(n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    p[-tail:], g[-tail:] = torch.randn(tail, device="cuda").bfloat16(), torch.randn(tail, device="cuda").bfloat16()
    small, opt = p[-tail:].clone(), tt.AdamW([p])
    twin = tt.AdamW([small])
    for _ in range(2):
        opt.step([g])
        twin.step([g[-tail:].clone()])
    assert torch.equal(p[-tail:], small) and not bool(p[:n - tail].any())
    for a, b in zip(opt.moments(), twin.moments()):
        assert torch.equal(a[n - tail:n], b[:tail])


def test_adamw_8_bit_more_than_2_to_31_elements():
    """Zero gradients but for the tail, whose moments the first step sets to (1 - b1) g and (1 - b2) g^2, to within a step of their codes (2^-3, and
    2^-4 of the root)."""
    torch.manual_seed(0)
    n, tail = (1 << 31) + 5000, 9096
    p, g = (torch.zeros(n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    g[-tail:] = (1 + torch.rand(tail, device="cuda")).bfloat16()
    opt = tt.AdamW([p], state_bits=8)
    opt.step([g])
    want = g[-tail:].float()
    flat, codes = opt._m[n - tail:n], opt._v[n - tail:n]
    assert bool((flat > 0).all()) and bool((codes > 0).all()) and not bool(opt._m[:n - tail].any()) and not bool(opt._v[:n - tail].any())
    small = tt.AdamW([torch.zeros(tail, device="cuda", dtype=torch.bfloat16)], state_bits=8)
    small._m[:tail], small._v[:tail] = flat, codes
    at = (n - tail) // 256
    blocks = small._ms.numel()
    small._ms.copy_(opt._ms[at:at + blocks])
    small._vs.copy_(opt._vs[at:at + blocks])
    m, v = (t[:tail] for t in small.moments())
    assert bool(((m - 0.1 * want).abs() <= 0.1 * want * 2 ** -3 * 1.001).all())
    assert bool(((v.sqrt() - 0.001 ** 0.5 * want).abs() <= 0.001 ** 0.5 * want * 2 ** -4 * 1.001).all())

"""Forward-mode derivatives: the differentiable operators have none, and refuse dual tensors instead of returning a result without a tangent."""
import pytest
import torch
from torch.autograd import forward_ad

import triton_tenstorrent_b200 as tt


def calls(device, dual):
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g).bfloat16().to(device)  # noqa: E731
    x, w, b, head, q = rn(4, 64), rn(64), rn(64), rn(16, 64), rn(1, 1, 128, 64)
    y = torch.arange(4).to(device)
    lse = torch.zeros(4).to(device)
    return [lambda: tt.layer_norm(dual(x), w, b), lambda: tt.layer_norm(x, dual(w)), lambda: tt.layer_norm(x, w, dual(b)), lambda: tt.layer_norm_with_stats(dual(x)),
            lambda: tt.layer_norm_backward(dual(x), x, w, lse, lse + 1), lambda: tt.linear_cross_entropy(dual(x), head, y),
            lambda: tt.linear_cross_entropy(x, dual(head), y), lambda: tt.linear_cross_entropy_with_lse(dual(x), head, y),
            lambda: tt.linear_cross_entropy(dual(x.clone().requires_grad_(True)), head, y), lambda: tt.attention(q, dual(q), q, True, 0.125)]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_dual_tensors_are_refused(device):
    with forward_ad.dual_level():
        for call in calls(device, lambda t: forward_ad.make_dual(t, torch.ones_like(t))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.gpu
def test_tensors_without_a_tangent_pass_inside_a_dual_level():
    want = [call() for call in calls("cuda", lambda t: t)]
    with forward_ad.dual_level():
        got = [call() for call in calls("cuda", lambda t: t)]
    flat = lambda rs: [t for r in rs for t in (r if isinstance(r, tuple) else (r,))]  # noqa: E731
    assert all(torch.equal(p, q) for p, q in zip(flat(want), flat(got)))

"""The operators of a training step together, as a user's program puts them: norm -> attention -> residual -> norm -> linear cross entropy -> backward
-> AdamW, against the same step in 64-bit torch operations.

Rounding: h, the attention's operands and results, and the gradients that flow between the operators are bf16, half a unit of 2^-8 each.  About ten
such roundings lie between the loss and the first parameters, so that a gradient's relative error (in the 2-norm; roundings of different
elements are independent) stays below 10 * 2^-8 = 0.04, and the loss, an average over the tokens, below 2^-8 of itself."""
import pytest
import torch

import triton_tenstorrent_b200 as tt

Z, S, H, D, V = 2, 200, 4, 64, 1003          # a length that is no multiple of a tile, an odd vocabulary
C = H * D


def build(seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    p = {"embed": rn(V, C) * 0.5, "norm1.w": 1 + 0.1 * rn(C), "norm1.b": 0.1 * rn(C), "norm2.w": 1 + 0.1 * rn(C), "norm2.b": 0.1 * rn(C), "head": rn(V, C) * 0.08}
    p = {k: (v if "norm" in k else v.bfloat16()).requires_grad_(True) for k, v in p.items()}
    tokens = torch.randint(0, V, (Z, S), generator=g, device="cuda")
    targets = torch.randint(0, V, (Z, S), generator=g, device="cuda")
    targets[0, :60] = -100                    # a prompt without loss
    targets[1, 150:] = -100                   # padding
    return p, tokens, targets


def heads(x):
    return x.view(Z, S, H, D).transpose(1, 2)


def forward(p, tokens, targets):
    x = p["embed"][tokens]
    n = heads(tt.layer_norm(x, p["norm1.w"], p["norm1.b"])).contiguous()
    a = tt.attention(n, n, n, True, D ** -0.5)
    x = x + a.transpose(1, 2).reshape(Z, S, C)
    return tt.linear_cross_entropy(tt.layer_norm(x, p["norm2.w"], p["norm2.b"]), p["head"], targets)


def exact(p, tokens, targets):
    def norm(x, w, b):
        c = x - x.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    x = p["embed"][tokens]
    n = heads(norm(x, p["norm1.w"], p["norm1.b"]))
    score = n @ n.transpose(-1, -2) * D ** -0.5
    score = score.masked_fill(torch.ones(S, S, dtype=torch.bool, device="cuda").triu(1), float("-inf"))
    x = x + (torch.softmax(score, -1) @ n).transpose(1, 2).reshape(Z, S, C)
    logits = norm(x, p["norm2.w"], p["norm2.b"]) @ p["head"].t()
    return torch.nn.functional.cross_entropy(logits.view(-1, V), targets.view(-1), ignore_index=-100)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_training_step(bits):
    p, tokens, targets = build()
    loss = forward(p, tokens, targets)
    loss.backward()
    q = {k: v.detach().double().requires_grad_(True) for k, v in p.items()}
    want = exact(q, tokens, targets)
    want.backward()
    assert abs(float(loss.detach()) - float(want.detach())) <= 2.0 ** -8 * float(want.detach())
    for k in p:
        assert p[k].grad.dtype == p[k].dtype
        assert float((p[k].grad.double() - q[k].grad).norm()) <= 0.04 * float(q[k].grad.norm()), k
    # the update, from the same gradients: the first step moves every parameter by lr g / (|g| + eps)
    before = {k: v.detach().clone() for k, v in p.items()}
    opt = tt.AdamW(list(p.values()), lr=1e-2, weight_decay=0.1, master_weights=True, state_bits=bits)
    opt.step()
    for master, k in zip(opt.split(opt.master), p):
        g, old = p[k].grad.double(), before[k].double()
        new = old * (1 - 1e-3) - 1e-2 * g / (g.abs() + 1e-8)
        got = p[k].detach().double() if p[k].dtype == torch.float32 else master.double()
        # fp32: a few units of the parameter and of the update, whose bias corrections cancel to within 2^-24 / (1 - beta2)
        assert float((got - new).abs().max()) <= 2.0 ** -22 * float(old.abs().max()) + 1e-2 * 2.0 ** -13
    assert tt.device_status() == 0 and opt.step_count() == 1
    opt.zero_grad()
    after = forward(p, tokens, targets)
    assert bool(after.isfinite())


@pytest.mark.gpu
def test_step_replayed_from_a_graph():
    """Gradients and update captured into one graph: every replay is a step of its own."""
    p, tokens, targets = build(1)
    leaves = list(p.values())
    q, _, _ = build(1)
    opts = [tt.AdamW(list(x.values()), lr=1e-2, state_bits=8, master_weights=True) for x in (p, q)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):            # one eager pass on the capturing stream: allocations and first-use lookups
        torch.autograd.grad(forward(p, tokens, targets), leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        loss = forward(p, tokens, targets)
        opts[0].step(torch.autograd.grad(loss, leaves))
    for _ in range(3):
        graph.replay()
    for _ in range(3):
        eager = forward(q, tokens, targets)
        opts[1].step(torch.autograd.grad(eager, list(q.values())))
    torch.cuda.synchronize()
    assert opts[0].step_count() == opts[1].step_count() == 3
    # torch's gradient of the embedding lookup adds with atomics, in an order of its own: equal up to that
    assert abs(float(loss.detach()) - float(eager.detach())) <= 1e-3 * float(eager.detach())
    for name in p:
        if name != "embed":
            assert float((p[name].detach().float() - q[name].detach().float()).norm()) <= 0.02 * float(q[name].detach().float().norm())
    assert tt.device_status() == 0

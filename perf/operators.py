"""Workloads of the operators that a training step needs next to attention and the matrix products: layer norm with its
gradients, the cross entropy of a linear output layer with its gradients, and the AdamW step over a list of tensors.

Each case is a dict of plain values.  `own` selects the framework's kernels; otherwise the same results are computed from
elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
IGNORE = -100
BLOCK = 256          # elements that share a scale in the 8-bit optimiser states


# ---------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------
def norm_case(name, direction, rows, cols, dtype, weight):
    return {"name": name, "op": "layer_norm", "direction": direction, "rows": rows, "cols": cols, "dtype": dtype, "weight": weight}


def loss_case(name, direction, tokens, dim, vocab, dtype, ignored):
    return {"name": name, "op": "linear_cross_entropy", "direction": direction, "tokens": tokens, "dim": dim, "vocab": vocab,
            "dtype": dtype, "ignored": ignored}


def adam_case(name, width, layers, extra, dtype, grad, bits, master):
    return {"name": name, "op": "adamw", "width": width, "layers": layers, "extra": extra, "dtype": dtype, "grad": grad, "bits": bits,
            "master": master}


def listed():
    return [
        # one token of a decoder that generates text: latency
        norm_case("norm one token", "forward", 1, 4096, "bf16", "bf16"),
        # the activations of a prompt batch, normalised on the way into a matmul
        norm_case("norm prompt", "forward", 16384, 4096, "bf16", "bf16"),
        # a training step's norm, forward and backward, weights kept in 32 bits
        norm_case("norm training", "training", 8192, 8192, "bf16", "fp32"),
        # an odd row length and row count in 32 bits
        norm_case("norm odd fp32", "training", 5003, 1537, "fp32", "fp32"),
        # scoring a short answer against a mid-sized vocabulary
        loss_case("loss scoring", "forward", 61, 1024, 32000, "fp16", 0.0),
        # scoring a long document, every token's loss
        loss_case("loss document", "forward", 4096, 2048, 65536, "bf16", 0.0),
        # fine-tuning: the prompt's tokens carry no loss; an odd vocabulary
        loss_case("loss fine-tuning", "training", 2047, 2048, 49999, "fp16", 0.4),
        # pre-training: every token carries a loss
        loss_case("loss pre-training", "training", 8192, 4096, 128000, "bf16", 0.0),
        # the optimiser of a small network: launch latency
        adam_case("adamw small", 64, 2, 1000, "fp32", "fp32", 32, False),
        # 32-bit states and parameters
        adam_case("adamw 32-bit states", 1024, 12, 32000 * 1024, "fp32", "fp32", 32, False),
        # 8-bit states, 16-bit parameters updated in place
        adam_case("adamw 8-bit states", 1536, 12, 32001 * 1536, "bf16", "bf16", 8, False),
        # 8-bit states, 32-bit master copies behind 16-bit parameters
        adam_case("adamw 8-bit master", 1000, 8, 7919 * 1000, "bf16", "fp32", 8, True),
    ]


def log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "linear_cross_entropy", "adamw"])
    if op == "layer_norm":
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        cols = log_int(rng, 64, 16384)
        rows = log_int(rng, 1, max(1, min(32768, (1 << 26) // cols)))
        c = norm_case("", rng.choice(["forward", "training"]), rows, cols, dtype, rng.choice([dtype, "fp32"]))
    elif op == "linear_cross_entropy":
        dim = 8 * log_int(rng, 16, 512)
        vocab = log_int(rng, 500, 128000)
        tokens = log_int(rng, 1, max(1, min(16384, int(2.0e12 / (dim * vocab)))))
        c = loss_case("", rng.choice(["forward", "training"]), tokens, dim, vocab, rng.choice(["bf16", "fp16"]), rng.choice([0.0, 0.1, 0.7]))
    else:
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        width = log_int(rng, 32, 1536)
        grad = rng.choice([dtype, "fp32"])
        c = adam_case("", width, rng.randint(1, 12), log_int(rng, 1, 1 << 25), dtype, grad, rng.choice([32, 8]), dtype != "fp32" and rng.random() < 0.5)
    del c["name"]
    return c


def shapes(case):
    """The parameter shapes of a decoder with two norms, four attention projections and a two-layer feed-forward part in each layer, and
    one tensor of `extra` elements (its embedding)."""
    w = case["width"]
    layer = [(w,), (w,), (w, w), (w, w), (w, w), (w, w), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
    return [(case["extra"],)] + layer * case["layers"]


def offsets(sizes):
    """Where each tensor begins in a flat buffer whose tensors start at multiples of BLOCK elements, and the buffer's length."""
    at, total = [], 0
    for n in sizes:
        at.append(total)
        total += -(-n // BLOCK) * BLOCK
    return at, total


# ---------------------------------------------------------------------------------------------
# The 8-bit states: BLOCK consecutive elements share a 32-bit scale; a code has 4 exponent bits and 3 (first moment, with a sign) or 4 (root
# of the second moment) mantissa bits, value(c) = (1 + mantissa / 2^bits) * 2^exponent, value(0) = 0; the largest code is left to NaN.
# Rounding is stochastic, with 16 random bits that a hash draws from (seed, step, tensor, element).
# ---------------------------------------------------------------------------------------------
def code_values(bits):
    c = torch.arange(1 << (4 + bits), dtype=torch.float64)
    v = (1 + torch.remainder(c, 1 << bits) / (1 << bits)) * torch.exp2(torch.floor(c / (1 << bits)))
    v[0] = 0.0
    return v


def top_value(bits):
    return (2.0 - 2.0 ** (1 - bits)) * 2.0 ** 15


def mix(x):
    """32-bit hash of whole numbers held in 64 bits."""
    x = x & 0xFFFFFFFF
    x = x ^ (x >> 16)
    x = (x * 0xDDB3D743) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0xB504F335) & 0xFFFFFFFF
    return x ^ (x >> 16)


def salts(count, seed, step):
    """One 32-bit salt per tensor of the list."""
    base = mix(torch.tensor((seed + step * 0x9E3779B9) & 0xFFFFFFFF, dtype=torch.int64))
    return mix(base + torch.arange(count, dtype=torch.int64))


def decode(codes, scales, bits):
    mag = (codes & ((1 << (4 + bits)) - 1)).to(torch.int32)
    value = ((mag << (23 - bits)) + (127 << 23)).view(torch.float32)
    value = torch.where(mag == 0, torch.zeros_like(value), value)
    if bits == 3:
        value = torch.where(codes >= 128, -value, value)
    return (value.view(-1, BLOCK) * scales[:, None]).view(-1)


def encode(x, random16, bits):
    """Codes and scales of finite x >= 0 (root of the second moment) or of any sign (first moment)."""
    mag = x.abs().view(-1, BLOCK)
    top = torch.full_like(mag[:, 0], top_value(bits))
    peak = mag.amax(dim=1)
    scales = peak / top
    inverse = torch.where(peak > 0, top / peak, torch.zeros_like(peak))
    y = torch.minimum(mag * inverse[:, None], top[:, None]).view(-1)
    least = 1 + 2.0 ** -bits
    raw = (y.view(torch.int32) - (127 << 23) + (random16 << (7 - bits)).to(torch.int32)) >> (23 - bits)
    small = ((2 * random16 + 1).to(torch.float32) * (least * 2.0 ** -17) < y).to(torch.int32)
    code = torch.where(y < least, small, raw)
    if bits == 3:
        code = torch.where(x < 0, code + 128, code)
    return code.to(torch.uint8), scales


# ---------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*size, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(*size, generator=g, device=dev) * scale + shift).to(dtype)

    s = {"case": case}
    if case["op"] == "layer_norm":
        t, wt = DTYPES[case["dtype"]], DTYPES[case["weight"]]
        rows, cols = case["rows"], case["cols"]
        s["x"] = randn(rows, cols, dtype=t, scale=1.5, shift=0.3)
        s["w"] = randn(cols, dtype=wt, scale=0.2, shift=1.0)
        s["b"] = randn(cols, dtype=wt, scale=0.2)
        s["dy"] = randn(rows, cols, dtype=t) if case["direction"] == "training" else None
    elif case["op"] == "linear_cross_entropy":
        t = DTYPES[case["dtype"]]
        T, D, V = case["tokens"], case["dim"], case["vocab"]
        s["h"] = randn(T, D, dtype=t)
        s["w"] = randn(V, D, dtype=t, scale=2.0 / math.sqrt(D))     # logits of about N(0, 4)
        y = torch.randint(0, V, (T,), generator=g, device=dev)
        masked = torch.rand(T, generator=g, device=dev) < case["ignored"]
        s["y"] = torch.where(masked, torch.full_like(y, IGNORE), y)
        if case["direction"] == "training":
            s["h"].requires_grad_(True)
            s["w"].requires_grad_(True)
    else:
        sh = shapes(case)
        sizes = [math.prod(x) for x in sh]
        at, total = offsets(sizes)
        t, gt = DTYPES[case["dtype"]], DTYPES[case["grad"]]
        live = torch.zeros(total, dtype=torch.bool, device=dev)
        for a, n in zip(at, sizes):
            live[a:a + n] = True
        p32 = randn(total, scale=0.05) * live
        s["p"] = p32.to(t)
        # gradients whose size differs from element to element by factors of ten, as between the rows of an embedding
        s["g"] = (randn(total) * torch.exp(randn(total, scale=1.5)) * 1e-3 * live).to(gt)
        m = randn(total, scale=3e-4) * torch.exp(randn(total)) * live
        v = (torch.exp(randn(total, scale=1.5)) * 1e-3 * live).square()
        s["master"] = p32 if case["master"] else None
        s["step"] = 1 + seed % 1000      # steps taken so far
        s["seed"] = 7 + seed % 3
        if case["bits"] == 8:
            zero = torch.zeros(total, dtype=torch.int64, device=dev)
            s["m"], s["ms"] = encode(m, zero + 32768, 3)
            s["r"], s["rs"] = encode(v.sqrt(), zero + 32768, 4)
        else:
            s["m"], s["v"] = m, v
        blocks = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor([-(-n // BLOCK) for n in sizes])).to(dev)
        s["tensor_of_block"] = blocks
        s["first"] = torch.tensor(at, device=dev)
        s["hyper"] = dict(lr=3e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
        if own:
            from triton_tenstorrent_b200 import AdamW

            views = [s["p"][a:a + n].view(x) for a, n, x in zip(at, sizes, sh)]
            s["grads"] = [s["g"][a:a + n].view(x) for a, n, x in zip(at, sizes, sh)]
            opt = AdamW(views, state_bits=case["bits"], master_weights=case["master"], seed=s["seed"], **s["hyper"])
            held = {"step": s["step"], "exp_avg": s["m"]}
            held.update({"exp_avg_scale": s["ms"], "exp_avg_sq_root": s["r"], "exp_avg_sq_root_scale": s["rs"]} if case["bits"] == 8 else {"exp_avg_sq": s["v"]})
            if case["master"]:
                held["master"] = p32
            opt.load_state_dict(held)
            s["opt"] = opt
    return s


# ---------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------
def run(s):
    return {"layer_norm": run_norm, "linear_cross_entropy": run_loss, "adamw": run_adamw}[s["case"]["op"]](s)


def run_norm(s):
    x, w, b, dy, eps = s["x"], s["w"], s["b"], s["dy"], 1e-5
    if own:
        import triton_tenstorrent_b200 as tt

        if dy is None:
            return tt.layer_norm(x, w, b, eps)
        y, mean, rstd = tt.layer_norm_with_stats(x, w, b, eps)
        dx, dw, db = tt.layer_norm_backward(dy, x, w, mean, rstd)
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    xf, wf = x.float(), w.float()
    centred = xf - xf.mean(dim=1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(dim=1, keepdim=True) + eps)
    hat = centred * rstd
    y = (hat * wf + b.float()).to(x.dtype)
    if dy is None:
        return y
    df = dy.float()
    u = df * wf
    dx = rstd * (u - u.mean(dim=1, keepdim=True) - hat * (u * hat).mean(dim=1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dw": (df * hat).sum(dim=0).to(w.dtype), "db": df.sum(dim=0).to(w.dtype)}


def run_loss(s):
    h, w, y = s["h"], s["w"], s["y"]
    training = s["case"]["direction"] == "training"
    if own:
        import triton_tenstorrent_b200 as tt

        if not training:
            return tt.linear_cross_entropy(h, w, y, ignore_index=IGNORE, reduction="none")
        loss = tt.linear_cross_entropy(h, w, y, ignore_index=IGNORE)
        dh, dw = torch.autograd.grad(loss, (h, w))
        return {"loss": loss.detach(), "dh": dh, "dw": dw}
    h, w = h.detach(), w.detach()
    valid = y != IGNORE
    target = torch.where(valid, y, torch.zeros_like(y))[:, None]
    hf, wf = torch.where(valid[:, None], h.float(), torch.zeros((), device=h.device)), w.float()
    logits = hf @ wf.t()
    peak = logits.amax(dim=1, keepdim=True)
    weight = torch.exp(logits - peak)
    total = weight.sum(dim=1, keepdim=True)
    losses = torch.where(valid, (torch.log(total) + peak - logits.gather(1, target))[:, 0], torch.zeros((), device=h.device))
    if not training:
        return losses
    count = valid.sum().clamp(min=1).float()
    loss = losses.sum() / count
    del logits
    weight /= total
    weight.scatter_add_(1, target, -torch.ones_like(total))
    weight *= (valid.float() / count)[:, None]
    return {"loss": loss, "dh": (weight @ wf).to(h.dtype), "dw": (weight.t() @ hf).to(w.dtype)}


def run_adamw(s):
    case = s["case"]
    if own:
        opt = s["opt"]
        opt.step(s["grads"])
        m, v = opt.moments()
        return {"p": s["p"], "m": m, "v": v, **({"master": opt.master} if case["master"] else {})}
    hy = s["hyper"]
    lr, (b1, b2), eps, wd = hy["lr"], hy["betas"], hy["eps"], hy["weight_decay"]
    s["step"] += 1
    step = s["step"]
    p = s["master"] if case["master"] else s["p"].float()
    g = s["g"].float()
    if case["bits"] == 8:
        m = decode(s["m"], s["ms"], 3)
        r = decode(s["r"], s["rs"], 4)
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    root = torch.sqrt(v)
    p = p * (1 - lr * wd) - (m / (root * (1 / math.sqrt(1 - b2 ** step)) + eps)) * (lr / (1 - b1 ** step))
    if case["master"]:
        s["master"].copy_(p)
    s["p"].copy_(p)
    if case["bits"] == 8:
        salt = salts(s["first"].numel(), s["seed"], step).to(p.device)
        within = torch.arange(p.numel(), device=p.device).view(-1, BLOCK) - s["first"][s["tensor_of_block"]][:, None]
        h = mix(within + salt[s["tensor_of_block"]][:, None]).view(-1)
        s["m"], s["ms"] = encode(m, h & 0xFFFF, 3)
        s["r"], s["rs"] = encode(root, h >> 16, 4)
        m = decode(s["m"], s["ms"], 3)
        r = decode(s["r"], s["rs"], 4)
        v = r * r
    else:
        s["m"], s["v"] = m, v
    return {"p": s["p"], "m": m, "v": v, **({"master": s["master"]} if case["master"] else {})}


# ---------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "layer_norm":
        n, c = case["rows"] * case["cols"], case["cols"]
        e, we = SIZE[case["dtype"]], SIZE[case["weight"]]
        if case["direction"] == "forward":
            return {"bytes": 2 * n * e + 2 * c * we, "flops": 8 * n}
        return {"bytes": 4 * n * e + 4 * c * we, "flops": 20 * n}
    if case["op"] == "linear_cross_entropy":
        T, D, V, e = case["tokens"], case["dim"], case["vocab"], SIZE[case["dtype"]]
        kept = T * (1 - case["ignored"])
        once = (T + V) * D * e + 8 * T
        if case["direction"] == "forward":
            return {"bytes": once + 4 * T, "flops": 2 * kept * D * V}
        return {"bytes": 2 * once, "flops": 6 * kept * D * V}
    n = sum(math.prod(x) for x in shapes(case))
    state = 2 * 8 if case["bits"] == 32 else 2 * (2 + 8 / BLOCK) + 8      # read and written; the 8-bit states also returned as values
    return {"bytes": n * (2 * SIZE[case["dtype"]] + SIZE[case["grad"]] + state + (8 if case["master"] else 0) - (SIZE[case["dtype"]] if case["master"] else 0)), "flops": 20 * n}


# ---------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        x, w, b = s["x"].double(), s["w"].double(), s["b"].double()
        n = x.shape[1]
        mean = x.sum(1, keepdim=True) / n
        sigma = torch.sqrt(((x - mean) ** 2).sum(1, keepdim=True) / n + 1e-5)
        xh = (x - mean) / sigma
        if s["dy"] is None:
            return xh * w + b
        dy = s["dy"].double()
        dxh = dy * w
        dx = (n * dxh - dxh.sum(1, keepdim=True) - xh * (dxh * xh).sum(1, keepdim=True)) / (n * sigma)
        return {"y": xh * w + b, "dx": dx, "dw": (dy * xh).sum(0), "db": dy.sum(0)}
    if case["op"] == "linear_cross_entropy":
        h, w, y = s["h"].detach().double(), s["w"].detach().double(), s["y"]
        kept = torch.nonzero(y >= 0)[:, 0]
        hk, yk = h[kept], y[kept]
        logits = hk @ w.t()
        lse = torch.logsumexp(logits, 1)
        rows = torch.arange(len(kept), device=h.device)
        each = lse - logits[rows, yk]
        if case["direction"] == "forward":
            out = torch.zeros(h.shape[0], dtype=torch.float64, device=h.device)
            out[kept] = each
            return out
        count = max(1, len(kept))
        logits -= lse[:, None]
        prob = logits.exp_()
        prob[rows, yk] -= 1
        prob /= count
        dh = torch.zeros_like(h)
        dh[kept] = prob @ w
        return {"loss": each.sum() / count, "dh": dh, "dw": prob.t() @ hk}
    hy, t = s["hyper"], s["step"] + 1
    (b1, b2), lr = hy["betas"], hy["lr"]
    g = s["g"].double()
    if case["bits"] == 8:
        values3, values4 = code_values(3).to(g.device), code_values(4).to(g.device)
        per = torch.arange(g.numel(), device=g.device) // BLOCK
        c = s["m"].long()
        m = torch.where(c > 127, -1.0, 1.0).double() * values3[c & 127] * s["ms"].double()[per]
        v = (values4[s["r"].long()] * s["rs"].double()[per]) ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    old = (s["master"] if case["master"] else s["p"]).double()
    p = old - lr * hy["weight_decay"] * old - lr * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + hy["eps"])
    # a stochastically rounded state is one of two neighbours, which of them turns on the last bit next to a border: no value in 64 bits
    states = {"m": None, "v": None} if case["bits"] == 8 else {"m": m, "v": v}
    return {"p": p, **states, **({"master": p} if case["master"] else {})}

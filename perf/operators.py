"""Work of the gated feed-forward block and of its 8-bit activation checkpoints, as cases that can be timed and checked.

A case names an operator and its sizes; `prepare` makes what a user's program holds before the call, `run` is one
pass through the operator, `work` its bytes and operations, `exact` its result in 64 bits.  With `own` true, `run`
calls the package's operators; otherwise it evaluates the same formulas with elementary torch operations.

  act    x -> 8-bit codes and one power-of-two scale per 1 x 128 block (saved in the forward pass), and back
  ffn    h = f(x Wg^T) * (x Wu^T)
  bwd    the gradients of x, Wg and Wu from dh and the 8-bit checkpoints of x, g = x Wg^T and u = x Wu^T
  step   a training step's share of the block: save x, forward with checkpoints, backward
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ACTS = ("silu", "gelu", "gelu_tanh", "relu")
BLOCK = 128


def listed():
    return [
        # the activations of a few sequences that are decoded together: launch latency counts
        {"name": "act 16x4096 bf16", "op": "act", "rows": 16, "cols": 4096, "pad": 0, "dtype": "bf16"},
        # the activations of a large training batch
        {"name": "act 65536x4096 bf16", "op": "act", "rows": 65536, "cols": 4096, "pad": 0, "dtype": "bf16"},
        # an odd width whose last block is short, rows that are a slice of a wider matrix
        {"name": "act 4099x5461 fp16 slice", "op": "act", "rows": 4099, "cols": 5461, "pad": 11, "dtype": "fp16"},
        # full-precision activations (norms, router inputs) of a mid-sized batch
        {"name": "act 4096x8192 fp32", "op": "act", "rows": 4096, "cols": 8192, "pad": 0, "dtype": "fp32"},
        # one token of one sequence: the weights are read once, nothing else matters
        {"name": "ffn 1 token bf16", "op": "ffn", "m": 1, "k": 4096, "f": 14336, "act": "silu", "dtype": "bf16"},
        # sixteen sequences decoded together
        {"name": "ffn 16 tokens fp16", "op": "ffn", "m": 16, "k": 4096, "f": 14336, "act": "gelu", "dtype": "fp16"},
        # a large decoding batch or a short prompt, ragged
        {"name": "ffn 125 tokens bf16", "op": "ffn", "m": 125, "k": 4096, "f": 14336, "act": "silu", "dtype": "bf16"},
        # a long prompt
        {"name": "ffn 4096 tokens bf16", "op": "ffn", "m": 4096, "k": 4096, "f": 14336, "act": "silu", "dtype": "bf16"},
        # a fine-tuning batch of few tokens: the gradients of the weights are most of what is written
        {"name": "bwd 500 tokens bf16", "op": "bwd", "m": 500, "k": 4096, "f": 14336, "act": "silu", "dtype": "bf16"},
        # a training batch
        {"name": "bwd 8192 tokens bf16", "op": "bwd", "m": 8192, "k": 4096, "f": 14336, "act": "silu", "dtype": "bf16"},
        # a small model with an odd hidden width and an odd number of tokens
        {"name": "step 1023 tokens fp16 odd", "op": "step", "m": 1023, "k": 1048, "f": 2731, "act": "gelu_tanh", "dtype": "fp16"},
        # a training step of a larger model
        {"name": "step 4096 tokens bf16", "op": "step", "m": 4096, "k": 4096, "f": 14336, "act": "silu", "dtype": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("act", "ffn", "ffn", "bwd", "step"))
    if op == "act":
        cols = _spread(rng, 100, 16384)
        rows = _spread(rng, 1, max(1, 65536 * 4096 // cols))
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        if dtype == "fp32":
            rows = max(1, rows // 2)
        return {"op": op, "rows": rows, "cols": cols, "pad": rng.choice((0, 0, 8, 3)), "dtype": dtype}
    k = 8 * _spread(rng, 64, 1024)
    f = _spread(rng, 512, 28672)
    most = {"ffn": 4096, "bwd": 8192, "step": 4096}[op] * 4096 * 14336 // (k * f)
    m = _spread(rng, 1, max(1, min(most, 16384)))
    return {"op": op, "m": m, "k": k, "f": f, "act": rng.choice(ACTS), "dtype": rng.choice(("bf16", "fp16"))}


# ---- plain forms: elementary operations in 32 bits, rounded once -----------------------------------


def plain_save(x):
    """Codes (e4m3) and scales (fp32, a power of two) of each 1 x 128 block: the smallest 2^e >= 2^-126 with
    amax <= 448 * 2^e over the block's finite values, 1 for a block of zeros; infinities and NaN are stored as NaN."""
    x = x.float()
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    xb = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).view(rows, blocks, BLOCK)
    amax = torch.where(torch.isfinite(xb), xb.abs(), torch.zeros_like(xb)).amax(dim=2)
    part, power = torch.frexp(amax)                                        # amax = part * 2^power, 448 = 0.875 * 2^9
    e = (power + (part > 0.875).to(power.dtype) - 9).clamp(min=-126)
    e = torch.where(amax > 0, e, torch.zeros_like(e))
    scale = ((e + 127) << 23).to(torch.int32).view(torch.float32)
    back = ((127 - e) << 23).to(torch.int32).view(torch.float32)
    codes = (xb * back[:, :, None]).to(torch.float8_e4m3fn).view(rows, blocks * BLOCK)[:, :cols]
    return codes.contiguous(), scale


def plain_restore(codes, scale, dtype):
    """codes * scale; what would round beyond the type's largest value takes that value."""
    rows, cols = codes.shape
    y = codes.float() * scale.repeat_interleave(BLOCK, dim=1)[:, :cols]
    top = torch.finfo(dtype).max
    return y.clamp(-top, top).to(dtype)


def plain_act(g, act):
    """f(g) and f'(g)."""
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if act == "gelu":
        p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * p, p + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        a, b = math.sqrt(2.0 / math.pi), 0.044715
        t = torch.tanh(a * (g + b * g * g * g))
        return 0.5 * g * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * g * (1.0 - t * t) * a * (1.0 + 3.0 * b * g * g)
    return g.clamp(min=0), (g > 0).to(g.dtype)


def plain_ffn(x, wg, wu, act):
    """h, and the two projections."""
    x32 = x.float()
    g, u = x32 @ wg.float().t(), x32 @ wu.float().t()
    return (plain_act(g, act)[0] * u).to(x.dtype), g, u


def plain_bwd(dh, wg, wu, xq, xs, gq, gs, uq, us, act):
    x, g, u = (plain_restore(q, s, torch.float32) for q, s in ((xq, xs), (gq, gs), (uq, us)))
    a, da = plain_act(g, act)
    dh = dh.float()
    dg, du = dh * u * da, dh * a
    dx = dg @ wg.float() + du @ wu.float()
    return tuple(t.to(wg.dtype) for t in (dx, dg.t() @ x, du.t() @ x))


# ---- cases -----------------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, rows, cols, scale, dtype):
    return (torch.randn(rows, cols, generator=gen, device="cuda") * scale).to(dtype)


def _inputs(case, seed):
    gen, dtype = _gen(seed), DTYPES[case["dtype"]]
    if case["op"] == "act":
        # rows of very different size, as the residual stream has them, and channels that stand out
        wide = torch.randn(case["rows"], case["cols"] + case["pad"], generator=gen, device="cuda")
        wide *= torch.exp(torch.randn(case["rows"], 1, generator=gen, device="cuda"))
        wide[:, :: 257] *= 30.0
        return {"x": wide.to(dtype)[:, :case["cols"]], "dtype": dtype}
    m, k, f = case["m"], case["k"], case["f"]
    s = {"act": case["act"]}
    s["wg"], s["wu"] = (_normal(gen, f, k, k ** -0.5, dtype) for _ in range(2))
    x = _normal(gen, m, k, 1.0, dtype)
    if case["op"] != "bwd":
        s["x"] = x
    if case["op"] != "ffn":
        s["dh"] = _normal(gen, m, f, 0.1, dtype)
    if case["op"] == "bwd":
        s["xq"], s["xs"] = plain_save(x)
        s["gq"], s["gs"] = plain_save(_normal(gen, m, f, 1.0, torch.float32))
        s["uq"], s["us"] = plain_save(_normal(gen, m, f, 1.0, torch.float32))
    return s


def prepare(case, seed):
    return {"op": case["op"], **_inputs(case, seed)}


def run(s):
    if own:
        from tilebench_b200.benchmarks.layers.act_checkpoint_fp8 import impl_cuda as save
        from tilebench_b200.benchmarks.layers.act_restore_fp8 import impl_cuda as restore
        from tilebench_b200.benchmarks.layers.ffn_gated import impl_cuda as ffn
        from tilebench_b200.benchmarks.layers.ffn_gated_bwd import impl_cuda as bwd
        if s["op"] == "act":
            q, scale = save.run(s["x"])
            return restore.run(q, scale, s["dtype"]), scale
        if s["op"] == "ffn":
            return ffn.run(s["x"], s["wg"], s["wu"], s["act"])
        if s["op"] == "bwd":
            return bwd.run(s["dh"], s["wg"], s["wu"], s["xq"], s["xs"], s["gq"], s["gs"], s["uq"], s["us"], s["act"])
        xq, xs = save.run(s["x"])
        h, gq, gs, uq, us = ffn.run(s["x"], s["wg"], s["wu"], s["act"], checkpoint=True)
        return (h, *bwd.run(s["dh"], s["wg"], s["wu"], xq, xs, gq, gs, uq, us, s["act"]))
    if s["op"] == "act":
        q, scale = plain_save(s["x"])
        return plain_restore(q, scale, s["dtype"]), scale
    if s["op"] == "ffn":
        return plain_ffn(s["x"], s["wg"], s["wu"], s["act"])[0]
    if s["op"] == "bwd":
        return plain_bwd(s["dh"], s["wg"], s["wu"], s["xq"], s["xs"], s["gq"], s["gs"], s["uq"], s["us"], s["act"])
    h, g, u = plain_ffn(s["x"], s["wg"], s["wu"], s["act"])
    return (h, *plain_bwd(s["dh"], s["wg"], s["wu"], *plain_save(s["x"]), *plain_save(g), *plain_save(u), s["act"]))


def work(case):
    if case["op"] == "act":
        n, size = case["rows"] * case["cols"], DTYPES[case["dtype"]].itemsize
        scales = case["rows"] * -(-case["cols"] // BLOCK) * 4
        # saving reads x and writes the codes and scales, restoring reads those and writes x
        return {"bytes": 2 * n * (size + 1) + 2 * scales, "flops": 4 * n}
    m, k, f = case["m"], case["k"], case["f"]
    weights, x, hidden = 2 * 2 * f * k, m * k, m * f
    if case["op"] == "ffn":
        return {"bytes": weights + 2 * x + 2 * hidden, "flops": 4 * m * k * f}
    if case["op"] == "bwd":
        scales = 4 * m * (-(-k // BLOCK) + 2 * -(-f // BLOCK))
        return {"bytes": 2 * weights + 3 * x + 4 * hidden + scales, "flops": 8 * m * k * f}
    return {"bytes": 2 * weights + 4 * x + 4 * hidden, "flops": 12 * m * k * f}


# ---- the definition in 64 bits ---------------------------------------------------------------------


def _stored(x):
    """(values that the 8-bit codes stand for, scales) in 64 bits, by the spacing of the code's numbers."""
    x = x.double()
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    of = torch.arange(cols, device=x.device) // BLOCK
    size = torch.where(torch.isfinite(x), x.abs(), x.new_zeros(()))
    amax = x.new_zeros(rows, blocks).scatter_reduce(1, of.expand(rows, cols), size, "amax")
    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -140) / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= amax, e - 1, e)           # the logarithm may be off at a power of two
    e = torch.where(448.0 * torch.exp2(e) < amax, e + 1, e).clamp(min=-126)
    scale = torch.where(amax > 0, torch.exp2(e), torch.ones_like(e))
    y = x / scale[:, of]
    # normal codes have three bits after the leading one, below 2^-6 the spacing stays 2^-9
    spacing = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    y = torch.round(y / spacing) * spacing
    y = torch.where(torch.isfinite(x), y, torch.full_like(y, math.nan))
    return y * scale[:, of], scale


def _top(v, dtype):
    return v.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max)


def _act64(g, act):
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if act == "gelu":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        z = math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)
        s = torch.sigmoid(2 * z)                                             # (1 + tanh z) / 2
        return g * s, s + g * 2 * s * (1 - s) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * g ** 2)
    return torch.relu(g), torch.heaviside(g, g.new_zeros(()))


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "act":
        value, scale = _stored(s["x"])
        return _top(value, s["dtype"]), scale
    wg, wu = s["wg"].double(), s["wu"].double()
    h = None
    if case["op"] == "bwd":
        def held(q, scale):
            of = torch.arange(q.shape[1], device=q.device) // BLOCK
            return q.to(torch.float64) * scale.double()[:, of]
        x, g, u = held(s["xq"], s["xs"]), held(s["gq"], s["gs"]), held(s["uq"], s["us"])
    else:
        x = s["x"].double()
        g, u = torch.einsum("mk,fk->mf", x, wg), torch.einsum("mk,fk->mf", x, wu)
        h = _act64(g, case["act"])[0] * u
        if case["op"] == "ffn":
            return h
        x, g, u = (_stored(t)[0] for t in (x, g, u))
    dh = s["dh"].double()
    a, da = _act64(g, case["act"])
    dg, du = dh * da * u, dh * a
    grads = (torch.einsum("mf,fk->mk", dg, wg) + torch.einsum("mf,fk->mk", du, wu),
             torch.einsum("mf,mk->fk", dg, x), torch.einsum("mf,mk->fk", du, x))
    return grads if h is None else (h, *grads)

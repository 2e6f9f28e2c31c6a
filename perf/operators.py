"""The operators of the training step around the MoE layer that this repository measures: the router's balance loss, and
activations kept in 8 bits between forward and backward.

``own = False`` computes every operator in its plain form, from elementary torch operations; ``own = True`` makes the calls
a user of ``cute_kernels`` makes.  Sizes: the workloads of bench.py (a layer of 8 experts of 4096 x 14336
with 8192 tokens, 64 experts of 2048 x 1408 with 16384 tokens, rows of 4096), and odd ones around them.

8-bit form (the int8 microscaling format with blocks of 32): a block of 32 consecutive elements of a row (the last one of a
row may be shorter) has one power-of-two step, the smallest for which every rounded element lies in [-127, 127].
"""

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kernel-hyperdrive_amd")
_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZES = {"fp32": 4, "fp16": 2, "bf16": 2}
_EPS = 1e-5
BLOCK = 32


def listed():
    return [
        # router of a short micro-batch: all latency
        {"name": "balance-64x8", "op": "balance", "tokens": 64, "experts": 8, "top_k": 2, "dtype": "bf16", "padding": 0.0},
        # the 8-expert layer of the benchmark
        {"name": "balance-8192x8", "op": "balance", "tokens": 8192, "experts": 8, "top_k": 2, "dtype": "bf16", "padding": 0.0},
        # the 64-expert layer of the benchmark, a padded batch
        {"name": "balance-16384x64-padded", "op": "balance", "tokens": 16384, "experts": 64, "top_k": 6, "dtype": "bf16", "padding": 0.2},
        # many fine-grained experts, a router kept in fp32, a long ragged batch
        {"name": "balance-65521x160-fp32", "op": "balance", "tokens": 65521, "experts": 160, "top_k": 8, "dtype": "fp32", "padding": 0.05},
        # what a caller keeps itself: a few rows, written and read back
        {"name": "checkpoint-64x4096", "op": "checkpoint", "rows": 64, "width": 4096, "dtype": "bf16"},
        # the hidden states of a whole batch
        {"name": "checkpoint-16384x4096", "op": "checkpoint", "rows": 16384, "width": 4096, "dtype": "bf16"},
        # separate gate and up projections, odd rows whose last block is short
        {"name": "swiglu-1001x1419-fp16", "op": "swiglu", "rows": 1001, "width": 1419, "dtype": "fp16"},
        # one projection for both halves, the fine-grained experts' routed rows
        {"name": "swiglu-unchunked-24576x1408", "op": "swiglu_unchunked", "rows": 24576, "width": 1408, "dtype": "bf16"},
        # the same at the 8-expert layer's width: the largest activation of the benchmark
        {"name": "swiglu-unchunked-16384x14336", "op": "swiglu_unchunked", "rows": 16384, "width": 14336, "dtype": "bf16"},
        # the norm of a few tokens
        {"name": "rmsnorm-64x4096", "op": "rmsnorm", "rows": 64, "width": 4096, "dtype": "bf16"},
        # the benchmark's norm
        {"name": "rmsnorm-16384x4096", "op": "rmsnorm", "rows": 16384, "width": 4096, "dtype": "bf16"},
        # residual stream kept in fp32, an odd number of rows
        {"name": "residual-rmsnorm-4099x2048-fp32", "op": "residual_rmsnorm", "rows": 4099, "width": 2048, "dtype": "fp32"},
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["balance", "balance", "checkpoint", "swiglu", "swiglu_unchunked", "rmsnorm", "residual_rmsnorm"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if op == "balance":
        experts = _log(rng, 2, 256)
        return {"op": op, "tokens": _log(rng, 1, 65536), "experts": experts, "top_k": rng.randint(1, min(8, experts)),
                "dtype": dtype, "padding": rng.choice([0.0, 0.0, 0.1, 0.5])}
    width = _log(rng, 33, 16384)
    if rng.random() < 0.6:
        width = (width + 31) // 32 * 32
    # no more elements than a quarter of the largest listed case has
    rows = _log(rng, 1, min(32768, max(1, 60_000_000 // width)))
    return {"op": op, "rows": rows, "width": width, "dtype": dtype}


def work(case):
    """Bytes: every input read once, every output written once, and the 8-bit form written and read once, since the
    backward is another call than the forward.  Flops: the arithmetic of the formulas, an exponential counted as one."""
    s = _SIZES[case["dtype"]]
    if case["op"] == "balance":
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        masks = 2 * T if case["padding"] else 0
        # forward: logits, ids; backward: logits, gradient
        return {"bytes": 3 * T * E * s + 8 * T * k + 8 * E + masks, "flops": 14 * T * E}
    n, rows, H = case["rows"] * case["width"], case["rows"], case["width"]
    kept = n + rows * -(-H // BLOCK)  # codes and one step per block
    if case["op"] == "checkpoint":
        return {"bytes": 2 * n * s + 2 * kept, "flops": 4 * n}
    if case["op"] in ("swiglu", "swiglu_unchunked"):
        return {"bytes": 6 * n * s + 4 * kept, "flops": 25 * n}
    streams = 6 if case["op"] == "residual_rmsnorm" else 4
    if case["op"] == "residual_rmsnorm":
        streams += 1  # the gradient of the sum
    return {"bytes": streams * n * s + 2 * kept + 8 * rows + 3 * H * s, "flops": 18 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _randn(g, *shape, dtype, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def _activation(g, rows, width, dtype):
    """Hidden states as blocks see them: unit rows, a few channels that stand far out, and a sixteenth of the rows padding."""
    x = torch.randn(rows, width, generator=g, device="cuda")
    channels = torch.randint(0, width, (max(1, width // 256),), generator=g, device="cuda")
    x[:, channels] *= 20.0
    if rows > 16:
        x[torch.randint(0, rows, (rows // 16,), generator=g, device="cuda")] = 0.0
    return x.to(dtype)


def prepare(case, seed):
    if own and _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, op = _DTYPES[case["dtype"]], case["op"]
    if op == "balance":
        T, E, k = case["tokens"], case["experts"], case["top_k"]
        # a few experts are popular: per-expert offsets on top of the tokens' own preferences
        logits = _randn(g, T, E, dtype=dtype) + _randn(g, E, dtype=dtype)
        mask = None
        if case["padding"]:
            mask = torch.rand(T, generator=g, device="cuda") >= case["padding"]
        # the losses' weights; fp16 training scales its loss, or gradients of 1e-7 would vanish in the type
        scale = min(65536, 16 * T) if dtype == torch.float16 else 1
        return {"op": op, "logits": logits.requires_grad_(own), "selected": logits.detach().topk(k, dim=-1).indices,
                "mask": mask, "weights": (torch.tensor(0.01 * scale, device="cuda"), torch.tensor(0.001 * scale, device="cuda"))}
    rows, H = case["rows"], case["width"]
    if op == "checkpoint":
        return {"op": op, "x": _activation(g, rows, H, dtype)}
    dy = _randn(g, rows, H, dtype=dtype)
    if op == "swiglu":
        return {"op": op, "gate": _randn(g, rows, H, dtype=dtype, scale=2.0).requires_grad_(own),
                "up": _randn(g, rows, H, dtype=dtype).requires_grad_(own), "dy": dy}
    if op == "swiglu_unchunked":
        return {"op": op, "x": _randn(g, rows, 2 * H, dtype=dtype, scale=1.5).requires_grad_(own), "dy": dy}
    weight = _randn(g, H, dtype=dtype, scale=0.1, shift=1.0).requires_grad_(own)
    x = _activation(g, rows, H, dtype)
    if op == "rmsnorm":
        return {"op": op, "x": x.requires_grad_(own), "weight": weight, "dy": dy}
    return {"op": op, "x": _randn(g, rows, H, dtype=dtype, scale=0.1).requires_grad_(own), "residual": x.requires_grad_(own),
            "weight": weight, "dy": dy, "dsum": _randn(g, rows, H, dtype=dtype)}


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


def _run_own(s):
    import cute_kernels as ck

    op, grad = s["op"], torch.autograd.grad
    if op == "balance":
        balance, z, counts = ck.moe_balance_loss_cute(s["logits"], s["selected"], s["mask"])
        (d_logits,) = grad((balance, z), s["logits"], s["weights"])
        return {"balance": balance.detach(), "z": z.detach(), "counts": counts, "d_logits": d_logits}
    if op == "checkpoint":
        codes, scales = ck.mx8_quantize_cute(s["x"])
        return {"x": ck.mx8_dequantize_cute(codes, scales, s["x"].dtype)}
    if op == "swiglu":
        y = ck.swiglu_cute(s["gate"], s["up"], checkpoint_8bit=True)
        d_gate, d_up = grad(y, (s["gate"], s["up"]), s["dy"])
        return {"y": y.detach(), "d_gate": d_gate, "d_up": d_up}
    if op == "swiglu_unchunked":
        y = ck.swiglu_unchunked_cute(s["x"], checkpoint_8bit=True)
        (d_x,) = grad(y, s["x"], s["dy"])
        return {"y": y.detach(), "d_x": d_x}
    if op == "rmsnorm":
        y = ck.rmsnorm_cute(s["x"], s["weight"], _EPS, checkpoint_8bit=True)
        d_x, d_weight = grad(y, (s["x"], s["weight"]), s["dy"])
        return {"y": y.detach(), "d_x": d_x, "d_weight": d_weight}
    y, total = ck.fused_residual_add_rmsnorm_cute(s["x"], s["residual"], s["weight"], _EPS, checkpoint_8bit=True)
    d_x, d_residual, d_weight = grad((y, total), (s["x"], s["residual"], s["weight"]), (s["dy"], s["dsum"]))
    return {"y": y.detach(), "sum": total.detach(), "d_x": d_x, "d_residual": d_residual, "d_weight": d_weight}


def _plain_balance(s):
    z = s["logits"].float()
    T, E = z.shape
    k = s["selected"].size(1)
    mask = torch.ones(T, device=z.device) if s["mask"] is None else s["mask"].float()
    n = mask.sum().clamp(min=1.0)
    top = z.max(dim=1, keepdim=True).values
    e = torch.exp(z - top)
    total = e.sum(dim=1, keepdim=True)
    p = e / total
    lse = (top + torch.log(total)).squeeze(1)
    hits = torch.zeros(T, E, device=z.device).scatter_add_(1, s["selected"], mask.unsqueeze(1).expand(T, k))
    counts = hits.sum(dim=0)
    mean_p = (p * mask.unsqueeze(1)).sum(dim=0) / n
    share = counts / (n * k)
    balance = E * (share * mean_p).sum()
    z_loss = (mask * lse * lse).sum() / n
    # the shares less their mean, in 64 bits: the gradient is their difference from a mean that lies close to them
    centred = (share.double() - share.double().mean()).float()
    inner = centred - (p * centred).sum(dim=1, keepdim=True)
    g_b, g_z = s["weights"]
    d = p * (g_b * E / n * inner + g_z * 2 / n * lse.unsqueeze(1)) * mask.unsqueeze(1)
    return {"balance": balance, "z": z_loss, "counts": counts.to(torch.int32), "d_logits": d.to(s["logits"].dtype)}


def _plain_8bit(x):
    """The values the 8-bit form of the fp32 rows ``x`` stands for."""
    rows, H = x.shape
    pad = -H % BLOCK
    if pad:
        x = torch.cat([x, x.new_zeros(rows, pad)], dim=1)
    blocks = x.view(rows, -1, BLOCK)
    # exponent of the largest magnitude, one more where it would round to 128 steps
    bits = blocks.abs().amax(dim=2, keepdim=True).view(torch.int32)
    exponent = ((bits + 0x10000) >> 23).clamp(7, 254)
    step, inverse = ((exponent - 6) << 23).view(torch.float32), ((260 - exponent) << 23).view(torch.float32)
    kept = (blocks * inverse).round().clamp(-127, 127) * step
    return kept.view(rows, -1)[:, :H]


def _plain_checkpoint(s):
    return {"x": _plain_8bit(s["x"].float()).to(s["x"].dtype)}


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


def _swiglu_backward(gate, up, dy):
    gate, up, dy = _plain_8bit(gate), _plain_8bit(up), dy.float()
    sig = _sigmoid(gate)
    return dy * up * sig * (1.0 + gate * (1.0 - sig)), dy * gate * sig


def _plain_swiglu(s):
    gate, up, dtype = s["gate"].float(), s["up"].float(), s["dy"].dtype
    y = up * gate * _sigmoid(gate)
    d_gate, d_up = _swiglu_backward(gate, up, s["dy"])
    return {"y": y.to(dtype), "d_gate": d_gate.to(dtype), "d_up": d_up.to(dtype)}


def _plain_swiglu_unchunked(s):
    H, dtype = s["dy"].size(1), s["dy"].dtype
    up, gate = s["x"][:, :H].float(), s["x"][:, H:].float()
    y = up * gate * _sigmoid(gate)
    d_gate, d_up = _swiglu_backward(gate, up, s["dy"])
    return {"y": y.to(dtype), "d_x": torch.cat([d_up, d_gate], dim=1).to(dtype)}


def _plain_norm(x, weight, dy):
    """(y, d_x, d_weight) in fp32 of rows ``x`` (fp32), the backward from their 8-bit form."""
    weight, dy = weight.float(), dy.float()
    r = torch.rsqrt((x * x).mean(dim=1, keepdim=True) + _EPS)
    kept = _plain_8bit(x)
    g = dy * weight
    d_x = r * (g - kept * (r * r * (g * kept).mean(dim=1, keepdim=True)))
    return x * r * weight, d_x, (dy * kept * r).sum(dim=0)


def _plain_rmsnorm(s):
    dtype = s["x"].dtype
    y, d_x, d_weight = _plain_norm(s["x"].float(), s["weight"], s["dy"])
    return {"y": y.to(dtype), "d_x": d_x.to(dtype), "d_weight": d_weight.to(dtype)}


def _plain_residual_rmsnorm(s):
    dtype = s["x"].dtype
    total = (s["x"].float() + s["residual"].float()).to(dtype)  # the sum is rounded first: it is the next residual
    y, d_x, d_weight = _plain_norm(total.float(), s["weight"], s["dy"])
    # the norm's gradient and the sum's own, added and rounded once; both terms of the sum get it
    d = (d_x + s["dsum"].float()).to(dtype)
    return {"y": y.to(dtype), "sum": total, "d_x": d, "d_residual": d, "d_weight": d_weight.to(dtype)}


_PLAIN = {"balance": _plain_balance, "checkpoint": _plain_checkpoint, "swiglu": _plain_swiglu,
          "swiglu_unchunked": _plain_swiglu_unchunked, "rmsnorm": _plain_rmsnorm,
          "residual_rmsnorm": _plain_residual_rmsnorm}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def _exact_8bit(x):
    rows, H = x.shape
    padded = torch.nn.functional.pad(x, (0, -H % BLOCK)).unflatten(1, (-1, BLOCK))
    largest = padded.abs().amax(2, keepdim=True)
    mantissa, exponent = torch.frexp(largest)  # largest = mantissa * 2^exponent, mantissa in [1/2, 1)
    # 127 steps of 2^(exponent - 7) reach 127/128 * 2^exponent; from 255/256 on the largest rounds to 128 of them
    exponent = torch.where(mantissa >= 255 / 256, exponent + 1, exponent)
    exponent = torch.where(largest > 0, exponent, torch.zeros_like(exponent)).clamp(min=-119, max=128)
    step = ((exponent.long() - 7 + 1023) << 52).view(torch.float64)  # 2^(exponent - 7), to the last bit
    return (torch.clamp(torch.round(padded / step), -127, 127) * step).flatten(1)[:, :H]


def _exact_swiglu(gate, up, dy):
    y = up * torch.nn.functional.silu(gate)
    gate, up = _exact_8bit(gate), _exact_8bit(up)
    s = torch.sigmoid(gate)
    return y, dy * up * (s + gate * s * (1 - s)), dy * torch.nn.functional.silu(gate)


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    with torch.no_grad():
        if op == "balance":
            z = s["logits"].detach().double()
            real = torch.ones(z.size(0), dtype=torch.bool, device=z.device) if s["mask"] is None else s["mask"]
            n, E = max(1, int(real.sum())), z.size(1)
            p, lse = torch.softmax(z, 1) * real[:, None], torch.logsumexp(z, 1) * real
            counts = torch.bincount(s["selected"][real].flatten(), minlength=E)
            f = counts.double() / (n * s["selected"].size(1))
            g_b, g_z = (w.double() for w in s["weights"])
            d = p * (g_b * E / n * (f - (torch.softmax(z, 1) @ f)[:, None]) + 2 * g_z / n * lse[:, None])
            return {"balance": E * (f * p.sum(0) / n).sum(), "z": lse.square().sum() / n, "counts": counts.int(),
                    "d_logits": d}
        if op == "checkpoint":
            return {"x": _exact_8bit(s["x"].double())}
        dy = s["dy"].double()
        if op == "swiglu":
            y, d_gate, d_up = _exact_swiglu(s["gate"].detach().double(), s["up"].detach().double(), dy)
            return {"y": y, "d_gate": d_gate, "d_up": d_up}
        if op == "swiglu_unchunked":
            up, gate = s["x"].detach().double().chunk(2, dim=1)
            y, d_gate, d_up = _exact_swiglu(gate, up, dy)
            return {"y": y, "d_x": torch.cat([d_up, d_gate], 1)}
        x = s["x"].detach()
        if op == "residual_rmsnorm":
            x = (x.double() + s["residual"].detach().double()).to(x.dtype)
        x, w = x.double(), s["weight"].detach().double()
        rms = (x.square().mean(1, keepdim=True) + _EPS).sqrt()
        kept = _exact_8bit(x)
        normal = kept / rms
        d_normal = dy * w
        d_x = (d_normal - normal * (d_normal * normal).mean(1, keepdim=True)) / rms
        d_weight = (dy * normal).sum(0)
        if op == "rmsnorm":
            return {"y": x / rms * w, "d_x": d_x, "d_weight": d_weight}
        d = d_x + s["dsum"].double()
        return {"y": x / rms * w, "sum": x, "d_x": d, "d_residual": d, "d_weight": d_weight}

"""Activations in 8 bits (cute_kernels/kernels/mx8.py): the form itself bit for bit, and the operators whose backward works
from it against their formulas in 64 bits, through the public functions.

Tolerances.  A result is the formula in 64 bits, evaluated in fp32 and rounded once to its type: half a step of that type,
``finfo.eps / 2`` of the value (plus half of fp16's smallest step, 2^-25), and the fp32 evaluation's own error.  That one is
relative to the sum of the magnitudes that are added, ``scale``: every fp32 operation is off by 2^-24, the exponential and
the reciprocal by a few times that (for |x| <= 16 the fast exponential by |x| 2^-24 = 2^-20 more), sums of n terms by n times
that.  The multiples are stated at each test."""

import pytest
import torch

from helpers import DTYPES, announce, randn

pytestmark = pytest.mark.gpu


def assert_rounded(actual, exact, dtype, evaluation, scale=None, what="", lost=0.0):
    """|actual - exact| <= half a step of `dtype` at the value + `evaluation` * scale (default: the value's magnitude) + lost."""
    a, e = actual.detach().cpu().double(), exact.double()
    assert a.shape == e.shape and actual.dtype == dtype, f"{what}: {actual.shape} {actual.dtype}"
    scale = e.abs() if scale is None else scale.double()
    # a value one evaluation error further out may lie in the next binade: the half step is taken there
    allowed = torch.finfo(dtype).eps / 2 * (e.abs() + evaluation * scale) + evaluation * scale + lost
    if dtype == torch.float16:
        allowed = allowed + 2.0 ** -25
    elif dtype == torch.bfloat16 or dtype == torch.float32:
        allowed = allowed + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = (a - e).abs()
    wrong = ~((off <= allowed) | (a.isnan() & e.isnan()))
    assert not wrong.any(), (
        f"{what}: {int(wrong.sum())} of {wrong.numel()} elements, worst {float((off / allowed)[wrong].max()):.2f} times the bound"
    )


# ---- the definition, in 64 bits and apart from the package -----------------------------------------------------------
def encode64(x):
    """(codes, scale bytes) of rows by the definition: int64 tensors."""
    H = x.size(-1)
    blocks = torch.nn.functional.pad(x.double(), (0, -H % 32)).unflatten(-1, (-1, 32))
    finite = blocks.isfinite().all(-1)
    largest = torch.where(finite.unsqueeze(-1), blocks, 0.0).abs().amax(-1)
    mantissa, exponent = torch.frexp(largest)  # largest = mantissa * 2^exponent, 1/2 <= mantissa < 1
    scale = exponent.long() + 126 + (mantissa >= 255 / 256).long()  # 127.5 steps of 2^(exponent - 7) round to 128
    scale = torch.where(largest > 0, scale, 0).clamp(7, 254)
    step = torch.pow(2.0, (scale - 133).double()).unsqueeze(-1)
    codes = (torch.where(finite.unsqueeze(-1), blocks, 0.0) / step).round().clamp(-127, 127).long()
    return codes.flatten(-2)[..., :H], torch.where(finite, scale, 255)


def decode64(codes, scales):
    steps = torch.where(scales == 255, float("nan"), torch.pow(2.0, (scales - 133).double()))
    return codes.double() * steps.repeat_interleave(32, -1)[..., : codes.size(-1)]


def kept64(x):
    return decode64(*encode64(x.cpu()))


def rows_like_activations(shape, dtype, seed):
    """Rows of unit size with channels that stand far out, tiny and zero rows."""
    x = randn(shape, torch.float32, seed)
    x[..., ::37] *= 30.0
    if x.dim() > 1 and x.size(0) > 4:
        x[1] = 0.0
        x[2] *= 2.0 ** -20
        x[3, ..., :40] = 0.0
    return x.to(dtype)


# ---- the form itself ------------------------------------------------------------------------------------------------------
SHAPES = [(1,), (31,), (4096,), (0, 64), (3, 0), (1, 1), (5, 7), (5, 8), (7, 31), (7, 32), (7, 33), (9, 72), (3, 5, 1419),
          (37, 4096), (130, 1416), (2, 65536), (300, 4104)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize_and_dequantize(gpu, dtype, shape):
    from cute_kernels import mx8_dequantize_cute, mx8_dequantize_torch, mx8_quantize_cute, mx8_quantize_torch

    announce("mx8", dtype, shape)
    x = rows_like_activations(shape, dtype, 1)
    codes, scales = mx8_quantize_cute(x.to(gpu))
    assert codes.dtype == torch.int8 and scales.dtype == torch.uint8 and codes.shape == x.shape
    want_codes, want_scales = encode64(x)
    assert torch.equal(codes.cpu().long(), want_codes) and torch.equal(scales.cpu().long(), want_scales)
    torch_codes, torch_scales = mx8_quantize_torch(x)
    assert torch.equal(codes.cpu(), torch_codes) and torch.equal(scales.cpu(), torch_scales)
    values = mx8_dequantize_cute(codes, scales, dtype)
    want = decode64(want_codes, want_scales)
    assert values.dtype == dtype and torch.equal(values.cpu().double(), want)  # exact: seven magnitude bits
    assert torch.equal(values.cpu(), mx8_dequantize_torch(codes.cpu(), scales.cpu(), dtype))
    # half a step, which is at most 1/127 of the block's largest magnitude
    if x.numel():
        step = torch.pow(2.0, (want_scales - 133).double()).repeat_interleave(32, -1)[..., : x.size(-1)]
        assert ((want - x.double()).abs() <= step / 2).all()
    # writing what was read changes nothing
    again_codes, again_scales = mx8_quantize_cute(values)
    again = mx8_dequantize_cute(again_codes, again_scales, dtype)
    assert torch.equal(again, values)


def test_known_blocks(gpu):
    """Blocks whose codes follow by hand from the definition."""
    from cute_kernels import mx8_dequantize_cute, mx8_quantize_cute

    announce("mx8 known blocks")
    inf, nan = float("inf"), float("nan")

    def block(*head):
        return list(head) + [0.0] * (32 - len(head))

    tiny = 2.0 ** -126
    rows = [
        (block(1.0, -1.0, 0.5, 1 / 64, 1 / 128, 3 / 128, -3 / 128), 127, (64, -64, 32, 1, 0, 2, -2)),  # ties go to even
        (block(127 / 64, 1.0), 127, (127, 64)),
        (block(127.4 / 64, 1.0), 127, (127, 64)),
        (block(127.5 / 64, 1.0), 128, (64, 32)),  # 127.5 would round to 128: the next exponent
        (block(-127.5 / 64, 1.0), 128, (-64, 32)),
        (block(), 7, (0, 0)),
        (block(tiny, -3 * tiny, tiny / 2, 1.5 * tiny), 7, (1, -3, 0, 2)),  # the smallest step
        (block(tiny / 4), 7, (0,)),
        (block(127 * 2.0 ** 121, -(2.0 ** 127)), 254, (127, -64)),
        (block(3.4e38, -3.4e38, 2.0 ** 120), 254, (127, -127, 0)),  # 127.9 steps: saturated
        (block(1.0, nan, 2.0), 255, (0, 0, 0)),
        (block(1.0, -inf, 2.0), 255, (0, 0, 0)),
        (block(nan, inf), 255, (0, 0)),
    ]
    x = torch.tensor([r[0] for r in rows], dtype=torch.float32)
    codes, scales = mx8_quantize_cute(x.to(gpu))
    for i, (_, scale, head) in enumerate(rows):
        assert int(scales[i, 0]) == scale, (i, int(scales[i, 0]), scale)
        assert codes[i].cpu().tolist() == block(*head), (i, codes[i].cpu().tolist()[: len(head)])
    values = mx8_dequantize_cute(codes, scales, torch.float32).cpu()
    bad = torch.tensor([r[1] == 255 for r in rows])
    assert values[bad].isnan().all() and values[~bad].isfinite().all()
    # a bad block stays in its row and its 32 columns
    x = randn((4, 100), torch.bfloat16, 2)
    x[1, 40] = nan
    x[3, 99] = inf
    values = mx8_dequantize_cute(*mx8_quantize_cute(x.to(gpu)), torch.bfloat16).cpu()
    want = torch.zeros(4, 100, dtype=torch.bool)
    want[1, 32:64] = True
    want[3, 96:] = True
    assert torch.equal(values.isnan(), want)


def test_fp16_end_of_range(gpu):
    """65504 is kept as 64 steps of 1024 = 65536, which fp16 does not have: it is read back as the largest finite number."""
    from cute_kernels import mx8_dequantize_cute, mx8_quantize_cute

    announce("mx8 fp16 range")
    x = torch.zeros(2, 32, dtype=torch.float16)
    x[0, 0], x[0, 1], x[1, 5] = 65504.0, -65504.0, 2.0 ** -24
    codes, scales = mx8_quantize_cute(x.to(gpu))
    values = mx8_dequantize_cute(codes, scales, torch.float16).cpu()
    assert values[0, 0] == 65504.0 and values[0, 1] == -65504.0 and values[1, 5] == 2.0 ** -24
    assert mx8_dequantize_cute(codes, scales, torch.float32).cpu()[0, 0] == 65536.0


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_of_the_pair(gpu, dtype):
    from cute_kernels import mx8_quantize_cute

    announce("mx8 layouts", dtype)
    x = randn((64, 96), dtype, 3)
    xg = x.to(gpu)
    for view, host in [(xg.t(), x.t()), (xg[:, ::2], x[:, ::2]), (xg[::3, 8:72], x[::3, 8:72])]:
        codes, scales = mx8_quantize_cute(view)
        want = encode64(host.contiguous())
        assert torch.equal(codes.cpu().long(), want[0]) and torch.equal(scales.cpu().long(), want[1])
    flat = randn((64 * 96 + 3,), dtype, 4)
    shifted = flat.to(gpu)[3:].view(64, 96)  # contiguous, but no row starts on a packet
    codes, scales = mx8_quantize_cute(shifted)
    want = encode64(flat[3:].view(64, 96))
    assert torch.equal(codes.cpu().long(), want[0]) and torch.equal(scales.cpu().long(), want[1])


# ---- SwiGLU ---------------------------------------------------------------------------------------------------------------
def swiglu64(gate, up):
    return up * gate * torch.sigmoid(gate)


def check_swiglu_grads(gate, up, dy, d_gate, d_up, dtype, what):
    """Gradients at the kept values.  fp32 evaluation: sigmoid (exponential, addition, reciprocal, |x| <= 16: 2^-20 for the
    fast forms), then at most eight operations: 2^-19 of the magnitudes added.  Beyond x = -87.3 the sigmoid is below 2^-126,
    fp32's smallest normal number, and the 16-bit types' reciprocal of 1 + exp(-x) gives 0 for it: 2^-126 of its factors are lost."""
    g, u, d = kept64(gate), kept64(up), dy.double()
    s = torch.sigmoid(g)
    assert_rounded(d_up, d * g * s, dtype, 2.0 ** -19, what=f"{what} d_up", lost=2.0 ** -126 * (d * g).abs())
    assert_rounded(d_gate, d * u * (s + g * s * (1 - s)), dtype, 2.0 ** -19, (d * u).abs() * (s + (g * s * (1 - s)).abs()),
                   what=f"{what} d_gate", lost=2.0 ** -126 * (d * u).abs() * (1 + g.abs()))


def check_swiglu_output(gate, up, y, dtype):
    """The output is that of the exact inputs, evaluated as swiglu_cute evaluates it.  (Not compared with swiglu_cute's bits:
    the compiler may form an fp16 product and its rounding in one instruction in one kernel and in two in the other, and
    rounding through fp32 can differ from rounding at once by the last bit.)  fp32 takes 1 - r as the sigmoid of a negative
    gate, which is off by 2^-24 whatever its size: 2^-23 of the factors."""
    g, u = gate.double(), up.double()
    lost = (2.0 ** -23 if dtype == torch.float32 else 2.0 ** -126) * (g * u).abs()
    assert_rounded(y, swiglu64(g, u), dtype, 2.0 ** -19, what="y", lost=lost)


SWIGLU_SHAPES = [(1,), (70,), (0, 32), (1, 1), (5, 31), (3, 32), (7, 40), (2, 3, 72), (37, 513), (33, 1408), (150, 1419)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SWIGLU_SHAPES)
def test_swiglu(gpu, dtype, shape):
    from cute_kernels import swiglu_cute

    announce("swiglu 8-bit", dtype, shape)
    gate, up, dy = randn(shape, dtype, 5, 2.0), rows_like_activations(shape, dtype, 6), randn(shape, dtype, 7)
    g = gate.to(gpu, copy=True).requires_grad_(True)
    u = up.to(gpu, copy=True).requires_grad_(True)
    y = swiglu_cute(g, u, checkpoint_8bit=True)
    check_swiglu_output(gate, up, y, dtype)
    y.backward(dy.to(gpu))
    assert g.grad.shape == gate.shape and u.grad.shape == gate.shape
    check_swiglu_grads(gate, up, dy, g.grad, u.grad, dtype, "swiglu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(2,), (140,), (0, 64), (1, 2), (5, 62), (3, 64), (7, 80), (2, 3, 144), (37, 1026), (33, 2816)])
def test_swiglu_unchunked(gpu, dtype, shape):
    from cute_kernels import swiglu_unchunked_cute

    announce("swiglu_unchunked 8-bit", dtype, shape)
    half = (*shape[:-1], shape[-1] // 2)
    x, dy = rows_like_activations(shape, dtype, 8), randn(half, dtype, 9)
    xg = x.to(gpu, copy=True).requires_grad_(True)
    y = swiglu_unchunked_cute(xg, checkpoint_8bit=True)
    up, gate = x.chunk(2, dim=-1)
    check_swiglu_output(gate, up, y, dtype)
    y.backward(dy.to(gpu))
    assert xg.grad.shape == x.shape
    d_up, d_gate = xg.grad.chunk(2, dim=-1)
    check_swiglu_grads(gate.contiguous(), up.contiguous(), dy, d_gate, d_up, dtype, "unchunked")


@pytest.mark.parametrize("dtype", DTYPES)
def test_swiglu_activation_is_recomputed_at_the_kept_values(gpu, dtype):
    """What the experts' backward takes from the same pass.  fp32 evaluation: as for the forward, 2^-19."""
    from cute_kernels import _C
    from cute_kernels.kernels.mx8 import kept_pair, new_kept

    announce("swiglu activation", dtype)
    for rows, h in [(5, 32), (5, 37), (65, 136)]:
        x, dy = rows_like_activations((rows, 2 * h), dtype, 10), randn((rows, h), dtype, 11)
        kept = new_kept(2 * rows, h, gpu)
        _C.mx8_quantize(x.to(gpu).view(rows, 2, h), *kept_pair(kept, (rows, 2, h)))
        dx = torch.empty(rows, 2 * h, dtype=dtype, device=gpu)
        act = torch.empty(rows, h, dtype=dtype, device=gpu)
        _C.swiglu_unchunked_backward_mx8(kept, dy.to(gpu), dx, act)
        up, gate = x.chunk(2, dim=-1)
        assert_rounded(act, swiglu64(kept64(gate.contiguous()), kept64(up.contiguous())), dtype, 2.0 ** -19, what="act",
                       lost=2.0 ** -126 * (kept64(gate.contiguous()) * kept64(up.contiguous())).abs())
        check_swiglu_grads(gate.contiguous(), up.contiguous(), dy, dx[:, h:], dx[:, :h], dtype, "with act")


def test_swiglu_layouts_and_single_gradients(gpu):
    from cute_kernels import swiglu_cute, swiglu_unchunked_cute

    announce("swiglu 8-bit layouts")
    dtype = torch.bfloat16
    gate, up, dy = randn((48, 64), dtype, 12), randn((48, 64), dtype, 13), randn((48, 64), dtype, 14)
    for change in (lambda t: t.t(), lambda t: t[:, ::2], lambda t: t.reshape(-1)[3:3 + 40 * 64].view(40, 64)):
        g = gate.to(gpu, copy=True).requires_grad_(True)
        u = up.to(gpu, copy=True).requires_grad_(True)
        y = swiglu_cute(change(g), change(u), checkpoint_8bit=True)
        d_gate, d_up = torch.autograd.grad(y, (g, u), change(dy.to(gpu)))
        grads = [torch.zeros_like(gate), torch.zeros_like(up)]
        check_swiglu_grads(change(gate).contiguous(), change(up).contiguous(), change(dy).contiguous(),
                           change(d_gate), change(d_up), dtype, "layout")
        assert all(t.shape == d.shape for t, d in zip(grads, (d_gate, d_up)))
    # one operand without a gradient; a broadcast gradient (stride 0) of a sum
    g = gate.to(gpu, copy=True).requires_grad_(True)
    swiglu_cute(g, up.to(gpu), checkpoint_8bit=True).sum().backward()
    check = torch.ones_like(dy)
    s = torch.sigmoid(kept64(gate))
    assert_rounded(g.grad, kept64(up) * (s + kept64(gate) * s * (1 - s)), dtype, 2.0 ** -19,
                   kept64(up).abs() * (s + (kept64(gate) * s * (1 - s)).abs()) * check.double(), "sum")
    # without a gradient to come nothing is kept, and the result is the same
    with torch.no_grad():
        assert torch.equal(swiglu_cute(g, up.to(gpu), checkpoint_8bit=True), swiglu_cute(g, up.to(gpu)))
    x = randn((8, 64), dtype, 15).to(gpu)
    assert torch.equal(swiglu_unchunked_cute(x, checkpoint_8bit=True), swiglu_unchunked_cute(x))


# ---- RMSNorm --------------------------------------------------------------------------------------------------------------
def check_norm(x, weight, dy, dsum, eps, y, dx, dw, dtype, what):
    """x: the rows as normalised (rounded sum).  fp32 evaluation: a lane adds at most 64 squares, the lanes and waves of a
    team 6 + 16 more: 1/rms within 50 * 2^-24, y two operations more, the products of dx thrice that and their own sums:
    2^-16 of the magnitudes added.  dw: every row's product as dx's, and `rows` additions of them."""
    H = x.size(-1)
    x64, d = x.double().reshape(-1, H), dy.double().reshape(-1, H)
    w = torch.ones(H, dtype=torch.float64) if weight is None else weight.double()
    r = torch.rsqrt(x64.square().mean(-1, keepdim=True) + eps)
    assert_rounded(y.reshape(-1, H), x64 * r * w, dtype, 2.0 ** -18, what=f"{what} y")
    k = kept64(x.reshape(-1, H))
    g = d * w
    mean, mean_size = (g * k).mean(-1, keepdim=True), (g * k).abs().mean(-1, keepdim=True)
    want, size = r * (g - k * r * r * mean), r * (g.abs() + k.abs() * r * r * mean_size)
    if dsum is not None:
        want, size = want + dsum.double().reshape(-1, H), size + dsum.double().reshape(-1, H).abs()
    assert_rounded(dx.reshape(-1, H), want, dtype, 2.0 ** -16, size, f"{what} dx")
    if dw is not None:
        terms = d * k * r
        evaluation = 2.0 ** -17 + (terms.size(0) + 64) * 2.0 ** -24
        assert_rounded(dw, terms.sum(0), dtype, evaluation, terms.abs().sum(0), f"{what} dw")


NORM_SHAPES = [(1,), (100,), (0, 64), (1, 1), (3, 8), (5, 33), (4, 512), (9, 520), (2, 3, 1024), (37, 4096), (3, 4104),
               (2, 8191), (2, 16384), (3, 16392), (2, 40001), (2, 65536), (700, 72)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("has_weight", [True, False])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_rmsnorm(gpu, dtype, has_weight, shape):
    from cute_kernels import rmsnorm_cute

    announce("rmsnorm 8-bit", dtype, has_weight, shape)
    x, dy = rows_like_activations(shape, dtype, 16), randn(shape, dtype, 17)
    weight = randn(shape[-1:], dtype, 18, 0.1, 1.0) if has_weight else None
    xg = x.to(gpu, copy=True).requires_grad_(True)
    wg = weight.to(gpu, copy=True).requires_grad_(True) if has_weight else None
    y = rmsnorm_cute(xg, wg, 1e-5, checkpoint_8bit=True)
    y.backward(dy.to(gpu))
    assert y.shape == x.shape and xg.grad.shape == x.shape
    check_norm(x, weight, dy, None, 1e-5, y, xg.grad, wg.grad if has_weight else None, dtype, "rmsnorm")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("has_weight", [True, False])
@pytest.mark.parametrize("shape", [(100,), (0, 64), (1, 1), (5, 33), (9, 520), (2, 3, 1024), (37, 4096), (3, 4104), (2, 8191),
                                   (3, 16392), (2, 40001), (2, 65536)])
def test_fused_residual_add_rmsnorm(gpu, dtype, has_weight, shape):
    from cute_kernels import fused_residual_add_rmsnorm_cute

    announce("residual rmsnorm 8-bit", dtype, has_weight, shape)
    x, residual = randn(shape, dtype, 19, 0.3), rows_like_activations(shape, dtype, 20)
    dy, dsum = randn(shape, dtype, 21), randn(shape, dtype, 22)
    weight = randn(shape[-1:], dtype, 23, 0.1, 1.0) if has_weight else None
    total = (x.float() + residual.float()).to(dtype)

    def leaves():
        return (x.to(gpu, copy=True).requires_grad_(True), residual.to(gpu, copy=True).requires_grad_(True),
                weight.to(gpu, copy=True).requires_grad_(True) if has_weight else None)

    for use in ("both", "output", "sum"):
        xg, rg, wg = leaves()
        y, s = fused_residual_add_rmsnorm_cute(xg, rg, wg, 1e-5, checkpoint_8bit=True)
        assert torch.equal(s.detach().cpu(), total)
        if use == "sum":
            s.backward(dsum.to(gpu))
            assert torch.equal(xg.grad.cpu(), dsum) and torch.equal(rg.grad.cpu(), dsum)
            assert wg is None or not wg.grad.any()
            continue
        if use == "both":
            torch.autograd.backward((y, s), (dy.to(gpu), dsum.to(gpu)))
        else:
            y.backward(dy.to(gpu))
        assert torch.equal(xg.grad, rg.grad)
        check_norm(total, weight, dy, dsum if use == "both" else None, 1e-5, y, xg.grad, wg.grad if has_weight else None,
                   dtype, f"residual {use}")


def test_rmsnorm_bad_rows_stay_alone(gpu):
    """A NaN poisons its own row's gradients and the weight's, not the other rows; default eps; an unaligned row start."""
    from cute_kernels import rmsnorm_cute

    announce("rmsnorm 8-bit bad rows")
    dtype = torch.bfloat16
    x, dy, weight = randn((6, 96), dtype, 24), randn((6, 96), dtype, 25), randn((96,), dtype, 26, 0.1, 1.0)
    x[2, 50] = float("nan")
    xg = x.to(gpu, copy=True).requires_grad_(True)
    y = rmsnorm_cute(xg, weight.to(gpu), None, checkpoint_8bit=True)
    y.backward(dy.to(gpu))
    keep = [0, 1, 3, 4, 5]
    assert y[2].isnan().all() and xg.grad[2].isnan().all()
    check_norm(x[keep], weight, dy[keep], None, torch.finfo(dtype).eps, y[keep], xg.grad[keep], None, dtype, "others")
    flat = randn((4 * 96 + 1,), dtype, 27)
    shifted = flat.to(gpu)[1:].view(4, 96).requires_grad_(True)
    wg = weight.to(gpu, copy=True).requires_grad_(True)
    y = rmsnorm_cute(shifted, wg, 1e-6, checkpoint_8bit=True)
    dx, dw = torch.autograd.grad(y, (shifted, wg), dy[:4].to(gpu))
    check_norm(flat[1:].view(4, 96), weight, dy[:4], None, 1e-6, y, dx, dw, dtype, "shifted")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rmsnorm_of_far_off_rows(gpu, dtype):
    """Rows of 2^55 and of 2^-55: their squares, and everything the results are made of, are ordinary fp32 numbers, but (1 / rms)^3
    is not.  The bounds are those of rows of size one."""
    from cute_kernels import rmsnorm_cute

    announce("rmsnorm 8-bit far off", dtype)
    for exponent in (55, -55):
        for H in (72, 4104):
            x = (randn((5, H), torch.float32, 50) * 2.0 ** exponent).to(dtype)
            dy, weight = randn((5, H), dtype, 51), randn((H,), dtype, 52, 0.1, 1.0)
            xg, wg = x.to(gpu, copy=True).requires_grad_(True), weight.to(gpu, copy=True).requires_grad_(True)
            y = rmsnorm_cute(xg, wg, 0.0, checkpoint_8bit=True)
            y.backward(dy.to(gpu))
            check_norm(x, weight, dy, None, 0.0, y, xg.grad, wg.grad, dtype, f"2^{exponent} H={H}")


def test_rmsnorm_of_more_rows_than_a_launch_holds(gpu):
    """2^24 + 5 rows of 64 lanes each are more than the 2^30 lanes one launch of the forward takes."""
    if gpu.type != "cuda":
        pytest.skip("too many rows for the emulation")
    from cute_kernels import rmsnorm_cute

    announce("rmsnorm 8-bit many rows")
    B, H = 2 ** 24 + 5, 40
    x = torch.randn(B, H, dtype=torch.bfloat16, device=gpu, generator=torch.Generator(gpu).manual_seed(53)).requires_grad_(True)
    dy = torch.randn(B, H, dtype=torch.bfloat16, device=gpu, generator=torch.Generator(gpu).manual_seed(54))
    y = rmsnorm_cute(x, None, 1e-5, checkpoint_8bit=True)
    (dx,) = torch.autograd.grad(y, x, dy)
    for rows in (slice(0, 300), slice(2 ** 24 - 300, B)):
        part = x[rows].detach().clone().requires_grad_(True)
        want = rmsnorm_cute(part, None, 1e-5, checkpoint_8bit=True)
        assert torch.equal(y[rows], want)
        assert torch.equal(dx[rows], torch.autograd.grad(want, part, dy[rows])[0])


@pytest.mark.parametrize("H", [65536, 65530])
def test_offsets_beyond_32_bits(gpu, H):
    """Rows behind the 2^32-nd element: the same bits as the same rows in a small tensor."""
    if gpu.type != "cuda":
        pytest.skip("too large for the emulation")
    import cute_kernels as ck

    announce("8-bit offsets", H)
    B, dtype = 2 ** 16 + 40, torch.bfloat16
    x = torch.empty(B, H, dtype=dtype, device=gpu)
    x[:-30].fill_(0.5)
    x[-30:] = randn((30, H), dtype, 55).to(gpu)
    x.requires_grad_(True)
    weight, dy = randn((H,), dtype, 56, 0.1, 1.0).to(gpu), randn((30, H), dtype, 57).to(gpu)
    tail = x[-30:].detach().clone().requires_grad_(True)
    codes, scales = ck.mx8_quantize_cute(x)
    want = ck.mx8_quantize_cute(tail)
    assert torch.equal(codes[-30:], want[0]) and torch.equal(scales[-30:], want[1])
    assert torch.equal(ck.mx8_dequantize_cute(codes, scales, dtype)[-30:], ck.mx8_dequantize_cute(*want, dtype))
    del codes, scales
    for call in (lambda v: ck.swiglu_unchunked_cute(v, checkpoint_8bit=True),
                 lambda v: ck.rmsnorm_cute(v, weight, 1e-5, checkpoint_8bit=True)):
        y, want = call(x), call(tail)
        assert torch.equal(y[-30:], want)
        grad = torch.zeros_like(y)
        grad[-30:] = dy[:, : y.size(-1)]
        (dx,) = torch.autograd.grad(y, x, grad)
        assert torch.equal(dx[-30:], torch.autograd.grad(want, tail, dy[:, : y.size(-1)].contiguous())[0])
        assert not dx[-2000:-30].any()
        del y, grad, dx


# ---- differences ------------------------------------------------------------------------------------------------------------
def test_gradients_against_differences(gpu):
    """The gradients are those of the operators at the kept values.  x is made of values that are kept exactly (multiples of
    a step, each block with a 127), and the operator itself is differenced in 64 bits: step 1e-5, error 1e-9 or so of
    second order; fp32 results are held to 2^-16 of the largest gradient."""
    from cute_kernels import rmsnorm_cute, swiglu_unchunked_cute

    announce("differences")
    g = torch.Generator().manual_seed(28)
    x = torch.randint(-127, 128, (2, 64), generator=g).double()
    x[:, ::32] = 127
    x = x / 64
    dy = torch.randn(2, 64, generator=g).double()
    w = 1 + 0.1 * torch.randn(64, generator=g).double()

    def norm(v):
        return (v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * w.float().double() * dy.float().double()).sum()

    def glu(v):
        up, gate = v.chunk(2, dim=-1)
        return (swiglu64(gate, up) * dy[:, :32].float().double()).sum()

    def differences(f):
        out = torch.zeros_like(x)
        for i in range(x.size(0)):
            for j in range(x.size(1)):
                e = torch.zeros_like(x)
                e[i, j] = 1e-5
                out[i, j] = (f(x + e) - f(x - e)) / 2e-5
        return out

    xg = x.float().to(gpu, copy=True).requires_grad_(True)
    y = rmsnorm_cute(xg, w.float().to(gpu), 1e-5, checkpoint_8bit=True)
    (dx,) = torch.autograd.grad(y, xg, dy.float().to(gpu))
    want = differences(norm)
    assert (dx.cpu().double() - want).abs().max() <= 2.0 ** -16 * want.abs().max()
    (dx,) = torch.autograd.grad(swiglu_unchunked_cute(xg, checkpoint_8bit=True), xg, dy[:, :32].float().to(gpu))
    want = differences(glu)
    assert (dx.cpu().double() - want).abs().max() <= 2.0 ** -16 * want.abs().max()


# ---- routing weights' gradient, and the experts -----------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (5, 2, 33), (7, 3, 64), (65, 2, 1000), (33, 6, 2048)])
def test_combine_backward_gates(gpu, dtype, shape):
    """fp32 evaluation: a lane adds at most 8 * ceil(H / 512) products, the wave 6 more."""
    from cute_kernels import mx8_quantize_cute
    from cute_kernels.kernels.scattermoe.ops import moe_combine_backward_gates_mx8

    announce("combine gates 8-bit", dtype, shape)
    T, k, H = shape
    y, dy = randn(shape, dtype, 29), randn((T, H), dtype, 30)
    codes, scales = mx8_quantize_cute(y.to(gpu))
    d_gates = torch.empty(T, k, dtype=dtype, device=gpu)
    moe_combine_backward_gates_mx8(codes, scales, dy.to(gpu), d_gates)
    terms = kept64(y) * dy.double().unsqueeze(1)
    evaluation = (8 * -(-H // 512) + 8) * 2.0 ** -24
    assert_rounded(d_gates, terms.sum(-1), dtype, evaluation, terms.abs().sum(-1), "d_gates")


def _layer(gpu, dtype, T, H, I, E, k, seed):
    import cute_kernels as ck

    moe = ck.MoE_HIP(num_experts=E, num_experts_per_tok=k, hidden_size=H, intermediate_size=I,
                     activation_function=ck.swiglu_unchunked_cute, is_glu=True, add_bias=False, std=0.05)
    with torch.no_grad():
        for i, p in enumerate(moe.parameters()):
            p.copy_(randn(p.shape, torch.float32, seed + i, 0.1))
    return moe.to(device=gpu, dtype=dtype), randn((T, H), dtype, seed + 10), randn((T, H), dtype, seed + 11)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(100, 64, 128, 4, 2), (33, 72, 40, 3, 1)])
def test_moe_layer(gpu, dtype, shape):
    """The layer with ``checkpoint_8bit``: the output is the ordinary layer's bit for bit, and the gradients are those of the
    experts' formulas (plain torch in 64 bits, every intermediate the layer stores rounded to its type) at the kept values.
    Products of 16-bit rounded terms: each intermediate is off by half a step where the two sides' last bits differ, sums of
    up to 128 such terms grow as their root: 4 steps of the type's eps norm-wise, 1e-5 for fp32 (sums of fp32 products)."""
    T, H, I, E, k = shape
    announce("layer 8-bit", dtype, shape)
    moe, x, dy = _layer(gpu, dtype, T, H, I, E, k, 31)
    xg = x.to(gpu, copy=True).requires_grad_(True)
    y_plain, _ = moe(xg)
    moe.checkpoint_8bit = True
    y, _ = moe(xg)
    if dtype != torch.float32:  # (fp32 layers take the separate products without the option: same sums, same order)
        assert torch.equal(y, y_plain)
    with torch.no_grad():
        assert torch.equal(moe(xg)[0], y)  # nothing is kept without a gradient to come
        _, gates, selected = moe._compute_routing_weights(xg)
    y.backward(dy.to(gpu))

    rounded = lambda t: t.to(dtype).double()
    w_fc, w_proj = moe.c_fc.weight.detach().cpu().double(), moe.c_proj.weight.detach().cpu().double()
    x64, d64, gates, selected = x.double(), dy.double(), gates.cpu().double(), selected.cpu()
    d_x_rows = torch.zeros(T, k, H, dtype=torch.float64)
    d_fc, d_proj = torch.zeros_like(w_fc), torch.zeros_like(w_proj)
    d_gates = torch.zeros(T, k, dtype=torch.float64)
    for e in range(E):
        t, slot = (selected == e).nonzero(as_tuple=True)
        h = rounded(x64[t] @ w_fc[e].t())
        up, gate = h.chunk(2, dim=-1)
        out = rounded(rounded(swiglu64(gate, up)) @ w_proj[e].t())
        d_gates[t, slot] = (kept64(out.to(dtype)) * d64[t]).sum(-1)
        grad = rounded(d64[t] * gates[t, slot].unsqueeze(1))
        ku, kg = kept64(up.contiguous().to(dtype)), kept64(gate.contiguous().to(dtype))
        s = torch.sigmoid(kg)
        d_act = rounded(grad @ w_proj[e])
        d_h = rounded(torch.cat([d_act * kg * s, d_act * ku * (s + kg * s * (1 - s))], dim=1))
        d_proj[e] = grad.t() @ rounded(ku * kg * s)
        d_fc[e] = d_h.t() @ x64[t]
        d_x_rows[t, slot] = rounded(d_h @ w_fc[e])
    # the router adds its own gradient to x: softmax over the k logits, then its linear
    router = gates * (d_gates - (gates * d_gates).sum(-1, keepdim=True))
    d_logits = torch.zeros(T, E, dtype=torch.float64).scatter_(1, selected, rounded(router))
    d_x = d_x_rows.sum(1) + rounded(d_logits @ moe.gate.weight.detach().cpu().double())
    tol = 1e-5 if dtype == torch.float32 else 4 * torch.finfo(dtype).eps
    for name, got, want in [("d_x", xg.grad, d_x), ("d_fc", moe.c_fc.weight.grad, d_fc),
                            ("d_proj", moe.c_proj.weight.grad, d_proj)]:
        error = float((got.cpu().double() - want).norm() / want.norm())
        assert error <= tol, f"{name}: {error:.2e} of the norm, allowed {tol:.1e}"


def test_moe_layer_saves_less(gpu):
    """What a call leaves behind for its backward: the 8-bit tensors and the routing, no 16-bit rows."""
    announce("layer 8-bit memory")
    moe, x, _ = _layer(gpu, torch.bfloat16, 256, 256, 384, 4, 2, 41)

    def saved(layer):
        seen = {}

        def pack(t):
            if t.dtype in (torch.bfloat16, torch.int8, torch.uint8) and not isinstance(t, torch.nn.Parameter):
                seen[t.data_ptr()] = t.numel() * t.element_size()
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            layer(x.to(gpu).requires_grad_(True))
        weights = sum(p.numel() * 2 for p in layer.parameters())
        return sum(seen.values()), weights

    plain, _ = saved(moe)
    moe.checkpoint_8bit = True
    kept, _ = saved(moe)
    rows = 512 * (2 * 384 + 256) + 512 * 384
    assert kept < plain - rows  # a byte an element less (the scale bytes aside), two for the activation


def test_moe_layer_refuses_what_it_cannot_keep(gpu):
    import cute_kernels as ck

    announce("layer 8-bit refusals")
    x = randn((8, 64), torch.bfloat16, 51).to(gpu)
    for activation, bias in [(ck.swiglu_unchunked_cute, True), (torch.nn.functional.gelu, False)]:
        moe = ck.MoE_HIP(num_experts=2, num_experts_per_tok=1, hidden_size=64, intermediate_size=32,
                         activation_function=activation, is_glu=activation is ck.swiglu_unchunked_cute, add_bias=bias,
                         std=0.02).to(device=gpu, dtype=torch.bfloat16)
        moe.checkpoint_8bit = True
        with pytest.raises(ValueError, match="checkpoint_8bit"):
            moe(x)


# ---- streams and graphs -----------------------------------------------------------------------------------------------------
def _step(gpu, leaves, dy):
    """norm -> SwiGLU -> norm with a residual, all kept in 8 bits; returns the output and the gradients."""
    from cute_kernels import fused_residual_add_rmsnorm_cute, rmsnorm_cute, swiglu_unchunked_cute

    x, w = leaves
    a = rmsnorm_cute(x, w, 1e-5, checkpoint_8bit=True)
    b = swiglu_unchunked_cute(torch.cat([a, x], dim=-1), checkpoint_8bit=True)
    y, s = fused_residual_add_rmsnorm_cute(b, x, w, 1e-5, checkpoint_8bit=True)
    return (y.detach(), s.detach(), *torch.autograd.grad((y, s), leaves, (dy, dy)))


def test_side_stream_and_captured_step(gpu):
    if gpu.type != "cuda":
        pytest.skip("streams and graphs need the GPU")
    announce("8-bit step on streams and in graphs")
    dtype = torch.bfloat16

    def fresh(seed):
        return (randn((130, 1056), dtype, seed).to(gpu).requires_grad_(True),
                randn((1056,), dtype, seed + 1, 0.1, 1.0).to(gpu).requires_grad_(True)), randn((130, 1056), dtype, seed + 2).to(gpu)

    inputs = [fresh(100 + 10 * i) for i in range(4)]
    expected = [[t.clone() for t in _step(gpu, *i)] for i in inputs]
    torch.cuda.synchronize()
    # two streams at once
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for stream, i in zip(streams, inputs):
        with torch.cuda.stream(stream):
            results.append([_step(gpu, *i) for _ in range(5)][-1])
    torch.cuda.synchronize()
    for got, want in zip(results, expected):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # two graphs of the same step over static inputs, replayed in turn with other inputs and eager work between
    statics, graphs = [], []
    for n in range(2):
        static = fresh(200 + n)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(gpu, *static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _step(gpu, *static)
        statics.append((static, out))
        graphs.append(graph)
    for turn in range(4):
        for n in (0, 1):
            (leaves, dy), out = statics[n]
            (src, src_dy), want = inputs[(turn + n) % 4], expected[(turn + n) % 4]
            with torch.no_grad():
                leaves[0].copy_(src[0])
                leaves[1].copy_(src[1])
                dy.copy_(src_dy)
        for n in (0, 1):
            graphs[n].replay()
        _step(gpu, *inputs[turn])
        torch.cuda.synchronize()
        for n in (0, 1):
            want = expected[(turn + n) % 4]
            assert all(torch.equal(a, b) for a, b in zip(statics[n][1], want)), (turn, n)


def test_results_repeat_bit_for_bit(gpu):
    announce("8-bit step repeats")
    leaves = (randn((600, 544), torch.float32, 301).to(gpu).requires_grad_(True),
              randn((544,), torch.float32, 302, 0.1, 1.0).to(gpu).requires_grad_(True))
    dy = randn((600, 544), torch.float32, 303).to(gpu)
    first = _step(gpu, leaves, dy)
    for _ in range(2):
        assert all(torch.equal(a, b) for a, b in zip(first, _step(gpu, leaves, dy)))


def _every_operator(gpu, dtype):
    """All results and gradients of the operators with an 8-bit checkpoint, the pair and the balance loss."""
    import cute_kernels as ck

    out = []
    x, res = randn((37, 200), dtype, 401).to(gpu).requires_grad_(True), randn((37, 200), dtype, 402).to(gpu).requires_grad_(True)
    w = randn((200,), dtype, 403, 0.1, 1.0).to(gpu).requires_grad_(True)
    dy = randn((37, 200), dtype, 404).to(gpu)
    for weight in (w, None):
        leaves = (x, w) if weight is not None else (x,)
        y = ck.rmsnorm_cute(x, weight, None, checkpoint_8bit=True)
        out += [y, *torch.autograd.grad(y, leaves, dy)]
        y, s = ck.fused_residual_add_rmsnorm_cute(x, res, weight, 1e-6, checkpoint_8bit=True)
        out += [y, s, *torch.autograd.grad((y, s), (*leaves, res), (dy, dy))]
    y = ck.swiglu_cute(x.t(), res.t(), checkpoint_8bit=True)
    out += [y, *torch.autograd.grad(y, (x, res), dy.t())]
    y = ck.swiglu_unchunked_cute(x, checkpoint_8bit=True)
    out += [y, *torch.autograd.grad(y, x, dy[:, :100])]
    y = ck.swiglu_unchunked_cute(x[3], checkpoint_8bit=True)
    out += [y, *torch.autograd.grad(y, x, dy[3, :100])]
    codes, scales = ck.mx8_quantize_cute(x)
    out += [codes, scales, ck.mx8_dequantize_cute(codes, scales, dtype), *ck.mx8_quantize_cute(x[0])]
    ids = x.detach().float().topk(3, dim=-1).indices
    mask = (torch.arange(37) % 5 != 0).to(gpu)
    for chosen in (ids, None):
        balance, z, counts = ck.moe_balance_loss_cute(x, chosen, mask, top_k=3)
        out += [balance, z, counts, *torch.autograd.grad(2 * balance + z, x)]
    return [t.detach() for t in out]


@pytest.mark.parametrize("dtype", DTYPES)
def test_compiled_and_python_host_paths_agree(gpu, dtype, monkeypatch):
    """Eager calls on GPU tensors go through csrc/autograd.cpp, traced ones through the Python autograd functions and their
    custom ops: the same kernels on the same buffers, bit for bit."""
    from cute_kernels import _native
    from cute_kernels.utils import set_cute_tracing

    announce("host paths", dtype)
    if gpu.type == "cuda":
        assert _native.functions_for(torch.zeros(1, device=gpu)) is not None
    eager = _every_operator(gpu, dtype)
    if gpu.type == "cuda":
        monkeypatch.setattr(_native, "functions_for", lambda tensor: None)
        python = _every_operator(gpu, dtype)
        assert all(torch.equal(a, b) for a, b in zip(eager, python))
        monkeypatch.undo()
        assert _native.functions_for(torch.zeros(1, device=gpu)) is not None
    set_cute_tracing(True)
    try:
        assert _native.functions_for(torch.zeros(1, device=gpu)) is None
        traced = _every_operator(gpu, dtype)
    finally:
        set_cute_tracing(False)
    assert len(traced) == len(eager) and all(torch.equal(a, b) for a, b in zip(eager, traced))


def test_no_second_derivative(gpu):
    """The gradients of the kernels say nothing about how they depend on their inputs: differentiating through them is an
    error, also where the other terms of a sum could be differentiated."""
    import cute_kernels as ck

    announce("no second derivative")
    x, res = randn((5, 64), torch.float32, 60).to(gpu), randn((5, 64), torch.float32, 61).to(gpu)
    ids = torch.tensor([[0], [1], [2], [3], [4]], device=gpu)
    calls = [
        lambda v: ck.rmsnorm_cute(v, None, 1e-5, checkpoint_8bit=True).square().sum(),
        lambda v: ck.fused_residual_add_rmsnorm_cute(v, res, None, 1e-5, checkpoint_8bit=True)[0].square().sum(),
        lambda v: ck.swiglu_cute(v, res, checkpoint_8bit=True).square().sum(),
        lambda v: ck.swiglu_unchunked_cute(v, checkpoint_8bit=True).square().sum(),
        lambda v: ck.moe_balance_loss_cute(v, ids)[0].square(),
    ]
    for call in calls:
        v = x.clone().requires_grad_(True)
        (first,) = torch.autograd.grad(call(v), v)
        (again,) = torch.autograd.grad(call(v), v, create_graph=True)
        assert torch.equal(first, again.detach())
        with pytest.raises(RuntimeError):
            torch.autograd.grad(again.square().sum(), v)
        if gpu.type == "cuda":
            (again,) = torch.autograd.grad(call(v), v, create_graph=True)
            with pytest.raises(RuntimeError, match="no derivative of its own"):
                torch.autograd.grad((again.square() + v.pow(3)).sum(), v)


@pytest.fixture
def fresh_dynamo():
    torch._dynamo.reset()
    yield
    torch._dynamo.reset()


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_torch_compile(gpu, dtype, backend, fresh_dynamo):
    """Whole calls traced without a break: forward and backward the eager call's bit for bit (the same kernels)."""
    import cute_kernels as ck

    announce("8-bit under torch.compile", dtype)
    x, res, dy = (randn((33, 136), dtype, 70 + i).to(gpu) for i in range(3))
    weight = randn((136,), dtype, 73, 0.1, 1.0).to(gpu)
    ids = torch.arange(66, device=gpu).view(33, 2) % 136

    def norm(a, b, w):
        return ck.rmsnorm_cute(a, w, 1e-5, checkpoint_8bit=True)

    def residual(a, b, w):
        return ck.fused_residual_add_rmsnorm_cute(a, b, w, 1e-5, checkpoint_8bit=True)

    def glu(a, b, w):
        return ck.swiglu_cute(a, b, checkpoint_8bit=True)

    def unchunked(a, b, w):
        return ck.swiglu_unchunked_cute(a, checkpoint_8bit=True)

    def balance(a, b, w):
        return ck.moe_balance_loss_cute(a, ids, None)

    def pair(a, b, w):
        codes, scales = ck.mx8_quantize_cute(a)
        return codes, scales, ck.mx8_dequantize_cute(codes, scales, dtype)

    for function in (norm, residual, glu, unchunked, balance, pair):
        runs = []
        for call in (function, torch.compile(function, fullgraph=True, backend=backend)):
            leaves = [t.clone().requires_grad_(True) for t in (x, res, weight)]
            out = call(*leaves)
            out = list(out) if isinstance(out, tuple) else [out]
            through = [o for o in out if o.requires_grad]
            grads = []
            if through:
                seeds = [dy[tuple(slice(0, n) for n in o.shape)] if o.dim() else torch.ones_like(o) for o in through]
                grads = torch.autograd.grad(through, leaves, seeds, allow_unused=True)
            runs.append([t.detach() for t in (*out, *grads) if t is not None])
        assert len(runs[0]) == len(runs[1]), function.__name__
        assert all(torch.equal(a, b) for a, b in zip(*runs)), function.__name__


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_compiled_moe_layer(gpu, dtype, fresh_dynamo):
    """The layer with ``checkpoint_8bit`` and the balance loss on its logits, whole under torch.compile.  Sums of a few terms
    between the kernels may be rounded in another place than the eager call's: two steps of the type norm-wise."""
    announce("8-bit layer under torch.compile", dtype)
    moe, x, dy = _layer(gpu, dtype, 100, 64, 128, 4, 2, 80)
    moe.checkpoint_8bit = True
    mask = (torch.arange(100) % 7 != 0).to(gpu)

    def step(module, x):
        out, logits = module(x)
        balance, z, counts = moe.balance_loss(logits, mask)
        return out, balance + z, counts

    runs = []
    for call in (step, torch.compile(step, fullgraph=True)):
        xg = x.to(gpu, copy=True).requires_grad_(True)
        out, loss, counts = call(moe, xg)
        grads = torch.autograd.grad((out, loss), (xg, *moe.parameters()), (dy.to(gpu), torch.ones_like(loss)))
        runs.append([t.detach().double() for t in (out, loss, counts, *grads)])
    for a, b in zip(*runs):
        assert (a - b).norm() <= 2 * torch.finfo(dtype).eps * b.norm()

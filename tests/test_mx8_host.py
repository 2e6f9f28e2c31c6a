"""The 8-bit checkpoints and the balance loss without a GPU: refusals of the C entry points and of the Python functions, the
buffer layout, the reference forms against hand-made values, the kernels' registers, and the GPU tests' bodies on the CPU
emulation of the kernels (every operand in front of, or right behind, an inaccessible page)."""

import inspect

import pytest
import torch

import test_gpu_moe_balance as B
import test_gpu_mx8 as X
from test_abi_errors import ALIGN, BF16, DTYPE, F32, NULL, OK, P, SHAPE, WORKSPACE, lib  # noqa: F401 (lib: a fixture)
from test_emulated_device import (  # noqa: F401 (fixtures)
    emulated,
    emulated_lanes_reversed,
    library,
    library_with_lanes_reversed,
)


# ---- refusals of the C entry points ----------------------------------------------------------------------------------------
def test_pair_argument_checks(lib):  # noqa: F811
    f = lib.ck_mx8_quantize
    assert f(P, P, P, -1, 64, BF16, None) == SHAPE
    assert f(P, P, P, 4, -64, BF16, None) == SHAPE
    assert f(P, P, P, 4, 64, 7, None) == DTYPE
    assert f(P, None, P, 4, 64, BF16, None) == NULL
    assert f(P, P, None, 4, 64, BF16, None) == NULL
    assert f(P + 1, P, P, 4, 64, BF16, None) == ALIGN
    assert f(P, P, P, 1 << 29, 32, BF16, None) == SHAPE  # 2^31 pieces
    assert f(P, P, P, 1 << 40, 1, BF16, None) == SHAPE
    assert f(P, P, P, 1, 1 << 40, BF16, None) == SHAPE
    assert f(None, None, None, 0, 64, BF16, None) == OK
    assert f(None, None, None, 4, 0, BF16, None) == OK
    g = lib.ck_mx8_dequantize
    assert g(P, P, P, 4, -64, BF16, None) == SHAPE
    assert g(P, P, None, 4, 64, BF16, None) == NULL
    assert g(None, P, P, 4, 64, BF16, None) == NULL
    assert g(P, P, P + 1, 4, 64, F32, None) == ALIGN
    assert g(P, P, P, 4, 64, 3, None) == DTYPE
    assert g(None, None, None, 0, 64, BF16, None) == OK


def test_swiglu_argument_checks(lib):  # noqa: F811
    f = lib.ck_swiglu_forward_mx8
    #        gate up ldx y  gc uc ldc gs us lds rows H dtype stream
    assert f(P, P, 64, P, P, P, 64, P, P, 2, 4, 64, 7, None) == DTYPE
    assert f(P, P, 63, P, P, P, 64, P, P, 2, 4, 64, BF16, None) == SHAPE  # rows that overlap
    assert f(P, P, 64, P, P, P, 63, P, P, 2, 4, 64, BF16, None) == SHAPE
    assert f(P, P, 64, P, P, P, 64, P, P, 1, 4, 64, BF16, None) == SHAPE
    assert f(P, None, 64, P, P, P, 64, P, P, 2, 4, 64, BF16, None) == NULL
    assert f(P, P, 64, P, P, P, 64, None, P, 2, 4, 64, BF16, None) == NULL
    assert f(P, P + 1, 64, P, P, P, 64, P, P, 2, 4, 64, BF16, None) == ALIGN
    assert f(P, P, 64, P, P, P, 64, P, P, 2, 0, 64, BF16, None) == OK
    g = lib.ck_swiglu_backward_mx8
    #        gc uc ldc gs us lds dy dg du ldx act rows H dtype stream
    assert g(P, P, 64, P, P, 2, P, P, P, 63, None, 4, 64, BF16, None) == SHAPE
    assert g(P, P, 64, P, P, 2, P, None, P, 64, None, 4, 64, BF16, None) == NULL
    assert g(P, P, 64, P, P, 2, P, P, P, 64, P + 1, 4, 64, BF16, None) == ALIGN
    assert g(P, P, 64, P, P, 2, P, P, P, 64, None, -4, 64, BF16, None) == SHAPE
    h = lib.ck_moe_combine_backward_gates_mx8
    assert h(P, P, P, P, 4, 0, 64, BF16, None) == SHAPE
    assert h(P, None, P, P, 4, 2, 64, BF16, None) == NULL
    assert h(P, P, P, P + 1, 4, 2, 64, BF16, None) == ALIGN
    assert h(P, P, P, P, 4, 2, 64, 9, None) == DTYPE
    assert h(None, None, None, None, 0, 2, 64, BF16, None) == OK


def test_rmsnorm_argument_checks(lib):  # noqa: F811
    f = lib.ck_rmsnorm_forward_mx8
    #        x res w  y  sum codes scales rstd B H eps dtype stream
    assert f(P, None, P, P, None, P, P, P, 4, 65537, 1e-5, BF16, None) == SHAPE
    assert f(P, None, P, P, None, P, P, P, 1 << 31, 64, 1e-5, BF16, None) == SHAPE
    assert f(P, None, P, P, None, P, P, None, 4, 64, 1e-5, BF16, None) == NULL  # 1 / rms is always kept
    assert f(P, P, P, P, None, P, P, P, 4, 64, 1e-5, BF16, None) == NULL  # a residual, and nowhere for the sum
    assert f(P, None, P + 1, P, None, P, P, P, 4, 64, 1e-5, BF16, None) == ALIGN
    assert f(P, None, P, P, None, P, P, P + 2, 4, 64, 1e-5, BF16, None) == ALIGN
    assert f(P, None, P, P, None, P, P, P, 4, 64, 1e-5, 5, None) == DTYPE
    assert f(None, None, None, None, None, None, None, None, 0, 64, 1e-5, BF16, None) == OK
    g = lib.ck_rmsnorm_backward_mx8
    need = lib.ck_rmsnorm_backward_mx8_workspace_size(4, 64, BF16)
    assert need >= 64 * 4 and lib.ck_rmsnorm_backward_mx8_workspace_size(0, 64, BF16) == 0
    #        codes scales w dy rstd dsum dx dw ws bytes B H dtype stream
    assert g(P, P, P, P, P, None, P, None, P, need, 4, 64, BF16, None) == NULL  # weight, no weight_grad
    assert g(P, P, P, P, P, None, P, P, None, 0, 4, 64, BF16, None) == WORKSPACE
    assert g(P, P, P, P, P, None, P, P, P, need - 1, 4, 64, BF16, None) == WORKSPACE
    assert g(P, P, P, P, P, None, P, P, P + 4, need, 4, 64, BF16, None) == WORKSPACE
    assert g(P, P, None, P, P, None, None, None, None, 0, 4, 64, BF16, None) == NULL
    assert g(P, P, None, P, P, P + 1, P, None, None, 0, 4, 64, BF16, None) == ALIGN
    assert g(P, P, None, P, P, None, P, None, None, 0, 4, 65537, BF16, None) == SHAPE
    assert g(None, None, None, None, None, None, None, None, None, 0, 0, 64, BF16, None) == OK
    # both alignments of the operands fit the workspace that is asked for
    for H in (1, 8, 500, 1024, 1500, 2048, 4096, 8192, 9000, 16384, 20000, 65536):
        for rows in (1, 3, 1000, 100000):
            assert lib.ck_rmsnorm_backward_mx8_workspace_size(rows, H, F32) >= (H + 31) // 32 * 128


def test_balance_loss_argument_checks(lib):  # noqa: F811
    f = lib.ck_moe_balance_loss_forward
    #        logits ld ids mask balance z counts shares ws bytes T E k dtype stream
    ok = [P, 8, P, None, P, P, P, P, None, 0, 64, 8, 2, BF16, None]

    def with_(**changes):
        names = ["logits", "ld", "ids", "mask", "balance", "z", "counts", "shares", "ws", "bytes", "T", "E", "k", "dtype", "stream"]
        return f(*[changes.get(n, v) for n, v in zip(names, ok)])

    assert with_(ld=7) == SHAPE and with_(T=-1) == SHAPE and with_(E=0) == SHAPE and with_(k=0) == SHAPE
    assert with_(k=9) == SHAPE and with_(E=1025, ld=1025) == SHAPE and with_(T=1 << 30) == SHAPE  # 2^31 selections
    assert with_(dtype=4) == DTYPE
    assert with_(logits=None) == NULL and with_(ids=None) == NULL and with_(z=None) == NULL and with_(shares=None) == NULL
    assert with_(logits=P + 1) == ALIGN
    need = lib.ck_moe_balance_loss_workspace_size(100000, 8)
    assert need > 0 and lib.ck_moe_balance_loss_workspace_size(64, 8) == 0
    assert with_(T=100000) == WORKSPACE and with_(T=100000, ws=P, bytes=need - 1) == WORKSPACE
    g = lib.ck_moe_balance_loss_backward
    #        logits ld mask shares gb gz d T E dtype stream
    assert g(P, 7, None, P, P, P, P, 64, 8, BF16, None) == SHAPE
    assert g(P, 8, None, None, P, P, P, 64, 8, BF16, None) == NULL
    assert g(P, 8, None, P, P, P, P + 1, 64, 8, F32, None) == ALIGN
    assert g(P, 8, None, P, P, P, P, 64, 8, 9, None) == DTYPE
    assert g(None, 8, None, None, None, None, None, 0, 8, BF16, None) == OK


# ---- refusals of the Python functions ----------------------------------------------------------------------------------------
def test_functions_refuse_cpu_tensors_and_bad_operands():
    import cute_kernels as ck

    x = torch.randn(4, 64, requires_grad=True)
    w = torch.ones(64)
    for call in (lambda: ck.mx8_quantize_cute(x), lambda: ck.swiglu_cute(x, x, checkpoint_8bit=True),
                 lambda: ck.swiglu_unchunked_cute(x, checkpoint_8bit=True),
                 lambda: ck.rmsnorm_cute(x, w, 1e-5, checkpoint_8bit=True),
                 lambda: ck.fused_residual_add_rmsnorm_cute(x, x, w, 1e-5, checkpoint_8bit=True),
                 lambda: ck.mx8_dequantize_cute(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 2, dtype=torch.uint8),
                                                torch.float32),
                 lambda: ck.moe_balance_loss_cute(x, torch.zeros(4, 2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
    for eps in (None, 1e-5):
        with pytest.raises(ValueError, match="memory_efficient"):
            ck.rmsnorm_cute(x, w, eps, memory_efficient=True, checkpoint_8bit=True)
        with pytest.raises(ValueError, match="memory_efficient"):
            ck.fused_residual_add_rmsnorm_cute(x, x, w, eps, memory_efficient=True, checkpoint_8bit=True)
    with pytest.raises(AssertionError, match="hidden size"):
        ck.rmsnorm_cute(x, torch.ones(32), 1e-5, checkpoint_8bit=True)
    with pytest.raises(AssertionError, match="same dtype"):
        ck.rmsnorm_cute(x, w.half(), 1e-5, checkpoint_8bit=True)
    with pytest.raises(ValueError, match="longest supported row"):
        ck.rmsnorm_cute(torch.randn(1, 65537, requires_grad=True), None, 1e-5, checkpoint_8bit=True)
    with pytest.raises(AssertionError, match="same shape"):
        ck.swiglu_cute(x, x[:2], checkpoint_8bit=True)
    with pytest.raises(AssertionError, match="same shape"):
        ck.fused_residual_add_rmsnorm_cute(x, x[:2], w, 1e-5, checkpoint_8bit=True)
    with pytest.raises(AssertionError, match="even"):
        ck.swiglu_unchunked_cute(torch.randn(4, 63, requires_grad=True), checkpoint_8bit=True)


def test_binding_refuses_what_the_library_cannot_see(emulated):  # noqa: F811
    from cute_kernels import _C

    x = torch.randn(4, 64)
    codes, scales = torch.empty(4, 64, dtype=torch.int8), torch.empty(4, 2, dtype=torch.uint8)
    kept = torch.empty(_C.mx8_kept_offsets(4, 64, True)[2], dtype=torch.int8)
    for bad in (lambda: _C.mx8_quantize(x.t(), codes, scales), lambda: _C.mx8_quantize(x, codes[:2], scales),
                lambda: _C.mx8_quantize(x, codes.to(torch.uint8), scales), lambda: _C.mx8_quantize(x, codes, scales[:, :1]),
                lambda: _C.mx8_quantize(x.double(), codes, scales),
                lambda: _C.mx8_dequantize(codes, scales, x[:2]),
                lambda: _C.rmsnorm_forward_mx8(x, None, None, x.clone(), None, kept[:-1], 1e-5),
                lambda: _C.rmsnorm_forward_mx8(x, x, None, x.clone(), None, kept, 1e-5),
                lambda: _C.rmsnorm_forward_mx8(x, None, torch.ones(63), x.clone(), None, kept, 1e-5),
                lambda: _C.rmsnorm_backward_mx8(kept, torch.ones(64), x, None, x.clone(), None, None),
                lambda: _C.swiglu_forward_mx8(x, x[:2], x.clone(), kept),
                lambda: _C.swiglu_unchunked_backward_mx8(kept, x, x.clone()),
                lambda: _C.moe_balance_loss_forward(x, torch.zeros(4, 2), None, x[0, 0], x[0, 0], x[0], x[0], None)):
        with pytest.raises(ValueError):
            bad()


# ---- layout and reference forms -------------------------------------------------------------------------------------------------
def test_kept_buffer_layout():
    from cute_kernels import _C
    from cute_kernels.kernels.mx8 import kept_pair, new_kept

    assert _C.mx8_kept_offsets(3, 33, False) == (112, 118, 118)  # 99 codes, 6 scale bytes from 112 on
    assert _C.mx8_kept_offsets(3, 33, True) == (112, 128, 140)  # three floats from 128 on
    assert _C.mx8_kept_offsets(0, 64, True) == (0, 0, 0) and _C.mx8_kept_offsets(5, 0, False) == (0, 0, 0)
    kept = new_kept(6, 40, torch.device("cpu"))
    codes, scales = kept_pair(kept, (3, 2, 40))
    assert codes.shape == (3, 2, 40) and scales.shape == (3, 2, 2) and scales.dtype == torch.uint8
    scales.fill_(200)
    codes.fill_(1)
    assert kept[:240].eq(1).all() and kept[240:252].view(torch.uint8).eq(200).all() and kept.numel() == 252


@pytest.mark.parametrize("dtype", X.DTYPES)
@pytest.mark.parametrize("shape", [(7,), (3, 33), (5, 4, 96), (0, 8), (40, 1000)])
def test_reference_forms(dtype, shape):
    """mx8_*_torch and moe_balance_loss_torch, what the GPU results are also held to, against the definitions in 64 bits."""
    import cute_kernels as ck

    x = X.rows_like_activations(shape, dtype, 3)
    codes, scales = ck.mx8_quantize_torch(x)
    want = X.encode64(x)
    assert torch.equal(codes.long(), want[0]) and torch.equal(scales.long(), want[1])
    assert torch.equal(ck.mx8_dequantize_torch(codes, scales, dtype).double(), X.decode64(*want))
    logits, selected, mask = B.case(50, 12, 3, dtype, 4, 0.3)
    z = logits.double().requires_grad_(True)
    balance, z_loss, counts = ck.moe_balance_loss_torch(z, selected, mask)
    (d,) = torch.autograd.grad(0.5 * balance + 0.25 * z_loss, z)
    want = B.reference(logits, selected, mask, 0.5, 0.25)
    assert torch.equal(counts.long(), want[2])
    assert abs(float(balance) - float(want[0])) < 1e-6 and abs(float(z_loss) - float(want[1])) < 1e-5
    assert (d - want[3]).abs().max() < 1e-7


# ---- registers ------------------------------------------------------------------------------------------------------------------
def test_kernels_do_not_spill():
    """Streaming kernels, and RMSNorm up to 16384 elements a row (teams of up to 512 lanes, and 1024 lanes with two units): a
    kernel that spills runs several times slower without any other sign.  (Wider rows leave a lane more sums of the weight's
    gradient than its 128 registers hold beside the rest.)"""
    from cute_kernels._build import kernel_resources

    for source in ("mx8.hip", "moe_balance.hip"):
        spilling = sorted(n for n, r in kernel_resources(source).items() if r.get("scratch", 0) > 0)
        assert not spilling, spilling
    kernels = kernel_resources("mx8_rmsnorm.hip")
    narrow = {n: r for n, r in kernels.items() if "Li1024E" not in n or "Li1024ELi2E" in n}
    assert len(narrow) > 60
    spilling = sorted(n for n, r in narrow.items() if r.get("scratch", 0) > 0)
    assert not spilling, spilling


# ---- the GPU tests' bodies on the emulated device -----------------------------------------------------------------------------------
BF, F16, FP32 = torch.bfloat16, torch.float16, torch.float32
CASES = []


def case(function, **arguments):
    label = function.__name__[5:] + "-" + "-".join(str(v).replace("torch.", "") for v in arguments.values())
    CASES.append(pytest.param(function, arguments, id=label[:90]))


for dtype in (BF, F16, FP32):
    for shape in [(31,), (5, 7), (7, 33), (9, 72), (3, 5, 141)]:
        case(X.test_quantize_and_dequantize, dtype=dtype, shape=shape)
    case(X.test_layouts_of_the_pair, dtype=dtype)
    case(X.test_swiglu, dtype=dtype, shape=(37, 513))
    case(X.test_swiglu_activation_is_recomputed_at_the_kept_values, dtype=dtype)
    case(X.test_rmsnorm, dtype=dtype, has_weight=True, shape=(9, 520))
    case(X.test_fused_residual_add_rmsnorm, dtype=dtype, has_weight=True, shape=(5, 33))
    case(X.test_combine_backward_gates, dtype=dtype, shape=(65, 2, 1000))
    case(B.test_masked_and_odd_rows, dtype=dtype)
    case(B.test_layouts, dtype=dtype)
    case(B.test_balance_loss, dtype=dtype, padding=0.3, shape=(700, 16, 4))
case(X.test_known_blocks)
case(X.test_fp16_end_of_range)
case(X.test_swiglu_unchunked, dtype=BF, shape=(33, 2816))
case(X.test_swiglu_layouts_and_single_gradients)
for shape in [(1, 1), (4, 512), (2, 3, 1024), (3, 4104), (2, 8191)]:
    case(X.test_rmsnorm, dtype=BF, has_weight=True, shape=shape)
case(X.test_rmsnorm, dtype=FP32, has_weight=False, shape=(3, 4104))
case(X.test_rmsnorm_bad_rows_stay_alone)
case(X.test_rmsnorm_of_far_off_rows, dtype=BF)
case(X.test_rmsnorm_of_far_off_rows, dtype=FP32)
case(X.test_no_second_derivative)
case(X.test_gradients_against_differences)
case(X.test_moe_layer, dtype=BF, shape=(100, 64, 128, 4, 2))
case(X.test_compiled_and_python_host_paths_agree, dtype=BF)
for shape in [(1, 1, 1), (3, 2, 1), (4097, 8, 2), (513, 64, 6), (130, 160, 8), (65, 513, 2)]:
    case(B.test_balance_loss, dtype=FP32, padding=0.0, shape=shape)
case(B.test_even_load_loses_nothing_to_cancellation)
case(B.test_no_tokens)
case(B.test_against_differences)
case(B.test_refusals)


def _run(function, device, arguments, monkeypatch):
    if "monkeypatch" in inspect.signature(function).parameters:
        arguments = dict(arguments, monkeypatch=monkeypatch)
    function(device, **arguments)


@pytest.mark.parametrize("function,arguments", CASES)
def test_gpu_test_body_on_the_emulated_device(emulated, monkeypatch, function, arguments):  # noqa: F811
    _run(function, emulated, arguments, monkeypatch)


@pytest.mark.parametrize("function,arguments", [c for c in CASES if "float16" not in c.id or "bfloat16" in c.id])
def test_results_do_not_depend_on_the_order_of_the_lanes(emulated_lanes_reversed, monkeypatch, function, arguments):  # noqa: F811
    _run(function, emulated_lanes_reversed, arguments, monkeypatch)

"""The router's balance loss, z-loss and expert counts (cute_kernels/kernels/scattermoe/balance.py) against their formulas in
64 bits, through the public function.

Tolerances.  Losses are fp32.  A probability is within a dozen fp32 operations of its formula (difference from the maximum,
exponential, reciprocal, product), its row's sum of E terms besides: 2^-19 of the loss.  z squares a log-sum-exp that is a
sum of the maximum and a logarithm: 2^-19 of the two magnitudes.  Gradients: the same for p, and the difference in brackets
relative to the magnitudes it is made of, then rounded once to the logits' type.  lse itself is such a difference where the
maximum is negative (max + log sum can be near 0), so its magnitude is |max| + log sum.  The difference from the maximum is
itself rounded, to 2^-24 of it, and an error there is a relative one of the exponential: 2^-24 |logit - max| of p besides."""

import pytest
import torch

from helpers import DTYPES, announce, randn
from test_gpu_mx8 import assert_rounded

pytestmark = pytest.mark.gpu


def reference(logits, selected, mask, g_balance, g_z):
    """(balance, z, counts, d_logits, the magnitudes d_logits is a difference of) in 64 bits."""
    z = logits.double()
    T, E = z.shape
    k = selected.size(1)
    real = torch.ones(T, dtype=torch.bool) if mask is None else mask
    n = max(1, int(real.sum()))
    ids = selected[real].flatten()
    counts = torch.bincount(ids[(ids >= 0) & (ids < E)], minlength=E)
    f = counts.double() / (n * k)
    dead = (z <= torch.finfo(logits.dtype).min).all(1)
    p = torch.where((real & ~dead).unsqueeze(1), torch.softmax(z, 1), 0.0)
    lse = torch.where(real & ~dead, torch.logsumexp(z, 1), 0.0)
    top = torch.where(real & ~dead, z.amax(1) if T else lse, 0.0)
    balance = E * (f * p.sum(0) / n).sum()
    centred = f - f.mean()
    inner = centred - (p @ centred).unsqueeze(1)
    d = p * (g_balance * E / n * inner + g_z * 2 / n * lse.unsqueeze(1))
    size = p * (abs(g_balance) * E / n * (centred.abs() + (p @ centred.abs()).unsqueeze(1)) +
                abs(g_z) * 2 / n * (top.abs() + (lse - top).abs()).unsqueeze(1))
    size = size * (1 + torch.where(p > 0, top.unsqueeze(1) - z, 0.0) / 32)  # 2^-19 / 32 = 2^-24
    return balance, lse.square().sum() / n, counts, d, size


def check(gpu, logits, selected, mask, dtype, g_balance=0.5, g_z=0.25, ids_type=torch.int64, call=None):
    from cute_kernels import moe_balance_loss_cute

    lead = logits.shape[:-1]
    z = logits.to(gpu, copy=True).requires_grad_(True)
    balance, z_loss, counts = (call or moe_balance_loss_cute)(
        z, selected.to(ids_type).to(gpu), None if mask is None else mask.to(gpu))
    assert balance.shape == () and z_loss.shape == () and balance.dtype == z_loss.dtype == torch.float32
    (d,) = torch.autograd.grad(g_balance * balance + g_z * z_loss, z)
    assert d.shape == logits.shape and d.dtype == dtype and counts.dtype == torch.int32
    E, k = logits.size(-1), selected.size(-1)
    want = reference(logits.reshape(-1, E), selected.reshape(-1, k).long(), None if mask is None else mask.reshape(-1),
                     g_balance, g_z)
    assert torch.equal(counts.cpu().long(), want[2])
    balance, z_loss = balance.detach(), z_loss.detach()
    assert abs(float(balance) - float(want[0])) <= 2.0 ** -19 * float(want[0]) + 1e-30
    assert abs(float(z_loss) - float(want[1])) <= 2.0 ** -19 * float(want[1]) + 1e-30
    assert_rounded(d.reshape(-1, E), want[3], dtype, 2.0 ** -19, want[4], "d_logits")
    assert lead == d.shape[:-1]
    return balance.detach(), z_loss.detach(), counts, d


def case(T, E, k, dtype, seed, padding=0.0, scale=1.0):
    logits = (randn((T, E), torch.float32, seed, scale) + randn((E,), torch.float32, seed + 1)).to(dtype)
    selected = logits.float().topk(k, dim=-1).indices if T else torch.empty(0, k, dtype=torch.int64)
    mask = None
    if padding:
        mask = torch.rand(T, generator=torch.Generator().manual_seed(seed + 2)) >= padding
    return logits, selected, mask


# tokens per launch form: one workgroup up to 4096 (E <= 8) .. 64 (E > 256) tokens, then many
SHAPES = [(1, 1, 1), (1, 8, 2), (3, 2, 1), (64, 8, 2), (65, 5, 3), (4096, 8, 2), (4097, 8, 2), (700, 16, 4), (511, 64, 6),
          (513, 64, 6), (2500, 60, 6), (300, 100, 8), (130, 160, 8), (257, 256, 8), (70, 333, 3), (66, 512, 5), (65, 513, 2),
          (200, 1000, 7), (130, 1024, 8), (9000, 3, 3)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("padding", [0.0, 0.3])
@pytest.mark.parametrize("shape", SHAPES)
def test_balance_loss(gpu, dtype, padding, shape):
    announce("balance", dtype, padding, shape)
    check(gpu, *case(*shape, dtype, 1, padding), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_only_one_of_the_losses_is_used(gpu, dtype):
    from cute_kernels import moe_balance_loss_cute

    announce("balance, one loss", dtype)
    logits, selected, mask = case(300, 24, 3, dtype, 5, 0.2)
    for which, weights in ((0, (1.0, 0.0)), (1, (0.0, 1.0))):
        z = logits.to(gpu, copy=True).requires_grad_(True)
        (d,) = torch.autograd.grad(moe_balance_loss_cute(z, selected.to(gpu), mask.to(gpu))[which], z)
        want = reference(logits, selected, mask, *weights)
        assert_rounded(d, want[3], dtype, 2.0 ** -19, want[4], "one loss")


def test_even_load_loses_nothing_to_cancellation(gpu):
    """Counts that differ by one in ten thousand: f_e - sum f p is a thousandth of a per cent of f, and is still held to the
    magnitudes of the *centred* shares (`reference`), not to those of f itself."""
    announce("balance, even load")
    T, E, k = 10007, 16, 2
    logits = randn((T, E), torch.float32, 6)
    selected = (torch.arange(T * k) % E).view(T, k)
    out = check(gpu, logits, selected, None, torch.float32, g_z=0.0)
    assert abs(float(out[0]) - 1.0) < 1e-4  # the loss of an even load


@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_and_odd_rows(gpu, dtype):
    """Padding may hold anything; a dropped slot counts nowhere; experts masked by -inf or the type's lowest value; a row
    of -inf alone; logits far out."""
    announce("balance, odd rows", dtype)
    inf = float("inf")
    logits, selected, _ = case(40, 12, 2, dtype, 7)
    mask = torch.ones(40, dtype=torch.bool)
    mask[3:9] = False
    dirty, dirty_ids = logits.clone(), selected.clone()
    dirty[3] = float("nan")
    dirty[4] = inf
    dirty[5, 2] = -inf
    dirty[6] = torch.finfo(dtype).max
    dirty_ids[3:9] = torch.tensor([10 ** 12, -(10 ** 12)])
    clean = check(gpu, logits, selected, mask, dtype)
    other = [t.detach() for t in _run(gpu, dirty, dirty_ids, mask)]
    assert all(torch.equal(a, b) for a, b in zip(clean, other))
    assert not other[3][3:9].any()
    ids = selected.clone()
    ids[10, 0], ids[11, 1], ids[12] = -1, 12, torch.tensor([2 ** 40, -7])
    check(gpu, logits, ids, None, dtype)
    odd = logits.clone()
    odd[0, 5:] = -inf
    odd[1, :11] = torch.finfo(dtype).min
    odd[2] = torch.finfo(dtype).min
    odd[20] = -inf
    odd[21, 0] = 80.0
    odd[22] = 500.0
    check(gpu, odd, selected, None, dtype)
    # no token counts: zeros
    nothing = _run(gpu, odd, selected, torch.zeros(40, dtype=torch.bool))
    assert not any(t.any() for t in nothing)
    # a NaN in a counting row is a NaN in the losses, and in that row's gradient alone
    bad = logits.clone()
    bad[7, 3] = float("nan")
    balance, z, counts, d = _run(gpu, bad, selected, None)
    assert balance.isnan() and z.isnan()
    assert d[7].isnan().all() and d[torch.arange(40) != 7].isfinite().all()


def _run(gpu, logits, selected, mask):
    from cute_kernels import moe_balance_loss_cute

    z = logits.to(gpu, copy=True).requires_grad_(True)
    balance, z_loss, counts = moe_balance_loss_cute(z, selected.to(gpu), None if mask is None else mask.to(gpu))
    (d,) = torch.autograd.grad(0.5 * balance + 0.25 * z_loss, z)
    return balance.detach(), z_loss.detach(), counts, d


def test_no_tokens(gpu):
    from cute_kernels import moe_balance_loss_cute

    announce("balance, no tokens")
    z = torch.empty(0, 8, device=gpu, requires_grad=True)
    balance, z_loss, counts = moe_balance_loss_cute(z, torch.empty(0, 2, dtype=torch.int64, device=gpu))
    (d,) = torch.autograd.grad(balance + z_loss, z)
    assert float(balance) == 0.0 and float(z_loss) == 0.0 and not counts.any() and d.shape == (0, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(gpu, dtype):
    """Leading dimensions, int32 ids, logits that are a column range or every other column of a wider matrix, unaligned rows."""
    from cute_kernels import moe_balance_loss_cute

    announce("balance layouts", dtype)
    logits, selected, mask = case(6 * 35, 16, 2, dtype, 8, 0.2)
    check(gpu, logits.view(6, 35, 16), selected.view(6, 35, 2), mask.view(6, 35), dtype, ids_type=torch.int32)
    wide, ids, _ = case(50, 56, 2, dtype, 9)
    for change in (lambda t: t[:, 8:24], lambda t: t[:, 3:19], lambda t: t[:, ::2], lambda t: t[::2, :20], lambda t: t[:16, :16].t()):
        part = change(wide)
        ids = part.float().topk(2, dim=-1).indices
        z = wide.to(gpu, copy=True).requires_grad_(True)
        balance, z_loss, counts = moe_balance_loss_cute(change(z), ids.to(gpu))
        (d,) = torch.autograd.grad(balance + z_loss, z)
        want = reference(part, ids, None, 1.0, 1.0)
        assert torch.equal(counts.cpu().long(), want[2])
        assert abs(float(balance) - float(want[0])) <= 2.0 ** -19 * float(want[0])
        assert_rounded(change(d), want[3], dtype, 2.0 ** -19, want[4], "layout")
        left = d.clone()
        change(left).zero_()
        assert not left.any()
    # an expanded row: one token's logits for all (stride 0)
    row = randn((1, 8), dtype, 10)
    z = row.to(gpu, copy=True).requires_grad_(True)
    many = torch.arange(40).remainder(8).view(20, 2)
    balance, z_loss, _ = moe_balance_loss_cute(z.expand(20, 8), many.to(gpu))
    want = reference(row.expand(20, 8), many, None, 1.0, 0.0)
    assert abs(float(balance) - float(want[0])) <= 2.0 ** -19 * float(want[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_selected_by_the_logits_and_the_layers_method(gpu, dtype):
    import cute_kernels as ck

    announce("balance of the layer", dtype)
    # distinct logits: topk leaves the order of ties open
    logits = torch.stack([torch.randperm(24, generator=torch.Generator().manual_seed(i)) for i in range(90)]).to(dtype) / 8
    ids = logits.float().topk(3, dim=-1).indices
    a = ck.moe_balance_loss_cute(logits.to(gpu), top_k=3)
    b = ck.moe_balance_loss_cute(logits.to(gpu), ids.to(gpu))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    moe = ck.MoE_HIP(num_experts=8, num_experts_per_tok=2, hidden_size=64, intermediate_size=128,
                     activation_function=ck.swiglu_unchunked_cute, is_glu=True, add_bias=False, std=0.05)
    with torch.no_grad():
        for i, p in enumerate(moe.parameters()):
            p.copy_(randn(p.shape, torch.float32, 60 + i, 0.1))
    moe = moe.to(device=gpu, dtype=dtype)
    moe.checkpoint_8bit = True
    x = randn((2, 50, 64), dtype, 63).to(gpu).requires_grad_(True)
    mask = torch.ones(2, 50, dtype=torch.bool, device=gpu)
    mask[1, 30:] = False
    y, router_logits = moe(x)
    balance, z, counts = moe.balance_loss(router_logits, mask)
    with torch.no_grad():
        _, _, selected = moe._compute_routing_weights(x.view(-1, 64))
    want = reference(router_logits.detach().cpu(), selected.cpu(), mask.view(-1).cpu(), 1.0, 1.0)
    assert torch.equal(counts.cpu().long(), want[2]) and int(counts.sum()) == 80 * 2
    assert abs(float(balance) - float(want[0])) <= 2.0 ** -19 * float(want[0])
    # the whole step as it would be used: the auxiliary losses add their gradient to the router's
    (d_gate,) = torch.autograd.grad(y.float().sum() + 0.01 * balance + 0.001 * z, moe.gate.weight, retain_graph=True)
    (d_plain,) = torch.autograd.grad(y.float().sum(), moe.gate.weight, retain_graph=True)
    (d_aux,) = torch.autograd.grad(100 * balance + 10 * z, moe.gate.weight)
    exact = reference(router_logits.detach().cpu(), selected.cpu(), mask.view(-1).cpu(), 100.0, 10.0)[3].t() @ x.detach().cpu().double().view(-1, 64)
    assert (d_aux.cpu().double() - exact).norm() <= 4 * torch.finfo(dtype).eps * exact.norm() + 1e-5 * exact.norm()
    assert d_gate.isfinite().all() and d_plain.isfinite().all()


def test_against_differences(gpu):
    """Central differences of the losses in 64 bits at a few logits, step 1e-5: their second-order error is 1e-9 or so."""
    from cute_kernels import moe_balance_loss_cute

    announce("balance differences")
    logits, selected, mask = case(12, 6, 2, torch.float32, 11, 0.2)
    z = logits.to(gpu, copy=True).requires_grad_(True)
    balance, z_loss, _ = moe_balance_loss_cute(z, selected.to(gpu), mask.to(gpu))
    (d,) = torch.autograd.grad(balance + 0.1 * z_loss, z)

    def loss(v):
        b, zz, *_ = reference(v, selected, mask, 1.0, 1.0)
        return float(b + 0.1 * zz)

    want = torch.zeros(12, 6, dtype=torch.float64)
    for t in range(12):
        for e in range(6):
            step = torch.zeros(12, 6, dtype=torch.float64)
            step[t, e] = 1e-5
            want[t, e] = (loss(logits.double() + step) - loss(logits.double() - step)) / 2e-5
    assert (d.cpu().double() - want).abs().max() <= 1e-8 + 2.0 ** -19 * want.abs().max()


def test_refusals(gpu):
    from cute_kernels import moe_balance_loss_cute

    announce("balance refusals")
    z = torch.randn(4, 8, device=gpu)
    ids = torch.zeros(4, 2, dtype=torch.int64, device=gpu)
    with pytest.raises(ValueError):
        moe_balance_loss_cute(z)
    with pytest.raises(ValueError):
        moe_balance_loss_cute(z, ids[:3])
    with pytest.raises(ValueError):
        moe_balance_loss_cute(z, ids, top_k=3)
    with pytest.raises(ValueError):
        moe_balance_loss_cute(z, ids.float())
    with pytest.raises(ValueError):
        moe_balance_loss_cute(z, ids, torch.ones(4, device=gpu))
    with pytest.raises(ValueError):
        moe_balance_loss_cute(z, ids, torch.ones(3, dtype=torch.bool, device=gpu))
    with pytest.raises(ValueError):
        moe_balance_loss_cute(z.double(), ids)
    with pytest.raises(RuntimeError):
        moe_balance_loss_cute(torch.randn(4, 1025, device=gpu), ids)
    with pytest.raises(RuntimeError):
        moe_balance_loss_cute(z[:, :1].contiguous(), ids)  # two experts of one


def test_streams_and_graphs(gpu):
    if gpu.type != "cuda":
        pytest.skip("streams and graphs need the GPU")
    from cute_kernels import moe_balance_loss_cute

    announce("balance graphs")

    def step(z, ids, mask):
        balance, z_loss, counts = moe_balance_loss_cute(z, ids, mask)
        (d,) = torch.autograd.grad(balance + z_loss, z)
        return balance.detach(), z_loss.detach(), counts, d

    def fresh(seed, T, E, k):
        logits, ids, mask = case(T, E, k, torch.bfloat16, seed, 0.3)
        return logits.to(gpu).requires_grad_(True), ids.to(gpu), mask.to(gpu)

    for T, E, k in ((6000, 16, 2), (100, 16, 2)):  # many workgroups and one
        inputs = [fresh(20 + i, T, E, k) for i in range(3)]
        expected = [[t.clone() for t in step(*i)] for i in inputs]
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        torch.cuda.synchronize()
        results = []
        for stream, i in zip(streams, inputs):
            with torch.cuda.stream(stream):
                results.append([step(*i) for _ in range(5)][-1])
        torch.cuda.synchronize()
        for got, want in zip(results, expected):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        statics, graphs = [], []
        for n in range(2):
            static = fresh(30 + n, T, E, k)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(*static)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step(*static)
            statics.append((static, out))
            graphs.append(graph)
        for turn in range(4):
            for n in (0, 1):
                with torch.no_grad():
                    for a, b in zip(statics[n][0], inputs[(turn + n) % 3]):
                        a.copy_(b)
            for n in (0, 1):
                graphs[n].replay()
            step(*inputs[turn % 3])
            torch.cuda.synchronize()
            for n in (0, 1):
                assert all(torch.equal(a, b) for a, b in zip(statics[n][1], expected[(turn + n) % 3])), (turn, n)


def test_offsets_beyond_32_bits(gpu):
    """Only tokens behind the 2^32-nd logit count: the losses are those of these tokens alone.  One workgroup holds them all in
    either call, in another order: sums of 300 terms (300 * 2^-24 of them), the gradient rounded to bf16 behind that."""
    if gpu.type != "cuda":
        pytest.skip("too large for the emulation")
    from cute_kernels import moe_balance_loss_cute

    announce("balance offsets")
    T, E, k = 2 ** 22 + 1000, 1024, 2
    logits, ids, _ = case(300, E, k, torch.bfloat16, 41, 0.0)
    z = torch.zeros(T, E, dtype=torch.bfloat16, device=gpu)
    z[-300:] = logits.to(gpu)
    selected = torch.zeros(T, k, dtype=torch.int64, device=gpu)
    selected[-300:] = ids.to(gpu)
    mask = torch.zeros(T, dtype=torch.bool, device=gpu)
    mask[-300:] = True
    small = logits.to(gpu).requires_grad_(True)
    want = moe_balance_loss_cute(small, ids.to(gpu))
    (want_d,) = torch.autograd.grad(want[0] + want[1], small)
    z.requires_grad_(True)
    got = moe_balance_loss_cute(z, selected, mask)
    (d,) = torch.autograd.grad(got[0] + got[1], z)
    assert torch.equal(got[2], want[2])
    for a, b in zip(got[:2], want[:2]):
        assert abs(float(a) - float(b)) <= 300 * 2.0 ** -24 * abs(float(b))
    # the sums reach a token's gradient through nothing but the counts: the same bits
    assert torch.equal(d[-300:], want_d) and not d[:-300].any()

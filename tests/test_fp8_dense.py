"""Dense layers in 8-bit floating point: rounding to blocks, products,
gradients from 8-bit checkpoints, refusals.

Tolerances. What is stored has to be equal to the bit. A product of k terms
adds in 32 bits: each addition is off by at most a step of 2^-23 of what it
adds up to (half a step where it rounds, a whole one where it truncates), so
the sum by at most (k + 8) * 2^-23 * sum |a||b|; the result's own rounding is
half a step of its type. A sigmoid is at most 1/4 as steep, and its own
exp and division are off by less than 2^-20 of it.
"""

import threading

import pytest
import torch

from elasticdl_amd.ops import (
    fp8,
    native_available,
    reference,
    require_native,
)
from elasticdl_amd.ops.fp8 import fp8_dense, quantize_fp8, quantize_fp8_weight
from test_embedding_ops import Elsewhere

TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def randn(*shape, seed=0, dtype=torch.float32, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g).to(dtype).to(device)


def values(x, tile=False):
    """q(x) in 64 bits, by the reference on the CPU."""
    x = x.detach().cpu()
    q, s = reference.fp8_quantize(x, tile)
    return reference.fp8_values(q, s, x.shape[1]).double()


def product_bound(a, b, k, extra, dtype):
    """How far a b^T may be off; extra is what is added to it."""
    bound = ((k + 8) * 2.0 ** -23) * (a.abs() @ b.abs().t() + extra)
    if dtype != torch.float32:
        pad = lambda t: torch.nn.functional.pad(t.abs(), (0, -t.shape[1] % 8)).view(t.shape[0], -1, 8)  # noqa: E731
        a, b = pad(a), pad(b)
        for at in range(0, a.shape[0], 16):
            rows = a[at:at + 16].unsqueeze(1)
            bound[at:at + 16] += 7 * 2.0 ** -13 * sum(
                (rows[:, :, g] * b[:, g]).amax(-1) for g in range(a.shape[1]))
    return bound


def check(got, want, bound, dtype):
    got = got.detach().cpu()
    assert got.dtype == dtype
    bound = bound + half_step(dtype) * (want.abs() + bound) \
        + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), \
        f"off by {float((off / bound).max())} of what is allowed"


# ------------------------------- rounding ---------------------------------
def test_block_values_against_a_plain_rounding():
    """Against e4m3 written out: the nearest of 2^e * (1 + m/8) and of the
    multiples of 2^-9, ties to the even one."""
    x = torch.cat([randn(3, 256), randn(3, 256, seed=1) * 1e-4])
    grid = [0.0] + [m * 2.0 ** -9 for m in range(1, 8)]
    for e in range(-6, 9):
        grid += [2.0 ** e * (1 + m / 8) for m in range(8)]
    grid = torch.tensor(grid[:-1], dtype=torch.float64)  # 480 is NaN's
    assert grid[-1] == 448
    for row, got in zip(x, quantize_fp8(x).dequantize()):
        for blk in range(2):
            v = row[blk * 128:][:128].double()
            e = -126
            while v.abs().max() > 448 * 2.0 ** e:
                e += 1
            u = (v / 2.0 ** e).abs()
            d = (u.unsqueeze(1) - grid).abs()
            near = d.min(1).values.unsqueeze(1) == d
            even = torch.arange(len(grid)) % 2 == 0
            pick = torch.where(near.sum(1) > 1, (near & even).int().argmax(1),
                               near.int().argmax(1))
            want = grid[pick] * 2.0 ** e * torch.sign(v)
            assert torch.equal(got[blk * 128:][:128].double(), want)


def test_scale_slots_are_a_permutation_of_each_64_rows():
    s = reference.fp8_scale_slots(256)
    assert torch.equal(s.view(4, 64).sort(1).values,
                       torch.arange(256).view(4, 64))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("tile", [False, True])
def test_values_that_are_not_finite_stay_with_themselves(device, tile):
    x = randn(130, 300)
    want = quantize_fp8(x * 1.0, tile).dequantize()
    y = x.clone()
    bad = [(0, 0, float("inf")), (5, 130, float("-inf")),
           (129, 299, float("nan"))]
    for r, c, v in bad:
        y[r, c] = v
        x[r, c] = 0.0
    want = quantize_fp8(x, tile).dequantize()
    got = quantize_fp8(y.to(device), tile).dequantize().cpu()
    for r, c, _ in bad:
        assert torch.isnan(got[r, c])
        got[r, c] = 0.0
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (129, 127), (64, 1000),
                                   (300, 257), (2, 8192), (1000, 24)])
def test_quantise_is_the_reference_to_the_bit(shape, dtype, tile):
    from elasticdl_amd.ops import _C

    x = randn(*shape, dtype=dtype) * torch.exp(randn(shape[1], seed=1) * 3).to(dtype)
    q, s, qt, st = _C.fp8_quantize(x.cuda(), tile, True, True)
    for a, b, src in ((q, s, x), (qt, st, x.t())):
        wq, ws = reference.fp8_quantize(src, tile)
        slots = reference.fp8_scale_slots(src.shape[0])
        assert torch.equal(a.cpu(), wq)
        assert torch.equal(b.cpu()[:, slots], ws[:, slots])
    only = _C.fp8_quantize(x.cuda(), tile, False, True)
    assert only[0] is None and torch.equal(only[2], qt)


@pytest.mark.gpu
def test_quantise_extremes_to_the_bit():
    x = torch.tensor([0.0, -0.0, 1e-45, -1e-40, 3e38, -3.4028235e38, 448.0,
                      449.0, 464.0, 480.0, 2.0 ** -126, 1.75, 1.7500001,
                      2.0 ** -149, 1.0, 2.0 ** -130])
    x = torch.cat([x.repeat_interleave(128).view(16, 128),
                   x.view(16, 1).expand(16, 128) * randn(16, 128)])
    q, s = reference.fp8_quantize(x, False)
    got = quantize_fp8(x.cuda())
    slots = reference.fp8_scale_slots(32)
    assert torch.equal(got.scale.cpu()[:, slots], s[:, slots])
    assert torch.equal(got.data.cpu(), q)  # NaN's byte too


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1])
def test_quantise_takes_strided_rows(offset):
    base = randn(40, 600, dtype=torch.bfloat16).cuda()
    x = base[::2, offset:offset + 300]
    got = quantize_fp8(x).dequantize()
    assert torch.equal(got, quantize_fp8(x.contiguous()).dequantize())
    assert torch.equal(got.cpu().double(), values(x))
    t = base.t()  # neighbours in a row are strided: copied
    assert torch.equal(quantize_fp8(t).dequantize().cpu().double(), values(t))


# ------------------------------- products ---------------------------------
SIZES = [(1, 16, 1), (2, 129, 17), (16, 640, 400), (17, 624, 400),
         (33, 100, 7), (128, 128, 128), (129, 1000, 130), (257, 257, 513),
         (1003, 384, 64), (40, 2049, 300)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["none", "relu", "sigmoid"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward(m, k, n, act, device):
    dtype = TYPES[(m + k + n) % 3]
    x = randn(m, k, dtype=dtype, device=device)
    w = (randn(n, k, seed=1) / k ** 0.5).to(dtype).to(device)
    b = None if n % 2 else randn(n, seed=2, dtype=dtype, device=device)
    xq, wq = values(x), values(w, True)
    add = torch.zeros(n).double() if b is None else b.cpu().double()
    z = xq @ wq.t() + add
    bound = product_bound(xq, wq, k, add.abs(), dtype)
    want = z
    if act == "relu":
        want = z.clamp(min=0)
    if act == "sigmoid":
        want = torch.sigmoid(z)
        bound = bound / 4 + 2.0 ** -20 * want
    with torch.no_grad():
        y = fp8_dense(x, w, b, act)
        check(y, want, bound, dtype)
        check(fp8_dense(x, quantize_fp8_weight(w), b, act), want, bound, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(4096, 256, 4096), (4000, 400, 4100),
                                   (130, 8192, 130)])
def test_forward_of_large_products(m, k, n):
    """One workgroup's tile of 256, edges of it, and a split contraction."""
    x = randn(m, k, dtype=torch.bfloat16)
    w = (randn(n, k, seed=1) / k ** 0.5).bfloat16()
    b = randn(n, seed=2)
    xq, wq = values(x), values(w, True)
    rows = torch.arange(0, m, max(1, m // 17))
    with torch.no_grad():
        y = fp8_dense(x.cuda(), w.cuda(), b.cuda(), "relu")
        one = fp8_dense(x.cuda()[:1], w.cuda(), b.cuda(), "relu")
    z = xq[rows] @ wq.t() + b.double()
    bound = product_bound(xq[rows], wq, k, b.double().abs(), torch.bfloat16)
    check(y[rows.cuda()], z.clamp(min=0), bound, torch.bfloat16)
    check(one, z[:1].clamp(min=0), bound[:1], torch.bfloat16)


@pytest.mark.parametrize("device", DEVICES)
def test_leading_dimensions_and_no_rows(device):
    w = randn(24, 40, device=device)
    x = randn(3, 5, 40, device=device)
    y = fp8_dense(x, w)
    assert y.shape == (3, 5, 24)
    assert torch.equal(y.view(15, 24), fp8_dense(x.view(15, 40), w))
    assert fp8_dense(x[0, 0], w).shape == (24,)
    empty = torch.zeros(0, 40, device=device, requires_grad=True)
    w.requires_grad_(True)
    y = fp8_dense(empty, w, None, "relu")
    assert y.shape == (0, 24)
    dx, dw = torch.autograd.grad(y.sum(), (empty, w))
    assert dx.shape == (0, 40) and not dw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 5, 16, 17])
def test_few_rows_of_strided_and_odd_inputs(m):
    base = randn(2 * m, 700, dtype=torch.float16).cuda()
    w = quantize_fp8_weight(randn(33, 301, seed=1).cuda())
    with torch.no_grad():
        for x in (base[::2, 3:304], base[:1, 3:304].expand(m, 301)):
            got = fp8_dense(x, w)
            xq = values(x)
            wq = w.dequantize().cpu().double()
            check(got, xq @ wq.t(), product_bound(xq, wq, 301, 0.0, torch.float16),
                  torch.float16)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("m", [3, 40])
def test_not_finite_inputs_spoil_their_own_rows(device, m):
    x = randn(m, 200)
    x[1, 150] = float("inf")
    x[2, 3] = float("nan")
    w = randn(20, 200, seed=1)
    with torch.no_grad():
        y = fp8_dense(x.to(device), w.to(device)).cpu()
        clean = fp8_dense(torch.nan_to_num(x, 0.0, 0.0, 0.0).to(device),
                          w.to(device)).cpu()
    assert torch.isnan(y[1:3]).all()
    keep = [r for r in range(m) if r not in (1, 2)]
    assert torch.equal(y[keep], clean[keep])


# ------------------------------- gradients --------------------------------
def whole_numbers(*shape, seed, most=4, device="cpu", dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most, most + 1, shape, generator=g).to(dtype).to(device)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("m,k,n", [(1, 16, 3), (50, 130, 40), (129, 100, 257),
                                   (700, 64, 128)])
def test_gradients_of_whole_numbers_are_exact(m, k, n, act, device):
    """Whole numbers up to 16 are e4m3's own values and their sums here are
    exact, so the layer and its gradients are the plain layer's, and
    differences of a step of one are the gradients."""
    leaf = lambda *s, seed: whole_numbers(*s, seed=seed, device=device).requires_grad_(True)  # noqa: E731
    x, w, b = leaf(m, k, seed=0), leaf(n, k, seed=1), leaf(n, seed=2)
    dy = whole_numbers(m, n, seed=3, device=device)
    y = fp8_dense(x, w, b, act)
    got = torch.autograd.grad(y, (x, w, b), dy)
    z = (x.detach().cpu().double() @ w.detach().cpu().double().t()
         + b.detach().cpu().double())
    dz = dy.cpu().double() * ((z > 0) if act == "relu" else 1.0)
    assert torch.equal(y.detach().cpu().double(),
                       z.clamp(min=0) if act == "relu" else z)
    want = (dz @ w.detach().cpu().double(), dz.t() @ x.detach().cpu().double(),
            dz.sum(0))
    for a, c in zip(got, want):
        assert torch.equal(a.cpu().double(), c)
    if act == "none":
        with torch.no_grad():
            loss = lambda p, q: float((fp8_dense(p, q, b) * dy).double().sum())  # noqa: E731
            base = loss(x, w)
            for r, c in ((0, 0), (m - 1, k - 1), (m // 2, k // 3)):
                p = x.detach().clone()
                p[r, c] += 1
                assert loss(p, w) - base == float(got[0][r, c])
            q = w.detach().clone()
            q[n - 1, k // 2] += 1
            assert loss(x, q) - base == float(got[1][n - 1, k // 2])


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("act", ["none", "relu", "sigmoid"])
@pytest.mark.parametrize("m,k,n", [(1, 40, 1), (100, 624, 400), (257, 130, 17),
                                   (2050, 77, 130)])
def test_gradients_against_the_formula(m, k, n, act, device):
    dtype = TYPES[(m + n) % 3]
    x = randn(m, k, dtype=dtype, device=device).requires_grad_(True)
    w = (randn(n, k, seed=1) / k ** 0.5).to(device).requires_grad_(True)
    b = randn(n, seed=2, dtype=dtype, device=device).requires_grad_(True)
    dy = randn(m, n, seed=3, dtype=dtype, device=device)
    y = fp8_dense(x, w, b, act)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    # the gradient before the activation, in 32 bits as it is rounded from
    dz = dy.cpu().float()
    if act == "relu":
        dz = dz * (y.detach().cpu() > 0)
    elif act == "sigmoid":
        o = y.detach().cpu().float()
        dz = dz * o * (1 - o)
    zr, zc = values(dz), values(dz.t())
    wq, xc = values(w, True), values(x.detach().t())
    check(dx, zr @ wq, product_bound(zr, wq.t(), n, 0.0, dtype), dtype)
    check(dw, zc @ xc.t(), product_bound(zc, xc, m, 0.0, torch.float32),
          torch.float32)
    check(db, dz.double().sum(0), (m + 8) * 2.0 ** -23 * dz.double().abs().sum(0),
          dtype)


# ----------------------------- relu's gates -------------------------------
def gates(x, w, b, rows):
    """Which outputs of these rows let a gradient through. The bias's gradient
    of 2^i in the i-th of 24 rows is their bits, exact in 32 bits."""
    b = b.requires_grad_(True)
    y = fp8_dense(x, w, b, "relu")
    found = []
    for at in range(0, len(rows), 24):
        part = rows[at:at + 24]
        powers = 2.0 ** torch.arange(-9, len(part) - 9)
        dy = torch.zeros_like(y)
        dy[part] = powers.to(y.dtype).to(y.device).unsqueeze(1)
        db, = torch.autograd.grad(y, b, dy, retain_graph=True)
        bits = (db.cpu() * 512).long().unsqueeze(0)
        found.append((bits >> torch.arange(len(part)).unsqueeze(1)) & 1)
    return torch.cat(found).bool()


GATE_SIZES = [(1, 64, 17), (33, 136, 40), (300, 640, 130),
              (130, 4096, 72),      # a split contraction
              (2041, 512, 2053),    # many tiles, and edges of them
              (4100, 192, 4097)]


def some(m):
    return torch.arange(0, m, max(1, m // 200))


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", GATE_SIZES)
def test_relu_gates_of_products_that_cancel(m, k, n, dtype, device):
    """In eight groups of eight neighbours two products of 448^2 cancel beside
    six of up to 1/4, and some columns have no weights. Every sum is a multiple
    of 1/4 below 2^21, so exact in 32 bits in any order, and the gates are
    those of 64 bits."""
    g = torch.Generator().manual_seed(m + n)
    x, w = torch.zeros(m, k), torch.zeros(n, k)
    for at in range(0, 8 * (k // 64) * 8, (k // 64) * 8):
        for t in (x, w):
            t[:, at:at + 6] = torch.randint(-1, 2, (len(t), 6), generator=g) / 2
        x[:, at + 6:at + 8] = 448.0
        w[:, at + 6] = 448.0 - 896.0 * torch.randint(0, 2, (n,), generator=g)
        w[:, at + 7] = -w[:, at + 6]
    b = torch.randint(-1, 2, (n,), generator=g) / 4
    w[3::7], b[3::7] = 0.0, 0.0
    assert torch.equal(values(w, True), w.double())  # e4m3 holds them
    rows = some(m)
    z = x[rows].double() @ w.double().t() + b.double()
    got = gates(x.to(dtype).to(device), w.to(dtype).to(device), b.to(device),
                rows)
    assert torch.equal(got, z > 0)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n", GATE_SIZES)
def test_relu_gates_of_columns_of_unlike_size(m, k, n, dtype, device):
    """Columns between 2^-8 and 2^8 times the others' size; a gate may differ
    where the sum is within its 32 bits' error of zero."""
    x = randn(m, k, seed=m, dtype=dtype)
    size = 2.0 ** torch.randint(-8, 9, (n, 1),
                                generator=torch.Generator().manual_seed(n))
    w = (randn(n, k, seed=1) * size / k ** 0.5).to(dtype)
    b = randn(n, seed=2) * size.view(-1) * 0.1
    b[3::7] = 0.0
    w[3::7] = 0.0
    rows = some(m)
    xq, wq = values(x[rows]), values(w, True)
    z = xq @ wq.t() + b.double()
    bound = product_bound(xq, wq, k, b.double().abs(), torch.float32)
    got = gates(x.to(device), w.to(device), b.to(device), rows)
    assert bool(((got == (z > 0)) | (z.abs() <= bound)).all())
    assert bool((z.abs() > bound).float().mean() > 0.8)


@pytest.mark.parametrize("device", DEVICES)
def test_only_what_is_asked_for_is_kept(device):
    x = randn(200, 128, dtype=torch.bfloat16, device=device)
    w = randn(64, 128, seed=1, dtype=torch.bfloat16, device=device)
    b = randn(64, seed=2, dtype=torch.bfloat16, device=device)
    dy = randn(200, 64, seed=3, dtype=torch.bfloat16, device=device)
    both = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(fp8_dense(*both, "relu"), both, dy)
    kept = []

    def pack(t):
        kept.append(t)
        return t

    for i in range(3):
        args = [x, w, b]
        args[i] = args[i].clone().requires_grad_(True)
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            y = fp8_dense(*args, "relu")
        assert torch.equal(torch.autograd.grad(y, args[i], dy)[0], want[i])
    # the last two keep: x^T's bytes with the batch up to 256, its scales, and
    # bits (on the CPU a byte each); and for the bias the bits alone
    assert sum(t.numel() for t in kept[-1:]) <= 200 * 64
    kept.clear()
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        fp8_dense(x, w.requires_grad_(True), b, "none")
    assert sum(t.numel() * t.element_size() for t in kept) == 128 * 256 + 2 * 256


@pytest.mark.parametrize("device", DEVICES)
def test_gradient_that_is_an_expanded_number(device):
    x = randn(30, 50, device=device).requires_grad_(True)
    w = randn(20, 50, seed=1, device=device)
    a, = torch.autograd.grad(fp8_dense(x, w).sum(), x)
    c, = torch.autograd.grad(fp8_dense(x, w), x, torch.ones(30, 20, device=device))
    assert torch.equal(a, c)


@pytest.mark.gpu
def test_captured_training_step_replays():
    x = randn(300, 200, dtype=torch.bfloat16).cuda()
    w = randn(130, 200, seed=1, dtype=torch.bfloat16).cuda().requires_grad_(True)
    b = randn(130, seed=2, dtype=torch.bfloat16).cuda().requires_grad_(True)
    x.requires_grad_(True)
    dy = randn(300, 130, seed=3, dtype=torch.bfloat16).cuda()

    def step():
        y = fp8_dense(x, w, b, "relu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for i in range(4):
        with torch.no_grad():
            x.copy_(randn(300, 200, seed=10 + i, dtype=torch.bfloat16).cuda())
            dy.copy_(randn(300, 130, seed=20 + i, dtype=torch.bfloat16).cuda())
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()  # eager, between the replays
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_on_a_stream_of_its_own():
    x = randn(500, 256, dtype=torch.bfloat16).cuda()
    w = randn(384, 256, seed=1, dtype=torch.bfloat16).cuda()
    with torch.no_grad():
        want = fp8_dense(x, w, None, "relu")
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = fp8_dense(x, w, None, "relu")
        side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_same_call_twice_gives_the_same_bits():
    x = randn(3000, 400, dtype=torch.bfloat16).cuda().requires_grad_(True)
    w = randn(400, 400, seed=1, dtype=torch.bfloat16).cuda().requires_grad_(True)
    dy = randn(3000, 400, seed=3, dtype=torch.bfloat16).cuda()
    runs = []
    for _ in range(2):
        y = fp8_dense(x, w, None, "relu")
        runs.append((y.detach(), *torch.autograd.grad(y, (x, w), dy)))
    for a, c in zip(*runs):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_outputs_and_checkpoints_past_32_bit_offsets():
    # whole numbers: e4m3 holds them, and every sum is below 2^24, so exact
    m, k, n = (1 << 24) - 200, 130, 200
    g = torch.Generator(device="cuda").manual_seed(0)

    def whole(*shape, most):
        return torch.randint(-most, most + 1, shape, generator=g,
                             device="cuda", dtype=torch.int8).bfloat16()

    x, w, b = whole(m, k, most=2), whole(n, k, most=2), whole(n, most=3)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = fp8_dense(*leaves, "relu")
    dy = whole(m, n, most=1)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    x, w, b = (t.detach().float() for t in leaves)
    want_w = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    want_b = torch.zeros(n, dtype=torch.float64, device="cuda")
    step = 1 << 20
    for at in range(0, m, step):
        z = x[at:at + step] @ w.t() + b
        assert torch.equal(y.detach()[at:at + step],
                           z.clamp(min=0).bfloat16())
        dz = dy[at:at + step].float() * (z > 0)
        assert torch.equal(dx[at:at + step], (dz @ w).bfloat16())
        want_w += (dz.t() @ x[at:at + step]).double()
        want_b += dz.double().sum(0)
    assert torch.equal(dw, want_w.bfloat16())
    assert torch.equal(db, want_b.bfloat16())


@pytest.mark.gpu
def test_gradients_of_more_rows_than_can_be_transposed():
    """Only x^T's form has a limit of rows; x's and the bias's gradients do
    not use it."""
    m, k, n = (1 << 24) - 128, 8, 3
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randint(-2, 3, (m, k), generator=g, device="cuda",
                      dtype=torch.int8).bfloat16().requires_grad_(True)
    w = whole_numbers(n, k, seed=1, most=2, device="cuda", dtype=torch.bfloat16)
    b = whole_numbers(n, seed=2, device="cuda").requires_grad_(True)
    y = fp8_dense(x, w, b, "relu")
    dy = torch.randint(-1, 2, (m, n), generator=g, device="cuda",
                       dtype=torch.int8).bfloat16()
    dx, db = torch.autograd.grad(y, (x, b), dy)
    z = x.detach().float() @ w.float().t() + b.detach()
    dz = dy.float() * (z > 0)
    # whole numbers below 2^24, and below 2^8 in dx: exact
    assert torch.equal(dx, (dz @ w.float()).bfloat16())
    assert torch.equal(db.double(), dz.double().sum(0))
    with pytest.raises(RuntimeError, match="too many rows"):
        fp8_dense(x, w.requires_grad_(True))


@pytest.mark.gpu
def test_one_row_of_more_outputs_than_a_launch_has_threads_for():
    n = 1 << 26
    w = (torch.arange(n, device="cuda") % 17 - 8).bfloat16().view(n, 1)
    x = torch.full((1, 1), 3.0, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():  # whole numbers: exact
        y = fp8_dense(x, quantize_fp8_weight(w))
    assert torch.equal(y, (w * 3).view(1, n))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 300])
def test_two_graphs_of_a_laid_out_weight(m):
    layers = []
    for i in range(2):
        w = randn(200, 300, seed=i, dtype=torch.bfloat16).cuda()
        b = randn(200, seed=5 + i).cuda()
        layers.append((quantize_fp8_weight(w), b))
    x = randn(m, 300, seed=9, dtype=torch.bfloat16).cuda()
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            fp8_dense(x, *layers[0], "relu")
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graphs, held = [], []
        for w, b in layers:
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1]):
                held.append(fp8_dense(x, w, b, "relu"))
        for r, i in enumerate((0, 1, 1, 0, 1)):
            x.copy_(randn(m, 300, seed=20 + r, dtype=torch.bfloat16).cuda())
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(held[i], fp8_dense(x, *layers[i], "relu"))


@pytest.mark.gpu
def test_threads_at_once():
    jobs = []
    for i in range(4):
        x = randn(700, 256 + 64 * i, seed=i, dtype=torch.bfloat16).cuda()
        w = randn(384, 256 + 64 * i, seed=9 + i, dtype=torch.bfloat16).cuda()

        def step(x=x.requires_grad_(True), w=w.requires_grad_(True)):
            y = fp8_dense(x, w, None, "relu")
            return (y.detach(),
                    *torch.autograd.grad(y, (x, w), torch.ones_like(y)))

        jobs.append((step, step()))
    torch.cuda.synchronize()
    bad = []

    def work(step, want):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = step()
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        bad.append("differs")
        except Exception as e:  # shown by the test
            bad.append(e)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


# ------------------------------- refusals ---------------------------------
def test_refusals():
    x, w = torch.randn(4, 32), torch.randn(8, 32)
    with pytest.raises(ValueError, match="activation"):
        fp8_dense(x, w, None, "gelu")
    with pytest.raises(ValueError, match="takes 32"):
        fp8_dense(x[:, :31], w)
    with pytest.raises(TypeError, match="float32"):
        fp8_dense(x.double(), w)
    with pytest.raises(TypeError, match="float32"):
        fp8_dense(x, w.double())
    with pytest.raises(TypeError, match="bias"):
        fp8_dense(x, w, torch.zeros(8).double())
    with pytest.raises(ValueError, match="bias"):
        fp8_dense(x, w, torch.zeros(7))
    with pytest.raises(ValueError, match="two dimensions"):
        fp8_dense(x, w[0])
    with pytest.raises(ValueError, match="no columns"):
        fp8_dense(x[:, :0], w[:, :0])
    with pytest.raises(ValueError, match="no rows"):
        fp8_dense(x, w[:0])
    with pytest.raises(ValueError, match="two dimensions"):
        quantize_fp8(x[0])
    with pytest.raises(RuntimeError, match="no backward"):
        fp8_dense(x.requires_grad_(True), quantize_fp8_weight(w))
    y = fp8_dense(x, w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    assert repr(fp8.quantize_fp8(x)).startswith("Fp8Blocks")


@pytest.mark.skipif(not native_available(), reason="needs the extension")
def test_tensors_without_memory_are_refused():
    x, w, b = (Elsewhere(randn(*s)) for s in ((4, 32), (8, 32), (8,)))
    frozen = quantize_fp8_weight(randn(8, 32))
    frozen = fp8.Fp8Blocks(Elsewhere(frozen.data), Elsewhere(frozen.scale), 32)
    for call in (lambda: fp8_dense(x, w, b), lambda: fp8_dense(x, frozen),
                 lambda: require_native().fp8_quantize(x, False, True, False)):
        with pytest.raises(RuntimeError, match="no memory"):
            call()


@pytest.mark.gpu
def test_refuses_mixed_devices():
    x, w = torch.randn(4, 32), torch.randn(8, 32)
    with pytest.raises(ValueError, match="weight on"):
        fp8_dense(x.cuda(), w)
    with pytest.raises(ValueError, match="bias on"):
        fp8_dense(x.cuda(), w.cuda(), torch.zeros(8))


@pytest.mark.gpu
def test_refusals_on_a_gpu():
    x, w = randn(20, 256).cuda(), randn(64, 256).cuda()
    frozen = quantize_fp8_weight(w)
    room = torch.zeros(64 * 256 + 1, dtype=torch.uint8, device="cuda")
    odd = room[1:].view(64, 256)
    with pytest.raises(RuntimeError, match="16 bytes"):
        fp8_dense(x, fp8.Fp8Blocks(odd, frozen.scale, 256))
    with pytest.raises(RuntimeError, match="does not match"):
        fp8_dense(x, fp8.Fp8Blocks(frozen.data, frozen.scale[:1], 256))
    with pytest.raises(RuntimeError, match="bytes and scales"):
        fp8_dense(x, fp8.Fp8Blocks(frozen.data.float(), frozen.scale, 256))
    many = torch.zeros(1, 256, device="cuda").expand(1 << 24, -1)
    with pytest.raises(RuntimeError, match="too many rows"):
        fp8_dense(many, w.requires_grad_(True))

"""Embedding lookup, its gradient by sorted ids, and sums of rows by id.

Tolerances. A sum of n terms in 32 bits, in any order, is off by at most
n * 2^-24 * sum |terms| to first order (n + 8 here, for the products and the
factor that go into each term); the result's own rounding is half a step of
its type.
"""

import threading

import pytest
import torch

from elasticdl_amd.common.tensor_utils import deduplicate_indexed_slices
from elasticdl_amd.ops import native_available, require_native
from elasticdl_amd.ops.embedding import coalesce_rows, embedding_lookup

TYPES = [torch.float32, torch.bfloat16, torch.float16]
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
COMBINERS = [None, "sum", "mean", "sqrtn"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=gen(seed)).to(dtype)


def check(got, want, bound, dtype):
    got = got.detach().cpu()
    assert got.dtype == dtype and got.shape == want.shape
    half = torch.finfo(dtype).eps / 2
    bound = bound + half * (want.abs() + bound) \
        + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), \
        f"off by {float((off / bound).max())} of what is allowed"


def plain(table, ids, weights, combiner, scale, dy):
    """(out, dtable, dweights) and the sums of their terms' sizes, and how
    many terms a table's row has, in 64 bits."""
    t = table.double()
    v, d = t.shape
    b = ids.reshape(-1, 1) if combiner is None else ids
    live = (b >= 0).double()
    w = live if weights is None else torch.where(
        b >= 0, weights.double(), torch.zeros_like(live))
    n = live.sum(1).clamp(min=1)
    norm = {"mean": n, "sqrtn": n.sqrt()}.get(combiner, torch.ones_like(n))
    c = scale / norm
    rows = t[b.clamp(min=0).long()] * live.unsqueeze(2)
    out = (rows * w.unsqueeze(2)).sum(1) * c.unsqueeze(1)
    out_size = (rows * w.unsqueeze(2)).abs().sum(1) * c.abs().unsqueeze(1)
    g = dy.double().reshape(out.shape)
    part = (g * c.unsqueeze(1)).unsqueeze(1) * w.unsqueeze(2)
    at = b.clamp(min=0).long().reshape(-1)
    zero = lambda: torch.zeros(v, d, dtype=torch.float64)  # noqa: E731
    dt = zero().index_add_(0, at, part.reshape(-1, d))
    dt_size = zero().index_add_(0, at, part.abs().reshape(-1, d))
    terms = torch.zeros(v, dtype=torch.float64).index_add_(
        0, at, live.reshape(-1))
    each = rows * (g * c.unsqueeze(1)).unsqueeze(1)
    return out, out_size, dt, dt_size, terms, each.sum(2), each.abs().sum(2)


def run(v, d, bags, length, combiner, weighted, dtype, device, ids_dtype,
        scale=3.0, ragged=True, seed=0, hot=False):
    table = randn(v, d, seed=seed, dtype=dtype)
    u = torch.rand(bags, length, generator=gen(seed + 1))
    ids = ((u ** 6 if hot else u) * v).long().clamp(max=v - 1)
    if ragged:
        ends = torch.randint(0, length + 1, (bags, 1), generator=gen(seed + 2))
        ids = torch.where(torch.arange(length) < ends, ids, -1)
    ids = ids.to(ids_dtype)
    weights = None
    if weighted:
        weights = torch.rand(bags, length, generator=gen(seed + 3)) + 0.5
        weights = torch.where(ids >= 0, weights, torch.nan)  # never read
    if combiner is None:
        ids = ids if length > 1 else ids.reshape(-1)
    shape = (*ids.shape, d) if combiner is None else (bags, d)
    dy = randn(*shape, seed=seed + 4, dtype=dtype)
    out, out_size, dt, dt_size, terms, dw, dw_size = plain(
        table, ids, weights, combiner, scale, dy)
    leaf = table.to(device).requires_grad_(True)
    w_leaf = None if weights is None else weights.to(device).requires_grad_(True)
    got = embedding_lookup(leaf, ids.to(device), w_leaf, combiner, scale)
    eps = 2.0 ** -24
    check(got.reshape(-1, d), out, (length + 8) * eps * out_size, dtype)
    assert got.shape == shape
    leaves = (leaf,) if w_leaf is None else (leaf, w_leaf)
    grads = torch.autograd.grad(got, leaves, dy.to(device))
    check(grads[0], dt, (terms.unsqueeze(1) + 8) * eps * dt_size, dtype)
    if weighted:
        check(grads[1], dw, (d + 8) * eps * dw_size, torch.float32)
        assert not grads[1].cpu()[ids < 0].any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("combiner", COMBINERS)
@pytest.mark.parametrize("v,d,bags,length", [
    (1, 1, 1, 1), (5, 3, 7, 1), (100, 16, 39, 5), (50, 64, 20, 50),
    (1000, 17, 300, 9), (37, 130, 3, 200), (9, 513, 33, 3), (20, 1024, 5, 4)])
def test_lookup_and_gradients(v, d, bags, length, combiner, device):
    dtype = TYPES[(d + bags) % 3]
    ids_dtype = torch.int32 if d % 2 else torch.int64
    run(v, d, bags, length, combiner, combiner is not None, dtype, device,
        ids_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("combiner,weighted", [(None, False), ("mean", True)])
@pytest.mark.parametrize("v,d,bags,length,hot", [
    (3, 8, 2000, 5, False),        # runs over many chunks
    (1, 16, 3000, 7, False),       # one id for all of it
    (70000, 4, 4000, 3, True),     # over the one-workgroup sort, 17 bits
    (1 << 20, 2, 30000, 2, True),  # three passes
    (600, 256, 900, 10, True)])
def test_gradient_of_many_tokens(v, d, bags, length, hot, combiner, weighted):
    run(v, d, bags, length, combiner, weighted, TYPES[v % 3], "cuda",
        torch.int64, hot=hot)


@pytest.mark.parametrize("device", DEVICES)
def test_padding_and_empty_bags(device):
    table = randn(6, 4).to(device).requires_grad_(True)
    ids = torch.tensor([[-1, -1], [2, -7], [-1, 5]], device=device)
    for combiner in ("sum", "mean", "sqrtn"):
        out = embedding_lookup(table, ids, None, combiner, 2.0)
        assert torch.equal(out[0], torch.zeros(4, device=device))
        assert torch.equal(out[1], table[2] * 2)
        assert torch.equal(out[2], table[5] * 2)
    out = embedding_lookup(table, ids)
    assert out.shape == (3, 2, 4) and not out[ids < 0].any()
    g, = torch.autograd.grad(out.sum(), table)
    want = torch.zeros(6, 4)
    want[2] = want[5] = 1
    assert torch.equal(g.cpu(), want)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("combiner", [None, "mean"])
def test_no_ids(combiner, device):
    table = randn(6, 4).to(device).requires_grad_(True)
    for shape in ((0, 3), (2, 0)):
        ids = torch.zeros(shape, dtype=torch.int64, device=device)
        out = embedding_lookup(table, ids, None, combiner)
        assert out.shape == ((*shape, 4) if combiner is None else (shape[0], 4))
        assert not out.any()
        g, = torch.autograd.grad(out.sum(), table)
        assert g.shape == (6, 4) and not g.any()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("combiner", ["mean", "sqrtn"])
def test_weighted_norms_count_ids_and_weights_divide_before(combiner, device):
    """The documented way to norms by weights, with their gradient's term."""
    t = randn(9, 5, seed=1).to(device)
    ids = torch.tensor([[1, 4, 7, 4], [2, -1, -1, -1]], device=device)
    w = (torch.rand(2, 4, generator=gen(2)) + 0.5).to(device)
    live = ids >= 0
    n = live.sum(1, keepdim=True).float()
    want = torch.where(live.unsqueeze(2), t[ids.clamp(min=0)]
                       * w.unsqueeze(2), 0.0).sum(1)
    want = want / (n if combiner == "mean" else n.sqrt())
    got = embedding_lookup(t, ids, w, combiner)
    assert torch.allclose(got, want, rtol=1e-6, atol=1e-6)

    def normed(w):
        w = torch.where(live, w, 0.0)
        sums = w if combiner == "mean" else w.square()
        norm = sums.sum(1, keepdim=True)
        return w / (norm if combiner == "mean" else norm.sqrt())

    w.requires_grad_(True)
    a = embedding_lookup(t, ids, normed(w), "sum")
    b = (t[ids.clamp(min=0)].double() * normed(w.double()).unsqueeze(2)).sum(1)
    # a few roundings of 2^-24 of sums of at most 4 terms of size 3
    assert torch.allclose(a.double(), b, rtol=0, atol=64 * 2.0 ** -24)
    ga, = torch.autograd.grad(a.square().sum(), w)
    gb, = torch.autograd.grad(b.square().sum(), w)
    # 5 columns of products of such, and a quotient's two terms
    assert torch.allclose(ga, gb.float(), rtol=0, atol=2048 * 2.0 ** -24)



@pytest.mark.gpu
@pytest.mark.parametrize("bags", [2, 20000])
def test_ids_past_the_table_show_and_reach_nothing(bags):
    table = randn(10, 4).cuda().requires_grad_(True)
    ids = torch.arange(bags * 3, device="cuda").reshape(bags, 3) % 10
    ids[1, 2] = 10
    ids[0, 0] = 1 << 40
    w = torch.ones(bags, 3, device="cuda", requires_grad=True)
    out = embedding_lookup(table, ids, w, "sum")
    assert torch.isnan(out[:2]).all() and torch.isfinite(out[2:]).all()
    dt, dw = torch.autograd.grad(out, (table, w), torch.ones_like(out))
    assert dw[0, 0] == 0 and dw[1, 2] == 0
    count = torch.bincount(ids[ids < 10].reshape(-1), minlength=10)
    assert torch.equal(dt, count.float().unsqueeze(1).expand(10, 4))


def test_ids_past_the_table_raise_on_the_cpu():
    with pytest.raises(IndexError):
        embedding_lookup(randn(10, 4), torch.tensor([3, 10]))


@pytest.mark.parametrize("device", DEVICES)
def test_strided_tables(device):
    base = randn(40, 12, dtype=torch.bfloat16).to(device)
    ids = torch.tensor([[3, 0, 19, -1]] * 5, device=device)
    for table in (base[::2, 1:9], base[:20, ::2], base[:12].t(),
                  base[:1, :8].expand(20, 8)):
        want = embedding_lookup(table.clone(), ids[:, :2], None, "sum")
        assert torch.equal(embedding_lookup(table, ids[:, :2], None, "sum"),
                           want)
    leaf = base.clone().requires_grad_(True)
    out = embedding_lookup(leaf[::2, 1:9], ids, None, "mean")
    g, = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert g.shape == (40, 12) and not g[:, 0].any() and not g[1::2].any()
    assert g[[0, 6, 38], 1:9].ne(0).all()


@pytest.mark.parametrize("device", DEVICES)
def test_not_finite_rows_stay_with_their_bags(device):
    table = randn(8, 4)
    table[0] = float("inf")  # row 0 is what padding would read
    table[3, 1] = float("nan")
    ids = torch.tensor([[1, -1, -1], [2, 3, -1], [-1, -1, -1], [0, 4, 5]])
    out = embedding_lookup(table.to(device), ids.to(device), None, "sum").cpu()
    assert torch.equal(out[0], table[1]) and not out[2].any()
    assert torch.isnan(out[1, 1]) and torch.isfinite(out[1, [0, 2, 3]]).all()
    assert torch.isinf(out[3]).all()


@pytest.mark.parametrize("device", DEVICES)
def test_gradients_against_differences(device):
    """Small whole numbers, whose sums are exact: the change for a step of
    one is the gradient."""
    table = torch.randint(-4, 5, (7, 3), generator=gen(0)).float().to(device)
    ids = torch.tensor([[0, 3, 3, -1], [6, 6, 6, 6]], device=device)
    w = torch.randint(1, 5, (2, 4), generator=gen(1)).float().to(device)
    dy = torch.randint(-4, 5, (2, 3), generator=gen(2)).float().to(device)
    loss = lambda t, x: float((embedding_lookup(t, ids, x, "sqrtn", 2.0) * dy).double().sum())  # noqa: E731
    t, x = table.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gt, gx = torch.autograd.grad(
        embedding_lookup(t, ids, x, "sqrtn", 2.0), (t, x), dy)
    # sqrt(3) is not whole: bag 0's factor rounds, and each sum has 4 terms
    for r in range(7):
        for c in range(3):
            p = table.clone()
            p[r, c] += 1
            d = loss(p, w) - loss(table, w)
            assert abs(d - float(gt[r, c])) <= 16 * 2.0 ** -23 * 200
    for b in range(2):
        for i in range(4):
            p = w.clone()
            p[b, i] += 1
            d = loss(table, p) - loss(table, w)
            assert abs(d - float(gx[b, i])) <= 16 * 2.0 ** -23 * 200


@pytest.mark.gpu
@pytest.mark.parametrize("combiner", [None, "mean"])
def test_captured_lookup_and_gradient_replay(combiner):
    table = randn(500, 16).cuda().requires_grad_(True)
    ids = torch.randint(-1, 500, (300, 40), generator=gen(1)).cuda()
    shape = (300, 16) if combiner else (300, 40, 16)
    dy = randn(*shape, seed=2).cuda()

    def step():
        out = embedding_lookup(table, ids, None, combiner, 4.0)
        return out.detach(), torch.autograd.grad(out, table, dy)[0]

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
        ids.copy_(torch.randint(-1, 500, (300, 40), generator=gen(10 + i)))
        dy.copy_(randn(*shape, seed=20 + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert torch.equal(a, c)


@pytest.mark.gpu
def test_same_call_twice_gives_the_same_bits():
    table = randn(300, 32).cuda().requires_grad_(True)
    ids = torch.randint(0, 300, (20000, 6), generator=gen(1)).cuda()
    dy = randn(20000, 32, seed=2).cuda()
    values = randn(100000, 8, seed=3).cuda()
    flat = torch.randint(0, 50, (100000,), generator=gen(4)).cuda()
    runs = []
    for _ in range(2):
        out = embedding_lookup(table, ids, None, "mean")
        runs.append((torch.autograd.grad(out, table, dy)[0],
                     *coalesce_rows(values, flat)))
    for a, c in zip(*runs):
        assert torch.equal(a, c)


@pytest.mark.gpu
def test_on_a_stream_of_its_own():
    table = randn(3000, 32).cuda()
    ids = torch.randint(-1, 3000, (2000, 20), generator=gen(1)).cuda()
    want = embedding_lookup(table, ids, None, "mean")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = embedding_lookup(table, ids, None, "mean")
    side.synchronize()
    assert torch.equal(got, want)


@pytest.mark.gpu
def test_more_tokens_than_a_launch_has_threads():
    # 66 columns of 16 bits: 64 lanes a row, so 2^26 rows are 2^32 threads
    n, v, d = (1 << 26) + 1000, 1000, 66
    g = torch.Generator(device="cuda").manual_seed(0)
    table = torch.randint(-4, 5, (v, d), generator=g, device="cuda").bfloat16()
    ids = torch.randint(0, v, (n, 1), generator=g, device="cuda",
                        dtype=torch.int32)
    weights = torch.ones(n, 1, dtype=torch.bfloat16, device="cuda")
    weights[ids == 7] = 2.0
    leaves = table.requires_grad_(True), weights.requires_grad_(True)
    out = embedding_lookup(*leaves[:1], ids, leaves[1], "sum")
    dt, dw = torch.autograd.grad(out, leaves, torch.ones_like(out))
    sums = table.detach().float().sum(1)
    for at in (0, (1 << 25) - 500, (1 << 26) - 500, n - 1000):  # whole numbers
        part = ids[at:at + 1000, 0].long()
        row = table.detach()[part] * weights.detach()[at:at + 1000]
        assert torch.equal(out[at:at + 1000], row)
        assert torch.equal(dw[at:at + 1000, 0], sums[part].bfloat16())
    count = torch.bincount(ids[:, 0].long(), minlength=v).float()
    count[7] *= 2
    assert torch.equal(dt, count.bfloat16().unsqueeze(1).expand(-1, d))


@pytest.mark.gpu
def test_two_graphs_and_eager_calls_in_turn():
    tables = [randn(500, 16, seed=i).cuda().requires_grad_(True)
              for i in range(2)]
    ids = [torch.randint(-1, 500, (300, 40), generator=gen(i)).cuda()
           for i in range(2)]
    dy = randn(300, 16, seed=2).cuda()

    def step(i):
        out = embedding_lookup(tables[i], ids[i], None, "mean")
        return out.detach(), torch.autograd.grad(out, tables[i], dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, held = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            held.append(step(i))
    want = [step(0), step(1)]
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        for k in range(2):
            assert torch.equal(step(i)[k], want[i][k])
            assert torch.equal(held[i][k], want[i][k])


@pytest.mark.gpu
def test_threads_at_once():
    jobs = []
    for i in range(4):
        n = (500, 9000, 60000, 8000)[i]
        ids = torch.randint(0, 300, (n,), generator=gen(i)).cuda()
        values = randn(n, 12, seed=i).cuda()
        jobs.append((values, ids, coalesce_rows(values, ids)))
    torch.cuda.synchronize()
    bad = []

    def work(values, ids, want):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    got = coalesce_rows(values, ids)
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


# ----------------------------- sums by id ---------------------------------
@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n,d,low,high", [
    (0, 4, 0, 1), (1, 1, 5, 6), (3, 7, -4, 4), (6656, 8, 0, 1_300_000),
    (8192, 3, 0, 2), (8193, 16, 0, 100), (9000, 5, -(1 << 40), 1 << 40),
    (3000, 2, -(1 << 63), (1 << 63) - 1), (50000, 1, 0, 97_500_000),
    (20000, 130, 0, 700), (9000, 4, -(1 << 63), (1 << 63) - 1)])
def test_deduplicate(n, d, low, high, device):
    ids = torch.randint(low, high, (n,), generator=gen(n + d))
    dtype = TYPES[d % 3] if device == "cuda" else torch.float32
    values = randn(n, d, seed=1, dtype=dtype)
    rows, unique = deduplicate_indexed_slices(values.to(device), ids.to(device))
    want_ids, place, count = torch.unique(ids, return_inverse=True,
                                          return_counts=True)
    assert torch.equal(unique.cpu(), want_ids)
    zero = lambda: torch.zeros(len(want_ids), d, dtype=torch.float64)  # noqa: E731
    want = zero().index_add_(0, place, values.double())
    size = zero().index_add_(0, place, values.double().abs())
    check(rows, want, (count.unsqueeze(1) + 8) * 2.0 ** -24 * size, dtype)


LOW, HIGH = -(1 << 63), (1 << 63) - 1


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("ids", [
    [HIGH, LOW], [LOW, HIGH], [HIGH - 5, LOW + 3, HIGH, LOW, HIGH - 5],
    [LOW + (1 << 31) - 1, HIGH, LOW], [HIGH - (1 << 31) + 2, LOW, HIGH],
    [LOW, LOW + (1 << 31), HIGH], [LOW + 1, LOW, LOW + 1], [HIGH, HIGH - 1]])
@pytest.mark.parametrize("times", [1, 700])
def test_deduplicate_at_the_ends_of_int64(ids, times, device):
    """The two ends are neighbours modulo 2^64, and far apart."""
    ids = torch.tensor(ids).repeat(times)
    values = torch.arange(1.0, 2 * ids.numel() + 1).view(-1, 2) % 64
    rows, unique = deduplicate_indexed_slices(values.to(device), ids.to(device))
    want, place = torch.unique(ids, return_inverse=True)
    assert torch.equal(unique.cpu(), want)
    # whole numbers below 2^24: every sum is exact
    sums = torch.zeros(want.numel(), 2).index_add_(0, place, values)
    assert torch.equal(rows.cpu(), sums)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [2, 31, 33, 1024, 4095, 8191, 8192])
def test_deduplicate_of_few_ids_far_apart(n, device):
    known = torch.cat([torch.randint(LOW, HIGH, (n // 3 + 1,), generator=gen(n)),
                       torch.tensor([LOW, HIGH, 0, -1, 1 << 32, 1 << 31])])
    at = torch.randint(0, len(known), (n,), generator=gen(n + 1))
    at[torch.rand(n, generator=gen(n + 2)) < 0.3] = 0  # one of them often
    values = torch.randint(-8, 9, (n, 3), generator=gen(n + 3)).float()
    rows, unique = deduplicate_indexed_slices(values.to(device),
                                              known[at].to(device))
    want, place = torch.unique(known[at], return_inverse=True)
    assert torch.equal(unique.cpu(), want)
    # whole numbers below 2^24: every sum is exact
    sums = torch.zeros(want.numel(), 3).index_add_(0, place, values)
    assert torch.equal(rows.cpu(), sums)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("n", [8193, 10240, 12289, 65536, 100_001, 196_608,
                               196_609, 250_000])
@pytest.mark.parametrize("known", [2, 700, 100_000])
def test_deduplicate_of_many_ids_far_apart(n, known, device):
    """Chunks that are merged, whole and not, and behind them all 64 bits."""
    known = torch.randint(LOW, HIGH, (known,), generator=gen(known))
    known[:2] = torch.tensor([LOW, HIGH])
    at = torch.randint(0, len(known), (n,), generator=gen(n))
    at[torch.rand(n, generator=gen(n + 1)) < 0.2] = 1  # the last, often
    values = torch.randint(-8, 9, (n, 3), generator=gen(n + 2)).float()
    rows, unique = deduplicate_indexed_slices(values.to(device),
                                              known[at].to(device))
    want, place = torch.unique(known[at], return_inverse=True)
    assert torch.equal(unique.cpu(), want)
    # whole numbers below 2^24: every sum is exact
    sums = torch.zeros(want.numel(), 3).index_add_(0, place, values)
    assert torch.equal(rows.cpu(), sums)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [8192, 50_000])
def test_sums_of_ids_far_apart_have_the_same_bits_each_time(n):
    ids = torch.randint(LOW, HIGH, (n // 9,), generator=gen(0)).cuda()
    ids = ids[torch.randint(0, n // 9, (n,), generator=gen(1)).cuda()]
    values = randn(n, 5, seed=2).cuda()
    want = coalesce_rows(values, ids)
    # the order of equal ids is theirs: near ids with the same order agree
    near = torch.unique(ids, return_inverse=True)[1]
    same = coalesce_rows(values, near)
    assert torch.equal(want[0], same[0])
    for _ in range(5):
        for a, b in zip(coalesce_rows(values, ids), want):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_deduplicate_keeps_a_gradient_where_one_is_asked_for():
    values = randn(50, 3).cuda().requires_grad_(True)
    ids = torch.randint(0, 9, (50,), generator=gen(1)).cuda()
    rows, _ = deduplicate_indexed_slices(values, ids)
    g, = torch.autograd.grad(rows.sum(), values)
    assert torch.equal(g, torch.ones_like(g))
    with torch.no_grad():
        assert not deduplicate_indexed_slices(values, ids)[0].requires_grad


@pytest.mark.parametrize("device", DEVICES)
def test_deduplicate_under_transforms(device):
    """Tracing and torch.func see torch's own operators."""
    values = torch.arange(1.0, 13.0).view(6, 2).to(device)
    ids = torch.tensor([4, 1, 4, 0, 1, 4], device=device)
    other = torch.tensor([2, 2, 2, 7, 2, 3], device=device)
    traced = torch.jit.trace(deduplicate_indexed_slices, (values, ids))
    for a, b in zip(traced(values * 2, other),
                    deduplicate_indexed_slices(values * 2, other)):
        assert torch.equal(a, b)
    weight = torch.tensor([[1.0], [2.0], [3.0]], device=device)
    g = torch.func.grad(lambda v: (
        deduplicate_indexed_slices(v, ids)[0] * weight).sum())(values)
    assert torch.equal(g[:, 0].cpu(), torch.tensor([3.0, 2, 3, 1, 2, 3]))


@pytest.mark.gpu
def test_coalesce_of_strided_values():
    base = randn(100, 20).cuda()
    ids = torch.randint(0, 9, (200,), generator=gen(1)).cuda()[::2]
    a = coalesce_rows(base[:, 3:11], ids)
    b = coalesce_rows(base[:, 3:11].clone(), ids.clone())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
@pytest.mark.parametrize("n,d", [(400_000, 16), (70_000, 130), (300_000, 1)])
def test_runs_of_most_of_the_tokens(n, d):
    # whole numbers: every sum is exact
    values = torch.randint(-3, 4, (n, d), generator=gen(n)).float().cuda()
    for ids in (torch.full((n,), 12345), torch.arange(n) % 2 * 7,
                torch.where(torch.arange(n) < n - 9, 5, torch.arange(n))):
        rows, unique = coalesce_rows(values, ids.cuda())
        want, back = torch.unique(ids, return_inverse=True)
        assert torch.equal(unique.cpu(), want)
        sums = torch.zeros(want.numel(), d, dtype=torch.float64)
        sums.index_add_(0, back, values.cpu().double())
        assert torch.equal(rows.cpu().double(), sums)


@pytest.mark.gpu
@pytest.mark.parametrize("v,d", [(7, 3), (1000, 16), (1, 1)])
@pytest.mark.parametrize("bags", [30, 4000])
def test_gradient_of_padding_alone_is_zero(v, d, bags):
    for dtype in TYPES:
        table = randn(v, d, dtype=dtype).cuda().requires_grad_(True)
        ids = torch.full((bags, 3), -1, device="cuda")
        for last in (-1, v - 1):
            ids[-1, -1] = last
            out = embedding_lookup(table, ids, None, "sum")
            g, = torch.autograd.grad(out, table, torch.full_like(out, 2.0))
            want = torch.zeros_like(g)
            if last >= 0:
                want[last] = 2.0
            assert torch.equal(g, want)


# ------------------------------- refusals ---------------------------------
def test_refusals():
    table, ids = randn(6, 4), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="combiner"):
        embedding_lookup(table, ids, None, "max")
    with pytest.raises(ValueError, match="table is"):
        embedding_lookup(table[0], ids)
    with pytest.raises(ValueError, match="table is"):
        embedding_lookup(table[:0], ids)
    with pytest.raises(TypeError, match="table must"):
        embedding_lookup(table.double(), ids)
    with pytest.raises(TypeError, match="ids must"):
        embedding_lookup(table, ids.float())
    with pytest.raises(ValueError, match="bags"):
        embedding_lookup(table, ids[0], None, "sum")
    with pytest.raises(ValueError, match="need a combiner"):
        embedding_lookup(table, ids, torch.ones(2, 3))
    with pytest.raises(ValueError, match="shape"):
        embedding_lookup(table, ids, torch.ones(2, 2), "sum")
    with pytest.raises(TypeError, match="weights"):
        embedding_lookup(table, ids, torch.ones(2, 3).double(), "sum")
    with pytest.raises(ValueError, match="GPU"):
        coalesce_rows(table, ids[0])


class Elsewhere(torch.Tensor):
    """Stands for a tensor on a GPU, without memory of its own."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_wrapper_subclass(
            cls, t.shape, dtype=t.dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise RuntimeError(f"{func} is not what is tested")


@pytest.mark.skipif(not native_available(), reason="needs the extension")
def test_tensors_without_memory_are_refused():
    """Before a kernel would read from address 0; no GPU takes part."""
    table, ids = Elsewhere(randn(5, 4)), Elsewhere(torch.zeros(2, 3).long())
    weights = Elsewhere(randn(2, 3))
    for args in ((table, ids), (table, ids, weights, "sum")):
        with pytest.raises(RuntimeError, match="no memory"):
            embedding_lookup(*args)
    with pytest.raises(RuntimeError, match="no memory"):
        require_native().coalesce_rows(Elsewhere(randn(3, 4)),
                                       Elsewhere(torch.zeros(3).long()))


@pytest.mark.gpu
def test_refusals_on_a_gpu():
    table, ids = randn(6, 4).cuda(), torch.zeros(2, 3, dtype=torch.int64)
    with pytest.raises(ValueError, match="table on"):
        embedding_lookup(table, ids)
    values = randn(3, 4).cuda()
    with pytest.raises(RuntimeError, match="same GPU"):
        coalesce_rows(values, ids[0])
    with pytest.raises(RuntimeError, match="int64"):
        coalesce_rows(values, ids[0].int().cuda())
    with pytest.raises(RuntimeError, match="dim"):
        coalesce_rows(values[:2], ids[0].cuda())


@pytest.mark.gpu
def test_coalesce_refuses_to_be_captured():
    values, ids = randn(30, 4).cuda(), torch.arange(30).cuda() // 2
    want = coalesce_rows(values, ids)
    torch.cuda.synchronize()
    x = torch.zeros(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1.0)
        with pytest.raises(RuntimeError, match="captured"):
            coalesce_rows(values, ids)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, torch.ones(4, device="cuda"))
    for a, b in zip(coalesce_rows(values, ids), want):
        assert torch.equal(a, b)

"""More of the operators on rows in device memory (superkmeans_b200.ops): tensors that torch holds in other ways, paths and sums that
test_row_ops_gpu.py does not reach.  Its helpers and its counting of roundings are used here too."""
import pytest
import torch

from tests.test_row_ops_gpu import TYPES, U, as_index, check_product, close, ops, pitched, randn, rng, rounding, some_bytes, some_ids   # noqa: F401

pytestmark = pytest.mark.gpu


def test_tensors_without_memory(ops):
    """A storage that was freed, as sharded training does with parameters, is refused by the host; so is one freed before the backward pass."""
    table, ids = randn(rng(1), 20, 8), some_ids(rng(2), 30, 20)
    part = table[1:]
    table.untyped_storage().resize_(0)
    for call in (lambda: ops.lookup(part, ids), lambda: ops.quantize_rows(part), lambda: ops.lookup(part.requires_grad_(), ids)):
        with pytest.raises(ValueError, match="has no memory"):
            call()
    y, w = randn(rng(3), 30, 8), randn(rng(4), 30).requires_grad_()
    out = ops.from_clusters(y, ops.group_rows(ids, 20), w)
    y.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="has no memory"):
        out.sum().backward()


def test_imaginary_parts_of_conjugates(ops):
    z = torch.complex(randn(rng(5), 40, 1), randn(rng(6), 40, 1)).conj().imag
    plain, ids = -(-z), some_ids(rng(7), 40, 40)
    assert z.is_neg() and not plain.is_neg()
    groups = ops.group_rows(ids, 40)
    for f in (lambda t: ops.lookup(t, ids), lambda t: ops.lookup_grad(t, ids, 40), lambda t: ops.to_clusters(t, groups), lambda t: ops.quantize_rows(t).values,
              lambda t: ops.lookup(plain, ids[:1], 1.0, t[:1, 0]), lambda t: ops.from_clusters(plain[:1], ops.group_rows(ids[:1], 40), t[:1, 0])):
        assert torch.equal(f(z), f(plain))


def test_derivatives_carried_forward(ops):
    table, ids, w = randn(rng(8), 20, 8), some_ids(rng(9), 30, 20), randn(rng(10), 30)
    groups = ops.group_rows(ids, 20)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(table, table)
        rows = torch.autograd.forward_ad.make_dual(randn(rng(11), 30, 8), randn(rng(12), 30, 8))
        for call in (lambda: ops.lookup(dual, ids), lambda: ops.lookup(dual[1:], ids), lambda: ops.lookup(table, ids, 1.0, rows[:, 0].contiguous()), lambda: ops.to_clusters(rows, groups),
                     lambda: ops.from_clusters(rows, groups, w), lambda: ops.from_clusters(table.repeat(2, 1)[:30], groups, rows[:, 1].contiguous()), lambda: ops.quantize_rows(rows)):
            with pytest.raises(NotImplementedError, match="derivative forward"):
                call()
        assert torch.equal(ops.lookup(torch.autograd.forward_ad.unpack_dual(dual).primal, ids), ops.lookup(table, ids))
    assert torch.equal(ops.lookup(dual, ids), ops.lookup(table, ids))   # (the level has ended, and the derivative with it)


def test_where_torch_records_or_looks_on(ops):
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils._python_dispatch import TorchDispatchMode

    table, ids = randn(rng(13), 20, 8), some_ids(rng(14), 30, 20)
    want = ops.lookup(table, ids)
    for record in (lambda: torch.jit.trace(lambda t: ops.lookup(t, ids), (table,)), lambda: make_fx(lambda t: ops.lookup(t, ids))(table),
                   lambda: make_fx(lambda t: ops.lookup(t[1:], ids), tracing_mode="fake")(table), lambda: torch.func.vmap(lambda t: ops.lookup(t, ids))(table[None]),
                   lambda: torch.func.functionalize(lambda t: ops.lookup(t[1:], ids))(table)):
        with pytest.raises(NotImplementedError):
            record()

    class LooksOn(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with LooksOn():
        assert torch.equal(ops.lookup(table, ids), want)
        t = table.clone().requires_grad_()
        ops.lookup(t, ids).sum().backward()
    assert torch.equal(t.grad, ops.lookup_grad(torch.ones_like(want), ids, 20))
    for t in (table, table.clone().requires_grad_()):
        assert torch.equal(torch.compile(lambda t: ops.lookup(t + 0, ids) * 1, backend="eager")(t), want)
    with torch.inference_mode():
        assert torch.equal(ops.lookup(table, ids), want)


@pytest.mark.parametrize("n,m", [(300, 500), (2000, 1200)])   # (one CTA to a tile, and pairs)
def test_a_wait_that_ran_out_ends_no_other_launch(ops, n, m):
    """What a launch that gave up leaves behind must not end the waits of the next one, whether or not anybody was told, and on whatever stream: that
    one's own waits run their time (here all of it, as the injection stops its producer too)."""
    from superkmeans_b200 import _lib

    g = rng(15)
    x, w, xs, ws = some_bytes(g, n, 4096), some_bytes(g, m, 4096), torch.ones(n, device="cuda"), torch.ones(m, device="cuda")
    cycles = 100_000_000   # 50 ms at 2 GHz

    def gives_up(call):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        call()
        end.record()
        end.synchronize()
        return start.elapsed_time(end)

    def told():
        with pytest.raises(RuntimeError, match="gave up waiting"):
            ops.product_8bit(x, xs, w, ws)

    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    ops.product_8bit(x, xs, w, ws)
    torch.cuda.synchronize()
    _lib.check(_lib.lib.skm_debug_wait_injection(cycles, 1))
    try:
        assert gives_up(lambda: ops.product_8bit(x, xs, w, ws)) >= 40
        with torch.cuda.stream(busy):   # told while this stream has other work
            torch.cuda._sleep(2_000_000_000)
            told()
        with torch.cuda.stream(other):
            assert gives_up(lambda: ops.product_8bit(x, xs, w, ws)) >= 40
            assert not busy.query(), "the other stream should still be busy"
            told()
            with torch.cuda.graph(graph, stream=other):
                ops.product_8bit(x, xs, w, ws)
            for _ in range(3):
                assert gives_up(graph.replay) >= 40
            told()
    finally:
        _lib.check(_lib.lib.skm_debug_wait_injection(0, 0))
        torch.cuda.synchronize()
    ops.check_products()
    check_product(ops.product_8bit(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws, torch.float32)
    torch.cuda.synchronize()
    ops.check_products()


@pytest.mark.parametrize("n,k,small,roundings", [
    (4096, 1, 2.0**-25, 80),           # one launch: eight rows, the 64 eights of a warp, eight warps
    (1_300_000, 5, 2.0**-25, 50),      # tiles: eight rows, 32 eights, their factor; and eight tiles at most, or fours of them in 64 bits
    (1_024_000, 100_000, 2.0**-33, 50),   # (the rows of a tile add up to half a step of one: a chain of tiles loses them all)
])
@pytest.mark.parametrize("scaled", [False, True])
def test_sums_of_many_rows_keep_their_last_places(ops, n, k, small, roundings, scaled):
    """One row of ones and many of less than half of one's last place each, all for one id: a chain of sums in 32 bits stays at one."""
    grad = torch.full((n, 8), small, device="cuda")
    grad[0] = 1.0
    ids = torch.full((n,), k - 1, dtype=torch.int32, device="cuda")
    got = ops.lookup_grad(grad, ids, k, 1.0, torch.ones(n, device="cuda") if scaled else None)
    want = torch.zeros(k, 8, dtype=torch.float64, device="cuda")
    want[k - 1] = 1.0 + (n - 1) * small
    close(got, want, roundings * U * want)


@pytest.mark.parametrize("dtype,d", [(torch.float32, 3), (torch.float32, 1), (torch.bfloat16, 7), (torch.float16, 2)])
@pytest.mark.parametrize("k", [20, 3000])
def test_gradients_of_a_million_narrow_rows(ops, dtype, d, k):
    n = 1_300_000
    g = rng(n + d)
    ids, grad = some_ids(g, n, k, skew=True), randn(g, n, d, dtype=dtype)
    i = as_index(ids, k)
    held = i >= 0
    want = torch.zeros(k, d, dtype=torch.float64, device="cuda").index_add_(0, i[held], grad.double()[held])
    size = torch.zeros(k, d, dtype=torch.float64, device="cuda").index_add_(0, i[held], grad.double()[held].abs())
    for out in {dtype, torch.float32}:
        close(ops.lookup_grad(grad, ids, k, dtype=out), want, rounding(want, out, 50 * U * size))


# ---- paths of the product by cluster: tiles of 16, 32 and 64 rows, and pairs of CTAs with 128 columns (groups of 65 - 191 rows) or 256

GROUPED = [
    (200, 20, 77, 48), (3000, 120, 300, 64), (3001, 120, 129, 200), (2500, 50, 1000, 96),   # 10, 25 and 50 rows a group
    (12_000, 100, 520, 129), (12_000, 100, 521, 160), (9001, 70, 1024, 64),                 # 120 and 129: pairs, odd and even numbers of channels
    (20_000, 40, 528, 300), (20_000, 40, 521, 96), (16_384, 64, 1040, 128),                 # 500 and 256: rows or channels in lanes
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,e,m,d", GROUPED)
@pytest.mark.parametrize("skew", [False, True])
def test_product_by_cluster_of_every_type(ops, dtype, n, e, m, d, skew):
    g = rng(n + e + m)
    ids = some_ids(g, n, e, lost=0.1, skew=skew)
    ids[ids == e // 2] = -1   # (a cluster that nobody has)
    groups = ops.group_rows(ids, e)
    x, w, xs, ws = some_bytes(g, n, d), some_bytes(g, e, m, d), torch.exp(randn(g, n)) / 4096, torch.exp(randn(g, e, m)) / 64
    xs[int(groups.offsets[-1]):] = float("nan")   # rows of no cluster: zeros, whatever their scales
    pitch = -(-d // 16) * 16
    got = ops.product_8bit(pitched(x, pitch), xs, pitched(w, pitch), ws, groups.offsets, dtype=dtype)
    ends = groups.offsets.tolist()
    for c in range(e):
        a, b = ends[c], ends[c + 1]
        check_product(got[a:b], x[a:b], xs[a:b], w[c], ws[c], dtype)
    assert not got[ends[-1]:].any()
    assert torch.equal(ops.product_8bit(x, xs, w, ws, groups.offsets, dtype=dtype), got)   # (rows that are copied first)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m", [(40, 33), (9000, 520)])
def test_product_of_rows_ahead_of_the_first_cluster(ops, dtype, n, m):
    """Offsets of one's own may begin behind the first row and end before the last; clusters without rows lie at either end."""
    g = rng(n)
    x, w, xs, ws = some_bytes(g, n, 64), some_bytes(g, 5, m, 64), torch.exp(randn(g, n)) / 512, torch.exp(randn(g, 5, m)) / 512
    ends = [n // 10, n // 10, n // 2, n // 2, n - 3, n - 3]
    got = ops.product_8bit(x, xs, w, ws, torch.tensor(ends, dtype=torch.int32, device="cuda"), dtype=dtype)
    for c in range(5):
        check_product(got[ends[c]:ends[c + 1]], x[ends[c]:ends[c + 1]], xs[ends[c]:ends[c + 1]], w[c], ws[c], dtype)
    assert not got[:ends[0]].any() and not got[ends[-1]:].any()


# ---- gradients of scales and weights: eight lanes to a row and 32, chunks of 16 bytes and less, windows


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [2, 4, 8, 16, 20, 24, 33, 64, 72, 128, 136, 137, 256, 512, 768, 1024, 1032, 2048])
def test_lookup_scale_grad_of_every_width(ops, dtype, d):
    g = rng(d)
    n, k = 501, 40
    grad, table, ids = randn(g, n, d, dtype=dtype), randn(g, k, d, dtype=dtype), some_ids(g, n, k)
    i = as_index(ids, k)
    parts = torch.where((i >= 0)[:, None], grad.double() * table.double()[i.clamp(min=0)], 0.0) * 0.75
    want = parts.sum(1)
    close(ops.lookup_scale_grad(grad, table, ids, 0.75), want, rounding(want, torch.float32, (d + 2) * U * parts.abs().sum(1)))
    # and of the weights of the way back: <grad[i], y[position]>
    groups = ops.group_rows(ids[:500].reshape(250, 2), k)
    up, y, w = randn(g, 250, d, dtype=dtype), randn(g, 500, d, dtype=dtype), randn(g, 250, 2)
    there = (as_index(ids[:500], k) >= 0).reshape(250, 2)
    parts = torch.where(there[..., None], up.double()[:, None] * y.double()[groups.position.long()], 0.0)
    close(ops.from_clusters_grad(up, y, groups, w)[1], parts.sum(2), rounding(parts.sum(2), torch.float32, (d + 1) * U * parts.abs().sum(2)))


# ---- the radix sort of one pass


@pytest.mark.parametrize("k", [1024, 1500, 2046])
def test_many_pairs_of_few_thousand_clusters(ops, k):
    """(One pass: the clusters' first slots come out of the sort itself, and its list of clusters goes to the gradient.)"""
    n = 10_000_000
    ids = some_ids(rng(k), n, k, lost=0.1)
    i = as_index(ids, k)
    key = torch.where(i >= 0, i, k)
    order, position, offsets = ops.group_rows(ids, k)
    want = torch.argsort(key, stable=True)
    assert torch.equal(order.long(), want)
    assert torch.equal(position.long()[want], torch.arange(n, device="cuda"))
    counts = torch.bincount(key, minlength=k + 1)
    assert torch.equal(offsets.long()[1:], counts[:k].cumsum(0)) and int(offsets[0]) == 0
    grad = torch.randint(-8, 9, (n, 4), generator=rng(k + 1), device="cuda").float()
    sums = torch.zeros(k + 1, 4, dtype=torch.float64, device="cuda").index_add_(0, key, grad.double())[:k]
    assert torch.equal(ops.lookup_grad(grad, ids, k).double(), sums)   # (whole numbers of less than 2^24)


# ---- as they are used


def test_ids_that_an_engine_leaves_on_the_gpu(ops):
    """Assignments stay on the device: as int32 or as the uint32 that they are, for lookup, grouping and gradient."""
    import numpy as np

    from superkmeans_b200 import Engine

    n, k, d = 5000, 60, 32
    rows = np.random.default_rng(1).standard_normal((n, d)).astype(np.float32)
    engine = Engine(k, d)
    centroids = engine.train(rows)
    x, table = torch.from_numpy(rows).cuda(), torch.from_numpy(centroids).cuda()
    want = torch.from_numpy(engine.assign(rows, centroids).astype(np.int64)).cuda()
    for dtype in (torch.int32, torch.uint32):
        ids = torch.empty(n, dtype=dtype, device="cuda")
        engine.assign(x, table, n=n, on_device=True, out=ids)
        assert torch.equal(as_index(ids, k), want)
        assert torch.equal(ops.lookup(table, ids), table[want])
        groups = ops.group_rows(ids, k)
        assert torch.equal(groups.order.long(), torch.argsort(want, stable=True))
        back = ops.from_clusters(ops.to_clusters(x, groups), groups)
        assert torch.equal(back, x)
        assert torch.equal(ops.lookup_grad(x, ids, k), ops.lookup_grad(x, want, k))


def test_two_threads_that_may_fail(ops):
    """Every turn of both threads ends, and with the right result."""
    import threading

    from tests.test_row_ops_gpu import make_run, whole_run

    runs = [make_run(s) for s in (21, 22)]
    want = [whole_run(ops, *r, 9) for r in runs]
    grads = [ops.lookup_grad(r[0], r[1][:, 0], 9) for r in runs]
    torch.cuda.synchronize()
    done, wrong = [0, 0], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    if not torch.equal(whole_run(ops, *runs[i], 9), want[i]) or not torch.equal(ops.lookup_grad(runs[i][0], runs[i][1][:, 0], 9), grads[i]):
                        wrong.append((i, "another result"))
                    done[i] += 1
        except BaseException as e:
            wrong.append((i, e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and done == [30, 30]

"""Operators on rows in device memory (superkmeans_b200.ops) against plain implementations in 64 bits.

Tolerances count roundings.  A value rounded to a type with `eps` is off by at most eps / 2 of itself, and by half the smallest step
near zero; u = 2^-24 is that of fp32.  A sum of L products in fp32, in whatever order and whether or not products and sums are rounded
together, is off by at most (L + 1) u times the sum of the magnitudes (to first order; the factor 1.01 covers the rest).  Whole numbers
and rows that are only moved are compared exactly."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
STEP = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module", params=["short cuts", "ctypes"])
def ops(request):
    """Every test runs twice: with the short cuts of plain calls, and with all calls on the way through ctypes."""
    from superkmeans_b200 import ops

    class Nothing:
        def __getattr__(self, _):
            return lambda *_: None

    calls = ops._calls
    assert type(calls).__name__ == "module", "_ops_calls.so is not built"
    if request.param == "ctypes":
        ops._calls = Nothing()
    yield ops
    ops._calls = calls


def rng(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rounding(want, dtype, before=0.0):
    """How far a result may be from `want`: `before` in fp32, then one rounding to dtype."""
    half = torch.finfo(dtype).eps / 2
    return 1.01 * (before * (1 + half) + half * want.abs()) + STEP[dtype]


def close(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, worst {float((off - tol)[bad].max() if not off.isnan().any() else float('nan'))} over"


def some_ids(g, n, k, dtype=torch.int32, lost=0.1, skew=False):
    ids = torch.randint(0, k, (n,), generator=g, device="cuda")
    if skew:   # half of them the same
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < 0.5, min(3, k - 1), ids)
    if lost:
        none = torch.tensor([-1, k, -5, 2**31 - 1], device="cuda")[torch.randint(0, 4, (n,), generator=g, device="cuda")]
        ids = torch.where(torch.rand(n, generator=g, device="cuda") < lost, none, ids)
    return ids.to(torch.int32).view(torch.uint32) if dtype == torch.uint32 else ids.to(dtype)


def as_index(ids, k):
    """int64, -1 for none"""
    i = ids.view(torch.int32).long() if ids.dtype == torch.uint32 else ids.long()
    return torch.where((i >= 0) & (i < k), i, -1)


def plain_lookup(table, ids, scale, row_scales):
    i = as_index(ids, table.shape[0])
    rows = table.double()[i.clamp(min=0)] * float(np.float32(scale))
    if row_scales is not None:
        rows = rows * row_scales.double()[..., None]
    return torch.where((i >= 0)[..., None], rows, 0.0)


# ---- lookup


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,d", [(1, 1, 1), (2, 7, 3), (31, 10, 50), (257, 1000, 768), (1000, 33, 130), (5000, 4097, 129), (64, 5, 10_001), (999, 8, 17), (333, 50, 9), (2, 2, 33)])
@pytest.mark.parametrize("scale,scaled", [(1.0, False), (11.4, False), (0.5, True)])
def test_lookup(ops, dtype, n, k, d, scale, scaled):
    g = rng(n + d)
    table, ids = randn(g, k, d, dtype=dtype), some_ids(g, n, k)
    s = torch.exp(randn(g, n)) if scaled else None
    got = ops.lookup(table, ids, scale, s)
    want = plain_lookup(table, ids, scale, s)
    assert got.dtype == dtype
    if scale == 1.0 and not scaled:
        assert torch.equal(got, want.to(dtype))
    else:
        close(got, want, rounding(want, dtype, 2 * U * want.abs()))   # the factor's rounding and the product's
    assert not got[as_index(ids, k) < 0].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [5, 16, 33, 130, 257])
def test_scales_that_are_no_numbers_where_the_id_is_none(ops, dtype, d):
    """Padding may hold anything: zeros come out, and gradients of zero, exactly."""
    g = rng(31)
    n, k = 300, 20
    table, ids = randn(g, k, d, dtype=dtype), some_ids(g, n, k, lost=0.3)
    lost = (ids < 0) | (ids >= k)
    scales = torch.rand(n, generator=g, device="cuda")
    odd = scales.clone()
    odd[lost] = torch.tensor([float("inf"), float("-inf"), float("nan")], device="cuda").repeat(n)[: int(lost.sum())]
    out = ops.lookup(table, ids, 1.0, odd)
    assert lost.any() and not out[lost].any() and torch.equal(out, ops.lookup(table, ids, 1.0, scales))
    grad = randn(g, n, d, dtype=dtype)
    assert torch.equal(ops.lookup_grad(grad, ids, k, 1.0, odd), ops.lookup_grad(grad, ids, k, 1.0, scales))
    grad[lost] = float("nan")
    assert not ops.lookup_grad(grad, ids, k, 1.0, odd).isnan().any()
    assert not ops.lookup_scale_grad(grad, table, ids)[lost].any()


@pytest.mark.parametrize("id_dtype", [torch.int32, torch.uint32, torch.int64])
def test_ids_of_every_type_and_shape(ops, id_dtype):
    g = rng(3)
    table = randn(g, 40, 16)
    ids = some_ids(g, 60, 40, id_dtype).reshape(3, 4, 5)
    assert torch.equal(ops.lookup(table, ids), plain_lookup(table, ids, 1.0, None).float())
    if id_dtype == torch.int64:
        ids = ids.clone()
        ids[0, 0, :3] = torch.tensor([2**32, 2**32 + 1, -(2**40)], device="cuda")   # (their low words are ids)
        assert not ops.lookup(table, ids)[0, 0, :3].any()
    grouped = ops.group_rows(ids.reshape(-1), 40)
    assert int(grouped.offsets[-1]) == int((as_index(ids.reshape(-1), 40) >= 0).sum())
    one = ops.lookup(table, ids.reshape(-1)[7])
    assert one.shape == (16,)


def test_lookup_of_spread_out_and_narrowed_tables(ops):
    g = rng(4)
    wide, ids = randn(g, 50, 200, dtype=torch.bfloat16), some_ids(g, 300, 50)
    for table in (wide[:, 3:131], wide[:, 8:136], wide[::2, :77], wide[:, 1::2], wide.t()[:60], wide[:1].expand(50, 200), wide[4:5]):
        assert torch.equal(ops.lookup(table, ids), plain_lookup(table, ids, 1.0, None).to(torch.bfloat16))
    every_other = ids[::2]
    assert torch.equal(ops.lookup(wide, every_other), plain_lookup(wide, every_other, 1.0, None).to(torch.bfloat16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cut", [slice(1, 40), slice(3, 100), slice(7, 136), slice(5, 38)])
def test_slices_between_values_that_are_no_numbers(ops, dtype, cut):
    """Rows of odd places and lengths, cut out of larger ones: what lies beside them is neither read into results nor written over."""
    g = rng(40)
    d = cut.stop - cut.start

    def beside(n):
        room = torch.full((n, 150), float("nan"), device="cuda", dtype=dtype)
        room[:, cut] = randn(g, n, d, dtype=dtype)
        return room[:, cut]

    table, grad, ids = beside(30), beside(500), some_ids(g, 500, 30)
    s = torch.exp(randn(g, 500))
    plain = table.contiguous(), grad.contiguous()
    assert torch.equal(ops.lookup(table, ids), ops.lookup(plain[0], ids))
    assert torch.equal(ops.lookup(table, ids, 2.0, s), ops.lookup(plain[0], ids, 2.0, s))
    for k in (30, 5000):
        got, want = ops.lookup_grad(grad, ids, k, 1.0, s), ops.lookup_grad(plain[1], ids, k, 1.0, s)
        close(got, want.double(), rounding(want.double(), dtype, 1e-4) + want.double().abs() * torch.finfo(dtype).eps)
    close(ops.lookup_scale_grad(grad, table, ids), ops.lookup_scale_grad(*plain[::-1], ids).double(), 1e-4)
    groups = ops.group_rows(ids.reshape(250, 2), 30)
    x, w = beside(250), randn(g, 250, 2)
    assert torch.equal(ops.to_clusters(x, groups), ops.to_clusters(x.contiguous(), groups))
    assert torch.equal(ops.from_clusters(grad, groups, w), ops.from_clusters(plain[1], groups, w))
    for a, b in zip(ops.from_clusters_grad(x, grad, groups, w), ops.from_clusters_grad(x.contiguous(), plain[1], groups, w)):
        close(a, b.double(), 1e-4)
    for a, b in zip(ops.quantize_rows(x), ops.quantize_rows(x.contiguous())):
        assert torch.equal(a, b)


def test_rows_in_8_bits_leave_what_is_behind_them(ops):
    from superkmeans_b200 import _lib

    x = torch.randn(20, 39, device="cuda", dtype=torch.bfloat16)
    room, scales = torch.full((20, 48), 77, dtype=torch.int8, device="cuda"), torch.empty(20, device="cuda")
    _lib.check(_lib.lib.skm_op_quantize_rows(0, x.data_ptr(), 39, 2, 20, 39, room.data_ptr(), 48, scales.data_ptr(), torch.cuda.current_stream().cuda_stream))
    assert (room[:, 39:] == 77).all() and torch.equal(room[:, :39], ops.quantize_rows(x).values)


def test_values_that_are_no_numbers_stay_in_their_rows(ops):
    table = torch.ones(4, 32, device="cuda")
    table[1] = float("nan")
    table[2, 5] = float("inf")
    ids = torch.tensor([0, 1, 2, -1, 3], device="cuda")
    got = ops.lookup(table, ids, 2.0)
    assert (got[0] == 2).all() and got[1].isnan().all() and got[2, 5].isinf() and (got[3] == 0).all() and (got[4] == 2).all()
    grad = torch.ones(5, 32, device="cuda")
    grad[3] = float("nan")   # of the padding
    grad[1, 0] = float("inf")
    dt = ops.lookup_grad(grad, ids, 4)
    assert torch.isfinite(dt[[0, 2, 3]]).all() and dt[1, 0].isinf() and torch.isfinite(dt[1, 1:]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k,d", [(1, 1, 1), (5, 9, 3), (300, 7, 50), (2001, 300, 130), (4096, 1000, 64), (4097, 1000, 64), (9000, 20, 768), (20_011, 4097, 129), (100, 65_536, 32), (6000, 50, 17), (5001, 4000, 1003)])
@pytest.mark.parametrize("skew", [False, True])
def test_lookup_grad(ops, dtype, n, k, d, skew):
    g = rng(n + k)
    ids, grad, s = some_ids(g, n, k, skew=skew), randn(g, n, d, dtype=dtype), torch.exp(randn(g, n))
    i = as_index(ids, k)
    held = i >= 0
    for scale, scales in ((1.0, None), (3.7, s)):
        terms = grad.double() * float(np.float32(scale)) * (1.0 if scales is None else scales.double()[:, None])
        want = torch.zeros(k, d, dtype=torch.float64, device="cuda").index_add_(0, i[held], terms[held])
        size = torch.zeros(k, d, dtype=torch.float64, device="cuda").index_add_(0, i[held], terms[held].abs())
        count = torch.bincount(i[held], minlength=k)[:, None]
        for out in {dtype, torch.float32}:
            got = ops.lookup_grad(grad, ids, k, scale, scales, dtype=out)
            assert got.dtype == out
            close(got, want, rounding(want, out, (count + 2) * U * size))   # (two more for the factor)
            assert not got[count[:, 0] == 0].any()
        assert torch.equal(got, ops.lookup_grad(grad, ids, k, scale, scales, dtype=out))   # the same bits
    dots = ops.lookup_scale_grad(grad, randn(g, k, d, dtype=dtype), ids, 2.5)
    assert dots.dtype == torch.float32 and not dots[~held].any()


@pytest.mark.parametrize("n,k", [(200_000, 3), (150_000, 100_000)])
def test_lookup_grad_of_long_runs_and_of_many_rows(ops, n, k):
    g = rng(8)
    ids, grad = some_ids(g, n, k, lost=0.0, skew=True), torch.randint(-8, 9, (n, 24), generator=g, device="cuda").float()
    want = torch.zeros(k, 24, dtype=torch.float64, device="cuda").index_add_(0, ids.long(), grad.double())
    assert torch.equal(ops.lookup_grad(grad, ids, k).double(), want)   # (whole numbers: sums of less than 2^24 are exact)


def test_lookup_grad_of_nothing(ops):
    none = torch.full((37,), -1, dtype=torch.int32, device="cuda")
    assert not ops.lookup_grad(torch.ones(37, 8, device="cuda"), none, 12).any()
    assert not ops.lookup_grad(torch.ones(0, 8, device="cuda"), none[:0], 12).any()
    assert ops.lookup(torch.ones(3, 8, device="cuda"), none[:0]).shape == (0, 8)
    assert ops.lookup_scale_grad(torch.ones(0, 8, device="cuda"), torch.ones(3, 8, device="cuda"), none[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", TYPES)
def test_lookup_scale_grad(ops, dtype):
    g = rng(9)
    for n, k, d in ((1, 1, 1), (100, 7, 50), (333, 40, 1025)):
        grad, table, ids = randn(g, n, d, dtype=dtype), randn(g, k, d, dtype=dtype), some_ids(g, n, k)
        i = as_index(ids, k)
        parts = torch.where((i >= 0)[:, None], grad.double() * table.double()[i.clamp(min=0)], 0.0) * float(np.float32(1.3))
        want = parts.sum(1)
        close(ops.lookup_scale_grad(grad, table, ids, 1.3), want, rounding(want, torch.float32, (d + 2) * U * parts.abs().sum(1)))


def test_lookup_is_differentiable(ops):
    g = rng(10)
    table, ids, s = randn(g, 20, 12).requires_grad_(), some_ids(g, 60, 20).reshape(12, 5), torch.exp(randn(g, 12, 5)).requires_grad_()
    up = randn(g, 12, 5, 12)
    out = ops.lookup(table, ids, 1.5, s)
    got = torch.autograd.grad(out, (table, s), up)
    t, r = table.detach().double().requires_grad_(), s.detach().double().requires_grad_()
    i = as_index(ids, 20)
    plain = torch.where((i >= 0)[..., None], t[i.clamp(min=0)] * 1.5 * r[..., None], 0.0)
    want = torch.autograd.grad(plain, (t, r), up.double())
    for a, b in zip(got, want):
        close(a, b, 64 * U * b.abs().max())   # (60 terms at most)
    # against differences: the operator is linear in each argument
    for j, x in enumerate((table, s)):
        v = randn(g, *x.shape)
        moved = [x.detach() + h * v for h in (1, -1)]
        f = [ops.lookup(*((m, ids, 1.5, s.detach()) if j == 0 else (table.detach(), ids, 1.5, m))).double() for m in moved]
        slope = ((f[0] - f[1]) / 2 * up.double()).sum()
        assert abs(float(slope - (got[j].double() * v.double()).sum())) <= 1e-5 * float(((f[0] - f[1]).abs() * up.double().abs()).sum() + 1)
    # each alone, and gradients that come as one number spread out
    assert ops.lookup(table, ids).sum().backward() is None and table.grad is not None
    only = ops.lookup(table.detach(), ids, 1.0, s)
    only.sum().backward()
    assert s.grad is not None
    with torch.no_grad():
        assert not ops.lookup(table, ids).requires_grad


# ---- rows to their clusters and back


def plain_groups(ids, k):
    i = as_index(ids, k).reshape(-1).cpu()
    key = torch.where(i >= 0, i, k)
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel())
    counts = torch.bincount(key, minlength=k + 1)[:k]
    return order, position.reshape(ids.shape), torch.cat([torch.zeros(1, dtype=torch.int64), counts.cumsum(0)])


SORTS = [(1, 1), (2, 1), (33, 5), (1000, 65_536), (4095, 300), (4096, 1), (4097, 1), (5000, 2047), (5000, 2048), (70_000, 255), (140_001, 10_000), (300_000, 5_000_000), (1_100_000, 37), (700, 2**20 - 1), (700, 2**20), (4000, 3_000_000), (1, 3_000_000), (2, 65_536), (3000, 65_537), (150_000, 18_700), (150_000, 18_800), (10_000_000, 300),
         (9_000_000, 5000), (150_000, 47_700), (150_000, 48_000), (4097, 40_000), (700_000, 255), (700_000, 256), (606_209, 30_000), (700_000, 1023), (700_000, 1024), (20_000_003, 500)]


@pytest.mark.parametrize("n,k", SORTS)
@pytest.mark.parametrize("lost", [0.0, 0.2, 1.0])
def test_group_rows(ops, n, k, lost):
    ids = some_ids(rng(n), n, k, lost=lost, skew=n % 2 == 0)
    for got, want in zip(ops.group_rows(ids, k), plain_groups(ids, k)):
        assert got.dtype == torch.int32 and torch.equal(got.cpu().long(), want)


def test_group_rows_of_nothing_and_of_choices(ops):
    order, position, offsets = ops.group_rows(torch.empty(0, 3, dtype=torch.int64, device="cuda"), 5)
    assert order.shape == (0,) and position.shape == (0, 3) and not offsets.any() and offsets.shape == (6,)
    ids = some_ids(rng(2), 90, 7).reshape(30, 3)
    for got, want in zip(ops.group_rows(ids, 7), plain_groups(ids, 7)):
        assert torch.equal(got.cpu().long(), want)
    assert torch.equal(ops.group_rows(ids.t(), 7).order.cpu().long(), plain_groups(ids.t().contiguous(), 7)[0])


MOVES = [(1, 1, 1, 1), (3, 2, 4, 5), (64, 2, 16, 1024), (100, 3, 7, 129), (2000, 8, 300, 50), (5001, 2, 256, 768), (10, 70, 9, 2049), (1, 1, 3, 17), (777, 3, 20, 39)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m,k,d", MOVES)
def test_rows_to_clusters_and_back(ops, dtype, n, m, k, d):
    g = rng(n + m + d)
    ids = some_ids(g, n * m, k, lost=0.15).reshape(n, m)
    groups = ops.group_rows(ids, k)
    held = int(groups.offsets[-1])
    there = as_index(ids, k) >= 0
    x, y, w = randn(g, n, d, dtype=dtype), randn(g, n * m, d, dtype=dtype), randn(g, n, m)
    y[held:] = float("nan")   # slots of choices without a cluster are not looked at
    order, position = groups.order.long(), groups.position.long()

    rows = ops.to_clusters(x, groups)
    want = x[order // m]
    want[held:] = 0
    assert torch.equal(rows, want)

    parts = torch.where(there[..., None], w.double()[..., None] * torch.where(there[..., None], y.double()[position], 0.0), 0.0)
    out = parts.sum(1)
    close(ops.from_clusters(y, groups, w), out, rounding(out, dtype, (m + 1) * U * parts.abs().sum(1)))
    plain = torch.where(there[..., None], y.double()[position], 0.0)
    total = plain.sum(1)
    for got in (ops.from_clusters(y, groups), ops.to_clusters_grad(y, groups)):
        close(got, total, rounding(total, dtype, (m + 1) * U * plain.abs().sum(1)))

    up = randn(g, n, d, dtype=dtype)
    grad_y, grad_w = ops.from_clusters_grad(up, y, groups, w)
    want = w.double().reshape(-1)[order][:, None] * up.double()[order // m]
    want[held:] = 0
    close(grad_y, want, rounding(want, dtype, U * want.abs()))
    parts = torch.where(there[..., None], up.double()[:, None] * torch.where(there[..., None], y.double()[position], 0.0), 0.0)
    close(grad_w, parts.sum(2), rounding(parts.sum(2), torch.float32, (d + 1) * U * parts.abs().sum(2)))
    grad_y, none = ops.from_clusters_grad(up, y, groups)
    assert none is None
    want = up[order // m]
    want[held:] = 0
    assert torch.equal(grad_y, want)


def test_rows_spread_out(ops):
    g = rng(20)
    ids = some_ids(g, 80, 6).reshape(40, 2)
    groups = ops.group_rows(ids, 6)
    wide = randn(g, 40, 300, dtype=torch.bfloat16)
    tall = randn(g, 80, 300, dtype=torch.bfloat16)
    w = randn(g, 40, 2)
    for cut in (slice(1, 129), slice(8, 72), slice(2, 60), slice(0, 300, 2)):
        x, y = wide[:, cut], tall[:, cut]
        assert torch.equal(ops.to_clusters(x, groups), ops.to_clusters(x.contiguous(), groups))
        assert torch.equal(ops.from_clusters(y, groups, w), ops.from_clusters(y.contiguous(), groups, w))
        for a, b in zip(ops.from_clusters_grad(x, y, groups, w), ops.from_clusters_grad(x.contiguous(), y.contiguous(), groups, w)):
            close(a, b.double(), rounding(b.double(), a.dtype, 1e-5 * 300))
    assert torch.equal(ops.to_clusters(wide[:1].expand(40, 300), groups), ops.to_clusters(wide[:1].repeat(40, 1), groups))


def test_routing_is_differentiable(ops):
    g = rng(21)
    n, m, k, d = 30, 3, 5, 20
    ids = some_ids(g, n * m, k, lost=0.2).reshape(n, m)
    groups = ops.group_rows(ids, k)
    x, w = randn(g, n, d).requires_grad_(), torch.softmax(randn(g, n, m), 1).requires_grad_()
    up = randn(g, n, d)
    out = ops.from_clusters(ops.to_clusters(x, groups).square(), groups, w)
    got = torch.autograd.grad(out, (x, w), up)
    a, b = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    there = (as_index(ids, k) >= 0).double()
    plain = (a.square()[:, None] * (b * there)[..., None]).sum(1)
    for p, q in zip(got, torch.autograd.grad(plain, (a, b), up.double())):
        close(p, q, 64 * U * q.abs().max())
    # against differences, in x (a square: central differences are exact) and in w
    for j, t in enumerate((x, w)):
        v = randn(g, *t.shape)
        f = []
        for h in (0.5, -0.5):
            xx, ww = (x.detach() + h * v, w.detach()) if j == 0 else (x.detach(), w.detach() + h * v)
            f.append(ops.from_clusters(ops.to_clusters(xx, groups).square(), groups, ww).double())
        slope = ((f[0] - f[1]) * up.double()).sum()
        assert abs(float(slope - (got[j].double() * v.double()).sum())) <= 1e-5 * float(((f[0].abs() + f[1].abs()) * up.double().abs()).sum())
    # only one of the two wants a gradient
    y = ops.to_clusters(x.detach(), groups)
    assert torch.autograd.grad(ops.from_clusters(y, groups, w).sum(), w)[0].shape == w.shape
    y.requires_grad_()
    assert torch.autograd.grad(ops.from_clusters(y, groups, w.detach()).sum(), y)[0].shape == y.shape
    assert torch.autograd.grad(ops.from_clusters(y, groups).sum(), y)[0].shape == y.shape


def test_groups_that_do_not_belong_to_the_rows_write_nowhere_else(ops):
    # slots beyond the rows: passed over
    groups = ops.RowGroups(*(torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0, 1], [5, 1], [0, 9])))
    x = torch.ones(2, 8, device="cuda")
    assert torch.equal(ops.to_clusters(x, groups)[1], x[1])
    assert torch.equal(ops.from_clusters(x, groups), torch.tensor([[0.0], [1.0]], device="cuda").expand(2, 8))


# ---- products in 8 bits


def plain_quantize(x):
    x = x.float().cpu().numpy()
    most = np.abs(x).max(1)
    with np.errstate(divide="ignore", invalid="ignore"):
        inverse = np.where(most > 0, np.float32(127) / most, np.float32(0)).astype(np.float32)
    return np.rint(x * inverse[:, None]).astype(np.int8), (most / np.float32(127)).astype(np.float32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d", [(1, 1), (5, 3), (1000, 16), (77, 50), (300, 130), (129, 768), (64, 1025), (33, 2048), (9, 5001), (3, 20_000), (1000, 17), (500, 39), (64, 259)])
def test_quantize_rows(ops, dtype, n, d):
    g = rng(d)
    x = (randn(g, n, d) * torch.exp(2 * randn(g, n, 1))).to(dtype)
    if n > 2:
        x[1] = 0
    q, s = ops.quantize_rows(x)
    want_q, want_s = plain_quantize(x)
    assert q.dtype == torch.int8 and (n == 1 or q.stride(0) % 16 == 0)
    assert np.array_equal(q.cpu().numpy(), want_q) and np.array_equal(s.cpu().numpy(), want_s)


def test_quantize_rows_at_the_edges(ops):
    x = torch.tensor([[1e-44, -1e-45, 0.0, 5e-45], [1e-38, 3e-39, -1e-38, 2e-39], [3e38, -1e38, 1.0, 0.0], [float("inf"), 1.0, 2.0, 3.0], [float("nan"), 1.0, -2.0, 0.0],
                      [0.0, -0.0, 0.0, 0.0]], device="cuda")
    q, s = ops.quantize_rows(x)
    assert q[0].tolist() == [127, -18, 0, 73]   # 7, -1, 0, 4 smallest floats: 127 v / 7
    assert q[1].tolist() == [127, 38, -127, 25]
    assert q[2].tolist() == [127, -42, 0, 0] and abs(float(s[2]) * 127 - float(x[2, 0])) <= 2e-7 * 3e38
    for bad in (3, 4):
        assert s[bad].isnan() and not q[bad].any()
    assert float(s[5]) == 0 and not q[5].any()
    wide = torch.randn(40, 300, device="cuda", dtype=torch.bfloat16)
    for cut in (slice(1, 130), slice(8, 72), slice(0, 300, 3)):
        for a, b in zip(ops.quantize_rows(wide[:, cut]), ops.quantize_rows(wide[:, cut].contiguous())):
            assert torch.equal(a, b)


def some_bytes(g, *shape):
    return torch.randint(-127, 128, shape, generator=g, device="cuda").to(torch.int8)


def pitched(q, pitch):
    room = torch.full((*q.shape[:-1], pitch), 99, dtype=torch.int8, device=q.device)
    room[..., : q.shape[-1]] = q
    return room[..., : q.shape[-1]]


def check_product(got, x, xs, w, ws, dtype):
    want = (x.double() @ w.double().T) * xs.double()[:, None] * ws.double()
    close(got, want, rounding(want, dtype, 3 * U * want.abs()))   # the sum's conversion and two products


PRODUCTS = [(1, 1, 1), (1, 16_384, 768), (3, 5, 17), (16, 128, 128), (17, 129, 129), (33, 1000, 50), (64, 300, 4096), (128, 128, 256), (777, 1001, 130), (1000, 64, 16), (300, 4097, 640),
            (5, 100, 40_000), (300, 6000, 256), (4100, 1030, 200), (2000, 1001, 768), (70, 20_001, 33), (8197, 517, 130), (1000, 2048, 1100), (6000, 2000, 700), (20_000, 4112, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,m,d", PRODUCTS)
@pytest.mark.parametrize("aligned", [True, False])
def test_product(ops, dtype, n, m, d, aligned):
    g = rng(n + m + d)
    x, w, xs, ws = some_bytes(g, n, d), some_bytes(g, m, d), torch.exp(randn(g, n)) / 4096, torch.exp(randn(g, m)) / 4096
    pitch = -(-d // 16) * 16 + (16 if aligned else 5)
    check_product(ops.product_8bit(pitched(x, pitch), xs, pitched(w, pitch), ws, dtype=dtype), x, xs, w, ws, dtype)
    check_product(ops.product_8bit(x, xs, w, ws, dtype=dtype), x, xs, w, ws, dtype)


def test_product_of_the_largest_sums(ops):
    # -128 is a byte too: sums up to 128 * 128 * 131071, the largest that 32 bits hold
    d = 131_071
    x = torch.full((2, d), -128, dtype=torch.int8, device="cuda")
    x[1] = 127
    w = torch.full((3, d), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(3, device="cuda")
    got = ops.product_8bit(x, one[:2], w, one, dtype=torch.float32)
    assert torch.equal(got.double(), torch.tensor([[128.0 * 128 * d], [-127.0 * 128 * d]], device="cuda").double().float().double().expand(2, 3))


def test_product_of_scales_that_are_zero_or_no_number(ops):
    g = rng(5)
    x, w = some_bytes(g, 20, 64), some_bytes(g, 30, 64)
    xs, ws = torch.ones(20, device="cuda"), torch.ones(30, device="cuda")
    xs[3], xs[4], ws[7] = float("nan"), 0.0, float("nan")
    got = ops.product_8bit(x, xs, w, ws, dtype=torch.float32)
    assert got[3].isnan().all() and got[:, 7].isnan().all()
    keep = torch.ones(30, dtype=torch.bool)
    keep[7] = False
    assert not got[4, keep].any() and torch.isfinite(got[5:, keep]).all()


GROUPED = [(1, 1, 5, 16), (40, 3, 200, 100), (1000, 300, 64, 32), (3000, 7, 768, 768), (5000, 2, 130, 257), (20_000, 64, 100, 129), (30_000, 9, 301, 200), (9000, 40, 520, 96)]


@pytest.mark.parametrize("n,e,m,d", GROUPED)
@pytest.mark.parametrize("skew", [False, True])
@pytest.mark.parametrize("aligned", [True, False])
def test_product_by_cluster(ops, n, e, m, d, skew, aligned):
    g = rng(n + e)
    ids = some_ids(g, n, e, lost=0.2, skew=skew)
    groups = ops.group_rows(ids, e)
    x, w, xs, ws = some_bytes(g, n, d), some_bytes(g, e, m, d), torch.exp(randn(g, n)) / 4096, torch.exp(randn(g, e, m))
    pitch = -(-d // 16) * 16 + (0 if aligned else 3)
    got = ops.product_8bit(pitched(x, pitch), xs, pitched(w, pitch), ws, groups.offsets, dtype=torch.float32)
    ends = groups.offsets.tolist()
    for c in range(e):
        a, b = ends[c], ends[c + 1]
        check_product(got[a:b], x[a:b], xs[a:b], w[c], ws[c], torch.float32)
    assert not got[ends[-1]:].any()
    # matrices that do not follow one another, and one for all
    apart = torch.stack([w, w], 1)[:, 0]
    assert torch.equal(ops.product_8bit(x, xs, apart, ws, groups.offsets, dtype=torch.float32), got)


def test_product_of_nothing(ops):
    x, w, s = torch.zeros(0, 64, dtype=torch.int8, device="cuda"), torch.zeros(5, 64, dtype=torch.int8, device="cuda"), torch.zeros(5, device="cuda")
    assert ops.product_8bit(x, s[:0], w, s).shape == (0, 5)
    assert ops.product_8bit(w, s, x, s[:0]).shape == (5, 0)
    q, scales = ops.quantize_rows(torch.zeros(0, 9, device="cuda"))
    assert q.shape == (0, 9) and scales.shape == (0,)


def test_a_wait_that_runs_out_in_a_product_is_reported(ops):
    from superkmeans_b200 import _lib

    g = rng(6)
    x, w, xs, ws = some_bytes(g, 300, 8192), some_bytes(g, 500, 8192), torch.ones(300, device="cuda"), torch.ones(500, device="cuda")
    check_product(ops.product_8bit(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws, torch.float32)
    ops.check_products()
    for rows in (300, 10):
        _lib.check(_lib.lib.skm_debug_wait_injection(20_000_000, 1))
        try:
            ops.product_8bit(x[:rows], xs[:rows], w, ws)
            torch.cuda.synchronize()
            with pytest.raises(RuntimeError, match="gave up waiting"):
                ops.product_8bit(x[:rows], xs[:rows], w, ws)
        finally:
            _lib.check(_lib.lib.skm_debug_wait_injection(0, 0))
        ops.check_products()
        check_product(ops.product_8bit(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws, torch.float32)


def test_a_wait_that_ran_out_is_told_under_capture_and_after_it(ops):
    from superkmeans_b200 import _lib

    g = rng(8)
    x, w, xs, ws = some_bytes(g, 40, 4096), some_bytes(g, 200, 4096), torch.ones(40, device="cuda"), torch.ones(200, device="cuda")
    _lib.check(_lib.lib.skm_debug_wait_injection(20_000_000, 1))
    try:
        ops.product_8bit(x, xs, w, ws)
        torch.cuda.synchronize()
    finally:
        _lib.check(_lib.lib.skm_debug_wait_injection(0, 0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="gave up waiting"):
            ops.product_8bit(x, xs, w, ws)
    with pytest.raises(RuntimeError, match="gave up waiting"):
        ops.check_products()
    check_product(ops.product_8bit(x, xs, w, ws, dtype=torch.float32), x, xs, w, ws, torch.float32)
    ops.check_products()


# ---- refusals


def test_refusals(ops):
    x, ids, s = torch.ones(6, 8, device="cuda"), torch.zeros(6, dtype=torch.int32, device="cuda"), torch.ones(6, device="cuda")
    groups = ops.group_rows(ids, 3)
    q = torch.ones(6, 8, dtype=torch.int8, device="cuda")
    wrong = [
        lambda: ops.lookup(x.double(), ids), lambda: ops.lookup(x[0], ids), lambda: ops.lookup(x, ids.float()), lambda: ops.lookup(x, ids, 1.0, s.half()),
        lambda: ops.lookup(x, ids, 1.0, s[:5]), lambda: ops.lookup(x[:0], ids), lambda: ops.lookup(x[:, :0], ids), lambda: ops.lookup(x, ids.cpu()),
        lambda: ops.lookup_grad(x, ids[:5], 3), lambda: ops.lookup_grad(x, ids, 0), lambda: ops.lookup_grad(x, ids, 3, dtype=torch.bfloat16), lambda: ops.lookup_grad(x, ids, 2**31),
        lambda: ops.lookup_scale_grad(x, x[:, :5], ids), lambda: ops.lookup_scale_grad(x, x.half(), ids),
        lambda: ops.group_rows(ids, 0), lambda: ops.group_rows(ids.reshape(1, 2, 3), 3), lambda: ops.group_rows(ids[:, None][:, :0], 3), lambda: ops.group_rows(ids.bool(), 3),
        lambda: ops.to_clusters(x[:5], groups), lambda: ops.from_clusters(x[:5], groups), lambda: ops.from_clusters(x, groups, s[:5]), lambda: ops.from_clusters(x, groups, s.double()),
        lambda: ops.from_clusters_grad(x, x[:, :5], groups, s), lambda: ops.from_clusters_grad(x[:5], x, groups, s),
        lambda: ops.to_clusters(x, ops.RowGroups(ids, ids.long(), groups.offsets)), lambda: ops.to_clusters(x, ops.RowGroups(ids, ids, groups.offsets[:1])),
        lambda: ops.quantize_rows(x.long()), lambda: ops.product_8bit(x, s, q, s), lambda: ops.product_8bit(q, s, q[:, :5], s), lambda: ops.product_8bit(q, s[:5], q, s),
        lambda: ops.product_8bit(q, s, q, s, groups.offsets), lambda: ops.product_8bit(q, s, q.reshape(3, 2, 8), s.reshape(3, 2), groups.offsets.long()),
        lambda: ops.product_8bit(q, s, q.reshape(2, 3, 8), s.reshape(2, 3), groups.offsets), lambda: ops.product_8bit(q, s, q.reshape(3, 2, 8), s, groups.offsets),
    ]
    for i, call in enumerate(wrong):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


# ---- as they are used


def whole_run(ops, x, ids, weights, w, ws, k):
    groups = ops.group_rows(ids, k)
    q, s = ops.quantize_rows(ops.to_clusters(x, groups))
    y = ops.product_8bit(q, s, w, ws, groups.offsets, dtype=x.dtype)
    return ops.from_clusters(y, groups, weights)


def make_run(seed, n=500, m=2, k=9, d=96, c=64):
    g = rng(seed)
    return randn(g, n, d, dtype=torch.bfloat16), some_ids(g, n * m, k, lost=0.1).reshape(n, m), torch.softmax(randn(g, n, m), 1), some_bytes(g, k, c, d), torch.rand(k, c, generator=g, device="cuda") / 500


def test_a_matrix_for_each_cluster(ops):
    x, ids, weights, w, ws = make_run(1)
    got = whole_run(ops, x, ids, weights, w, ws, 9)
    q, s = plain_quantize(x)
    rows = torch.from_numpy(q).cuda().double() * torch.from_numpy(s).cuda().double()[:, None]
    i = as_index(ids, 9)
    want = torch.zeros(500, 64, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(want)
    for j in range(2):
        mats = (w.double() * ws.double()[..., None])[i[:, j].clamp(min=0)]
        part = torch.einsum("nd,ncd->nc", rows, mats) * (weights[:, j].double() * (i[:, j] >= 0))[:, None]
        want += part
        size += part.abs()
    half = torch.finfo(torch.bfloat16).eps / 2
    close(got, want, 1.02 * (half * size + half * want.abs()) + 8 * U * size)   # rounded behind the product and behind the sum


def test_from_training_to_a_codebook(ops):
    """Clusters of a training, their vectors looked up by assignment on the GPU, and one step along the gradient."""
    from superkmeans_b200 import SuperKMeans

    rows = np.random.default_rng(0).standard_normal((4000, 32)).astype(np.float32)
    km = SuperKMeans(50, 32, hierarchical=False, iters=5)
    table = torch.from_numpy(km.train(rows)).cuda()
    ids = torch.from_numpy(km.assign(rows, table.cpu().numpy()).astype(np.int64)).cuda()
    x = torch.from_numpy(rows).cuda()
    table.requires_grad_()
    loss = (ops.lookup(table, ids) - x).square().sum()
    loss.backward()
    # the gradient of the squared distances is 2 (count * centroid - sum), which the update of centroids makes zero
    from superkmeans_b200 import engine

    sums, counts, _ = engine.update_centroids(rows, ids.cpu().numpy().astype(np.uint32), 50)
    want = 2 * (counts[:, None] * table.detach().cpu().numpy().astype(np.float64) - sums)
    bound = 8 * (counts.max() + 4) * U * float(np.abs(rows).max() * counts.max() + 1)   # (both sums; a term is at most 4 max |x|)
    assert np.abs(table.grad.cpu().numpy() - want).max() <= bound


def test_on_another_stream_and_from_a_graph(ops):
    x, ids, weights, w, ws = make_run(2)
    table = randn(rng(3), 9, 96)
    want = whole_run(ops, x, ids, weights, w, ws, 9), ops.lookup_grad(x, ids[:, 0], 9), ops.lookup(table, ids)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        again = whole_run(ops, x, ids, weights, w, ws, 9), ops.lookup_grad(x, ids[:, 0], 9), ops.lookup(table, ids)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    graphs = []
    for _ in range(2):   # two graphs, replayed at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = whole_run(ops, x, ids, weights, w, ws, 9), ops.lookup_grad(x, ids[:, 0], 9), ops.lookup(table, ids)
        graphs.append((graph, out))
    new = make_run(4)
    new_table = randn(rng(5), 9, 96)
    want = whole_run(ops, *new, 9), ops.lookup_grad(new[0], new[1][:, 0], 9), ops.lookup(new_table, new[1])
    for to, v in zip((x, ids, weights, w, ws, table), (*new, new_table)):
        to.copy_(v)
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(side):
            graphs[0][0].replay()
        graphs[1][0].replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_first_calls_of_a_process_in_a_graph(ops):
    """What a call sets up for itself the first time (status words, sizes of shared memory) is no part of the graph."""
    import subprocess
    import sys

    code = """
import torch
from tests import test_row_ops_gpu as t
from superkmeans_b200 import ops
run = t.make_run(2)
grad, ids = t.randn(t.rng(1), 6000, 39, dtype=torch.bfloat16), t.some_ids(t.rng(3), 6000, 700)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = t.whole_run(ops, *run, 9), ops.lookup_grad(grad, ids, 700), ops.product_8bit(run[3][0], run[4][0], run[3][1], run[4][1])
graph.replay()
torch.cuda.synchronize()
want = t.whole_run(ops, *run, 9), ops.lookup_grad(grad, ids, 700), ops.product_8bit(run[3][0], run[4][0], run[3][1], run[4][1])
assert all(torch.equal(a, b) for a, b in zip(out, want))
ops.check_products()
print("captured")
"""
    root = __file__.rsplit("/tests/", 1)[0]
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


def test_backward_in_a_graph(ops):
    table = randn(rng(7), 9, 96, dtype=torch.bfloat16).requires_grad_()
    ids, up = some_ids(rng(8), 700, 9), randn(rng(9), 700, 96, dtype=torch.bfloat16)
    want = ops.lookup_grad(up, ids, 9)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = torch.autograd.grad(ops.lookup(table, ids), table, up)[0]
    grad.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(grad, want)


def test_offsets_beyond_32_bits(ops):
    """More than 2^31 values, and more than 2^32 bytes, in inputs and outputs."""
    n, d = 2_200_000, 1024
    table = torch.arange(2048, device="cuda", dtype=torch.float16)[:, None].expand(2048, d).contiguous()
    ids = (torch.arange(n, device="cuda") * 7919 % 2048).to(torch.int32)
    out = ops.lookup(table, ids)
    at = torch.cat([torch.arange(5), torch.randint(0, n, (2000,)), torch.arange(n - 5, n)]).cuda()
    assert torch.equal(out[at].float(), ids[at].float()[:, None].expand(-1, d))
    groups = ops.group_rows(ids, 2048)
    rows = ops.to_clusters(out, groups)
    assert torch.equal(rows[at][:, 0].float(), ids[groups.order[at].long()].float())
    del out
    back = ops.from_clusters(rows, groups)
    assert torch.equal(back[at].float(), ids[at].float()[:, None].expand(-1, d))
    del back
    q, s = ops.quantize_rows(rows)
    assert torch.equal(s[at], (rows[at][:, 0].double() / 127).float()) and (q[at][:, -1].bool() == s[at].bool()).all()
    got = ops.product_8bit(q, s, q[-3:], torch.ones(3, device="cuda"), dtype=torch.float32)
    close(got[at], (s[at].double() * 127 * 127 * d)[:, None].expand(-1, 3) * (s[at] != 0)[:, None], 4 * U * 2048 * 127 * d + 1e-30)
    del q
    g = ops.lookup_grad(rows, groups.order.remainder(16), 16, dtype=torch.float32)
    want = torch.zeros(16, dtype=torch.float64, device="cuda").index_add_(0, groups.order.long() % 16, ids[groups.order.long()].double())
    close(g[:, 0], want, n * U * want)


def test_from_two_threads(ops):
    import threading

    runs = [make_run(s) for s in (11, 12)]
    want = [whole_run(ops, *r, 9) for r in runs]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                if not torch.equal(whole_run(ops, *runs[i], 9), want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad

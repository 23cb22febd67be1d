"""Tensors that the operators on rows cannot take as they are (superkmeans_b200.ops): refused before anything is asked of their device, so that
no GPU is needed here."""
import pytest
import torch

from superkmeans_b200 import ops as _ops


@pytest.fixture(params=["short cuts", "ctypes"])
def ops(request, monkeypatch):
    if request.param == "ctypes":

        class Nothing:
            def __getattr__(self, _):
                return lambda *_: None

        monkeypatch.setattr(_ops, "_calls", Nothing())
    return _ops


def calls(ops, change):
    """Every operator with one of its tensors put through `change`: (what is changed, call)."""

    def make():
        x, ids, s = torch.ones(6, 8), torch.zeros(6, dtype=torch.int32), torch.ones(6)
        q = torch.ones(6, 8, dtype=torch.int8)
        groups = ops.RowGroups(torch.arange(6, dtype=torch.int32), torch.arange(6, dtype=torch.int32), torch.tensor([0, 6], dtype=torch.int32))
        return x, ids, s, q, groups

    def swapped(groups, i):
        parts = list(groups)
        parts[i] = change(parts[i])
        return ops.RowGroups(*parts)

    x, ids, s, q, groups = make()
    yield "table", lambda: ops.lookup(change(x), ids, 1.0, s)
    yield "ids", lambda: ops.lookup(x, change(ids))
    yield "row_scales", lambda: ops.lookup(x, ids, 1.0, change(s))
    yield "grad", lambda: ops.lookup_grad(change(x), ids, 3)
    yield "ids", lambda: ops.lookup_grad(x, change(ids), 3)
    yield "row_scales", lambda: ops.lookup_grad(x, ids, 3, 1.0, change(s))
    yield "table", lambda: ops.lookup_scale_grad(x, change(x), ids)
    yield "ids", lambda: ops.group_rows(change(ids), 3)
    yield "x", lambda: ops.to_clusters(change(x), groups)
    yield "y", lambda: ops.from_clusters(change(x), groups)
    yield "weights", lambda: ops.from_clusters(x, groups, change(s))
    yield "grad", lambda: ops.to_clusters_grad(change(x), groups)
    yield "y", lambda: ops.from_clusters_grad(x, change(x), groups, s)
    yield "weights", lambda: ops.from_clusters_grad(x, x, groups, change(s))
    for i, name in enumerate(groups._fields):
        yield name, lambda i=i: ops.to_clusters(x, swapped(groups, i))
        yield name, lambda i=i: ops.from_clusters(x, swapped(groups, i), s)
    yield "x", lambda: ops.quantize_rows(change(x))
    yield "x", lambda: ops.product_8bit(change(q), s, q, s)
    yield "w_scales", lambda: ops.product_8bit(q, s, q, change(s))


def part_of_a_freed_storage(t):
    room = torch.cat([t.reshape(-1)[:1], t.reshape(-1)])
    part = room[1:].view(t.shape)
    room.untyped_storage().resize_(0)
    return part


def part_of_a_shortened_storage(t):
    room = t.clone()
    room.untyped_storage().resize_(room.untyped_storage().nbytes() - room.element_size())
    return room


def zeros_without_memory(t):
    return torch._efficientzerotensor((*t.shape[:-1], t.shape[-1] + 1), dtype=t.dtype)[..., 1:]


@pytest.mark.parametrize("change", [part_of_a_freed_storage, part_of_a_shortened_storage, zeros_without_memory])
def test_tensors_without_memory_are_refused(ops, change):
    """(The address of a part of a storage that was freed is its distance from the storage's beginning: a kernel would follow it.)"""
    for name, call in calls(ops, change):
        with pytest.raises(ValueError, match=f"{name} has no memory"):
            call()


def test_empty_and_spread_out_tensors_have_memory(ops):
    x = torch.ones(3, 4)
    for t in (x, x[1:], x[:0], x.t(), x[:1].expand(5, 4), x[1, 2], torch.empty(0), torch.empty(5, 0), x[2:, 3:]):
        ops._check_ordinary(t=t)


def test_imaginary_parts_of_conjugates_are_read_with_their_sign(monkeypatch):
    """(A view, and a contiguous one where there is one column or one number: what lies in its memory has the other sign.)"""
    monkeypatch.setattr(_ops, "_on_gpu", lambda *_: None)
    part = torch.complex(torch.ones(5, 2), torch.arange(10.0).reshape(5, 2)).conj().imag
    assert part.is_neg()
    for t in (part, part[:, :1], part[1:2, :1]):
        rows, n, d, ld, _ = _ops._rows(t, "x")
        assert not rows.is_neg() and (n, d) == t.shape and torch.equal(rows.as_strided((n, d), (ld, 1)), -(-t))
        one = _ops._floats(t, "weights", t.shape, t)
        assert not one.is_neg() and one.is_contiguous() and torch.equal(one, -(-t))


def test_derivatives_carried_forward_are_refused(ops):
    """(A result without its tangent would be taken for a constant.)"""
    with torch.autograd.forward_ad.dual_level():

        def dual(t):
            return torch.autograd.forward_ad.make_dual(t, torch.ones_like(t)) if t.is_floating_point() else t

        seen = 0
        for name, call in calls(ops, dual):
            if name in ("table", "row_scales", "grad", "weights", "y", "w_scales"):
                seen += 1
                with pytest.raises(NotImplementedError, match=f"{name} carries a derivative forward"):
                    call()
        assert seen >= 10
        ops._check_ordinary(t=torch.ones(3), ids=torch.zeros(3, dtype=torch.int32))


def test_calls_are_refused_where_torch_records_them(ops):
    """(A trace would hold the allocation of the output and nothing else, and give back memory as it finds it.)"""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, ids = torch.ones(6, 8), torch.zeros(6, dtype=torch.int32)
    fs = [lambda t: ops.lookup(t, ids), lambda t: ops.lookup(t[1:], ids), lambda t: ops.lookup_grad(t, ids, 3), lambda t: ops.lookup_scale_grad(t, t, ids),
          lambda t: ops.group_rows(t[:, 0].int(), 3).order, lambda t: ops.to_clusters(t, (ids, ids, ids)), lambda t: ops.from_clusters(t, (ids, ids, ids)),
          lambda t: ops.to_clusters_grad(t, (ids, ids, ids)), lambda t: ops.from_clusters_grad(t, t, (ids, ids, ids)), lambda t: ops.quantize_rows(t).values,
          lambda t: ops.product_8bit(t.to(torch.int8), t[:, 0], t.to(torch.int8), t[:, 0])]
    for f in fs:
        with pytest.raises(NotImplementedError, match="not recorded"):
            torch.jit.trace(f, (x,))
        for how in (dict(tracing_mode="real"), dict(tracing_mode="fake"), dict(tracing_mode="symbolic"), dict(pre_dispatch=True)):
            with pytest.raises(NotImplementedError, match="not recorded"):
                make_fx(f, **how)(x)
        with pytest.raises(NotImplementedError, match="torch.func"):
            torch.func.functionalize(f)(x)
    for f in (fs[0], fs[2], fs[5], fs[9]):
        with pytest.raises(NotImplementedError, match="torch.func"):
            torch.func.vmap(f)(torch.ones(2, 6, 8))
        with pytest.raises(NotImplementedError, match="torch.func"):
            torch.func.jvp(f, (x,), (x,))
        with pytest.raises(NotImplementedError, match="torch.func"):
            torch.func.grad(lambda t: f(t).sum())(x)


def test_fake_tensors_are_refused(ops):
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        fake, ids = torch.empty(6, 8, device="cuda"), torch.empty(6, device="cuda", dtype=torch.int32)
        with pytest.raises(NotImplementedError, match="not recorded"):
            ops.lookup(fake[1:], ids)
    with pytest.raises(ValueError, match="table has no memory"):
        ops.lookup(fake, ids)


def test_modes_that_only_look_on_are_none_of_ours(ops):
    from torch.utils._python_dispatch import TorchDispatchMode

    class LooksOn(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    with LooksOn():
        ops._check_ordinary(t=torch.ones(3))
        with pytest.raises(ValueError, match="CUDA"):
            ops.lookup(torch.ones(3, 4), torch.zeros(2, dtype=torch.int32))


@pytest.mark.parametrize("dtype,d", [(0, 1), (0, 3), (0, 4), (1, 1), (1, 7), (2, 8)])
def test_the_workspace_of_narrow_rows_is_mostly_lists(dtype, d):
    """Two lists of n numbers and what sorts them, the ids' first slots, and for every 256 rows two of partial sums (8 floats, as rows are rounded up)."""
    from superkmeans_b200._lib import lib

    n, k = 100_000_000, 1000
    tiles = -(-n // 256)
    most = 2 * 4 * n + lib.skm_op_group_rows_workspace(n, k) + 4 * (k + 1) + tiles * 2 * 8 * 4
    assert lib.skm_op_lookup_grad_workspace(n, k, d, dtype) <= most + 5 * 256

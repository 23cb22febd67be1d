"""Refusals of the operators on rows in device memory, which need no GPU: the Python layer's, and the C ABI's, which come before any
work (the pointers here are never followed)."""
import ctypes as C

import pytest
import torch

from superkmeans_b200 import _lib, ops

lib = _lib.lib
AT = 4096   # an address that is only looked at


def refused(status, text):
    assert status == _lib.SKM_INVALID_ARGUMENT
    assert text in lib.skm_last_error(None).decode()


def test_tensors_must_be_on_a_gpu():
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int32)
    groups = ops.RowGroups(ids, ids, ids)
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: ops.lookup(x, ids), lambda: ops.lookup_grad(x, ids, 4), lambda: ops.lookup_scale_grad(x, x, ids), lambda: ops.group_rows(ids, 4),
                 lambda: ops.to_clusters(x, groups), lambda: ops.to_clusters_grad(x, groups), lambda: ops.from_clusters(x, groups), lambda: ops.from_clusters_grad(x, x, groups),
                 lambda: ops.quantize_rows(x), lambda: ops.product_8bit(q, s, q, s)):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    with pytest.raises(ValueError, match="torch tensor"):
        ops.lookup([[1.0]], ids)
    with pytest.raises(ValueError, match="dtype"):
        ops.product_8bit(q, s, q, s, dtype=torch.int32)


def test_lookup_refusals():
    def call(k=10, d=8, dtype=0, bits=32, n=3, table=AT, ids=AT, out=AT):
        return lib.skm_op_lookup(-1, table, d, dtype, k, d, ids, bits, n, 1.0, None, out, None)

    refused(call(k=0), "clusters")
    refused(call(k=2**31), "clusters")
    refused(call(d=0), "dimensionality")
    refused(call(d=2**20 + 1), "dimensionality")
    refused(call(dtype=3), "dtype")
    refused(call(bits=16), "ids_bits")
    refused(call(n=2**31), "2^31")
    refused(call(table=None), "NULL")
    refused(call(ids=None), "NULL")
    refused(call(out=None), "NULL")
    refused(lib.skm_op_lookup_scale_grad(-1, AT, 8, None, 8, 0, 10, 8, AT, 32, 3, 1.0, AT, None), "NULL")


def test_lookup_grad_refusals():
    need = lib.skm_op_lookup_grad_workspace(5000, 10, 8, 2)
    assert lib.skm_op_lookup_grad_workspace(100, 10, 8, 2) == 0   # (few pairs need none)

    def call(dtype=2, out_dtype=2, grad=AT, out=AT, workspace=AT, size=need, k=10):
        return lib.skm_op_lookup_grad(-1, grad, 8, dtype, k, 8, AT, 32, 5000, 1.0, None, out, out_dtype, workspace, size, None)

    refused(call(out_dtype=1), "fp32")
    refused(call(dtype=0, out_dtype=2), "fp32")
    refused(call(grad=None), "NULL")
    refused(call(out=None), "NULL")
    refused(call(size=need - 1), "workspace")
    refused(call(workspace=None), "workspace")
    refused(call(workspace=AT + 16), "workspace")
    refused(call(k=0), "clusters")


def test_grouping_refusals():
    n, k = 100_000, 5000
    need = lib.skm_op_group_rows_workspace(n, k)
    assert need > 0 and lib.skm_op_group_rows_workspace(100, k) == 0   # (few ids need none)

    def call(n=n, k=k, order=AT, position=AT, offsets=AT, workspace=AT, size=need, bits=64):
        return lib.skm_op_group_rows(-1, AT, bits, n, k, order, position, offsets, workspace, size, None)

    refused(call(k=0), "clusters")
    refused(call(bits=8), "ids_bits")
    refused(call(order=None), "NULL")
    refused(call(position=None), "NULL")
    refused(call(offsets=None), "NULL")
    refused(call(size=need - 1), "workspace")
    refused(call(n=2**31), "2^31")


def test_moving_refusals():
    def to(x=AT, order=AT, position=AT, offsets=AT, k=4, n=3, m=2, d=8, dtype=0, out=AT):
        return lib.skm_op_to_clusters(-1, x, 8, dtype, d, order, position, offsets, k, n, m, out, None)

    refused(to(x=None), "NULL")
    refused(to(order=None), "NULL")
    refused(to(position=None), "NULL")
    refused(to(offsets=None), "NULL")
    refused(to(out=None), "NULL")
    refused(to(m=0), "choice")
    refused(to(n=2**30, m=2), "2^31")
    refused(to(d=0), "dimensionality")
    refused(to(dtype=-1), "dtype")
    refused(lib.skm_op_from_clusters(-1, None, 8, 0, 8, AT, AT, AT, 4, 3, 2, None, AT, None), "NULL")

    def grad(grad=AT, y=AT, grad_y=AT, grad_weights=AT):
        return lib.skm_op_from_clusters_grad(-1, grad, 8, y, 8, 0, 8, AT, AT, AT, 4, 3, 2, None, grad_y, grad_weights, None)

    refused(grad(grad=None), "NULL")
    refused(grad(y=None), "NULL")
    refused(grad(grad_y=None, grad_weights=None), "NULL")


def test_product_refusals():
    def call(x=AT, ld=16, n=5, m=7, d=16, groups=0, offsets=None, out_dtype=0, workspace=None, size=0, scales=AT):
        return lib.skm_op_product_8bit(-1, x, ld, scales, AT, 16, scales, n, m, d, groups, offsets, AT, out_dtype, workspace, size, None)

    refused(call(d=0), "dimensionality")
    refused(call(d=131072), "dimensionality")
    refused(call(out_dtype=5), "dtype")
    refused(call(x=None), "NULL")
    refused(call(scales=None), "NULL")
    refused(call(groups=3), "offsets")
    refused(call(groups=3, offsets=AT), "workspace")   # (the list of tiles)
    refused(call(ld=17), "workspace")                  # (the copy of rows that do not begin on 16 bytes)
    refused(call(m=2**32), "too many")
    refused(call(n=2**31), "2^31")
    refused(lib.skm_op_quantize_rows(-1, AT, 8, 0, 4, 8, AT, 7, AT, None), "overlap")
    refused(lib.skm_op_quantize_rows(-1, None, 8, 0, 4, 8, AT, 16, AT, None), "NULL")


def test_pointers_between_values_are_refused():
    """(No kernel has loads for them: until they were refused such a call answered SKM_OK and left its output as it was.)"""
    def lookup(table=AT, ids=AT, scales=AT, out=AT, dtype=0, bits=32):
        return lib.skm_op_lookup(-1, table, 8, dtype, 10, 8, ids, bits, 3, 1.0, scales, out, None)

    refused(lookup(table=AT + 2), "aligned")
    refused(lookup(table=AT + 1, dtype=2), "aligned")
    refused(lookup(out=AT + 2), "aligned")
    refused(lookup(ids=AT + 4, bits=64), "aligned")
    refused(lookup(scales=AT + 2), "aligned")
    refused(lib.skm_op_lookup_grad(-1, AT + 2, 8, 0, 10, 8, AT, 32, 100, 1.0, None, AT, 0, None, 0, None), "aligned")
    refused(lib.skm_op_lookup_grad(-1, AT, 8, 2, 10, 8, AT, 32, 100, 1.0, None, AT + 2, 0, None, 0, None), "aligned")
    refused(lib.skm_op_lookup_scale_grad(-1, AT, 8, AT + 2, 8, 0, 10, 8, AT, 32, 3, 1.0, AT, None), "aligned")
    refused(lib.skm_op_lookup_scale_grad(-1, AT, 8, AT, 8, 1, 10, 8, AT, 32, 3, 1.0, AT + 2, None), "aligned")
    refused(lib.skm_op_group_rows(-1, AT, 32, 100, 10, AT, AT, AT + 2, None, 0, None), "aligned")
    refused(lib.skm_op_to_clusters(-1, AT + 2, 8, 0, 8, AT, AT, AT, 4, 3, 2, AT, None), "aligned")
    refused(lib.skm_op_to_clusters(-1, AT, 8, 0, 8, AT, AT + 2, AT, 4, 3, 2, AT, None), "aligned")
    refused(lib.skm_op_from_clusters(-1, AT, 8, 1, 8, AT, AT, AT, 4, 3, 2, AT + 2, AT, None), "aligned")
    refused(lib.skm_op_from_clusters(-1, AT, 8, 1, 8, AT, AT, AT, 4, 3, 2, None, AT + 1, None), "aligned")
    refused(lib.skm_op_from_clusters_grad(-1, AT, 8, AT + 1, 8, 1, 8, AT, AT, AT, 4, 3, 2, AT, AT, AT, None), "aligned")
    refused(lib.skm_op_from_clusters_grad(-1, AT, 8, AT, 8, 1, 8, AT, AT, AT, 4, 3, 2, AT, AT, AT + 2, None), "aligned")
    refused(lib.skm_op_quantize_rows(-1, AT + 2, 8, 0, 4, 8, AT, 16, AT, None), "aligned")
    refused(lib.skm_op_quantize_rows(-1, AT, 8, 0, 4, 8, AT, 16, AT + 1, None), "aligned")
    refused(lib.skm_op_product_8bit(-1, AT, 16, AT, AT, 16, AT + 2, 5, 7, 16, 0, None, AT, 0, None, 0, None), "aligned")
    refused(lib.skm_op_product_8bit(-1, AT, 16, AT, AT, 16, AT, 5, 7, 16, 0, None, AT + 2, 0, None, 0, None), "aligned")


def test_workspaces_grow_with_what_they_hold():
    assert lib.skm_op_product_8bit_workspace(AT, 16, AT, 16, 5, 7, 16, 0) == 0
    assert lib.skm_op_product_8bit_workspace(AT, 17, AT, 16, 5, 7, 16, 0) >= 5 * 16
    assert lib.skm_op_product_8bit_workspace(AT + 1, 16, AT, 16, 5, 7, 16, 0) >= 5 * 16
    assert lib.skm_op_product_8bit_workspace(AT, 16, AT, 18, 5, 7, 17, 3) >= 3 * 7 * 32
    for n, k in ((2**40, 5), (5000, 0), (5000, 2**63), (2**64 - 1, 2**64 - 1)):   # (refused sizes need nothing)
        assert lib.skm_op_group_rows_workspace(n, k) == 0 and lib.skm_op_lookup_grad_workspace(n, k, 8, 0) == 0
    assert lib.skm_op_product_8bit_workspace(AT, 17, AT, 17, 2**40, 2**40, 2**40, 2**63) == 0
    small, large = (lib.skm_op_group_rows_workspace(n, 100) for n in (5_000, 5_000_000))
    assert 0 < small < large
    assert lib.skm_op_lookup_grad_workspace(10_000, 10, 64, 0) >= 10_000 * 8 + 11 * 4


def test_signatures_take_64_bit_sizes():
    for name in ("skm_op_lookup", "skm_op_lookup_grad", "skm_op_group_rows", "skm_op_to_clusters", "skm_op_product_8bit"):
        assert C.c_uint64 in _lib.SIGNATURES[name][1]

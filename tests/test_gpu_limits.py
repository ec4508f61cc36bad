"""Sizes and strides at the edge of what the row-selection operators and
gradient clipping can index: refused before anything is launched, or right."""
from __future__ import annotations

import ctypes as C

import pytest
import torch

import spmvbench_b200 as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def at(t):
    return t.data_ptr()


def refused(status, what):
    message = S.load().spmvb_last_error().decode()
    assert status == 1 and what in message, (status, message)


@pytest.mark.parametrize("ld", [2 ** 58, 2 ** 60, 2 ** 62, 2 ** 63 - 1])
def test_strides_whose_extent_wraps_are_refused(ctx, ld):
    """17 rows 2^60 floats apart end 2^66 + 32 bytes on, which is 32 in 64 bits:
    a length that any buffer has."""
    lib = S.load()
    rows, width = 17, 8
    t = torch.zeros(rows, width, device=DEV)
    u, v, x = torch.zeros_like(t), torch.zeros_like(t), torch.zeros_like(t)
    i = torch.zeros(rows, dtype=torch.int32, device=DEV)
    w = torch.zeros(rows, device=DEV)
    torch.cuda.synchronize()
    E = S.Embedding(ctx, rows, width, max_tokens=rows)
    R = S.Router(ctx, width, 1, max_tokens=rows)
    for a, b in ((ld, width), (width, ld)):
        refused(lib.spmvb_embedding_lookup(E.handle, S.F32, rows, at(i), 1.0, at(t), a, at(u), b, None), "63 bits")
        refused(lib.spmvb_embedding_lookup_grad(E.handle, S.F32, rows, at(i), 1.0, at(t), a, S.F32, at(u), b, 0, None), "63 bits")
        refused(lib.spmvb_router_route_grad(R.handle, S.F32, rows, at(t), a, at(i), at(w), at(u), b, None), "63 bits")
        refused(lib.spmvb_router_dispatch(R.handle, S.F32, rows, width, at(i), at(t), a, rows, at(u), b, None), "63 bits")
        refused(lib.spmvb_router_dispatch_grad(R.handle, S.F32, rows, width, at(i), rows, at(t), a, at(u), b, None), "63 bits")
        refused(lib.spmvb_router_combine(R.handle, S.F32, rows, width, at(i), at(w), rows, at(t), a, at(u), b, None), "63 bits")
    refused(lib.spmvb_router_route(R.handle, S.F32, rows, at(t), ld, None, at(i), at(w), None, None, None, None), "63 bits")
    for lds in ((ld, width, width), (width, ld, width), (width, width, ld)):
        refused(lib.spmvb_router_combine_grad(R.handle, S.F32, rows, width, at(i), at(w), rows, at(t), lds[0], at(u), lds[1],
                                              at(v), lds[2], at(x), None), "63 bits")
    ctx.check()


def test_a_lone_row_may_have_any_stride(ctx):
    lib = S.load()
    t, u = torch.arange(8.0, device=DEV).view(1, 8), torch.zeros(1, 8, device=DEV)
    i = torch.zeros(1, dtype=torch.int32, device=DEV)
    E = S.Embedding(ctx, 1, 8, max_tokens=1)
    torch.cuda.synchronize()
    for ld in (8, 2 ** 40, 2 ** 63 - 1):
        u.zero_()
        torch.cuda.synchronize()
        assert lib.spmvb_embedding_lookup(E.handle, S.F32, 1, at(i), 1.0, at(t), ld, at(u), ld, None) == 0
        ctx.check()
        assert torch.equal(t, u)
    # A row of columns beside it in the same buffer is not its own.
    both = torch.arange(64.0, device=DEV).view(2, 32)
    E = S.Embedding(ctx, 1, 16, max_tokens=2)
    E.lookup(torch.zeros(2, dtype=torch.int32, device=DEV), both[:1, :16], both[:, 16:])
    assert torch.equal(both[1, 16:], both[0, :16]) and torch.equal(both[0, 16:], both[0, :16])


@pytest.mark.parametrize("sizes,dtype", [([2 ** 61], S.F64), ([2 ** 62], S.F32), ([2 ** 63 - 1], S.BF16), ([2 ** 63 - 1], S.F64),
                                         ([16, 2 ** 60 - 1], S.F64), ([2 ** 62 - 1] * 3, S.F16)])
def test_clip_sizes_whose_bytes_wrap_are_refused(ctx, sizes, dtype):
    """2^61 doubles are 2^64 bytes, 0 in 64 bits: a length that is in order for
    any pointer."""
    t = torch.zeros(16, device=DEV, dtype=torch.float64)
    n, out = len(sizes), C.c_void_p()
    refused(S.load().spmvb_clip_create(ctx.handle, n, (C.c_void_p * n)(*[at(t)] * n), (C.c_int64 * n)(*sizes),
                                       (C.c_int * n)(*[dtype] * n), C.byref(out)), "63 bits")
    assert not out.value


def test_a_timeout_does_not_swallow_the_report_of_an_index(ctx):
    """A wait that gave up and an index past the end, before the same check:
    both are reported, one after the other."""
    E = S.Embedding(ctx, 4, 8, max_tokens=1)
    out = torch.zeros(1, 8, device=DEV)
    E.lookup(torch.full((1,), 9, dtype=torch.int32, device=DEV), torch.ones(4, 8, device=DEV), out)
    assert S.load().spmvb_selftest_wait_timeout(ctx.handle) == 7
    with pytest.raises(S.SpmvbError) as e:
        ctx.check()
    assert e.value.status == 1 and "out of range" in str(e.value)
    ctx.check()


def test_rows_as_long_as_int32_holds(ctx):
    """Rows of 2^31 - 1 bf16 values, in every operator that moves rows: the
    count of their 16-byte words, and the place of the last, pass int32 on the
    way."""
    width = 2 ** 31 - 1

    def row(value):
        return torch.full((1, width), value, dtype=torch.bfloat16, device=DEV)

    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    x = torch.empty(1, width, dtype=torch.bfloat16, device=DEV).random_(0, 100)
    y = row(7.0)
    E = S.Embedding(ctx, 1, width, max_tokens=1)
    E.lookup(one, x, y)
    assert torch.equal(x, y)
    y.fill_(7.0)
    E.lookup_grad(one, x, y)
    assert torch.equal(x, y)
    E.close()
    R = S.Router(ctx, 4, 1, max_tokens=1)
    w = torch.ones(1, device=DEV)
    for call in (R.dispatch, lambda p, a, b: R.dispatch_grad(p, a, b), lambda p, a, b: R.combine(p, w, a, b)):
        y.fill_(7.0)
        call(one, x, y)
        assert torch.equal(x, y)
    y.fill_(7.0)
    ones, dw = row(1.0), torch.zeros(1, device=DEV)
    R.combine_grad(one, w, ones, x, y, dw)
    assert torch.equal(x, y)
    # The inner product with ones: the sum of x, each of the block's 256 threads'
    # terms in order, then a tree of 256.
    total = x.sum(dtype=torch.float64).item()
    assert abs(dw.item() - total) <= (width / 8 / 256 + 16) * 2.0 ** -24 * total
    ctx.check()
    # Give the blocks back: a later test measures its buffers against their allocation.
    del x, y, ones
    torch.cuda.empty_cache()


@pytest.mark.parametrize("code", [S.F16, S.BF16])
def test_matrices_refuse_16_bit_types_for_their_type(ctx, code):
    """Every entry point of the sparse matrices that takes a type, with all
    other arguments in order."""
    A = S.generate(2, seed=1, scale_rows=64)
    lib, out = S.load(), C.c_void_p()
    at_host = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    refused(lib.spmvb_matrix_create_csr(ctx.handle, code, A.m, A.n, A.nnz, at_host(A.rowptr), at_host(A.colind), at_host(A.values),
                                        C.byref(out)), "bad dtype")
    bounds = S.partition_rows(A.rowptr, 1)
    refused(lib.spmvb_dist_create(ctx.handle, 1, 0, None, code, A.m, A.nnz, at_host(A.rowptr), at_host(A.colind),
                                  at_host(A.values), at_host(bounds), C.byref(out)), "bad dtype")
    M = S.DeviceMatrix(ctx, A, S.F32)
    x, y = torch.zeros(A.n * 4, device=DEV), torch.zeros(A.m * 4, device=DEV)
    hx, hy, ms = S.generate_vector(1, A.n * 4).astype("float32"), S.generate_vector(2, A.m * 4), (C.c_double * 4)()
    h, k = M.handle, S.CSR_SCALAR
    for status in (lambda: lib.spmvb_spmv(h, k, 0, 0, at(x), at(y), code, None),
                   lambda: lib.spmvb_spmv_host(h, k, 0, 0, at_host(hx), at_host(hy), code, None),
                   lambda: lib.spmvb_spmv_time(h, k, 0, 0, at(x), at(y), code, 1, 0, None, ms),
                   lambda: lib.spmvb_spmm(h, 32, 0, 4, at(x), at(y), code, None),
                   lambda: lib.spmvb_spmm_host(h, 32, 0, 4, at_host(hx), at_host(hy), code, None)):
        refused(status(), "bad accumulator dtype")
    P = C.c_void_p()
    assert lib.spmvb_pipeline_create(h, 2, C.byref(P)) == 0
    refused(lib.spmvb_pipeline_submit(P, k, 0, 0, at_host(hx), at_host(hy), code), "bad accumulator dtype")
    assert lib.spmvb_pipeline_destroy(P) == 0
    M.close()


def test_reports_right_after_a_check_are_kept(ctx):
    """An index past the end on a stream that does not wait for the default
    one, enqueued as soon as a check that cleared the last report returns."""
    E = S.Embedding(ctx, 4, 8, max_tokens=1)
    side = torch.cuda.Stream()
    table, out = torch.ones(4, 8, device=DEV), torch.zeros(1, 8, device=DEV)
    bad = torch.full((1,), 9, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    E.lookup(bad, table, out, stream=side)
    for turn in range(200):
        with pytest.raises(S.SpmvbError):
            ctx.check()
        E.lookup(bad, table, out, stream=side)
    with pytest.raises(S.SpmvbError):
        ctx.check()
    ctx.check()

"""The product with an epilogue, what needs no GPU: refusals at the C boundary, before any launch."""
import ctypes as C

import pytest

from ixrun_amd import _lib


def _lanes(out_f=8, in_f=1024):
    return _lib.IxhLanes(3, out_f, in_f, 0x1000, _lib.lib().ixh_lanes_plane_words(out_f, in_f, 3), 0x1000, 0x1000, 0x1000, 64, 0x1000)


@pytest.mark.parametrize("change,code,needle", [
    (dict(ep=None), -1, "epilogue is NULL"), (dict(act=6), -1, "activation"), (dict(act=-1), -1, "activation"), (dict(x=None), -1, "NULL"),
    (dict(y=None), -1, "NULL"), (dict(m=0), -1, "m = 0"), (dict(m=4097), -1, "m = 4097"), (dict(m=2, ldx=1023), -1, "shorter"),
    (dict(m=2, ldy=7), -1, "shorter"), (dict(m=2, multiplier=0x1000, ld_multiplier=7), -1, "shorter"), (dict(m=2, residual=0x1000, ld_residual=7), -1, "shorter"),
    (dict(m=17, x=0x1008), -2, "16-byte"), (dict(m=17, ldx=1028), -2, "16-byte"), (dict(in_f=1020, m=17), -2, "16-byte"),
    (dict(m=16, in_f=4096, out_f=4096), -4, "workspace"), (dict(m=600, in_f=8192, out_f=8192), -4, "workspace"),
])
def test_malformed_products_are_refused(change, code, needle):
    lib = _lib.lib()
    a = dict(dict(in_f=1024, out_f=8, m=1, act=1, x=0x1000, ldx=None, y=0x1000, ldy=None, multiplier=None, ld_multiplier=0, residual=None,
                  ld_residual=0, ep=1), **change)
    lanes = _lanes(a["out_f"], a["in_f"])
    ep = _lib.IxhEpilogue(a["act"], a["multiplier"], a["ld_multiplier"], a["residual"], a["ld_residual"])
    rc = lib.ixh_lanes_product(C.byref(lanes), a["x"], a["ldx"] or a["in_f"], None, a["m"], C.byref(ep) if a["ep"] else None, a["y"],
                               a["ldy"] or a["out_f"], None, 0, None)
    assert rc == code and needle in lib.ixh_last_error().decode()


def test_product_scratch_is_that_of_the_product_by_itself():
    lib = _lib.lib()
    lanes = _lanes(4096, 4096)
    for m in (1, 5, 16, 17, 100, 4096):
        plain = lib.ixh_lanes_gemv_workspace_bytes if m <= 16 else lib.ixh_lanes_gemm_workspace_bytes
        assert lib.ixh_lanes_product_workspace_bytes(C.byref(lanes), m) == plain(C.byref(lanes), m)
    assert lib.ixh_lanes_product_workspace_bytes(C.byref(lanes), 0) == lib.ixh_lanes_product_workspace_bytes(C.byref(lanes), 4097) == 0


@pytest.mark.parametrize("change,needle", [
    (dict(v=None), "NULL"), (dict(y=None), "NULL"), (dict(m=-1), "-1 x"), (dict(out_f=0), "x 0"), (dict(ldv=7), "shorter"), (dict(ldy=7), "shorter"),
    (dict(act=9), "activation"), (dict(out_f=1 << 24, ldv=1 << 24, ldy=1 << 24), "2 x 16777216"),
])
def test_malformed_epilogues_are_refused(change, needle):
    lib = _lib.lib()
    a = dict(dict(v=0x1000, ldv=8, m=2, out_f=8, y=0x1000, ldy=8, act=1), **change)
    ep = _lib.IxhEpilogue(a["act"], None, 0, None, 0)
    assert lib.ixh_epilogue(a["v"], a["ldv"], a["m"], a["out_f"], C.byref(ep), a["y"], a["ldy"], None) == -1
    assert needle in lib.ixh_last_error().decode()
    assert lib.ixh_epilogue(None, 0, 0, 8, C.byref(_lib.IxhEpilogue(0, None, 0, None, 0)), None, 0, None) == 0


def test_parts_of_a_long_call_are_taken_at_any_stride():
    """Every part that StreamingLinear.product makes passes the boundary's look at the stride (the call ends at the missing scratch), and one
    row more does not."""
    from ixrun_amd.engine import MAX_FUSED_ROWS, MAX_PRODUCT_ROWS, _product_rows

    lib = _lib.lib()
    ep = _lib.IxhEpilogue(1, None, 0, None, 0)
    lanes = _lanes(8192, 8192)

    def code(rows, stride):
        assert lib.ixh_lanes_product_workspace_bytes(C.byref(lanes), rows) > 0  # (without which nothing is launched)
        return lib.ixh_lanes_product(C.byref(lanes), 0x1000, stride, None, rows, C.byref(ep), 0x1000, 8192, None, 0, None)

    borders = {(1 << 31) // rows // 8 * 8 + d for rows in range(130, MAX_PRODUCT_ROWS + 1, 7) for d in (-8, 0, 8)}
    for stride in sorted(borders | {8192, 524672, 1 << 20, 1 << 24}):
        rows = _product_rows(stride)
        if rows > 128:
            assert code(rows, stride) == -4, (rows, stride)
            assert rows == MAX_PRODUCT_ROWS or code(rows + 1, stride) == -2, (rows, stride)
    assert _product_rows(8192) == MAX_PRODUCT_ROWS and _product_rows(1 << 40) == MAX_FUSED_ROWS

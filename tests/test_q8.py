"""Refusals of the 8-bit entry points, in front of any launch (no GPU needed)."""
import pytest


@pytest.mark.parametrize("bad", [dict(x=None), dict(codes=None), dict(scale=None), dict(rows=-1), dict(width=0), dict(width=1025), dict(dtype=7)])
def test_rows_and_restore_refuse(bad):
    from gnn_amd import _lib
    lib = _lib.lib()
    a = dict(x=4096, codes=4096, scale=4096, rows=5, width=128, dtype=0)
    a.update(bad)
    assert lib.mgn_q8_rows(a["x"], a["dtype"], a["rows"], a["width"], 0, a["codes"], a["scale"], None) == -1
    assert b"mgn_q8_rows" in lib.mgn_last_error()
    assert lib.mgn_q8_restore(a["codes"], a["scale"], a["rows"], a["width"], a["dtype"], a["x"], None) == -1
    assert b"mgn_q8_restore" in lib.mgn_last_error()


def test_no_rows_are_no_work():
    from gnn_amd import _lib
    lib = _lib.lib()
    assert lib.mgn_q8_rows(None, 0, 0, 128, 0, None, None, None) == 0
    assert lib.mgn_q8_restore(None, None, 0, 128, 0, None, None) == 0


# G, codes, scale, W, ldw, koff, mask_codes, mask, res, GA, dW, lddw, db, scratch, rows, stream
LINEAR = [4096, 4096, 4096, 4096, 128, 0, 0, None, None, 4096, 4096, 128, 4096, 4096, 64, None]


@pytest.mark.parametrize("change", [{0: None}, {1: None}, {1: 4097}, {2: None}, {3: None}, {4: 127}, {4: 130}, {5: -1}, {5: 4}, {6: 1, 7: 4096}, {10: None},
                                    {11: 127}, {13: None}, {14: 0}, {14: 1 << 31}, {9: None, 6: 1}, {9: None, 7: 4096}, {9: None, 8: 4096}])
def test_linear_backward_refuses(change):
    from gnn_amd import _lib
    lib, a = _lib.lib(), list(LINEAR)
    for i, v in change.items():
        a[i] = v
    assert lib.mgn_train_linear_bwd_q8(*a) < 0
    assert b"mgn_train_linear_bwd_q8" in lib.mgn_last_error()


def test_edge_backward_refuses():
    from gnn_amd import _lib
    lib = _lib.lib()
    ok = [4096] * 20 + [10, 40, None]
    for change in ({0: None}, {0: 4098}, {1: None}, {3: None}, {6: None}, {20: 0}, {21: 0}, {20: 1 << 24}, {21: 1 << 24}):
        a = list(ok)
        for i, v in change.items():
            a[i] = v
        assert lib.mgn_train_edge_bwd_q8(*a) < 0, change

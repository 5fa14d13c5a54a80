"""Refusals of the token-order and 8-bit entry points: bad arguments are
answered before a device is touched.  No compute runs here."""
import ctypes as C

import numpy as np
import pytest

import qgmoe

INV = qgmoe.ERR_INVALID_ARG
ONE = C.c_void_p(256)  # a non-null, aligned pointer that no refused call follows
BIG = 1 << 30


def L():
    return qgmoe.lib()


@pytest.mark.parametrize("args", [
    (ONE, -1, 2, 4, ONE, ONE, ONE), (ONE, 4, 0, 4, ONE, ONE, ONE), (ONE, BIG, 2, 4, ONE, ONE, ONE),
    (ONE, 4, 2, 0, ONE, ONE, ONE), (ONE, 4, 2, 1025, ONE, ONE, ONE), (None, 4, 2, 4, ONE, ONE, ONE),
    (ONE, 4, 2, 4, None, ONE, ONE), (ONE, 4, 2, 4, ONE, None, ONE)])
def test_sort_refuses(args):
    assert L().qgmoe_sort_tokens(*args, None) == INV
    assert "sort_tokens" in qgmoe.last_error()


@pytest.mark.parametrize("T,k,H,a,b,null", [
    (-1, 2, 8, 0, 0, None), (4, 0, 8, 0, 0, None), (BIG, 2, 8, 0, 0, None), (4, 2, 0, 0, 0, None),
    (4, 2, (1 << 22) + 1, 0, 0, None), (4, 2, 8, 3, 0, None), (4, 2, 8, 0, 6, None),
    (4, 2, 8, -1, 0, None), (4, 2, 8, 0, 0, 0), (4, 2, 8, 0, 0, 1), (4, 2, 8, 0, 0, 2)])
def test_row_calls_refuse(T, k, H, a, b, null):
    p = [None if i == null else ONE for i in range(3)]
    assert L().qgmoe_gather_rows(p[0], a, T, k, H, p[1], p[2], b, None) == INV
    assert L().qgmoe_gather_rows_backward(p[0], a, T, k, H, p[1], p[2], b, None) == INV
    assert L().qgmoe_combine_rows(p[0], a, ONE, T, k, H, p[1], p[2], b, None) == INV
    assert L().qgmoe_combine_rows_backward(p[0], a, p[2], b, ONE, T, k, H, p[1], ONE, ONE,
                                           None) == INV


def test_combine_refuses_null_weights():
    assert L().qgmoe_combine_rows(ONE, 0, None, 4, 2, 8, ONE, ONE, 0, None) == INV
    # a gradient needs what it is computed from
    assert L().qgmoe_combine_rows_backward(ONE, 0, None, 0, ONE, 4, 2, 8, ONE, None, ONE, None) == INV
    assert L().qgmoe_combine_rows_backward(ONE, 0, ONE, 0, None, 4, 2, 8, ONE, ONE, None, None) == INV
    # nothing asked for, nothing done
    assert L().qgmoe_combine_rows_backward(ONE, 0, ONE, 0, ONE, 4, 2, 8, ONE, None, None, None) == 0


@pytest.mark.parametrize("dt,at", [(0, 258), (0, 257), (qgmoe.DT_F16, 257), (qgmoe.DT_BF16, 257)])
def test_rows_off_their_elements_are_refused(dt, at):
    odd = C.c_void_p(at)
    for a, b in ((odd, ONE), (ONE, odd)):
        assert L().qgmoe_gather_rows(a, dt, 4, 2, 8, ONE, b, dt, None) == INV
        assert "aligned" in qgmoe.last_error()
        assert L().qgmoe_gather_rows_backward(a, dt, 4, 2, 8, ONE, b, dt, None) == INV
        assert L().qgmoe_combine_rows(a, dt, ONE, 4, 2, 8, ONE, b, dt, None) == INV
    for p in ((odd, ONE, ONE), (ONE, odd, ONE), (ONE, ONE, odd)):
        assert L().qgmoe_combine_rows_backward(p[0], dt, p[1], dt, ONE, 4, 2, 8, ONE, p[2], ONE,
                                               None) == INV
        assert "aligned" in qgmoe.last_error()
    assert L().qgq8_quantize_rows(odd, dt, 4, 1, 8, None, ONE, 16, ONE, None) == INV
    assert "aligned" in qgmoe.last_error()


def test_no_tokens_need_no_pointers():
    assert L().qgmoe_gather_rows(None, 0, 0, 2, 8, None, None, 0, None) == 0
    assert L().qgmoe_combine_rows(None, 0, None, 0, 2, 8, None, None, 0, None) == 0
    assert L().qgq8_quantize_rows(None, 0, 0, 1, 8, None, None, 16, None, None) == 0


@pytest.mark.parametrize("T,k,K,dt,pair,codes,ld,scale", [
    (-1, 1, 8, 0, None, ONE, 16, ONE), (4, 2, 8, 0, None, ONE, 16, ONE),
    (4, 1, 0, 0, None, ONE, 16, ONE), (4, 1, 8, 3, None, ONE, 16, ONE),
    (4, 1, 17, 0, None, ONE, 16, ONE), (4, 1, 8, 0, None, ONE, 24, ONE),
    (4, 1, 8, 0, None, None, 16, ONE), (4, 1, 8, 0, None, C.c_void_p(264), 16, ONE),
    (4, 1, 8, 0, None, ONE, 16, None), (BIG, 2, 8, 0, ONE, ONE, 16, ONE)])
def test_quantize_rows_refuses(T, k, K, dt, pair, codes, ld, scale):
    assert L().qgq8_quantize_rows(ONE, dt, T, k, K, pair, codes, ld, scale, None) == INV


@pytest.mark.parametrize("g,o,i,q,s,sw", [
    (0, 8, 8, ONE, ONE, 0), (1025, 8, 8, ONE, ONE, 0), (1, 0, 8, ONE, ONE, 0),
    (1, 8, 0, ONE, ONE, 0), (1, 8, 131072, ONE, ONE, 0), (1, 7, 8, ONE, ONE, 1),
    (1024, 1 << 22, 8, ONE, ONE, 0), (1, 8, 8, None, ONE, 0), (1, 8, 8, ONE, None, 0)])
def test_create_refuses(g, o, i, q, s, sw):
    h = C.c_void_p()
    assert L().qgq8_create(g, o, i, q, s, sw, 0, 0, C.byref(h)) == INV
    assert not h.value
    assert L().qgq8_create(1, 8, 8, ONE, ONE, 0, 0, 0, None) == INV


def test_null_handles():
    assert L().qgq8_destroy(None) == 0
    assert L().qgq8_forward(None, ONE, 1, ONE) == INV
    assert L().qgq8_matmul_device(None, ONE, 16, ONE, 1, None, ONE, 0, None) == INV
    assert L().qgq8_forward_device(None, ONE, 0, 1, 1, None, None, ONE, 16, ONE, ONE, 0, None) == INV
    assert L().qgq8_sync(None, None) == INV


def test_python_refusals_of_host_arrays():
    import torch
    cpu = torch.zeros((4, 8))
    with pytest.raises(ValueError):
        qgmoe.sort_tokens(torch.zeros((4, 2), dtype=torch.int32), 3)
    with pytest.raises(ValueError):
        qgmoe.quantize_rows(cpu)
    q, s = np.zeros((8, 16), np.int8), np.zeros(8, np.float32)
    for a in ((q[0], s), (q, s[:4]), (q.astype(np.int32), s), (q, s.astype(np.float64)),
              (np.zeros((2, 8, 16), np.int8), s)):
        with pytest.raises(ValueError):
            qgmoe.Int8Linear(*a)

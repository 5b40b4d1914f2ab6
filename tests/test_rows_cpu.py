"""Refusals of the calls on rows of logits: every bad argument is answered
with a status before anything reaches a device (no kernel is launched; the
pointers are numbers)."""
import ctypes

import pytest

import pz_sampling as pz

L = pz._lib
P = 1 << 20  # stands for a device pointer
BAD, UNSUPPORTED, OK = 1, 6, 0


def process(rules=None, *, logits=P, dtype=0, B=2, V=100, ld=100, out=P * 4, out_dtype=0, ld_out=100, **r):
    R = pz.LogitsRules(**r) if rules is None else rules
    return L.pz_process_logits(logits, dtype, B, V, ld, ctypes.byref(R), out, out_dtype, ld_out, None, None)


@pytest.mark.parametrize("kw", [
    dict(logits=None), dict(out=None), dict(B=-1), dict(V=0), dict(ld=99), dict(ld_out=99), dict(dtype=2),
    dict(dtype=0, out_dtype=1), dict(dtype=1, out_dtype=2), dict(logits=P + 2), dict(out=P * 4 + 2),
    dict(out=P + 400), dict(out=P, ld_out=101), dict(out=P, dtype=1, out_dtype=0), dict(hist=P), dict(hist_off=P),
    dict(hist=P, hist_off=P), dict(bias_ids=P, bias_off=P), dict(bias_vals=P), dict(mask_index=P),
    dict(mask=P, mask_ld=3, mask_rows=2), dict(mask=P, mask_ld=4, mask_rows=1),
    dict(mask=P, mask_ld=4, mask_rows=0, mask_index=P), dict(mask=P + 2, mask_ld=4, mask_rows=2),
    dict(mask=P, mask_ld=4, mask_rows=2, mask_index=P + 1), dict(hist=P + 2, hist_off=P, cfg=P),
    dict(hist=P, hist_off=P + 1, cfg=P), dict(hist=P, hist_off=P, cfg=P + 2),
    dict(bias_ids=P, bias_off=P, bias_vals=P + 3),
], ids=str)
def test_process_refuses(kw):
    assert process(**kw) == BAD
    assert L.pz_last_error() == BAD and b"pz_process_logits" in L.pz_last_error_detail()


def test_process_limits_and_empty():
    assert L.pz_process_logits(P, 0, 1, 100, 100, None, P, 0, 100, None, None) == BAD
    assert process(V=(1 << 30) + 1, ld=1 << 31, ld_out=1 << 31) == UNSUPPORTED
    assert process(B=0) == OK


def target(**kw):
    d = dict(ids=P, values=P, ld_ids=4, ld_values=4, K=4, mode=0, temperature=1.0)
    d.update(kw)
    return pz.DistillTarget(**d)


def calls(t, *, logits=P, dtype=0, N=2, V=100, ld=100, loss=P, stats=P, grad=P * 4, ld_grad=100):
    t = None if t is None else ctypes.byref(t)
    return (L.pz_distill_forward(logits, dtype, N, V, ld, t, loss, stats, None),
            L.pz_distill_backward(logits, dtype, N, V, ld, t, stats, None, grad, ld_grad, None),
            L.pz_distill_loss_grad(logits, dtype, N, V, ld, t, loss, grad, ld_grad, None))


@pytest.mark.parametrize("kw", [dict(ids=None), dict(values=None), dict(K=0), dict(ld_ids=3), dict(ld_values=3),
                                dict(ids=P + 2), dict(values=P + 1), dict(n_list=P + 2), dict(weight=P + 2),
                                dict(mode=2), dict(temperature=0.0), dict(temperature=float("nan")),
                                dict(temperature=float("inf")), dict(temperature=-1.0)], ids=str)
def test_distill_refuses_targets(kw):
    assert calls(target(**kw)) == (BAD, BAD, BAD)
    assert b"pz_distill" in L.pz_last_error_detail()


@pytest.mark.parametrize("kw", [dict(logits=None), dict(N=-1), dict(V=0), dict(ld=99), dict(dtype=3),
                                dict(logits=P + 1)], ids=str)
def test_distill_refuses_rows(kw):
    assert calls(target(), **kw) == (BAD, BAD, BAD)


def test_distill_refuses_outputs_and_limits():
    assert calls(None) == (BAD, BAD, BAD)
    assert calls(target(), loss=None)[0] == BAD and calls(target(), loss=None)[2] == BAD
    assert calls(target(), loss=P + 2)[0] == BAD and calls(target(), loss=P + 2)[2] == BAD
    assert calls(target(), stats=None)[1] == BAD and calls(target(), stats=P + 4)[:2] == (BAD, BAD)
    for kw in (dict(grad=None), dict(ld_grad=99), dict(grad=P + 400), dict(grad=P, ld_grad=101), dict(grad=P * 4 + 2)):
        assert calls(target(), **kw)[1:] == (BAD, BAD)
    assert calls(target(K=1025, ld_ids=1025, ld_values=1025)) == (UNSUPPORTED,) * 3
    assert calls(target(), V=(1 << 20) + 1, ld=1 << 21, ld_grad=1 << 21, grad=P << 12) == (UNSUPPORTED,) * 3
    assert calls(target(), N=0) == (OK, OK, OK)


def test_structures_match_the_header():
    assert ctypes.sizeof(pz.LogitsRules) == 80 and ctypes.sizeof(pz.DistillTarget) == 64


def head(hidden=P, dtype=0, B=2, dim=64, ld_h=64, w=P * 2, ld_w=64, ws=P, V=100, out=P * 3, out_dtype=0, ld=100,
         q=P * 4, ld_q=64, s=P):
    return L.pz_lm_head_logits_i8(hidden, dtype, B, dim, ld_h, w, ld_w, ws, V, out, out_dtype, ld, q, ld_q, s, None)


@pytest.mark.parametrize("kw", [
    dict(hidden=None), dict(w=None), dict(ws=None), dict(out=None), dict(q=None), dict(s=None), dict(B=-1),
    dict(dim=0), dict(V=0), dict(ld_h=63), dict(ld_w=48), dict(ld_w=72), dict(ld_q=72), dict(ld_q=48), dict(ld=99),
    dict(dtype=2), dict(out_dtype=2), dict(w=P * 2 + 8), dict(q=P * 4 + 8), dict(hidden=P + 2), dict(out=P * 3 + 2),
    dict(ws=P + 2), dict(s=P + 2), dict(q=P + 16), dict(out=P * 2 - 64), dict(out=P * 4 + 48),
], ids=str)
def test_head_refuses(kw):
    assert head(**kw) == BAD
    assert b"_i8" in L.pz_last_error_detail()


def test_head_limits_and_empty():
    big = dict(dim=1 << 17, ld_h=1 << 17, ld_w=1 << 17, ld_q=1 << 17, hidden=1 << 30, w=1 << 31, out=1 << 32, q=1 << 33)
    assert head(**big) == UNSUPPORTED
    assert head(B=0) == OK
    assert L.pz_matmul_i8(P, 64, P, 0, P, 64, P, 10, 64, P, 0, 10, None) == OK
    assert L.pz_matmul_i8(P, 64, None, 2, P * 2, 64, P, 10, 64, P * 3, 0, 10, None) == BAD
    assert L.pz_quantize_rows_i8(P, 0, 0, 64, 64, P, 64, P, None) == OK
    assert L.pz_quantize_rows_i8(P, 0, 2, 64, 64, P, 60, P, None) == BAD


def test_sizes_that_32_bit_indexes_do_not_hold():
    """Rounded up to a vector or a tile they would wrap: an unwritten row with
    scale 0, a grid of a negative size."""
    top = (1 << 31) - 1
    far = 1 << 40
    for cols in (top, top - 14):
        assert L.pz_quantize_rows_i8(P, 0, 1, cols, 1 << 31, far, 1 << 31, P, None) == UNSUPPORTED
        assert b"2^31" in L.pz_last_error_detail()
    for n in (top, top - 254):
        assert L.pz_matmul_i8(P, 16, P, 1, far, 16, P, n, 16, far * 2, 0, 1 << 31, None) == UNSUPPORTED
        assert L.pz_matmul_i8(far, 16, P, n, P, 16, P, 1, 16, far * 2, 0, 1 << 31, None) == UNSUPPORTED
        assert b"2^31" in L.pz_last_error_detail()
    assert L.pz_quantize_rows_i8(P, 0, 0, top - 15, 1 << 31, far, 1 << 31, P, None) == OK
    assert L.pz_matmul_i8(P, 16, P, 0, far, 16, P, top - 255, 16, far * 2, 0, 1 << 31, None) == OK

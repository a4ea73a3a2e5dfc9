"""Without a GPU: what the operators for sorted rows, gradients and 8-bit rows refuse by their arguments alone, and the plain forms against one another."""
import ctypes as C
import importlib.util
import os
import re

import numpy as np
import pytest

import more_ops_common as M
import ops_common as R
from c0ven_b200 import MoEError, _lib, ops

P = 1 << 20  # an address nothing may look at


def refused(call, *words):
    with pytest.raises(MoEError) as e:
        call()
    assert e.value.status == _lib.MOE_BAD_ARGUMENT, e.value
    for w in words:
        assert w in str(e.value), e.value


SORT = dict(x_ptr=P, type=ops.F32, T=4, n_used=2, n_embd=64, inv_ptr=P, R=8, xs_ptr=P)
SORT_GRAD = dict(dxs_ptr=P, type=ops.F32, R=8, inv_ptr=P, T=4, n_used=2, n_embd=64, dx_ptr=P, w_ptr=P, x_ptr=P, dw_ptr=P)
COMBINE_GRAD = dict(dout_ptr=P, dout_type=ops.F32, y_ptr=P, y_type=ops.F16, R=8, inv_ptr=P, w_ptr=P, T=4, n_used=2, n_embd=64, dy_ptr=P, dw_ptr=P)
ROUTE_GRAD = dict(logits_ptr=P, type=ops.F32, T=8, n_experts=64, n_used=4, ids_ptr=P, dw_ptr=P, dlogits_ptr=P)
QUANTIZE = dict(x_ptr=P, type=ops.F32, T=4, K=64, codes_ptr=P, scales_ptr=P, R=4)


@pytest.mark.parametrize("change, word", [
    (dict(type=39), "type"), (dict(n_used=0), "n_used"), (dict(n_used=17), "n_used"), (dict(n_embd=0), "n_embd"), (dict(n_embd=60), "n_embd"),
    (dict(n_embd=(1 << 24) + 8), "n_embd"), (dict(T=1 << 31), "2^31"), (dict(R=1 << 31), "2^31")])
def test_sorted_rows_refuse(change, word):
    refused(lambda: ops.sort_rows_device(**(SORT | change)), word)
    refused(lambda: ops.sort_rows_grad_device(**(SORT_GRAD | change)), word)
    refused(lambda: ops.combine_rows_grad_device(**(COMBINE_GRAD | {("y_type" if k == "type" else k): v for k, v in change.items()})), word)


@pytest.mark.parametrize("call, args", [(ops.sort_rows_device, SORT), (ops.sort_rows_grad_device, SORT_GRAD)])
def test_strides_refused(call, args):
    refused(lambda: call(**(args | dict(stride=63))), "stride")
    refused(lambda: call(**(args | dict(stride=66))), "stride")  # rows of f32 not 16-byte aligned
    refused(lambda: call(**(args | dict(stride=68, type=ops.BF16))), "stride")
    refused(lambda: call(**(args | dict(stride=1 << 32))), "stride")


def test_gradients_refuse_what_lacks():
    g = lambda **k: ops.sort_rows_grad_device(**(SORT_GRAD | k))  # noqa: E731
    refused(lambda: g(dx_ptr=None, dw_ptr=None), "dx or dw")
    refused(lambda: g(x_ptr=None), "x is required")
    refused(lambda: g(dx_ptr=None, add_ptr=P), "add")
    c = lambda **k: ops.combine_rows_grad_device(**(COMBINE_GRAD | k))  # noqa: E731
    refused(lambda: c(dout_type=8), "dout_type")
    refused(lambda: c(dy_ptr=None, dw_ptr=None), "dy or dw")
    refused(lambda: c(y_ptr=None), "y is required")
    refused(lambda: c(w_ptr=None), "w is required")


@pytest.mark.parametrize("change, word", [
    (dict(n_experts=0), "n_experts"), (dict(n_experts=513), "n_experts"), (dict(n_used=0), "n_used"), (dict(n_used=17), "n_used"),
    (dict(n_experts=3), "n_used"), (dict(score=2), "score"), (dict(type=8), "logits_type"), (dict(stride=63), "stride"), (dict(stride=1 << 32), "stride"),
    (dict(dlogits_stride=63), "dlogits_stride"), (dict(dlogits_stride=1 << 32), "dlogits_stride"), (dict(T=(1 << 24) + 1), "T"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")])
def test_routing_gradient_refuses(change, word):
    refused(lambda: ops.route_logits_grad_device(**(ROUTE_GRAD | change)), word)
    assert _lib.lib().moe_route_logits_grad_device(None, P, 0, None, 8, P, P, P, 0, None) == _lib.MOE_BAD_ARGUMENT


@pytest.mark.parametrize("K", [0, 16, 48, 65568])
def test_row_lengths_refused(K):
    w = ops.I8Weights(1, 64, K, P, P)
    for call in (lambda: ops.i8_quantize_rows_device(**(QUANTIZE | dict(K=K))), lambda: ops.i8_dequantize_rows_device(P, P, 4, K, P, ops.F32),
                 lambda: ops.i8_product_device(w, P, P, 4, None, P, ops.F16), lambda: ops.i8_gate_up_device(w, P, P, 4, None, P, ops.F16)):
        refused(call, "multiple of 32")


def test_8_bit_rows_refused():
    q = lambda **k: ops.i8_quantize_rows_device(**(QUANTIZE | k))  # noqa: E731
    refused(lambda: q(type=39), "type")
    refused(lambda: q(stride=63), "stride")
    refused(lambda: q(stride=66), "stride")
    refused(lambda: q(type=ops.F16, stride=68), "stride")
    refused(lambda: q(R=5), "R be T")
    refused(lambda: q(inv_ptr=P, n_used=17), "n_used")
    refused(lambda: q(inv_ptr=P, n_used=0), "n_used")
    refused(lambda: q(T=1 << 31, R=1 << 31), "2^31")
    refused(lambda: ops.i8_dequantize_rows_device(P, P, 4, 64, P, 8), "type")
    refused(lambda: ops.i8_dequantize_rows_device(P, P, 1 << 31, 64, P, ops.F32), "2^31")


def test_products_refused():
    W = lambda **k: ops.I8Weights(*(dict(n_experts=4, n_out=64, n_in=64, codes_ptr=P, scales_ptr=P) | k).values())  # noqa: E731
    p = lambda w, **k: ops.i8_product_device(**(dict(weights=w, codes_ptr=P, scales_ptr=P, R=8, offsets_ptr=P, y_ptr=P, y_type=ops.F16) | k))  # noqa: E731
    g = lambda w, **k: ops.i8_gate_up_device(**(dict(weights=w, codes_ptr=P, scales_ptr=P, R=8, offsets_ptr=P, h_ptr=P, h_type=ops.F16) | k))  # noqa: E731
    for c in (p, g):
        refused(lambda: c(W(n_experts=0)), "n_experts")
        refused(lambda: c(W(n_experts=513)), "n_experts")
        refused(lambda: c(W(n_out=48)), "n_out")
        refused(lambda: c(W(n_out=0)), "n_out")
        refused(lambda: c(W(), offsets_ptr=None), "offsets")
        refused(lambda: c(W(), R=(1 << 24) + 1), "R")
        w = W()
        w.reserved = 1
        refused(lambda: c(w), "reserved")
    refused(lambda: p(W(), y_type=ops.F32), "y_type")
    refused(lambda: g(W(), h_type=ops.F32), "h_type")
    refused(lambda: g(W(n_out=96)), "multiple of 64")
    refused(lambda: g(W(), swiglu_limit=-1.0), "swiglu_limit")
    refused(lambda: g(W(), swiglu_limit=float("nan")), "swiglu_limit")
    assert _lib.lib().moe_i8_product_device(None, P, P, 8, P, P, ops.F16, None) == _lib.MOE_BAD_ARGUMENT and b"weights" in _lib.lib().moe_ops_error()
    assert C.sizeof(_lib.I8Weights) == 32


def test_nothing_to_do_needs_no_device():
    """Calls of no rows are no errors, and look at no buffer."""
    w = ops.I8Weights(4, 64, 64, P, P)
    ops.sort_rows_device(None, ops.F32, 0, 2, 64, None, 0, None)
    ops.sort_rows_device(P, ops.F32, 4, 2, 64, P, 0, None)
    ops.sort_rows_grad_device(None, ops.F32, 0, None, 0, 2, 64, dx_ptr=P)
    ops.combine_rows_grad_device(None, ops.F32, None, ops.F16, 0, None, P, 0, 2, 64, dy_ptr=P)
    ops.route_logits_grad_device(**(ROUTE_GRAD | dict(T=0)))
    ops.i8_quantize_rows_device(None, ops.F32, 0, 64, None, None, 0)
    ops.i8_dequantize_rows_device(None, None, 0, 64, None, ops.F32)
    ops.i8_product_device(w, None, None, 0, P, None, ops.F16)
    ops.i8_gate_up_device(w, None, None, 0, P, None, ops.F16)


@pytest.mark.parametrize("past", [1 << 32, -(1 << 32), 1 << 63])
def test_numbers_past_32_bits_are_refused(past):
    """None is cut down to its low bits, which alone would be a call that is allowed."""
    weights = dict(n_experts=1, n_out=64, n_in=64, codes_ptr=P, scales_ptr=P)
    w = ops.I8Weights(**weights)
    for call, a in ((ops.sort_rows_device, SORT | dict(T=0, stride=0)), (ops.sort_rows_grad_device, SORT_GRAD | dict(T=0, stride=0)),
                    (ops.combine_rows_grad_device, COMBINE_GRAD | dict(T=0)),
                    (ops.route_logits_grad_device, ROUTE_GRAD | dict(T=0, score=0, stride=0, dlogits_stride=0)),
                    (ops.i8_quantize_rows_device, QUANTIZE | dict(T=0, R=0, stride=0, inv_ptr=P, n_used=1)),
                    (ops.i8_dequantize_rows_device, dict(codes_ptr=P, scales_ptr=P, R=0, K=64, out_ptr=P, type=ops.F32)),
                    (ops.i8_product_device, dict(weights=w, codes_ptr=P, scales_ptr=P, R=0, offsets_ptr=P, y_ptr=P, y_type=ops.F16)),
                    (ops.i8_gate_up_device, dict(weights=w, codes_ptr=P, scales_ptr=P, R=0, offsets_ptr=P, h_ptr=P, h_type=ops.F16)), (ops.I8Weights, weights)):
        call(**a)
        for name, v in a.items():
            if isinstance(v, int) and not name.endswith("_ptr"):
                refused(lambda: call(**(a | {name: v + past})), "stride" if "stride" in name else "32 bits")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_the_plain_gradient_of_routing_agrees_with_differences(score, renorm):
    """Central differences of the weights in 64 bits, a step of 2^-16: off by its square times the third derivative (below 4), and by 2^-53 over it."""
    rng = np.random.default_rng(3)
    T, E, k, step = 4, 24, 5, 2.0 ** -16
    l, dw = rng.standard_normal((T, E)), rng.standard_normal((T, k))
    l[1, 7] = -np.inf
    ids = np.argsort(-l, 1)[:, :k].astype(np.int32)
    ids[2, 3:] = -1
    got, _ = M.route_grad(l, ids, dw, score, renorm, 2.5)
    for e in range(E):
        hi, lo = l.copy(), l.copy()
        hi[:, e] += step
        lo[:, e] -= step
        d = (M.weights_by_logits(hi, ids, score, renorm, 2.5) - M.weights_by_logits(lo, ids, score, renorm, 2.5)) / (2 * step)
        assert np.allclose((d * dw).sum(1), got[:, e], rtol=0, atol=1e-8)


def test_the_plain_weights_are_the_routings():
    rng = np.random.default_rng(4)
    l = rng.standard_normal((6, 32))
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            ids, w, _, _ = R.route(l, 5, score, None, 1, 1, renorm, 1.5)
            assert np.allclose(M.weights_by_logits(l, ids, score, renorm, 1.5), w, rtol=1e-13, atol=0)


def test_the_plain_forms_agree_with_the_cases_plain_forms():
    """Two independent readings of the definitions, on the host: the tests' and the measured cases'."""
    import torch

    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(os.path.dirname(__file__), "..", "perf", "more_operators.py"))
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((7, 160)) * np.exp2(rng.integers(-20, 20, (7, 1)))).astype(np.float32)
    x[3] = 0
    x[4] = np.float32(2.0) * np.arange(-80, 80) / 127  # quotients that lie on borders
    codes, scales = M.quantize(x)
    got = cases._quantize(torch.from_numpy(x))
    assert np.array_equal(got[0].numpy(), codes) and np.array_equal(got[1].numpy(), scales)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            l, dw = rng.standard_normal((9, 40)).astype(np.float32), rng.standard_normal((9, 6)).astype(np.float32)
            ids = np.argsort(-l, 1)[:, :6].astype(np.int32)
            c = dict(op="route_grad", score=score, type="f32", renorm=renorm, scale=2.5)
            out = cases._route_grad_plain(dict(case=c, logits=torch.from_numpy(l), ids=torch.from_numpy(ids), dw=torch.from_numpy(dw)))
            assert np.allclose(out.numpy(), M.route_grad(l.astype(np.float64), ids, dw, score, renorm, 2.5)[0], rtol=0, atol=1e-6)
    inv = np.array([[0, 3], [-1, 2], [1, -1]], np.int32)
    rows, w, dout = rng.standard_normal((4, 8)).astype(np.float32), rng.random((3, 2)).astype(np.float32), rng.standard_normal((3, 8)).astype(np.float32)
    g = cases._gathered(torch.from_numpy(rows), torch.from_numpy(inv)).numpy()
    assert np.array_equal(g, M.gathered(rows, inv).astype(np.float32))
    s = cases._scattered(torch.from_numpy(inv), torch.from_numpy(w[..., None] * dout[:, None]), 4).numpy()
    assert np.array_equal(s, M.sort(dout, inv, w, np.zeros((4, 8), np.float32)))


def test_the_header_says_what_may_be_in_place_and_how_far_numbers_go():
    """The operators' general rule on shared bytes names every output that a call's own text lets be an input, and the limits that the calls hold to."""
    header = open(os.path.join(os.path.dirname(__file__), "..", "include", "moe_layer.h")).read()
    part = header[header.index("/* Operators without a layer"):]
    rule, rest = part.split("*/", 1)
    rule, texts = " ".join(rule.replace("\n *", " ").split()), re.findall(r"/\*(.*?)\*/", rest, re.S)
    allowed = [pair for t in texts for pair in re.findall(r"(\w+_dev) may be (\w+_dev)", t)]
    assert len(allowed) == 3
    for out, of in allowed:
        assert f"{out} its {of}" in rule, (out, of)
    for limit, args in (("T and R are below 2^31", dict(T=1 << 31)), ("T and R are below 2^31", dict(R=1 << 31)), ("strides below 2^32", dict(stride=1 << 32)),
                        ("n_embd is at most 2^24", dict(n_embd=(1 << 24) + 8))):
        assert limit in rule
        refused(lambda: ops.sort_rows_device(**(SORT | args)))

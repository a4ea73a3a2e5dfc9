"""Without a GPU: what the operators without a layer refuse, by their arguments alone, before any device is asked."""
import ctypes as C

import numpy as np
import pytest

import ops_common as R
from c0ven_b200 import MoEError, _lib, ops

P = 1 << 20  # an address nothing may look at


def refused(call, *words):
    with pytest.raises(MoEError) as e:
        call()
    assert e.value.status == _lib.MOE_BAD_ARGUMENT, e.value
    for w in words:
        assert w in str(e.value), e.value


@pytest.mark.parametrize("change, word", [
    (dict(n_experts=0), "n_experts"), (dict(n_experts=513), "n_experts"), (dict(n_used=0), "n_used"), (dict(n_used=17), "n_used"),
    (dict(n_experts=4, n_used=5), "n_used"), (dict(score=2), "score"), (dict(n_groups=7, n_groups_used=1), "n_groups"),
    (dict(n_groups=64, n_groups_used=8, n_experts=128), "n_groups"), (dict(n_groups=8, n_groups_used=0), "n_groups_used"),
    (dict(n_groups=8, n_groups_used=9), "n_groups_used"), (dict(n_groups=32, n_groups_used=1, n_used=8), "n_groups_used"),
    (dict(type=8), "logits_type"), (dict(stride=63), "stride"), (dict(stride=1 << 32), "stride"), (dict(T=(1 << 24) + 1), "T"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(inv_ptr=None), "together"), (dict(offsets_ptr=None), "together"),
    (dict(work_bytes=4 * 64 * 5 - 1, T=100), "work")])
def test_routing_refuses(change, word):
    a = dict(logits_ptr=P, type=ops.F32, T=8, n_experts=64, n_used=4, ids_ptr=P, w_ptr=P, offsets_ptr=P, inv_ptr=P, work_ptr=P, work_bytes=1 << 20)
    refused(lambda: ops.route_logits_device(**(a | change)), word)


def test_work_bytes():
    assert ops.route_work_bytes(1, 64) == 4 * 64 * 2 and ops.route_work_bytes(33, 512) == 4 * 512 * 3
    assert ops.route_work_bytes(1 << 24, 512) == 4 * 512 * ((1 << 19) + 1)


@pytest.mark.parametrize("K", [0, 16, 48, 65568])
def test_row_lengths_refused(K):
    w = ops.Mx4Weights(1, 64, K, P, P)
    for call in (lambda: ops.mx4_quantize_rows_device(P, ops.F32, 4, K, P, P, 4), lambda: ops.mx4_dequantize_rows_device(P, P, 4, K, P, ops.F32),
                 lambda: ops.mx4_from_blocks_device(P, 4, K, P, P), lambda: ops.mx4_product_device(w, P, P, 4, None, P, ops.F16),
                 lambda: ops.mx4_gate_up_device(w, P, P, 4, None, P, P)):
        refused(call, "multiple of 32")


def test_rows_refused():
    q = lambda **k: ops.mx4_quantize_rows_device(**(dict(x_ptr=P, type=ops.F32, T=4, K=64, codes_ptr=P, scales_ptr=P, R=4) | k))  # noqa: E731
    refused(lambda: q(type=39), "type")
    refused(lambda: q(stride=63), "stride")
    refused(lambda: q(stride=66), "stride")          # rows of f32 not 16-byte aligned
    refused(lambda: q(type=ops.F16, stride=68), "stride")
    refused(lambda: q(R=5), "R be T")
    refused(lambda: q(inv_ptr=P, n_used=17), "n_used")
    refused(lambda: q(inv_ptr=P, n_used=0), "n_used")
    refused(lambda: q(T=1 << 31, R=1 << 31), "2^31")
    refused(lambda: ops.mx4_dequantize_rows_device(P, P, 4, 64, P, 8), "type")
    c = lambda **k: ops.combine_rows_device(**(dict(y_ptr=P, y_type=ops.F16, R=8, inv_ptr=P, w_ptr=P, T=4, n_used=2, n_embd=64, out_ptr=P) | k))  # noqa: E731
    refused(lambda: c(y_type=39), "y_type")
    refused(lambda: c(n_used=0), "n_used")
    refused(lambda: c(n_used=17), "n_used")
    refused(lambda: c(n_embd=60), "n_embd")
    refused(lambda: c(n_embd=0), "n_embd")


def test_products_refused():
    W = lambda **k: ops.Mx4Weights(*(dict(n_experts=4, n_out=64, n_in=64, codes_ptr=P, scales_ptr=P) | k).values())  # noqa: E731
    p = lambda w, **k: ops.mx4_product_device(**(dict(weights=w, codes_ptr=P, scales_ptr=P, R=8, offsets_ptr=P, y_ptr=P, y_type=ops.F16) | k))  # noqa: E731
    refused(lambda: p(W(n_experts=0)), "n_experts")
    refused(lambda: p(W(n_experts=513)), "n_experts")
    refused(lambda: p(W(n_out=48)), "n_out")
    refused(lambda: p(W(n_out=0)), "n_out")
    refused(lambda: p(W(), y_type=ops.F32), "y_type")
    refused(lambda: p(W(), offsets_ptr=None), "offsets")
    refused(lambda: p(W(), R=(1 << 24) + 1), "R")
    g = lambda w, **k: ops.mx4_gate_up_device(**(dict(weights=w, codes_ptr=P, scales_ptr=P, R=8, offsets_ptr=P, h_codes_ptr=P, h_scales_ptr=P) | k))  # noqa: E731
    refused(lambda: g(W(n_out=96)), "multiple of 64")
    refused(lambda: g(W(), swiglu_limit=-1.0), "swiglu_limit")
    refused(lambda: g(W(), swiglu_limit=float("nan")), "swiglu_limit")
    w = W()
    w.reserved = 1
    refused(lambda: p(w), "reserved")
    st = _lib.lib().moe_mx4_product_device(None, P, P, 8, P, P, ops.F16, None)
    assert st == _lib.MOE_BAD_ARGUMENT and b"weights" in _lib.lib().moe_ops_error()
    assert _lib.lib().moe_route_logits_device(None, P, 0, None, 8, P, P, None, None, None, 0, None) == _lib.MOE_BAD_ARGUMENT


def test_nothing_to_do_needs_no_device():
    """Calls of no rows are no errors, and look at no buffer."""
    w = ops.Mx4Weights(4, 64, 64, P, P)
    ops.mx4_quantize_rows_device(None, ops.F32, 0, 64, None, None, 0)
    ops.mx4_dequantize_rows_device(None, None, 0, 64, None, ops.F32)
    ops.mx4_from_blocks_device(None, 0, 64, None, None)
    ops.mx4_product_device(w, None, None, 0, P, None, ops.F16)
    ops.mx4_gate_up_device(w, None, None, 0, P, None, None)
    ops.combine_rows_device(None, ops.F16, 0, None, None, 0, 2, 64, None)


def test_messages_are_a_threads_own():
    import threading

    refused(lambda: ops.combine_rows_device(P, 39, 8, P, P, 4, 2, 64, P), "y_type")
    seen = []
    t = threading.Thread(target=lambda: seen.append(_lib.lib().moe_ops_error()))
    t.start()
    t.join()
    assert seen == [b""] and b"y_type" in _lib.lib().moe_ops_error()


def test_the_plain_forms_agree_with_the_cases_plain_forms():
    """Two independent readings of the definitions, on the host: the tests' and the measured cases'."""
    import importlib.util
    import os

    import torch

    spec = importlib.util.spec_from_file_location("operators", os.path.join(os.path.dirname(__file__), "..", "perf", "operators.py"))
    M = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(M)
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((7, 160)) * np.exp2(rng.integers(-20, 20, (7, 1)))).astype(np.float32)
    x[3, :32] = 0
    code, byte = R.quantize(x)
    codes, scales = R.pack(code, byte)
    mc, ms = M._quantize(torch.from_numpy(x))
    assert np.array_equal(ms.numpy(), scales)
    assert np.array_equal(M._values(mc, ms).numpy(), R.values(code, byte)) and np.array_equal(M._values(torch.from_numpy(codes), ms).numpy(), R.values(code, byte))
    for score, bias, groups, used, renorm in (("softmax", False, 1, 1, True), ("sigmoid", True, 8, 3, True), ("softmax", True, 4, 2, False), ("sigmoid", False, 16, 8, False)):
        c = dict(op="route", T=9, E=64, k=6, score=score, type="f32", bias=bias, groups=groups, used=used, renorm=renorm, scale=2.5)
        l = rng.standard_normal((9, 64)).astype(np.float32)
        b = (0.1 * rng.standard_normal(64)).astype(np.float32) if bias else None
        got = M._route_plain(dict(case=c, logits=torch.from_numpy(l), bias=None if b is None else torch.from_numpy(b)))
        ids, w, offsets, inv = R.route(l.astype(np.float64), 6, score, b, groups, used, renorm, 2.5)
        assert np.array_equal(got["ids"], ids) and np.array_equal(got["offsets"], offsets) and np.array_equal(got["inv"], inv)
        assert np.allclose(got["w"], w, rtol=2.0 ** -23, atol=0)


def test_scale_rows_fill_words():
    assert [ops.mx4_scale_row_bytes(k) for k in (32, 128, 160, 2880, 4096)] == [4, 4, 8, 92, 128]
    assert C.sizeof(_lib.Mx4Weights) == 32 and C.sizeof(_lib.RouteConfig) == 32


def test_a_files_mx_tensors_are_listed_and_no_layers(tmp_path):
    """ggml type 39: the table says where the blocks lie, as gguf-py does; a layer of them is refused with the reason."""
    gguf = pytest.importorskip("gguf")
    from c0ven_b200 import synth
    from c0ven_b200.layer import GgufFile, MoELayer

    layer = synth.make_layer(n_embd=256, n_ff=256, n_experts=32, n_used=4, gate_type=synth.Q8_0, seed=9)
    blocks = np.random.default_rng(9).integers(0, 255, (32, 256, 256 // 32 * 17), dtype=np.uint8)
    mx = dict(layer, gate_type=39, gate_exps=blocks, up_exps=blocks)
    synth.write_gguf(tmp_path / "mx.gguf", [mx])
    f = GgufFile(tmp_path / "mx.gguf")
    theirs = {t.name: t for t in gguf.GGUFReader(str(tmp_path / "mx.gguf")).tensors}
    ty, shape, offset, nbytes = f.tensors()["blk.0.ffn_gate_exps.weight"]
    t = theirs["blk.0.ffn_gate_exps.weight"]
    assert (ty, shape, offset, nbytes) == (39, (256, 256, 32), t.data_offset, t.n_bytes) and nbytes == blocks.size
    assert open(tmp_path / "mx.gguf", "rb").read()[offset:offset + nbytes] == blocks.tobytes()
    with pytest.raises(MoEError) as e:
        MoELayer.from_gguf(f, 0)
    assert "type 39" in str(e.value) and "does not decode" in str(e.value)
    with pytest.raises(MoEError) as e:
        MoELayer(mx)
    assert e.value.status == _lib.MOE_BAD_ARGUMENT
    f.close()


@pytest.mark.parametrize("past", [1 << 32, -(1 << 32), 1 << 63])
def test_numbers_past_32_bits_are_refused(past):
    """None is cut down to its low bits, which alone would be a call that is allowed."""
    route = dict(logits_ptr=P, type=ops.F32, T=0, n_experts=64, n_used=4, ids_ptr=P, w_ptr=P, score=0, n_groups=1, n_groups_used=1, stride=0)
    rows = dict(x_ptr=P, type=ops.F32, T=0, K=64, codes_ptr=P, scales_ptr=P, R=0, stride=0, inv_ptr=P, n_used=1)
    back = dict(codes_ptr=P, scales_ptr=P, R=0, K=64, out_ptr=P, type=ops.F32)
    blocks = dict(blocks_ptr=P, R=0, K=64, codes_ptr=P, scales_ptr=P)
    product = dict(weights=ops.Mx4Weights(1, 64, 64, P, P), codes_ptr=P, scales_ptr=P, R=0, offsets_ptr=P, y_ptr=P, y_type=ops.F16)
    gate_up = dict(weights=ops.Mx4Weights(1, 64, 64, P, P), codes_ptr=P, scales_ptr=P, R=0, offsets_ptr=P, h_codes_ptr=P, h_scales_ptr=P)
    combine = dict(y_ptr=P, y_type=ops.F16, R=0, inv_ptr=P, w_ptr=P, T=0, n_used=2, n_embd=64, out_ptr=P)
    weights = dict(n_experts=1, n_out=64, n_in=64, codes_ptr=P, scales_ptr=P)
    for call, a in ((ops.route_logits_device, route), (ops.mx4_quantize_rows_device, rows), (ops.mx4_dequantize_rows_device, back), (ops.mx4_from_blocks_device, blocks),
                    (ops.mx4_product_device, product), (ops.mx4_gate_up_device, gate_up), (ops.combine_rows_device, combine), (ops.Mx4Weights, weights),
                    (ops.route_work_bytes, dict(T=1, n_experts=64)), (ops.mx4_scale_row_bytes, dict(K=64))):
        if call is not ops.route_logits_device:  # which asks for the device before it finds that there is nothing to do
            call(**a)
        for name, v in a.items():
            if isinstance(v, int) and not name.endswith("_ptr"):
                refused(lambda: call(**(a | {name: v + past})), "stride" if name == "stride" else "32 bits")
    refused(lambda: ops.route_logits_device(**(route | dict(T=100, offsets_ptr=P, inv_ptr=P, work_ptr=P, work_bytes=-1))), "32 bits")
    refused(lambda: ops.status(timeout_ms=past), "32 bits")

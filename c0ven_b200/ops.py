"""The operators without a layer of include/moe_layer.h: routing of logits, rows sorted by expert as they are, as MX rows (microscaled 4-bit floating
point) or in 8-bit integers, the experts' products over those and the combine, and the gradients of routing, sorting and combine. All take device addresses and queue on `stream` (the default stream when None), as the layer's
device calls do; the shapes, limits and alignments are the header's, and a call that breaks them raises MoEError."""
from __future__ import annotations

import ctypes as C
import functools

from . import _lib
from .layer import MoEError

SOFTMAX, SIGMOID = 0, 1
F32, F16, BF16 = 0, 1, 30  # ggml's type numbers
BLOCK = 32                 # values an MX scale covers


def _need_words(bits: int):
    """bits: a call's numbers, or-ed together, of those of 64 bits what is above them. ctypes would cut one below 0 or past its width down to its
    low bits without a word."""
    if bits >> 32:
        raise MoEError(_lib.MOE_BAD_ARGUMENT, "a number is below 0 or past its 32 bits (a stride, work_bytes: 64)")


class I8Weights(_lib.I8Weights):
    """n_experts matrices of n_out rows of n_in values on the device, in 8-bit rows (addresses of their codes and f32 scales, one a row)."""

    def __init__(self, n_experts: int, n_out: int, n_in: int, codes_ptr: int, scales_ptr: int):
        _need_words(n_experts | n_out | n_in)
        super().__init__(n_experts, n_out, n_in, 0, codes_ptr, scales_ptr)


class Mx4Weights(_lib.Mx4Weights):
    """n_experts matrices of n_out rows of n_in values on the device, in MX rows (addresses of their codes and scales)."""

    def __init__(self, n_experts: int, n_out: int, n_in: int, codes_ptr: int, scales_ptr: int):
        _need_words(n_experts | n_out | n_in)
        super().__init__(n_experts, n_out, n_in, 0, codes_ptr, scales_ptr)


def _check(st: int):
    if st != _lib.MOE_OK:
        raise MoEError(st, _lib.lib().moe_ops_error().decode())


def route_work_bytes(T: int, n_experts: int) -> int:
    """Bytes of work that route_logits_device takes for the lists of T rows."""
    _need_words(T | n_experts)
    return _lib.lib().moe_route_work_bytes(T, n_experts)


@functools.lru_cache(maxsize=256)
def _route_config(*fields):
    return _lib.RouteConfig(*fields)


def route_logits_device(logits_ptr: int, type: int, T: int, n_experts: int, n_used: int, ids_ptr: int, w_ptr: int, *, score: int = SOFTMAX,
                        bias_ptr: int | None = None, n_groups: int = 1, n_groups_used: int = 1, renorm: bool = True, scale: float = 1.0,
                        stride: int = 0, offsets_ptr: int | None = None, inv_ptr: int | None = None, work_ptr: int | None = None,
                        work_bytes: int = 0, stream: int | None = None):
    """ids and w [T][n_used] from logits [T][n_experts]; with offsets_ptr and inv_ptr the lists of expert order too."""
    _need_words(type | T | n_experts | n_used | score | n_groups | n_groups_used | (stride | work_bytes) >> 64 << 32)
    c = _route_config(n_experts, n_used, score, n_groups, n_groups_used, 0 if renorm else 1, scale, type)
    _check(_lib.lib().moe_route_logits_device(C.byref(c), logits_ptr, stride, bias_ptr, T, ids_ptr, w_ptr, offsets_ptr, inv_ptr, work_ptr,
                                              work_bytes, stream))


def mx4_scale_row_bytes(K: int) -> int:
    """Bytes a row of K values has of scales: one per 32 values, rounded up to a multiple of four."""
    _need_words(K)
    return _lib.lib().moe_mx4_scale_row_bytes(K)


def mx4_quantize_rows_device(x_ptr: int, type: int, T: int, K: int, codes_ptr: int, scales_ptr: int, R: int, *, stride: int = 0,
                             inv_ptr: int | None = None, n_used: int = 1, stream: int | None = None):
    """Rows to MX rows: row t to row t, or to the n_used rows inv[t] names."""
    _need_words(type | T | K | R | n_used | stride >> 64 << 32)
    _check(_lib.lib().moe_mx4_quantize_rows_device(x_ptr, type, stride, T, K, inv_ptr, n_used, R, codes_ptr, scales_ptr, stream))


def mx4_dequantize_rows_device(codes_ptr: int, scales_ptr: int, R: int, K: int, out_ptr: int, type: int, stream: int | None = None):
    """What R MX rows stand for."""
    _need_words(R | K | type)
    _check(_lib.lib().moe_mx4_dequantize_rows_device(codes_ptr, scales_ptr, R, K, out_ptr, type, stream))


def mx4_from_blocks_device(blocks_ptr: int, R: int, K: int, codes_ptr: int, scales_ptr: int, stream: int | None = None):
    """R rows of a GGUF tensor of ggml type 39, in the file's blocks, to MX rows."""
    _need_words(R | K)
    _check(_lib.lib().moe_mx4_from_blocks_device(blocks_ptr, R, K, codes_ptr, scales_ptr, stream))


def mx4_product_device(weights: Mx4Weights, codes_ptr: int, scales_ptr: int, R: int, offsets_ptr: int | None, y_ptr: int, y_type: int,
                       stream: int | None = None):
    """y [R][n_out]: every MX row, in expert order, times its expert's matrix."""
    _need_words(R | y_type)
    _check(_lib.lib().moe_mx4_product_device(C.byref(weights), codes_ptr, scales_ptr, R, offsets_ptr, y_ptr, y_type, stream))


def mx4_gate_up_device(weights: Mx4Weights, codes_ptr: int, scales_ptr: int, R: int, offsets_ptr: int | None, h_codes_ptr: int,
                       h_scales_ptr: int, *, swiglu_limit: float = 0.0, stream: int | None = None):
    """MX rows h [R][n_out / 2] = swiglu of the gate and up products, every row with its expert's."""
    _need_words(R)
    _check(_lib.lib().moe_mx4_gate_up_device(C.byref(weights), codes_ptr, scales_ptr, R, offsets_ptr, swiglu_limit, h_codes_ptr, h_scales_ptr,
                                             stream))


def combine_rows_device(y_ptr: int, y_type: int, R: int, inv_ptr: int, w_ptr: int, T: int, n_used: int, n_embd: int, out_ptr: int, *,
                        residual_ptr: int | None = None, stream: int | None = None):
    """out [T][n_embd] f32: each row's results, weighted and summed in rank order, and its residual."""
    _need_words(y_type | R | T | n_used | n_embd)
    _check(_lib.lib().moe_combine_rows_device(y_ptr, y_type, R, inv_ptr, w_ptr, T, n_used, n_embd, residual_ptr, out_ptr, stream))


def sort_rows_device(x_ptr: int, type: int, T: int, n_used: int, n_embd: int, inv_ptr: int, R: int, xs_ptr: int, *, stride: int = 0,
                     w_ptr: int | None = None, stream: int | None = None):
    """xs [R][n_embd]: row t of x, times w[t][k] where there are weights, to row inv[t][k], for every k."""
    _need_words(type | T | n_used | n_embd | R | stride >> 64 << 32)
    _check(_lib.lib().moe_sort_rows_device(x_ptr, type, stride, T, n_used, n_embd, inv_ptr, w_ptr, R, xs_ptr, stream))


def sort_rows_grad_device(dxs_ptr: int, type: int, R: int, inv_ptr: int, T: int, n_used: int, n_embd: int, *, dx_ptr: int | None = None,
                          w_ptr: int | None = None, x_ptr: int | None = None, stride: int = 0, add_ptr: int | None = None, dw_ptr: int | None = None,
                          stream: int | None = None):
    """dx [T][n_embd] = (add +) what came back for each row, times w where there are weights, summed; dw [T][n_used] = <x[t], dxs[inv[t][k]]>."""
    _need_words(type | R | T | n_used | n_embd | stride >> 64 << 32)
    _check(_lib.lib().moe_sort_rows_grad_device(dxs_ptr, type, R, inv_ptr, w_ptr, x_ptr, stride, T, n_used, n_embd, add_ptr, dx_ptr, dw_ptr, stream))


def combine_rows_grad_device(dout_ptr: int, dout_type: int, y_ptr: int | None, y_type: int, R: int, inv_ptr: int, w_ptr: int | None, T: int, n_used: int,
                             n_embd: int, *, dy_ptr: int | None = None, dw_ptr: int | None = None, stream: int | None = None):
    """dy [R][n_embd]: row inv[t][k] = w[t][k] * dout[t]; dw [T][n_used] = <dout[t], y[inv[t][k]]>."""
    _need_words(dout_type | y_type | R | T | n_used | n_embd)
    _check(_lib.lib().moe_combine_rows_grad_device(dout_ptr, dout_type, y_ptr, y_type, R, inv_ptr, w_ptr, T, n_used, n_embd, dy_ptr, dw_ptr, stream))


def route_logits_grad_device(logits_ptr: int, type: int, T: int, n_experts: int, n_used: int, ids_ptr: int, dw_ptr: int, dlogits_ptr: int, *,
                             score: int = SOFTMAX, bias_ptr: int | None = None, renorm: bool = True, scale: float = 1.0, stride: int = 0,
                             dlogits_stride: int = 0, stream: int | None = None):
    """dlogits [T][n_experts] from dw, the gradient of route_logits_device's w, for the experts ids that it chose."""
    _need_words(type | T | n_experts | n_used | score | (stride | dlogits_stride) >> 64 << 32)
    c = _route_config(n_experts, n_used, score, 1, 1, 0 if renorm else 1, scale, type)
    _check(_lib.lib().moe_route_logits_grad_device(C.byref(c), logits_ptr, stride, bias_ptr, T, ids_ptr, dw_ptr, dlogits_ptr, dlogits_stride, stream))


def i8_quantize_rows_device(x_ptr: int, type: int, T: int, K: int, codes_ptr: int, scales_ptr: int, R: int, *, stride: int = 0,
                            inv_ptr: int | None = None, n_used: int = 1, stream: int | None = None):
    """Rows to 8-bit rows: row t to row t, or to the n_used rows inv[t] names."""
    _need_words(type | T | K | R | n_used | stride >> 64 << 32)
    _check(_lib.lib().moe_i8_quantize_rows_device(x_ptr, type, stride, T, K, inv_ptr, n_used, R, codes_ptr, scales_ptr, stream))


def i8_dequantize_rows_device(codes_ptr: int, scales_ptr: int, R: int, K: int, out_ptr: int, type: int, stream: int | None = None):
    """What R 8-bit rows stand for."""
    _need_words(R | K | type)
    _check(_lib.lib().moe_i8_dequantize_rows_device(codes_ptr, scales_ptr, R, K, out_ptr, type, stream))


def i8_product_device(weights: I8Weights, codes_ptr: int, scales_ptr: int, R: int, offsets_ptr: int | None, y_ptr: int, y_type: int,
                      stream: int | None = None):
    """y [R][n_out]: every 8-bit row, in expert order, times its expert's matrix."""
    _need_words(R | y_type)
    _check(_lib.lib().moe_i8_product_device(C.byref(weights), codes_ptr, scales_ptr, R, offsets_ptr, y_ptr, y_type, stream))


def i8_gate_up_device(weights: I8Weights, codes_ptr: int, scales_ptr: int, R: int, offsets_ptr: int | None, h_ptr: int, h_type: int, *,
                      swiglu_limit: float = 0.0, stream: int | None = None):
    """h [R][n_out / 2] = swiglu of the gate and up products, every row with its expert's."""
    _need_words(R | h_type)
    _check(_lib.lib().moe_i8_gate_up_device(C.byref(weights), codes_ptr, scales_ptr, R, offsets_ptr, swiglu_limit, h_ptr, h_type, stream))


def status(stream: int | None = None, timeout_ms: int = 0):
    """Waits for stream; raises MoEError where that runs out, or where a product on the device, on any stream, gave up one of its own waits since
    the calling thread last asked about this stream: products' results since then are not to be used."""
    _need_words(timeout_ms)
    _check(_lib.lib().moe_ops_status(timeout_ms, stream))

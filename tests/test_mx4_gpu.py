"""On a B200: rows to and from microscaled 4-bit floating point, the experts' products over them and the combine, against the
definitions in 64 bits."""
import numpy as np
import pytest

import ops_common as R
from c0ven_b200 import MoEError, _lib, ops

pytestmark = pytest.mark.gpu
TYPES = {"f32": ops.F32, "f16": ops.F16, "bf16": ops.BF16}


def dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def dev(a, type=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if type is None else t.to(dtype(type))).cuda()


def mx_buffers(rows, K, fill=0xEE):
    import torch

    return (torch.full((rows, K // 2), fill, dtype=torch.uint8, device="cuda"), torch.full((rows, R.scale_row_bytes(K)), fill, dtype=torch.uint8, device="cuda"))


def rows_of(rng, T, K):
    """Rows with all the sizes a type has room for, zeros, signed zeros and values on the borders between codes."""
    x = rng.standard_normal((T, K)) * np.exp2(rng.integers(-12, 13, (T, K // 32)).repeat(32, 1).astype(np.float64))
    b = x.reshape(T, -1, 32)
    b[0, 0] = 0
    b[-1, -1] = -0.0
    borders = np.array([4, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5, 6, 7, -7.5, 7.99, 0.2499, 0.2501, 2.4999, 2.5001, 4.999, 5.001, 0.125, -0.1])
    b[0, -1, :len(borders)] = borders * 0.125
    return x


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T, K", [(1, 32), (3, 96), (5, 2048), (2, 2080), (33, 2880), (1, 65536), (700, 160), (2501, 2080), (19001, 288)])
def test_quantize_rows_bit_for_bit(type, T, K):
    import torch

    rng = np.random.default_rng(T + K)
    x = dev(rows_of(rng, T, K).astype(np.float32), type)
    code, byte = R.quantize(x.double().cpu().numpy())
    codes, scales = mx_buffers(T + 1, K)
    ops.mx4_quantize_rows_device(x.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), T)
    torch.cuda.synchronize()
    want = R.pack(code, byte)
    assert np.array_equal(codes[:T].cpu().numpy(), want[0]) and np.array_equal(scales[:T].cpu().numpy(), want[1])
    assert (codes[T] == 0xEE).all() and (scales[T] == 0xEE).all()
    for out_type in ("f32", "bf16", "f16"):
        out = torch.empty((T, K), dtype=dtype(out_type), device="cuda")
        ops.mx4_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), T, K, out.data_ptr(), TYPES[out_type])
        v = R.values(code, byte)
        exact = torch.from_numpy(v).to(dtype(out_type)).double().numpy()  # rounded once; f32 and bf16 hold every value here
        assert np.array_equal(out.double().cpu().numpy(), exact)
        if out_type != "f16":
            assert np.array_equal(exact, v)


def test_quantize_extremes():
    """The largest and smallest scales, blocks with an infinity or NaN, denormals."""
    import torch

    rng = np.random.default_rng(1)
    x = rng.uniform(1, 2, (9, 64)).astype(np.float32)
    x[0] = np.finfo(np.float32).max
    x[1] = 2.0 ** -126 * x[1]
    x[2] = 2.0 ** -140
    x[3] = np.float32(2.0 ** -149)
    x[4, 3], x[4, 40] = np.inf, -np.inf
    x[5, 63] = np.nan
    x[6] *= np.float32(2.0 ** -125)
    x[7, :32] = 2.0 ** 120
    x[8] *= -1
    codes, scales = mx_buffers(9, 64)
    xd = dev(x)
    ops.mx4_quantize_rows_device(xd.data_ptr(), ops.F32, 9, 64, codes.data_ptr(), scales.data_ptr(), 9)
    code, byte = R.quantize(x)
    want = R.pack(code, byte)
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])
    assert byte[4, 0] == 255 and byte[4, 1] == 255 and byte[5, 0] != 255 and byte[5, 1] == 255 and byte[0, 0] == 252 and byte[3, 0] == 0
    out = torch.empty((9, 64), device="cuda")
    ops.mx4_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), 9, 64, out.data_ptr(), ops.F32)
    assert np.array_equal(out.cpu().numpy().astype(np.float64), R.values(code, byte), equal_nan=True)


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_quantize_extremes_of_16_bit_types(type):
    """An infinity or NaN of either sign at every place of a block, the type's largest and its denormals, magnitudes that differ in their last bit."""
    import torch

    rng = np.random.default_rng(2)
    bits = dev(rng.uniform(-2, 2, (32 * 4 + 8, 96)), type).view(torch.int16).cpu().numpy().view(np.uint16).copy()
    inf = 0x7C00 if type == "f16" else 0x7F80
    for place in range(32):
        for j, b in enumerate((inf, inf | 0x8000, inf | 1, 0xFFFF)):
            bits[4 * place + j, 32 + place] = b
    rest = bits[128:]
    rest[0] = inf - 1                                       # the largest finite value
    rest[1] = rng.integers(0, 4, 96)                        # denormals, zeros among them
    rest[2] = rng.integers(0, 4, 96) | 0x8000
    rest[3] = 1
    rest[4] = rng.integers(0, inf & ~(inf << 1), 96)        # all denormals
    rest[5] = rng.integers(0, inf, 96) | rng.integers(0, 2, 96) * 0x8000
    rest[6] = 0x8000
    rest[7] = rng.integers(inf - 3, inf, 96)
    x = torch.from_numpy(bits.view(np.int16)).view(dtype(type)).cuda()
    T = x.shape[0]
    code, byte = R.quantize(x.double().cpu().numpy())
    want = R.pack(code, byte)
    codes, scales = mx_buffers(T, 96)
    ops.mx4_quantize_rows_device(x.data_ptr(), TYPES[type], T, 96, codes.data_ptr(), scales.data_ptr(), T)
    torch.cuda.synchronize()
    assert (byte[:128, 1] == 255).all() and (byte[:128, 0] != 255).all() and (byte[128:] != 255).all()
    assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


@pytest.mark.parametrize("type", ["f32", "bf16"])
def test_quantize_scatters_strided_rows(type):
    """Every row to the places its assignments have; places of none and rows past R are left as they were."""
    import torch

    rng = np.random.default_rng(2)
    T, K, n, rows = 21, 224, 5, 90
    full = dev(rng.standard_normal((T, 256)).astype(np.float32), type)
    inv = rng.permutation(120)[:T * n].reshape(T, n).astype(np.int32)  # some at rows and past
    inv[3, 2], inv[4, :] = -1, -1
    codes, scales = mx_buffers(rows + 2, K)
    di = dev(inv)
    ops.status()
    ops.mx4_quantize_rows_device(full.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), rows, stride=256, inv_ptr=di.data_ptr(), n_used=n)
    torch.cuda.synchronize()
    c, s = R.pack(*R.quantize(full.double().cpu().numpy()[:, :K]))
    want_c, want_s = np.full((rows + 2, K // 2), 0xEE, np.uint8), np.full((rows + 2, R.scale_row_bytes(K)), 0xEE, np.uint8)
    for t in range(T):
        for r in inv[t]:
            if 0 <= r < rows:
                want_c[r], want_s[r] = c[t], s[t]
    assert np.array_equal(codes.cpu().numpy(), want_c) and np.array_equal(scales.cpu().numpy(), want_s)


def test_quantize_scatters_many_rows():
    import torch

    rng = np.random.default_rng(4)
    T, K, n = 5003, 1056, 3
    x = dev(rng.standard_normal((T, K)).astype(np.float32), "f16")
    inv = rng.permutation(T * n).reshape(T, n).astype(np.int32)
    codes, scales = mx_buffers(T * n, K)
    di = dev(inv)
    ops.mx4_quantize_rows_device(x.data_ptr(), ops.F16, T, K, codes.data_ptr(), scales.data_ptr(), T * n, inv_ptr=di.data_ptr(), n_used=n)
    torch.cuda.synchronize()
    c, s = R.pack(*R.quantize(x.double().cpu().numpy()))
    for j in range(n):
        assert np.array_equal(codes.cpu().numpy()[inv[:, j]], c) and np.array_equal(scales.cpu().numpy()[inv[:, j]], s)


def test_offsets_past_32_bits():
    """Rows, matrices and results whose places do not fit 32 bits: the last ones are right."""
    import torch

    rng = np.random.default_rng(5)
    T, K = 66000, 65536  # 8.6 GB of bf16, 2.2 GB of codes
    x = torch.zeros((T, K), dtype=torch.bfloat16, device="cuda")
    tail = dev(rng.standard_normal((3, K)).astype(np.float32), "bf16")
    x[-3:] = tail
    codes, scales = mx_buffers(T, K)
    ops.mx4_quantize_rows_device(x.data_ptr(), ops.BF16, T, K, codes.data_ptr(), scales.data_ptr(), T)
    c, s = R.quantize(tail.double().cpu().numpy())
    want = R.pack(c, s)
    assert np.array_equal(codes[-3:].cpu().numpy(), want[0]) and np.array_equal(scales[-3:].cpu().numpy(), want[1]) and (codes[:-3] == 0).all()
    x.fill_(7)
    ops.mx4_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), T, K, x.data_ptr(), ops.BF16)
    assert np.array_equal(x[-3:].double().cpu().numpy(), R.values(c, s)) and (x[:-3] == 0).all()
    # The same 4.3 thousand million values as results of 64 columns, two of which are summed.
    del codes, scales
    rows = T * K // 64
    inv, w = dev(np.array([[rows - 1, rows - 2]], np.int32)), torch.ones((1, 2), device="cuda")
    out = torch.empty((1, 64), device="cuda")
    ops.combine_rows_device(x.data_ptr(), ops.BF16, rows, inv.data_ptr(), w.data_ptr(), 1, 2, 64, out.data_ptr())
    assert torch.equal(out[0], (x.view(-1, 64)[-1].float() + x.view(-1, 64)[-2].float()))
    del x
    # Matrices of more than 2^32 bytes of codes, rows for the last alone.
    E, N, K = 512, 4128, 4128
    wc = torch.zeros((E, N, K // 2), dtype=torch.uint8, device="cuda")
    ws = torch.full((E, N, R.scale_row_bytes(K)), 127, dtype=torch.uint8, device="cuda")
    c1, s1, w1, xc, xs, xv = product_case(rng, 1, N, K, None, 40)
    wc[-1], ws[-1] = c1[0], s1[0]
    offsets = dev(np.array([0] * E + [40], np.int32))
    y = torch.empty((40, N), dtype=torch.float16, device="cuda")
    ops.mx4_product_device(ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), 40, offsets.data_ptr(), y.data_ptr(), ops.F16)
    ops.status()
    want = xv @ w1[0].T
    assert np.linalg.norm(y.double().cpu().numpy() - want) <= (2.0 ** -11 + 1e-5) * np.linalg.norm(want)
    del wc, ws, y
    # Results past 2^32 bytes, and past 2^32 values.
    rows, N, K = 1 << 20, 4128, 32
    (c1, s1), w1 = R.random_mx(rng, (1, N, K))
    xc, xs = torch.zeros((rows, K // 2), dtype=torch.uint8, device="cuda"), torch.full((rows, 4), 127, dtype=torch.uint8, device="cuda")
    (c2, s2), xv = R.random_mx(rng, (5, K), 125, 129)
    xc[-5:], xs[-5:] = dev(c2), dev(s2)
    y = torch.full((rows, N), 7.0, dtype=torch.float16, device="cuda")
    dc, ds = dev(c1), dev(s1)
    ops.mx4_product_device(ops.Mx4Weights(1, N, K, dc.data_ptr(), ds.data_ptr()), xc.data_ptr(), xs.data_ptr(), rows, None, y.data_ptr(), ops.F16)
    ops.status()
    want = xv @ w1[0].T
    assert np.linalg.norm(y[-5:].double().cpu().numpy() - want) <= (2.0 ** -11 + 1e-5) * np.linalg.norm(want) and (y[:-5] == 0).all()


def test_rows_of_a_files_blocks():
    import torch

    rng = np.random.default_rng(3)
    for rows, K in ((1, 32), (5, 160), (3, 9600)):
        code, byte = rng.integers(0, 16, (rows, K), dtype=np.uint8), rng.integers(0, 255, (rows, K // 32), dtype=np.uint8)
        b = code.reshape(rows, -1, 2, 16)
        blocks = np.concatenate([byte[..., None], b[:, :, 0] | b[:, :, 1] << 4], -1)  # the scale; low halves values 0 .. 15, high halves 16 .. 31
        codes, scales = mx_buffers(rows, K)
        bd = dev(blocks)
        ops.mx4_from_blocks_device(bd.data_ptr(), rows, K, codes.data_ptr(), scales.data_ptr())
        torch.cuda.synchronize()
        want = R.pack(code, byte)
        assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


def test_blocks_stand_for_what_gguf_py_says():
    import torch

    gguf = pytest.importorskip("gguf")
    blocks = np.random.default_rng(6).integers(0, 256, (50, 9 * 17), dtype=np.uint8)
    blocks[:, ::17] = np.random.default_rng(7).integers(1, 250, (50, 9))
    codes, scales = mx_buffers(50, 288)
    out, bd = torch.empty((50, 288), device="cuda"), dev(blocks)
    ops.mx4_from_blocks_device(bd.data_ptr(), 50, 288, codes.data_ptr(), scales.data_ptr())
    ops.mx4_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), 50, 288, out.data_ptr(), ops.F32)
    assert np.array_equal(out.cpu().numpy(), gguf.quants.dequantize(blocks, gguf.GGMLQuantizationType.MXFP4))


def product_case(rng, E, N, K, offsets, rows):
    """Weights and rows with their values: w (codes, scales) [E][N], x [rows]."""
    (wc, ws), w = R.random_mx(rng, (E, N, K))
    (xc, xs), x = R.random_mx(rng, (rows, K), 125, 129)
    # Bytes that fill a row's scales up are never read.
    ws[..., K // 32:] = 255
    xs[..., K // 32:] = 255
    return dev(wc), dev(ws), w, dev(xc), dev(xs), x


def by_expert(x, w, offsets, rows, absolute=False):
    out = np.zeros((rows, w.shape[1]))
    if absolute:
        x, w = np.abs(x), np.abs(w)
    for e in range(w.shape[0]):
        a, b = offsets[e], min(offsets[e + 1], rows)
        out[a:b] = x[a:b] @ w[e].T
    return out


def sum_bound(magnitude, K):
    """What an f32 sum of K products (exact themselves: two-bit significands) may be off by: a step of 2^-23 of the running sum a product,
    however the hardware orders or cuts them."""
    return K * 2.0 ** -23 * magnitude


SHAPES = [(1, 32, 32, [5]), (1, 64, 96, [1]), (1, 160, 256, [300]), (3, 128, 64, [0, 7, 130]), (8, 96, 544, [1, 0, 2, 64, 65, 0, 17, 1]),
          (5, 288, 2880, [16, 15, 0, 33, 1]), (2, 2080, 160, [129, 257]), (70, 64, 128, [1] * 70), (4, 32, 4096, [0, 0, 0, 3]), (512, 32, 32, [0, 1] * 256),
          (2, 256, 2880, [225, 33]), (1, 288, 1312, [1793]), (7, 544, 4128, [0, 448, 449, 1, 100, 17, 224]), (1, 32, 65536, [3]), (1, 65536, 32, [2]),
          # Enough rows an expert and items for pairs of CTAs.
          (1, 2080, 160, [900]), (3, 1056, 1312, [209, 0, 1100]), (7, 544, 2880, [0, 448, 449, 1, 100, 17, 1700]), (2, 8224, 96, [33, 64]), (2, 4128, 4064, [417, 16]),
          (1, 65536, 64, [40])]


@pytest.mark.parametrize("y_type", ["f16", "bf16"])
@pytest.mark.parametrize("E, N, K, counts", SHAPES)
def test_products(E, N, K, counts, y_type):
    import torch

    rng = np.random.default_rng(N + K)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used = int(offsets[-1])
    rows = used + 3  # rows of no expert behind the last
    wc, ws, w, xc, xs, x = product_case(rng, E, N, K, offsets, rows)
    y = torch.full((rows + 1, N), 7.0, dtype=dtype(y_type), device="cuda")
    od = dev(offsets)
    for at in (od.data_ptr(),) + ((None,) if E == 1 else ()):
        y[:] = 7.0
        r = rows if at else used
        ops.mx4_product_device(ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), r, at, y.data_ptr(), TYPES[y_type])
        ops.status()
        got, want, size = y.double().cpu().numpy(), by_expert(x, w, offsets, rows), by_expert(x, w, offsets, rows, True)
        assert (got[used:] == 7.0).all()
        off = np.abs(got[:used] - want[:used])
        assert (off <= HALF(y_type) * np.abs(want[:used]) + sum_bound(size[:used], K) * (1 + HALF(y_type)) + 2.0 ** -25).all(), off.max()
        # Taken together the roundings spread: no more than half a step, and the sums' own error is far below it.
        assert np.linalg.norm(off) <= (HALF(y_type) + 1e-5) * np.linalg.norm(want[:used])


def HALF(y_type):
    return R.HALF_STEP[y_type]


def test_offsets_that_say_too_much_are_cut_off():
    """Offsets past R, below 0 or falling: no row outside 0 .. R - 1 is read or written."""
    import torch

    rng = np.random.default_rng(11)
    E, N, K, rows = 4, 64, 64, 40
    wc, ws, w, xc, xs, x = product_case(rng, E, N, K, None, rows)
    y = torch.full((rows + 8, N), 7.0, dtype=torch.float16, device="cuda")
    for offsets, sound in (([0, 10, 20, 30, 1000], [0, 10, 20, 30, 40]), ([-5, 10, 20, 20, 2 ** 31 - 1], [0, 10, 20, 20, 40])):
        y[:] = 7.0
        od = dev(np.array(offsets, np.int32))
        ops.mx4_product_device(ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.F16)
        torch.cuda.synchronize()
        want = by_expert(x, w, np.array(sound), rows)
        got = y.double().cpu().numpy()
        assert (got[rows:] == 7.0).all()
        assert np.linalg.norm(got[:rows] - want) <= (2.0 ** -11 + 1e-5) * np.linalg.norm(want)
    od = dev(np.array([30, 20, 35, 10, 5], np.int32))
    ops.mx4_product_device(ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.F16)
    torch.cuda.synchronize()
    assert (y[rows:] == 7.0).all()


def test_nan_scales_reach_their_rows_alone():
    import torch

    rng = np.random.default_rng(12)
    E, N, K, rows = 2, 64, 320, 50
    wc, ws, w, xc, xs, x = product_case(rng, E, N, K, None, rows)
    xs[17, 3] = 255
    ws[1, 40, 9] = 255
    offsets = dev(np.array([0, 20, 50], np.int32))
    y = torch.empty((rows, N), dtype=torch.bfloat16, device="cuda")
    ops.mx4_product_device(ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), rows, offsets.data_ptr(), y.data_ptr(), ops.BF16)
    bad = torch.isnan(y).cpu().numpy()
    want = np.zeros((rows, N), bool)
    want[17] = True
    want[20:, 40] = True
    assert np.array_equal(bad, want)


@pytest.mark.parametrize("limit", [0.0, 2.0])
@pytest.mark.parametrize("E, F, K, counts", [(1, 32, 32, [5]), (3, 64, 96, [0, 7, 130]), (6, 96, 2880, [1, 0, 33, 64, 2, 0]), (2, 224, 256, [129, 257]), (1, 640, 544, [300]),
                                           (3, 288, 1312, [225, 0, 500]), (2, 160, 2880, [100, 40]),
                                           (1, 1056, 160, [900]), (3, 672, 1312, [209, 0, 1100]), (7, 288, 2880, [0, 448, 449, 1, 100, 17, 1700]), (2, 4128, 96, [33, 64])])
def test_gate_up(E, F, K, counts, limit):
    import torch

    rng = np.random.default_rng(F + K)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used = int(offsets[-1])
    rows = used + 3
    wc, ws, w, xc, xs, x = product_case(rng, E, 2 * F, K, offsets, rows)
    hc, hs = mx_buffers(rows, F)
    od = dev(offsets)
    ops.mx4_gate_up_device(ops.Mx4Weights(E, 2 * F, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), hc.data_ptr(),
                           hs.data_ptr(), swiglu_limit=limit)
    ops.status()
    assert (hc[used:] == 0xEE).all() and (hs[used:] == 0xEE).all()
    assert (hs[:used, F // 32:] == 0).all()
    code, byte = R.unpack(hc[:used].cpu().numpy(), hs[:used].cpu().numpy())
    v, size = by_expert(x, w, offsets, rows)[:used], by_expert(x, w, offsets, rows, True)[:used]
    g, u = v[:, :F], v[:, F:]
    h = R.swiglu(g, u, limit)
    # What h may be off by before it is rounded: the sums' errors through a function whose slopes are at most 1.1 |u| and |silu(g)|, at most g above
    # zero and 0.28 below, both of what the limit leaves; and the exponential and division, 2^-20 of it.
    e = sum_bound(size, K)
    eg, eu, top = e[:, :F], e[:, F:], limit or np.inf
    err = 1.1 * np.minimum(np.abs(u) + eu, top) * eg + np.clip(g + eg, 0.28, max(top, 0.28)) * eu + 2.0 ** -20 * np.abs(h) + 1e-38
    # A block's scale is the largest magnitude's, or a neighbour's where that lies within its error of a power of two.
    hb, eb = np.abs(h).reshape(used, -1, 32), err.reshape(used, -1, 32)
    lo, hi = ((hb - eb).clip(0).max(2), (hb + eb).max(2))
    blo, bhi = (np.where(m > 0, np.maximum(np.frexp(np.where(m > 0, m, 1))[1] - 3, -127) + 127, 0) for m in (lo, hi))
    assert ((byte >= blo) & (byte <= bhi)).all()
    # Each code is right for some value within the error: between the codes of the error's two ends.
    s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, axis=1)
    nearest = lambda a: np.sign(a) * R.E2M1[np.searchsorted([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.abs(a))]  # noqa: E731
    down, up = (h - err) / s, (h + err) / s
    got = R.E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    tie = 1e-9
    assert ((got >= nearest(down - tie)) & (got <= nearest(up + tie))).all()
    # That bound is the worst case's. Roundings spread: a sum is off by some 2^-23 of its terms' magnitudes, h by a K-th of err then, and a code
    # differs from h's own where a border lies that near: borders are half a scale apart or more, so of all codes 4 err / (K s) at most, which
    # is under two thousandths in each of these cases; five times that is allowed.
    assert 4 * (err / s).mean() / K < 2e-3
    assert (got == nearest(h / s)).mean() > 0.99


def test_products_on_a_stream_and_in_a_graph():
    import torch

    rng = np.random.default_rng(13)
    E, N, K, rows = 6, 128, 288, 100
    offsets = np.array([0, 3, 3, 40, 41, 90, 100], np.int32)
    wc, ws, w, xc, xs, x = product_case(rng, E, N, K, offsets, rows)
    od = dev(offsets)
    y, z = (torch.zeros((rows, N), dtype=torch.float16, device="cuda") for _ in range(2))
    weights = ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr())
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    ops.mx4_product_device(weights, xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.F16, stream=st.cuda_stream)
    torch.cuda.synchronize()
    want = by_expert(x, w, offsets, rows)
    assert np.linalg.norm(y.double().cpu().numpy() - want) <= (2.0 ** -11 + 1e-5) * np.linalg.norm(want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.mx4_product_device(weights, xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), z.data_ptr(), ops.F16, stream=torch.cuda.current_stream().cuda_stream)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    # Other rows and another split through the same graph.
    (c2, s2), x2 = R.random_mx(rng, (rows, K), 125, 129)
    s2[:, K // 32:] = 255
    xc.copy_(dev(c2)), xs.copy_(dev(s2)), od.copy_(dev(np.array([0, 0, 64, 64, 65, 66, 99], np.int32)))
    z.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    want = by_expert(x2, w, [0, 0, 64, 64, 65, 66, 99], rows)
    assert (z[99] == 7).all()
    assert np.linalg.norm(z[:99].double().cpu().numpy() - want[:99]) <= (2.0 ** -11 + 1e-5) * np.linalg.norm(want)


def test_products_side_by_side():
    """Two products and a routing on three streams at once, many times over: each has its own results."""
    import torch

    rng = np.random.default_rng(14)
    jobs = []
    for E, N, K, rows in ((6, 2080, 544, 900), (40, 128, 2080, 90)):
        offsets = np.sort(rng.integers(0, rows + 1, E + 1)).astype(np.int32)
        offsets[0], offsets[-1] = 0, rows
        wc, ws, w, xc, xs, x = product_case(rng, E, N, K, None, rows)
        jobs.append((torch.cuda.Stream(), ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr()), xc, xs, rows, dev(offsets), torch.zeros((rows, N), dtype=torch.float16, device="cuda"),
                     by_expert(x, w, offsets, rows), (wc, ws)))
    logits = dev(rng.standard_normal((500, 64)).astype(np.float32))
    ids, rw, st = torch.zeros((500, 4), dtype=torch.int32, device="cuda"), torch.zeros((500, 4), device="cuda"), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, w, xc, xs, rows, od, y, _, _ in jobs:
            ops.mx4_product_device(w, xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.F16, stream=s.cuda_stream)
        ops.route_logits_device(logits.data_ptr(), ops.F32, 500, 64, 4, ids.data_ptr(), rw.data_ptr(), stream=st.cuda_stream)
    for s, *_ in jobs:
        ops.status(s.cuda_stream)
    torch.cuda.synchronize()
    for *_, y, want, _ in jobs:
        assert np.linalg.norm(y.double().cpu().numpy() - want) <= (2.0 ** -11 + 1e-5) * np.linalg.norm(want)
    assert np.array_equal(ids.cpu().numpy(), R.route(logits.double().cpu().numpy(), 4)[0])


def test_same_bits_every_time():
    import torch

    rng = np.random.default_rng(15)
    E, N, K, rows = 4, 1088, 1312, 1300
    offsets = dev(np.array([0, 300, 301, 900, 1300], np.int32))
    wc, ws, _, xc, xs, _ = product_case(rng, E, N, K, None, rows)
    weights = ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr())
    y, first = torch.empty((rows, N), dtype=torch.bfloat16, device="cuda"), None
    (hc, hs), h_first = mx_buffers(rows, N // 2), None
    for _ in range(10):
        y.fill_(9)
        ops.mx4_product_device(weights, xc.data_ptr(), xs.data_ptr(), rows, offsets.data_ptr(), y.data_ptr(), ops.BF16)
        ops.mx4_gate_up_device(weights, xc.data_ptr(), xs.data_ptr(), rows, offsets.data_ptr(), hc.data_ptr(), hs.data_ptr())
        first, h_first = first if first is not None else y.clone(), h_first if h_first is not None else (hc.clone(), hs.clone())
        assert torch.equal(y, first) and torch.equal(hc, h_first[0]) and torch.equal(hs, h_first[1])


@pytest.mark.parametrize("y_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T, n, D", [(1, 1, 8), (1, 16, 2560), (7, 3, 4104), (300, 10, 64)])
def test_combine(T, n, D, y_type):
    import torch

    rng = np.random.default_rng(T + n + D)
    rows = T * n
    y = dev(rng.standard_normal((rows + 1, D)).astype(np.float32), y_type)
    y[rows] = float("nan")
    inv = rng.permutation(rows).reshape(T, n).astype(np.int32)
    if n > 2:
        inv[0, 1], inv[-1, 2] = -1, rows  # no expert, and past the end
        inv[T // 2, :] = -1
    w, res = rng.random((T, n)).astype(np.float32), rng.standard_normal((T, D)).astype(np.float32)
    yd, there = y.double().cpu().numpy(), (inv >= 0) & (inv < rows)
    terms = np.where(there, w, 0)[..., None].astype(np.float64) * yd[np.where(there, inv, 0)]
    want, size = terms.sum(1), np.abs(terms).sum(1)
    out = torch.full((T + 1, D), 7.0, device="cuda")
    di, dw, dr = dev(inv), dev(w), dev(res)
    ops.combine_rows_device(y.data_ptr(), TYPES[y_type], rows, di.data_ptr(), dw.data_ptr(), T, n, D, out.data_ptr())
    assert (out[T] == 7.0).all()
    bound = (n + 2) * 2.0 ** -24  # a rounding a term
    assert (np.abs(out[:T].double().cpu().numpy() - want) <= bound * size).all()
    ops.combine_rows_device(y.data_ptr(), TYPES[y_type], rows, di.data_ptr(), dw.data_ptr(), T, n, D, dr.data_ptr(), residual_ptr=dr.data_ptr())
    assert (np.abs(dr.double().cpu().numpy() - want - res) <= bound * (size + np.abs(res))).all()


def test_combine_of_no_results():
    import torch

    inv, w, res, out = torch.full((3, 2), -1, dtype=torch.int32, device="cuda"), torch.ones((3, 2), device="cuda"), torch.ones((3, 64), device="cuda"), torch.zeros((3, 64), device="cuda")
    ops.combine_rows_device(None, ops.F16, 0, inv.data_ptr(), w.data_ptr(), 3, 2, 64, out.data_ptr(), residual_ptr=res.data_ptr())
    assert (out == 1).all()


def test_memory_refused():
    import torch

    d, h = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda"), torch.zeros(1 << 16, dtype=torch.uint8)
    p, q = d.data_ptr(), h.data_ptr()
    for call, word in ((lambda: ops.mx4_quantize_rows_device(q, ops.F32, 4, 64, p, p, 4), "x is not device memory"),
                       (lambda: ops.mx4_quantize_rows_device(p + 4, ops.F32, 4, 64, p, p, 4), "x must be 16-byte aligned"),
                       (lambda: ops.mx4_quantize_rows_device(p, ops.F32, 4, 64, p, p + 2, 4), "scales must be 4-byte aligned"),
                       (lambda: ops.mx4_product_device(ops.Mx4Weights(2, 64, 64, p, q), p, p, 4, p, p, ops.F16), "weight scales is not device memory"),
                       (lambda: ops.mx4_product_device(ops.Mx4Weights(2, 64, 64, p, p), p, p, 4, p, p + 8, ops.F16), "y must be 16-byte aligned"),
                       (lambda: ops.mx4_gate_up_device(ops.Mx4Weights(2, 64, 64, p, p), p, p, 4, p, p, None), "h scales is required"),
                       (lambda: ops.combine_rows_device(p, ops.F16, 4, p, p, 2, 2, 64, q), "out is not device memory"),
                       (lambda: ops.mx4_from_blocks_device(q, 4, 64, p, p), "blocks is not device memory")):
        with pytest.raises(MoEError) as e:
            call()
        assert e.value.status == _lib.MOE_BAD_ARGUMENT and word in str(e.value)


@pytest.mark.parametrize("T", [1, 50, 700])
def test_a_block_put_together(T):
    """Router logits to the block's output by all the operators in their order, on one stream, twice from one graph: against the definition in
    64 bits on the same quantised rows."""
    import torch

    rng = np.random.default_rng(T)
    E, k, D, F = 16, 3, 160, 96
    logits, bias = rng.standard_normal((T, E)).astype(np.float32), (0.1 * rng.standard_normal(E)).astype(np.float32)
    x = rng.standard_normal((T, D)).astype(np.float32)
    w1c, w1s, w1, _, _, _ = product_case(rng, E, 2 * F, D, None, 1)
    w2c, w2s, w2, _, _, _ = product_case(rng, E, D, F, None, 1)
    rows = T * k
    ids, w = torch.empty((T, k), dtype=torch.int32, device="cuda"), torch.empty((T, k), device="cuda")
    offsets, inv = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty((T, k), dtype=torch.int32, device="cuda")
    work = torch.empty(ops.route_work_bytes(T, E), dtype=torch.uint8, device="cuda")
    (xc, xs), (hc, hs) = mx_buffers(rows, D), mx_buffers(rows, F)
    y, out = torch.empty((rows, D), dtype=torch.float16, device="cuda"), torch.empty((T, D), device="cuda")
    dl, db, dx = dev(logits), dev(bias), dev(x)
    up, down = ops.Mx4Weights(E, 2 * F, D, w1c.data_ptr(), w1s.data_ptr()), ops.Mx4Weights(E, D, F, w2c.data_ptr(), w2s.data_ptr())

    def block(st):
        ops.route_logits_device(dl.data_ptr(), ops.F32, T, E, k, ids.data_ptr(), w.data_ptr(), score=ops.SIGMOID, bias_ptr=db.data_ptr(), n_groups=4,
                                n_groups_used=2, scale=1.5, offsets_ptr=offsets.data_ptr(), inv_ptr=inv.data_ptr(), work_ptr=work.data_ptr(),
                                work_bytes=work.numel(), stream=st)
        ops.mx4_quantize_rows_device(dx.data_ptr(), ops.F32, T, D, xc.data_ptr(), xs.data_ptr(), rows, inv_ptr=inv.data_ptr(), n_used=k, stream=st)
        ops.mx4_gate_up_device(up, xc.data_ptr(), xs.data_ptr(), rows, offsets.data_ptr(), hc.data_ptr(), hs.data_ptr(), swiglu_limit=7.0, stream=st)
        ops.mx4_product_device(down, hc.data_ptr(), hs.data_ptr(), rows, offsets.data_ptr(), y.data_ptr(), ops.F16, stream=st)
        ops.combine_rows_device(y.data_ptr(), ops.F16, rows, inv.data_ptr(), w.data_ptr(), T, k, D, out.data_ptr(), residual_ptr=dx.data_ptr(), stream=st)

    def want(l, x):
        i, wt, off, place = R.route(l.astype(np.float64), k, "sigmoid", bias, 4, 2, True, 1.5)
        xe = np.empty((rows, D))
        xe[place.reshape(-1)] = np.repeat(R.values(*R.quantize(x)), k, 0)
        v = by_expert(xe, w1, off, rows)
        h = R.values(*R.quantize(R.swiglu(v[:, :F], v[:, F:], 7.0)))
        ye = by_expert(h, w2, off, rows)
        return x + (wt[..., None] * ye[place]).sum(1)

    block(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    first = out.clone()
    # y's rounding to f16, and the few values of h within an f32 sum's error of a border between two codes (a code further off: some 1e-6 of them
    # by a fifth of a block's size): a part in two thousand of the block's result, which the residual is no smaller than.
    assert np.linalg.norm(first.double().cpu().numpy() - want(logits, x)) <= 2e-3 * np.linalg.norm(want(logits, x))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block(torch.cuda.current_stream().cuda_stream)
    for seed in (None, 1, 2):
        if seed is not None:
            g = np.random.default_rng(seed)
            logits, x = g.standard_normal((T, E)).astype(np.float32), g.standard_normal((T, D)).astype(np.float32)
            dl.copy_(dev(logits)), dx.copy_(dev(x))
        graph.replay()
        torch.cuda.synchronize()
        if seed is None:
            assert torch.equal(out, first)  # the same bits, captured or not
        assert np.linalg.norm(out.double().cpu().numpy() - want(logits, x)) <= 2e-3 * np.linalg.norm(want(logits, x))


def check_h(hc, hs, h, err):
    """Each code of h's MX rows is right for some value within err of h's, each scale for some largest one."""
    rows, F = h.shape
    code, byte = R.unpack(hc.cpu().numpy(), hs.cpu().numpy())
    hb, eb = np.abs(h).reshape(rows, -1, 32), err.reshape(rows, -1, 32)
    lo, hi = ((hb - eb).clip(0).max(2), (hb + eb).max(2))
    blo, bhi = (np.where(m > 0, np.maximum(np.frexp(np.where(m > 0, m, 1))[1] - 3, -127) + 127, 0) for m in (lo, hi))
    assert ((byte >= blo) & (byte <= bhi)).all()
    s = np.repeat(np.exp2(byte.astype(np.float64) - 127), 32, axis=1)
    nearest = lambda a: np.sign(a) * R.E2M1[np.searchsorted([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.abs(a))]  # noqa: E731
    got = R.E2M1[code & 7] * np.where(code & 8, -1.0, 1.0)
    assert ((got >= nearest((h - err) / s - 1e-9)) & (got <= nearest((h + err) / s + 1e-9))).all()


def mx_of(v):
    """MX rows of values that the form holds exactly: (codes, scales) on the device."""
    code, byte = R.quantize(v)
    assert np.array_equal(R.values(code, byte), v)
    c, s = R.pack(code, byte)
    return dev(c), dev(s)


@pytest.mark.parametrize("copies", [1, 20])
def test_gates_far_below_zero(copies):
    """Where e^g is below f32's normal values and u so large that h is not: an MX scale can hold it. By single CTAs and, with many copies, by pairs."""
    import torch

    gates = -np.array([1, 48, 64, 96, 128, 192, 256, 384], np.float64)
    ups = np.array([0.5, 2.0 ** 40, 2.0 ** 101, 2.0 ** 124])
    g1, u1 = (a.reshape(-1).repeat(32) for a in np.meshgrid(gates, ups))
    u1 = u1 * np.tile(np.array([1, -1.5, 2, 0.5]), u1.size // 4)                     # a block's gates alike, its other factors not
    F, K, rows = g1.size * copies, 32, 40
    w = np.zeros((1, 2 * F, K))
    w[0, :F, 0], w[0, F:, 0] = np.tile(g1, copies), np.tile(u1, copies)              # a row's first value alone meets the matrix
    x = np.zeros((rows, K))
    x[:, 0] = np.tile([1, 0.5, 2, 1.5], rows // 4)
    (wc, ws), (xc, xs) = mx_of(w.reshape(-1, K)), mx_of(x)
    hc, hs = mx_buffers(rows, F)
    ops.mx4_gate_up_device(ops.Mx4Weights(1, 2 * F, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), rows, None, hc.data_ptr(), hs.data_ptr())
    ops.status()
    v = x @ w[0].T
    h = R.swiglu(v[:, :F], v[:, F:], 0.0)
    # g and u are exact. To g = -80 the exponential's argument is below 116 and rounds by 2^-18 of one, log2(e) is within 2^-25 of itself, and the four other
    # roundings are 2^-22 at most: 2^-17 covers it, and with it four exponentials of 2 ulp each. Below f32's normal values a step is 2^-149.
    check_h(hc, hs, h, 2.0 ** -17 * np.abs(h) + 2.0 ** -148)


def test_h_of_infinities_and_nans():
    """NaN scales, sums past f32 and NaN under a limit: a block of h with an infinity or NaN is NaN, the others are as ever."""
    import torch

    rng = np.random.default_rng(16)
    for E, F, rows, first in ((2, 64, 50, 20), (1, 4128, 208, 0)):                   # single CTAs; pairs
        K = 320
        wc, ws, w, xc, xs, x = product_case(rng, E, 2 * F, K, None, rows)
        xs[17, 3] = 255                                                              # a row
        ws[-1, 40, 9] = 255                                                          # a gate of the last expert
        ws[-1, F + 3, 0] = 255                                                       # an up row of it
        offsets = dev(np.array([0, first, rows][-E - 1:], np.int32))
        bad = np.zeros((rows, F), bool)
        bad[17] = True
        bad[first:, [3, 40]] = True
        w[-1, [40, F + 3]] = 0
        x[17] = 0
        off = [0, first, rows][-E - 1:]
        v, size = by_expert(x, w, off, rows), by_expert(x, w, off, rows, True)
        for limit in (0.0, 2.0):
            hc, hs = mx_buffers(rows, F)
            ops.mx4_gate_up_device(ops.Mx4Weights(E, 2 * F, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), rows, offsets.data_ptr(),
                                   hc.data_ptr(), hs.data_ptr(), swiglu_limit=limit)
            ops.status()
            code, byte = R.unpack(hc.cpu().numpy(), hs.cpu().numpy())
            block = bad.reshape(rows, -1, 32).any(2)
            assert np.array_equal(byte == 255, block) and (code[np.repeat(block, 32, axis=1)] == 0).all()
            h = R.swiglu(v[:, :F], v[:, F:], limit)
            got = R.values(code, byte)
            keep = ~np.repeat(block, 32, axis=1)
            # A value that is no border's differs by a step of its code at most: 2 of the scale, an eighth to a quarter of the largest.
            top = np.repeat(np.abs(h).reshape(rows, -1, 32).max(2), 32, axis=1)
            assert (np.abs(got - h)[keep] <= 0.26 * top[keep] + 1e-30).all()
    # Sums past f32, one value of the contraction alone: (g, u) of infinities, with and without a limit.
    inf = np.inf
    pairs = [(2.0, inf), (inf, 2.0), (-2.0, inf), (inf, -inf), (-192.0, -inf), (-inf, 2.0), (inf, 0.0), (2.0, 3.0)]
    F, K = 32 * len(pairs), 32
    big = 1.5 * 2.0 ** 100
    w, x = np.zeros((2 * F, K)), np.zeros((4, K))
    fill = lambda a: np.array([np.sign(p) * big if np.isinf(p) else p / 2.0 ** 60 for p in a]).repeat(32)  # noqa: E731
    w[:F, 0], w[F:, 0] = fill([p[0] for p in pairs]), fill([p[1] for p in pairs])
    x[:, 0] = 2.0 ** 60
    (wc, ws), (xc, xs) = mx_of(w), mx_of(x)
    for limit in (0.0, 7.0):
        hc, hs = mx_buffers(4, F)
        ops.mx4_gate_up_device(ops.Mx4Weights(1, 2 * F, K, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), 4, None, hc.data_ptr(), hs.data_ptr(), swiglu_limit=limit)
        ops.status()
        _, byte = R.unpack(hc.cpu().numpy(), hs.cpu().numpy())
        with np.errstate(invalid="ignore"):
            g, u = (np.array(a) for a in zip(*pairs))
            want = ~np.isfinite(R.swiglu(g, u, limit))
        assert want.sum() == (7 if limit == 0 else 1) and np.array_equal(byte == 255, np.tile(want, (4, 1)))


def run_both(E, N, K, offsets, rows, rng):
    """Product and gate_up of the same rows and matrices (2 F = N): y, h's codes and scales, filled with 7 and 0xEE before."""
    import torch

    wc, ws, w, xc, xs, x = product_case(rng, E, N, K, None, rows)
    y = torch.full((rows, N), 7.0, dtype=torch.float16, device="cuda")
    hc, hs = mx_buffers(rows, N // 2)
    od, weights = dev(np.asarray(offsets, np.int32)), ops.Mx4Weights(E, N, K, wc.data_ptr(), ws.data_ptr())
    ops.mx4_product_device(weights, xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.F16)
    ops.mx4_gate_up_device(weights, xc.data_ptr(), xs.data_ptr(), rows, od.data_ptr(), hc.data_ptr(), hs.data_ptr())
    ops.status()
    return y, hc, hs, w, x


def check_both(y, hc, hs, w, x, sound):
    """Every row with the expert that the sound offsets give it; rows of none as they were."""
    rows, N, K = y.shape[0], w.shape[1], w.shape[2]
    F, mine = N // 2, np.zeros(rows, bool)
    for e in range(w.shape[0]):
        mine[sound[e]:sound[e + 1]] = True
    v, size = by_expert(x, w, sound, rows), by_expert(x, w, sound, rows, True)
    got = y.double().cpu().numpy()
    off = 2.0 ** -11 * np.abs(v) + sum_bound(size, K) * (1 + 2.0 ** -11) + 2.0 ** -25
    assert (np.abs(got - v)[mine] <= off[mine]).all() and (got[~mine] == 7.0).all()
    g, u, e = v[:, :F], v[:, F:], sum_bound(size, K)
    h = R.swiglu(g, u, 0.0)
    err = 1.1 * (np.abs(u) + e[:, F:]) * e[:, :F] + np.maximum(g + e[:, :F], 0.28) * e[:, F:] + 2.0 ** -20 * np.abs(h) + 1e-38  # as in test_gate_up
    at = np.flatnonzero(mine)
    hc, hs = hc.cpu(), hs.cpu()
    check_h(hc[at], hs[at], h[at], err[at])
    assert (hc.numpy()[~mine] == 0xEE).all() and (hs.numpy()[~mine] == 0xEE).all()


@pytest.mark.parametrize("N, K, rows, offsets, sound", [
    (64, 64, 40, [30, 20, 35, 10, 5], [30, 30, 35, 35, 35]),
    (64, 64, 40, [-5, 12, 11, 10, 39], [0, 12, 12, 12, 39]),
    (2112, 64, 900, [700, 500, 820, 400, 3000], [700, 700, 820, 820, 900]),          # by pairs of CTAs
    (2112, 64, 900, [250, 900, 100, 2 ** 31 - 1, -2 ** 31], [250, 900, 900, 900, 900])])
def test_falling_offsets_count_as_the_one_before(N, K, rows, offsets, sound):
    check_both(*run_both(4, N, K, offsets, rows, np.random.default_rng(17)), sound)


def test_more_tiles_than_the_table_holds():
    """Tiles of many experts past the first 1,024, whose expert is searched for: some experts without rows on both sides, some of one row."""
    rng = np.random.default_rng(18)
    E = 512
    counts = rng.integers(0, 1400, E)
    counts[rng.random(E) < 0.3] = 0
    counts[rng.random(E) < 0.1] = 1
    counts[-1] = 0
    offsets = np.concatenate([[0], np.cumsum(counts)])
    tiles = np.cumsum(-(-counts // 208))
    at = int(np.searchsorted(tiles, 1024, side="right"))
    counts[at + 1:at + 3] = 0                                                         # behind the expert whose tile is number 1,024 too
    offsets = np.concatenate([[0], np.cumsum(counts)])
    tiles = np.cumsum(-(-counts // 208))
    assert tiles[-1] > 1100 and (counts[:at] == 0).sum() > 50 and (counts[at:] == 0).sum() > 20
    check_both(*run_both(E, 64, 32, offsets, int(offsets[-1]), rng), offsets)


def test_many_rows_of_a_files_blocks():
    import torch

    rng = np.random.default_rng(19)
    for rows, K in ((70001, 64), (300, 8224)):
        code, byte = rng.integers(0, 16, (rows, K), dtype=np.uint8), rng.integers(0, 256, (rows, K // 32), dtype=np.uint8)
        b = code.reshape(rows, -1, 2, 16)
        bd = dev(np.concatenate([byte[..., None], b[:, :, 0] | b[:, :, 1] << 4], -1))
        codes, scales = mx_buffers(rows, K)
        ops.mx4_from_blocks_device(bd.data_ptr(), rows, K, codes.data_ptr(), scales.data_ptr())
        torch.cuda.synchronize()
        want = R.pack(code, byte)
        assert np.array_equal(codes.cpu().numpy(), want[0]) and np.array_equal(scales.cpu().numpy(), want[1])


def test_a_give_up_is_told_to_everyone():
    """A product that gave up is told to every thread for every stream that it asks about, once each, whoever asks first; the count is raised by hand,
    since no sound product gives up."""
    import threading

    import torch

    def asked(stream):
        try:
            ops.status(stream)
        except MoEError as e:
            assert e.status == _lib.MOE_TIMEOUT and "gave up" in str(e)
            return True
        return False

    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    streams = (a.cuda_stream, b.cuda_stream, None)
    [asked(s) for s in streams]                               # what earlier ones left
    assert not any(asked(s) for s in streams)
    for _ in range(2):
        assert _lib.lib().moe_ops_note_give_up(b.cuda_stream) == _lib.MOE_OK
        b.synchronize()
        assert [asked(s) for s in streams] == [True] * 3      # a, whose work was sound, asks first: b is told all the same
        assert not any(asked(s) for s in streams)
        seen = []
        t = threading.Thread(target=lambda: seen.extend(asked(b.cuda_stream) for _ in range(2)))
        t.start()
        t.join()
        assert seen == [True, False]                          # a thread that has not asked before is told too
    # Two at once are one answer; a product after them is sound.
    for s in (a, b):
        assert _lib.lib().moe_ops_note_give_up(s.cuda_stream) == _lib.MOE_OK
    torch.cuda.synchronize()
    rng = np.random.default_rng(20)
    wc, ws, w, xc, xs, x = product_case(rng, 1, 64, 64, None, 5)
    y = torch.empty((5, 64), dtype=torch.float16, device="cuda")
    assert asked(a.cuda_stream)
    ops.mx4_product_device(ops.Mx4Weights(1, 64, 64, wc.data_ptr(), ws.data_ptr()), xc.data_ptr(), xs.data_ptr(), 5, None, y.data_ptr(), ops.F16, stream=a.cuda_stream)
    assert [asked(s) for s in streams] == [False, True, True]
    assert np.linalg.norm(y.double().cpu().numpy() - x @ w[0].T) <= (2.0 ** -11 + 1e-5) * np.linalg.norm(x @ w[0].T)


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("T, K", [(38001, 32), (38003, 96), (37999, 128), (38005, 160)])
def test_quantize_many_narrow_rows(type, T, K):
    """Rows of fewer threads than a warp, several a thread: some of a warp's rows are past the last."""
    import torch

    rng = np.random.default_rng(T)
    x = dev(rows_of(rng, T, K).astype(np.float32), type)
    want = R.pack(*R.quantize(x.double().cpu().numpy()))
    codes, scales = mx_buffers(T + 1, K)
    ops.mx4_quantize_rows_device(x.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), T)
    torch.cuda.synchronize()
    assert np.array_equal(codes[:T].cpu().numpy(), want[0]) and np.array_equal(scales[:T].cpu().numpy(), want[1])
    assert (codes[T] == 0xEE).all() and (scales[T] == 0xEE).all()
    out = torch.empty((T, K), device="cuda")
    ops.mx4_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), T, K, out.data_ptr(), ops.F32)
    assert np.array_equal(out.double().cpu().numpy(), R.values(*R.unpack(*want)))

"""On a B200: rows to and from 8-bit integers and the experts' products over them, against the definitions in 64 bits."""
import numpy as np
import pytest

import more_ops_common as M
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


def host(t):
    return t.double().cpu().numpy()


def buffers(rows, K):
    import torch

    return torch.full((rows, K), 0x6E, dtype=torch.int8, device="cuda"), torch.full((rows,), 7.0, device="cuda")


def rows_of(rng, T, K):
    """Rows of all sizes, of zeros, and with quotients on and beside the borders between codes."""
    x = rng.standard_normal((T, K)) * np.exp2(rng.integers(-30, 31, (T, 1)).astype(np.float64))
    if T > 1:
        x[1] = 0
        x[1, ::3] = -0.0
    b = (np.arange(K) % 127 + 0.5) * np.where(np.arange(K) % 2, 1, -1)  # of a largest of 127: exact borders
    x[0] = b
    x[0, 0] = 127.0
    if T > 2:
        x[2] = np.float32(b) * (1 + np.float32(2.0 ** -20) * rng.integers(-1, 2, K))
        x[2, K - 1] = -127.0
    if T > 3:
        x[3] = rng.integers(-254, 255, K) / 256 * 1.75  # many share a quotient with few bits
        x[3, K // 2] = 1.75
    return x


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T, K", [(1, 32), (3, 96), (5, 2048), (2, 2080), (33, 2880), (4, 4128), (3, 16384), (3, 16416), (1, 65536), (700, 160), (2501, 2080), (19001, 288), (6000, 64)])
def test_quantize_rows_bit_for_bit(type, T, K):
    import torch

    rng = np.random.default_rng(T + K)
    x = dev(np.clip(rows_of(rng, T, K), -6e4, 6e4).astype(np.float32), type)
    code, scale = M.quantize(host(x))
    codes, scales = buffers(T + 1, K)
    ops.i8_quantize_rows_device(x.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), T)
    torch.cuda.synchronize()
    assert np.array_equal(codes[:T].cpu().numpy(), code) and np.array_equal(scales[:T].cpu().numpy(), scale)
    assert (codes[T] == 0x6E).all() and scales[T] == 7.0
    for out_type in ("f32", "bf16", "f16"):
        out = torch.full((T + 1, K), 7.0, dtype=dtype(out_type), device="cuda")
        ops.i8_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), T, K, out.data_ptr(), TYPES[out_type])
        v = torch.from_numpy(code.astype(np.float32) * scale[:, None]).to(dtype(out_type))
        assert torch.equal(out[:T].cpu(), v) and (out[T] == 7.0).all()


def test_quantize_extremes():
    """The largest and smallest rows of f32, infinities and NaN at every place of a row, denormals."""
    import torch

    rng = np.random.default_rng(1)
    x = rng.uniform(-1, 1, (10 + 96, 96)).astype(np.float32)
    tiny = np.float32(2.0 ** -149)
    x[0] *= np.finfo(np.float32).max
    x[0, 5] = np.finfo(np.float32).max
    x[1] *= np.float32(2.0 ** -126)
    x[2] = tiny * rng.integers(-200, 201, 96)
    x[3] = tiny * rng.integers(-1, 2, 96)
    x[4] = tiny
    x[5] *= np.float32(1e-36)
    x[6] *= np.float32(1e-35)
    x[7] *= np.float32(2e-35)
    x[8] = 0
    x[8, 95] = tiny
    x[9, 1:] *= np.float32(1e-30)
    for i in range(96):
        x[10 + i, i] = (np.inf, -np.inf, np.nan)[i % 3]
    code, scale = M.quantize(x)
    codes, scales = buffers(106, 96)
    dx = dev(x)
    ops.i8_quantize_rows_device(dx.data_ptr(), ops.F32, 106, 96, codes.data_ptr(), scales.data_ptr(), 106)
    assert np.array_equal(codes.cpu().numpy(), code) and np.array_equal(scales.cpu().numpy(), scale, equal_nan=True)
    assert np.isnan(scale[10:]).all() and (code[10:] == 0).all() and scale[3] == 0 and abs(code[3]).max() == 127
    out = torch.empty((106, 96), device="cuda")
    ops.i8_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), 106, 96, out.data_ptr(), ops.F32)
    assert np.array_equal(out.cpu().numpy(), code.astype(np.float32) * scale[:, None], equal_nan=True)


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_quantize_every_pair_of_16_bit_numbers_near_a_border(type):
    """Rows whose largest has every significand, with every significand beside it: all quotients there can be, ties among them."""
    import torch

    bits = 7 if type == "bf16" else 10
    n = 1 << bits
    sig = 1 + np.arange(n) / n
    tops = 2 * sig[:: max(1, n // 256)]
    x = np.concatenate([np.repeat(tops[:, None], 32, 1), np.tile(sig * 0.5, (len(tops), 1)), np.tile(sig, (len(tops), 1))], 1).astype(np.float32)
    t = dev(x, type)
    T, K = x.shape
    code, scale = M.quantize(host(t))
    codes, scales = buffers(T, K)
    ops.i8_quantize_rows_device(t.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), T)
    assert np.array_equal(codes.cpu().numpy(), code) and np.array_equal(scales.cpu().numpy(), scale)
    q = 127 * host(t) / host(t).max(1, keepdims=True)
    assert (q - np.floor(q) == 0.5).sum() > 100


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("T, K, n", [(21, 224, 5), (5003, 1056, 3), (3, 20480, 16), (13, 2560, 8)])
def test_quantize_scatters_strided_rows(type, T, K, n):
    """Every row to the places its assignments have; places of none and rows past R are left as they were."""
    import torch

    rng = np.random.default_rng(2)
    rows = T * n * 3 // 4
    full = dev(rng.standard_normal((T, K + 32)).astype(np.float32), type)
    inv = rng.permutation(T * n)[:T * n].reshape(T, n).astype(np.int32)
    inv[1, n - 1], inv[2, :] = -1, -2 ** 31
    codes, scales = buffers(rows + 2, K)
    di = dev(inv)
    ops.i8_quantize_rows_device(full.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), rows, stride=K + 32, inv_ptr=di.data_ptr(), n_used=n)
    c, s = M.quantize(host(full)[:, :K])
    want_c, want_s = np.full((rows + 2, K), 0x6E, np.int8), np.full(rows + 2, 7.0, np.float32)
    for k in range(n):
        ok = (inv[:, k] >= 0) & (inv[:, k] < rows)
        want_c[inv[ok, k]], want_s[inv[ok, k]] = c[ok], s[ok]
    assert np.array_equal(codes.cpu().numpy(), want_c) and np.array_equal(scales.cpu().numpy(), want_s)


def product_case(rng, E, N, K, rows, largest=127):
    """Matrices and rows of codes over the whole range, -128 among them, and scales over some powers of two: host and device."""
    wc, c = rng.integers(-largest - (largest == 127), largest + 1, (E, N, K), dtype=np.int8), rng.integers(-largest - (largest == 127), largest + 1, (rows, K), dtype=np.int8)
    ws, s = ((rng.uniform(0.5, 2, n) * 2.0 ** -7 / np.sqrt(np.sqrt(K))).astype(np.float32) for n in ((E, N), (rows,)))
    return wc, ws, c, s


def weights_of(wc, ws):
    d = dev(wc), dev(ws)
    return ops.I8Weights(*wc.shape, d[0].data_ptr(), d[1].data_ptr()), d


SHAPES = [(1, 32, 32, [5]), (1, 64, 96, [1]), (1, 160, 256, [300]), (3, 128, 64, [0, 7, 130]), (8, 96, 544, [1, 0, 2, 64, 65, 0, 17, 1]),
          (5, 288, 2880, [16, 15, 0, 33, 1]), (2, 2080, 160, [129, 257]), (70, 64, 128, [1] * 70), (4, 32, 4096, [0, 0, 0, 3]), (512, 32, 32, [0, 1] * 256),
          (2, 256, 2880, [225, 33]), (1, 288, 1312, [1793]), (7, 544, 4128, [0, 448, 449, 1, 100, 17, 224]), (1, 32, 65536, [3]), (1, 65536, 32, [2]),
          # Enough rows an expert and items for pairs of CTAs; halves of 16, 48, 80, 96, 112 and 128 rows.
          (1, 2080, 160, [900]), (3, 1056, 1312, [209, 0, 1100]), (7, 544, 2880, [0, 448, 449, 1, 100, 17, 1700]), (2, 8224, 96, [33, 64]), (2, 4128, 4064, [417, 16]),
          (1, 65536, 64, [40]), (8, 1056, 544, [32, 96, 160, 192, 224, 256, 257, 511])]


@pytest.mark.parametrize("y_type", ["f16", "bf16"])
@pytest.mark.parametrize("E, N, K, counts", SHAPES)
def test_products_bit_for_bit(E, N, K, counts, y_type):
    """Sums are exact; a sum in f32 times two scales, each rounded, then the type: one right answer."""
    import torch

    rng = np.random.default_rng(N + K)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used = int(offsets[-1])
    rows = used + 3  # rows of no expert behind the last
    wc, ws, c, s = product_case(rng, E, N, K, rows)
    w, keep = weights_of(wc, ws)
    dc, ds, od = dev(c), dev(s), dev(offsets)
    want, named = M.product(c, s, wc, ws, offsets, rows)
    assert named[:used].all() and not named[used:].any()
    want = torch.from_numpy(want[:used]).to(dtype(y_type))
    for at in (od.data_ptr(),) + ((None,) if E == 1 else ()):
        y = torch.full((rows + 1, N), 7.0, dtype=dtype(y_type), device="cuda")
        ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), rows if at else used, at, y.data_ptr(), TYPES[y_type])
        ops.status()
        assert torch.equal(y[:used].cpu(), want) and (y[used:] == 7.0).all()


def test_sums_at_their_largest():
    """65,536 products of -128 by -128 are 2^30, and of 127 by -128 nearly as far below: 32 bits hold both."""
    import torch

    K = 65536
    wc, c = np.full((1, 64, K), -128, np.int8), np.full((40, K), -128, np.int8)
    c[1] = 127
    wc[0, 3] = 127
    one = lambda *n: np.ones(n, np.float32)  # noqa: E731
    w, keep = weights_of(wc, one(1, 64))
    dc, ds = dev(c), dev(one(40) * np.float32(2.0 ** -20))
    y = torch.empty((40, 64), dtype=torch.bfloat16, device="cuda")
    ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), 40, None, y.data_ptr(), ops.BF16)
    ops.status()
    want, _ = M.product(c, one(40) * np.float32(2.0 ** -20), wc, one(1, 64), [0, 40], 40)
    assert torch.equal(y.cpu(), torch.from_numpy(want).bfloat16()) and y[0, 0] == 1024


def swiglu_near(h, g, u, limit, type):
    """h within 2^-17 of its exact value (g, u are to the bit), then half a step of the type. To g = -80 the exponential's argument is below 116 and rounds by
    2^-18 of one, its factor is within 2^-26 of itself, and the other roundings, the approximate forms' among them, are 2^-21 at most; below, four exponentials of 2 ulp
    and six products."""
    want = R.swiglu(g, u, limit)
    least = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}[type] + 2.0 ** -148
    top = {"f16": 65504.0, "bf16": 3.3895313892515355e38}[type]
    over = np.abs(want) > top
    got = host(h)
    off = np.abs(np.where(over, 0.0, got) - np.where(over, 0.0, want))
    assert (off <= (2.0 ** -17 + R.HALF_STEP[type] * (1 + 2.0 ** -17)) * np.abs(want) + least).all(), off.max()
    assert (np.abs(got[over]) >= top).all() and (np.sign(got[over]) == np.sign(want[over])).all()


@pytest.mark.parametrize("h_type", ["f16", "bf16"])
@pytest.mark.parametrize("limited", [False, True])
@pytest.mark.parametrize("E, F, K, counts", [(1, 32, 32, [5]), (1, 64, 96, [1]), (3, 96, 544, [0, 7, 130]), (5, 288, 2880, [16, 15, 0, 33, 1]), (70, 32, 128, [1] * 70),
                                             (1, 544, 160, [1793]), (512, 32, 32, [0, 1] * 256), (1, 32768, 32, [40]), (3, 1056, 1312, [209, 0, 1100]),
                                             (8, 544, 544, [32, 96, 160, 192, 224, 256, 257, 511]), (2, 4128, 416, [417, 16]), (1, 32, 65536, [2]),
                                             # By pairs with a contraction long enough for two groups of epilogue warps.
                                             (2, 1056, 1696, [600, 217])])
def test_gate_up(E, F, K, counts, limited, h_type):
    import torch

    rng = np.random.default_rng(F + K)
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    used = int(offsets[-1])
    rows = used + 3
    wc, ws, c, s = product_case(rng, E, 2 * F, K, rows, 40)
    w, keep = weights_of(wc, ws)
    dc, ds, od = dev(c), dev(s), dev(offsets)
    v = M.product(c, s, wc, ws, offsets, rows)[0][:used].astype(np.float64)
    limit = float(np.float32(np.median(np.abs(v)))) if limited else 0.0
    h = torch.full((rows + 1, F), 7.0, dtype=dtype(h_type), device="cuda")
    ops.i8_gate_up_device(w, dc.data_ptr(), ds.data_ptr(), rows, od.data_ptr(), h.data_ptr(), TYPES[h_type], swiglu_limit=limit)
    ops.status()
    assert (h[used:] == 7.0).all()
    swiglu_near(h[:used], v[:, :F], v[:, F:], limit, h_type)


@pytest.mark.parametrize("h_type", ["f16", "bf16"])
@pytest.mark.parametrize("copies", [1, 20])
def test_gates_far_from_zero(copies, h_type):
    """Where e^g is below f32's normal values and u so large that h is not, and gates far above. By single CTAs and, with many copies, by pairs."""
    import torch

    gates = np.array([-1, -48, -64, -79.5, -80, -81, -96, -128, -192, -256, -384, 60, 100, 1e30, -1e30, 0])
    ups = np.array([0.5, 2.0 ** 40, -2.0 ** 101, 2.0 ** 124])
    g1, u1 = (np.tile(a.reshape(-1), 1) for a in np.meshgrid(gates, ups))  # 64 features
    g1, u1 = np.tile(g1, copies), np.tile(u1, copies)
    F, K, rows = g1.size, 32, 40
    wc, c = np.zeros((1, 2 * F, K), np.int8), np.zeros((rows, K), np.int8)
    wc[:, :, 3], c[:, 3] = 1, 1
    ws, s = np.concatenate([g1, u1])[None].astype(np.float32), np.tile(np.array([1, 0.5, 2, 1.5], np.float32), rows // 4)
    w, keep = weights_of(wc, ws)
    dc, ds = dev(c), dev(s)
    h = torch.empty((rows, F), dtype=dtype(h_type), device="cuda")
    ops.i8_gate_up_device(w, dc.data_ptr(), ds.data_ptr(), rows, None, h.data_ptr(), TYPES[h_type])
    ops.status()
    v = M.product(c, s, wc, ws, [0, rows], rows)[0].astype(np.float64)
    swiglu_near(h, v[:, :F], v[:, F:], 0.0, h_type)


def test_scales_of_nan_and_zero():
    """A row whose scale is NaN (a row that held an infinity) gives NaN in its own results alone, under a limit too; scale 0 gives zeros."""
    import torch

    rng = np.random.default_rng(16)
    for rows, N in ((40, 64), (40, 8256)):
        wc, ws, c, s = product_case(rng, 1, N, 160, rows)
        s[3], s[17], s[5] = np.nan, np.nan, 0.0
        w, keep = weights_of(wc, ws)
        dc, ds = dev(c), dev(s)
        y, h = torch.empty((rows, N), dtype=torch.float16, device="cuda"), torch.empty((rows, N // 2), dtype=torch.float16, device="cuda")
        ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), rows, None, y.data_ptr(), ops.F16)
        for limit in (0.0, 2.0):
            ops.i8_gate_up_device(w, dc.data_ptr(), ds.data_ptr(), rows, None, h.data_ptr(), ops.F16, swiglu_limit=limit)
            ops.status()
            for t in (y, h):
                bad = torch.isnan(t)
                assert bad[[3, 17]].all() and bad.sum() == 2 * t.shape[1] and (t[5] == 0).all()


@pytest.mark.parametrize("E, N, K, rows, offsets, sound", [
    (4, 64, 64, 40, [0, 10, 20, 30, 1000], [0, 10, 20, 30, 40]), (4, 64, 64, 40, [-5, 10, 20, 20, 2 ** 31 - 1], [0, 10, 20, 20, 40]),
    (4, 64, 64, 40, [0, 20, 5, 30, 25], [0, 20, 20, 30, 30]), (3, 4128, 64, 300, [0, 200, 100, 300], [0, 200, 200, 300]),
    (3, 64, 64, 40, [7, 9, 9, 30], [7, 9, 9, 30]), (2, 64, 64, 40, [0, 0, 0], [0, 0, 0])])
def test_offsets_that_say_too_much_are_cut_off(E, N, K, rows, offsets, sound):
    """Offsets past R, below 0 or falling: no row outside 0 .. R - 1 is read or written, rows before the first expert's are left."""
    import torch

    rng = np.random.default_rng(11)
    wc, ws, c, s = product_case(rng, E, N, K, rows)
    w, keep = weights_of(wc, ws)
    dc, ds, od = dev(c), dev(s), dev(np.array(offsets, np.int32))
    y = torch.full((rows + 8, N), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.BF16)
    ops.status()
    want, named = M.product(c, s, wc, ws, sound, rows)
    full = torch.where(torch.from_numpy(named)[:, None], torch.from_numpy(want), torch.tensor(7.0)).bfloat16()
    assert torch.equal(y[:rows].cpu(), full) and (y[rows:] == 7.0).all()


def test_more_tiles_than_the_table_holds():
    """Tiles past the 1,024 whose expert is looked up, of three experts, one of them without rows."""
    import torch

    rng = np.random.default_rng(12)
    offsets = np.array([0, 700, 700, 270001], np.int32)
    rows = int(offsets[-1])
    wc, ws, c, s = product_case(rng, 3, 32, 32, rows)
    w, keep = weights_of(wc, ws)
    dc, ds, od = dev(c), dev(s), dev(offsets)
    y = torch.empty((rows, 32), dtype=torch.float16, device="cuda")
    ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.F16)
    ops.status()
    assert torch.equal(y.cpu(), torch.from_numpy(M.product(c, s, wc, ws, offsets, rows)[0]).half())


def test_offsets_past_32_bits():
    """Rows, matrices and results whose places do not fit 32 bits: the last ones are right."""
    import torch

    rng = np.random.default_rng(5)
    T, K = 66000, 65536
    x = torch.zeros((T, K), dtype=torch.bfloat16, device="cuda")  # 8.6 GB, and 4.3 of codes
    x[-3:] = dev(rng.standard_normal((3, K)).astype(np.float32), "bf16")
    c, s = M.quantize(host(x[-3:]))
    codes, scales = buffers(T, K)
    ops.i8_quantize_rows_device(x.data_ptr(), ops.BF16, T, K, codes.data_ptr(), scales.data_ptr(), T)
    assert np.array_equal(codes[-3:].cpu().numpy(), c) and np.array_equal(scales[-3:].cpu().numpy(), s) and (codes[:-3] == 0).all() and (scales[:-3] == 0).all()
    # A product of the last rows alone, which begin past 2^32 bytes.
    wc, ws = rng.integers(-128, 128, (1, 64, K), dtype=np.int8), rng.uniform(1e-3, 1e-2, (1, 64)).astype(np.float32)
    w, keep = weights_of(wc, ws)
    od, y = dev(np.array([T - 3, T], np.int32)), torch.full((T, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.i8_product_device(w, codes.data_ptr(), scales.data_ptr(), T, od.data_ptr(), y.data_ptr(), ops.BF16)
    ops.status()
    assert torch.equal(y[-3:].cpu(), torch.from_numpy(M.product(c, s, wc, ws, [0, 3], 3)[0]).bfloat16()) and (y[:-3] == 7.0).all()
    x.fill_(7)
    ops.i8_dequantize_rows_device(codes.data_ptr(), scales.data_ptr(), T, K, x.data_ptr(), ops.BF16)
    assert torch.equal(x[-3:].cpu(), torch.from_numpy(c.astype(np.float32) * s[:, None]).bfloat16()) and (x[:-3] == 0).all()
    del x, codes, scales, y
    # Matrices of more than 2^32 bytes, rows for the last alone; results of more than 2^32 values.
    E, N, K = 512, 4128, 4128
    big, bs = torch.zeros((E, N, K), dtype=torch.int8, device="cuda"), torch.zeros((E, N), device="cuda")
    wc, ws, c, s = product_case(rng, 1, N, K, 40)
    big[-1], bs[-1] = dev(wc[0]), dev(ws[0])
    dc, ds, od = dev(c), dev(s), dev(np.array([0] * E + [40], np.int32))
    y, h = torch.empty((40, N), dtype=torch.bfloat16, device="cuda"), torch.empty((40, N // 2), dtype=torch.bfloat16, device="cuda")
    w = ops.I8Weights(E, N, K, big.data_ptr(), bs.data_ptr())
    ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), 40, od.data_ptr(), y.data_ptr(), ops.BF16)
    v = M.product(c, s, wc, ws, [0, 40], 40)[0]
    ops.status()
    assert torch.equal(y.cpu(), torch.from_numpy(v).bfloat16())
    del big
    N, rows = 65536, 70000
    wc, ws, c, s = product_case(rng, 1, N, 32, 5)
    w, keep = weights_of(wc, ws)
    dc, ds = torch.zeros((rows, 32), dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    dc[-5:], ds[-5:] = dev(c), dev(s)
    y = torch.empty((rows, N), dtype=torch.bfloat16, device="cuda")
    ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), rows, None, y.data_ptr(), ops.BF16)
    ops.status()
    assert torch.equal(y[-5:].cpu(), torch.from_numpy(M.product(c, s, wc, ws, [0, 5], 5)[0]).bfloat16()) and (y[:-5] == 0).all()


def test_products_side_by_side_and_the_same_bits():
    """Two streams at once, by pairs and by single CTAs; again and again to the same bits."""
    import torch

    rng = np.random.default_rng(13)
    jobs = []
    for E, N, K, rows in ((4, 1056, 544, 700), (64, 256, 288, 90)):
        wc, ws, c, s = product_case(rng, E, N, K, rows)
        offsets = np.sort(np.concatenate([[0, rows], rng.integers(0, rows, E - 1)])).astype(np.int32)
        w, keep = weights_of(wc, ws)
        jobs.append((w, keep, dev(c), dev(s), rows, dev(offsets), torch.from_numpy(M.product(c, s, wc, ws, offsets, rows)[0]).half().cuda(), torch.cuda.Stream()))
    torch.cuda.synchronize()
    ys = []
    for i in range(20):
        for w, _, dc, ds, rows, od, want, st in jobs:
            y = torch.empty_like(want)
            ops.i8_product_device(w, dc.data_ptr(), ds.data_ptr(), rows, od.data_ptr(), y.data_ptr(), ops.F16, stream=st.cuda_stream)
            ys.append((y, want))
    torch.cuda.synchronize()
    ops.status()
    assert all(torch.equal(y, want) for y, want in ys)


def test_memory_refused():
    """Host memory, and addresses that are not aligned."""
    import torch

    d, h = torch.zeros(1 << 16, device="cuda"), torch.zeros(4096)
    p, q = d.data_ptr(), h.data_ptr()
    w = ops.I8Weights(1, 64, 64, p, p)
    calls = [lambda a, b: ops.i8_quantize_rows_device(a, ops.F32, 4, 64, b, p, 4), lambda a, b: ops.i8_dequantize_rows_device(a, p, 4, 64, b, ops.F32),
             lambda a, b: ops.i8_product_device(w, a, p, 4, None, b, ops.F16), lambda a, b: ops.i8_gate_up_device(w, a, p, 4, None, b, ops.F16),
             lambda a, b: ops.i8_product_device(ops.I8Weights(1, 64, 64, a, p), p, p, 4, None, b, ops.F16)]
    for call in calls:
        for a, b, word in ((q, p, "not device memory"), (p, q, "not device memory"), (p + 2, p, "aligned"), (p, p + 2, "aligned"), (None, p, "required"), (p, None, "required")):
            with pytest.raises(MoEError) as e:
                call(a, b)
            assert e.value.status == _lib.MOE_BAD_ARGUMENT and word in str(e.value)
    with pytest.raises(MoEError) as e:
        ops.i8_product_device(ops.I8Weights(1, 64, 64, p, q), p, p, 4, None, p, ops.F16)
    assert "weight scales" in str(e.value)


@pytest.mark.parametrize("T", [1, 50, 700])
def test_a_block_put_together(T):
    """Routing, rows in 8 bits to expert order, the experts' products and the combine, plain and replayed from a graph with other inputs."""
    import torch

    rng = np.random.default_rng(T)
    E, k, D, F = 32, 4, 288, 160
    rows = T * k
    wc1, ws1, _, _ = product_case(rng, E, 2 * F, D, 1, 40)
    wc2, ws2, _, _ = product_case(rng, E, D, F, 1, 40)
    ws1, ws2 = ws1 / 8, ws2 / 8
    (w1, keep1), (w2, keep2) = weights_of(wc1, ws1), weights_of(wc2, ws2)
    logits, x = rng.standard_normal((T, E)).astype(np.float32), rng.standard_normal((T, D)).astype(np.float32)
    dl, dx = dev(logits), dev(x)
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    ids, w, offsets, inv, out = i32(T, k), f32(T, k), i32(E + 1), i32(T, k), f32(T, D)
    work = torch.empty(ops.route_work_bytes(T, E), dtype=torch.uint8, device="cuda")
    (xc, xs), (hc, hs) = buffers(rows, D), buffers(rows, F)
    h, y = torch.empty((rows, F), dtype=torch.bfloat16, device="cuda"), torch.empty((rows, D), dtype=torch.bfloat16, device="cuda")

    def block(st):
        p = lambda t: t.data_ptr()  # noqa: E731
        ops.route_logits_device(p(dl), ops.F32, T, E, k, p(ids), p(w), offsets_ptr=p(offsets), inv_ptr=p(inv), work_ptr=p(work), work_bytes=work.numel(), stream=st)
        ops.i8_quantize_rows_device(p(dx), ops.F32, T, D, p(xc), p(xs), rows, inv_ptr=p(inv), n_used=k, stream=st)
        ops.i8_gate_up_device(w1, p(xc), p(xs), rows, p(offsets), p(h), ops.BF16, swiglu_limit=7.0, stream=st)
        ops.i8_quantize_rows_device(p(h), ops.BF16, rows, F, p(hc), p(hs), rows, stream=st)
        ops.i8_product_device(w2, p(hc), p(hs), rows, p(offsets), p(y), ops.BF16, stream=st)
        ops.combine_rows_device(p(y), ops.BF16, rows, p(inv), p(w), T, k, D, p(out), residual_ptr=p(dx), stream=st)

    def want(logits, x):
        _, wt, off, place = R.route(logits.astype(np.float64), k)
        c, s = M.quantize(x)
        at = place.reshape(-1)
        ce, se = np.empty((rows, D), np.int8), np.empty(rows, np.float32)
        ce[at], se[at] = np.repeat(c, k, 0), np.repeat(s, k)
        v = M.product(ce, se, wc1, ws1, off, rows)[0].astype(np.float64)
        hb = torch.from_numpy(R.swiglu(v[:, :F], v[:, F:], 7.0)).bfloat16().double().numpy()
        ye = M.product(*M.quantize(hb), wc2, ws2, off, rows)[0].astype(np.float64)
        return x + (wt[..., None] * ye[place]).sum(1), np.linalg.norm((wt[..., None] * ye[place]).sum(1))

    block(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    ops.status()
    first = out.clone()
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
            assert torch.equal(out, first)
        ref, size = want(logits, x)
        # y's rounding to bf16 (2^-8 of each), and the values of h within 2^-17 of a border between two of bf16 (one in some 2^8), a step of which, 2^-8, may move
        # its row's scale or a code by one: 2^-7 of a row's largest for one in 2^8 values, below 2^-8 in all.
        assert np.linalg.norm(host(out) - ref) <= 2.0 ** -7 * size + 2.0 ** -22 * np.linalg.norm(ref)

"""On a B200: forms of the sorted rows', gradients' and 8-bit rows' kernels that only longer steps or other row lengths take, against the definitions in 64 bits."""
import numpy as np
import pytest

import more_ops_common as M
import test_i8_gpu as I
import test_sort_rows_gpu as S
from c0ven_b200 import ops

pytestmark = pytest.mark.gpu
TYPES = S.TYPES


# --- the routing's gradient: warps that take one row after another ------------------------------------------------------


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T, E, n", [(19001, 64, 8), (20011, 33, 16), (38001, 200, 4), (19500, 512, 10)])
def test_route_grad_of_more_rows_than_warps(T, E, n, score, renorm, type):
    """148 * 16 CTAs of 8 warps are 18,944: warps take a second row, and a third, whatever the form. Rows of few assignments follow rows of many, so that what a
    row leaves in the columns' memory would be seen."""
    import torch

    rng = np.random.default_rng(T + n)
    l, ids = S.route_case(rng, T, E, n, type, 3.0)
    kept = torch.from_numpy(rng.random((T, n)) < np.where(np.arange(T) // 18944 % 2, 0.2, 0.9)[:, None]).cuda()
    ids = torch.where(kept, ids, -1)
    dw = rng.standard_normal((T, n)).astype(np.float32)
    dd = S.dev(dw)
    dd[~kept] = float("nan")
    out = torch.full((T + 1, E), 7.0, dtype=S.dtype(type), device="cuda")
    ops.route_logits_grad_device(l.data_ptr(), TYPES[type], T, E, n, ids.data_ptr(), dd.data_ptr(), out.data_ptr(), score=S.TYPES_OF_SCORE[score], renorm=renorm, scale=2.5)
    S.check_route_grad(S.host(out[:T]), S.host(l), ids.cpu().numpy(), dw, score, renorm, 2.5, type)
    assert (out[T] == 7.0).all()


# --- gradients by 16 and by 32 threads a row ------------------------------------------------------------------------------


def additions(D):
    """Of a sum over D columns one after another, at most: a thread's share, by 32 threads a row at least where there are as many octets, and exchanges after it."""
    octets = D // 8
    threads = min(32, 1 << max(0, (octets - 1).bit_length()))
    return 8 * -(-octets // threads) + 5 + 8


def gathered64(rows, inv):
    """rows[inv] on the device, zeros where an entry names none: [T][n][D]."""
    import torch

    there = (inv >= 0) & (inv < len(rows))
    return torch.where(there[..., None], rows.double()[torch.where(there, inv, 0).long()], torch.zeros((), dtype=torch.float64, device="cuda"))


# Rows of 17 to 32 octets by 32 threads; so the rows' and weights' gradients of longer rows from 2,368 rows on, and all gradients where no more threads fit
# (264, 1,032 and 1,320 columns of 2,368 rows and more). Rows of 9 to 16 octets by 16.
HALF_AND_WHOLE_WARPS = [(2370, 3, 2560), (2370, 8, 2560), (2368, 11, 2560), (2369, 16, 2560), (2400, 2, 264), (2401, 16, 1032), (2500, 7, 1320), (37, 4, 136), (51, 10, 200),
                        (9, 13, 256), (1501, 6, 256), (50, 1, 72), (33, 16, 128), (5003, 5, 72), (1501, 9, 128)]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T, n, D", HALF_AND_WHOLE_WARPS)
def test_gradients_by_half_and_whole_warps(T, n, D, type):
    import torch

    rng = np.random.default_rng(T + n + D)
    g = torch.Generator(device="cuda").manual_seed(T + n)
    rows = max(1, T * n - T * n // 7)
    randn = lambda s, t=type: torch.randn(s, generator=g, device="cuda").to(S.dtype(t))  # noqa: E731
    inv = S.dev(S.places(rng, T, n, rows))
    x, dxs, y, dout, w = randn((T, D)), randn((rows, D)), randn((rows, D)), randn((T, D), "f32"), randn((T, n), "f32")
    dx, dw = torch.full((T + 1, D), 7.0, dtype=S.dtype(type), device="cuda"), torch.full((T + 1, n), 7.0, device="cuda")
    ops.sort_rows_grad_device(dxs.data_ptr(), TYPES[type], rows, inv.data_ptr(), T, n, D, dx_ptr=dx.data_ptr(), w_ptr=w.data_ptr(), x_ptr=x.data_ptr(), dw_ptr=dw.data_ptr())
    v = gathered64(dxs, inv)
    f = w.double()[..., None]
    S.near(S.host(dx[:T]), S.host((f * v).sum(1)), S.host((f * v).abs().sum(1)), type, n + 2)
    terms = x.double()[:, None] * v
    S.near(S.host(dw[:T]), S.host(terms.sum(2)), S.host(terms.abs().sum(2)), "f32", additions(D))
    assert (dx[T] == 7.0).all() and (dw[T] == 7.0).all()
    alone = torch.full((T, D), 7.0, dtype=S.dtype(type), device="cuda")
    ops.sort_rows_grad_device(dxs.data_ptr(), TYPES[type], rows, inv.data_ptr(), T, n, D, dx_ptr=alone.data_ptr(), w_ptr=w.data_ptr())
    assert torch.equal(alone, dx[:T])  # a column's sum has one order
    del v, terms
    dy, dw = y.clone(), torch.full((T + 1, n), 7.0, device="cuda")
    ops.combine_rows_grad_device(dout.data_ptr(), ops.F32, dy.data_ptr(), TYPES[type], rows, inv.data_ptr(), w.data_ptr(), T, n, D, dy_ptr=dy.data_ptr(), dw_ptr=dw.data_ptr())
    terms = dout.double()[:, None] * gathered64(y, inv)
    S.near(S.host(dw[:T]), S.host(terms.sum(2)), S.host(terms.abs().sum(2)), "f32", additions(D))
    want, there = y.clone(), (inv >= 0) & (inv < rows)
    want[inv[there].long()] = (w[..., None] * dout[:, None])[there].to(S.dtype(type))
    assert torch.equal(dy, want) and (dw[T] == 7.0).all()


# --- 8-bit rows: several rows a thread --------------------------------------------------------------------------------------


def quantized64(x):
    """Codes and scales of rows x on the device, in 64 bits: the quotient's rounding makes no border between two codes of what is none."""
    import torch

    x = x.double()
    top = x.abs().amax(1)
    bad = ~torch.isfinite(top)
    safe = torch.where(bad | (top == 0), torch.ones_like(top), top)
    codes = torch.round(127 * torch.where(bad[:, None], torch.zeros_like(x), x) / safe[:, None])
    scales = torch.where(bad, torch.full_like(top, float("nan")), top).float() / torch.full_like(top, 127, dtype=torch.float32)
    return codes.to(torch.int8), scales


def same(codes, scales, want):
    import torch

    return torch.equal(codes, want[0]) and torch.equal(scales.view(torch.int32)[~torch.isnan(want[1])], want[1].view(torch.int32)[~torch.isnan(want[1])]) and \
        torch.equal(torch.isnan(scales), torch.isnan(want[1]))


# Calls of 606,208 octets and more whose rows have 4, 8, 12 and 16: four threads a row, eight, four, three and two rows a thread at the same time.
SHORT_ROWS = [(151_553, 32), (75_787, 64), (50_533, 96), (37_891, 128)]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T, K", SHORT_ROWS)
def test_quantize_many_short_rows(T, K, type):
    """As they lie; rows of ordinary sizes, and among them rows of zeros, of f32's ends, denormals, infinities and NaN, so that a thread's rows differ in kind."""
    import torch

    rng = np.random.default_rng(K)
    x = I.rows_of(rng, T, K).astype(np.float32) if type != "f16" else np.clip(I.rows_of(rng, T, K), -6e4, 6e4).astype(np.float32)
    plain = S.dev(x, type)
    odd = x.copy()
    pick = rng.integers(0, 40, T)
    odd[pick == 1] *= np.float32(2.0 ** -100)
    odd[pick == 2] *= np.float32(2.0 ** 70)
    odd[pick == 3] = 0
    odd[np.flatnonzero(pick == 4), rng.integers(0, K, (pick == 4).sum())] = np.inf
    odd[np.flatnonzero(pick == 5), rng.integers(0, K, (pick == 5).sum())] = np.nan
    odd[pick == 6] = np.float32(2.0 ** -149) * rng.integers(-200, 201, ((pick == 6).sum(), K))
    for t in (plain, S.dev(odd, type)):
        codes, scales = I.buffers(T + 1, K)
        ops.i8_quantize_rows_device(t.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), T)
        assert same(codes[:T], scales[:T], quantized64(t))
        assert (codes[T] == 0x6E).all() and scales[T] == 7.0


@pytest.mark.parametrize("type", ["f32", "bf16"])
@pytest.mark.parametrize("T, K", SHORT_ROWS)
def test_quantize_scatters_many_short_rows(T, K, type):
    """To two places each, some of none, from rows that lie apart; rows no entry names are left as they were."""
    import torch

    rng, n = np.random.default_rng(K + 1), 2
    rows = T * n * 7 // 8
    full = S.dev(rng.standard_normal((T, K + 8)).astype(np.float32), type)
    inv = S.dev(S.places(rng, T, n, rows, 0.05))
    codes, scales = I.buffers(rows + 1, K)
    ops.i8_quantize_rows_device(full.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), rows, stride=K + 8, inv_ptr=inv.data_ptr(), n_used=n)
    want, (c, s) = I.buffers(rows + 1, K), quantized64(full[:, :K])
    for k in range(n):
        there = (inv[:, k] >= 0) & (inv[:, k] < rows)
        want[0][inv[there, k].long()], want[1][inv[there, k].long()] = c[there], s[there]
    assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])


def test_the_device_form_of_the_definition_is_the_hosts():
    rng = np.random.default_rng(3)
    x = I.rows_of(rng, 500, 96).astype(np.float32)
    x[7, 3], x[8, 4] = np.inf, np.nan
    c, s = quantized64(S.dev(x))
    want = M.quantize(x)
    assert np.array_equal(c.cpu().numpy(), want[0]) and np.array_equal(s.cpu().numpy(), want[1], equal_nan=True)


@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_quantize_every_significand_by_every_other(type):
    """Rows whose largest has every significand of the type, in [2, 4), and beside it all significands of each of the nine powers of two below."""
    n = 1 << (7 if type == "bf16" else 10)
    sig = 1 + np.arange(n) / n
    x = np.concatenate([np.repeat(2 * sig[:, None], 32, 1)] + [np.tile(sig * 2.0 ** -j, (n, 1)) for j in range(9)], 1).astype(np.float32)
    t = S.dev(x, type)
    T, K = x.shape
    assert K % 32 == 0 and np.array_equal(S.host(t), x)  # nothing was rounded
    codes, scales = I.buffers(T, K)
    ops.i8_quantize_rows_device(t.data_ptr(), TYPES[type], T, K, codes.data_ptr(), scales.data_ptr(), T)
    assert same(codes, scales, quantized64(t))


# --- products: the same bits again ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("y_type", ["f16", "bf16"])
@pytest.mark.parametrize("E, T, k, D, F", [(512, 100, 10, 2048, 512), (16, 300, 4, 2560, 768), (1, 1, 1, 288, 64)])
def test_gate_up_rows_and_product_repeat_themselves(E, T, k, D, F, y_type):
    """Gate and up, its result in 8-bit rows, the product: twenty times over on buffers that held something else, bit for bit."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(E)
    rows = T * k
    w1, w2 = (torch.randint(-40, 41, s, generator=g, device="cuda", dtype=torch.int8) for s in ((E, 2 * F, D), (E, D, F)))
    s1, s2 = (0.01 + 0.01 * torch.rand(s, generator=g, device="cuda") for s in ((E, 2 * F), (E, D)))
    c, s = torch.randint(-127, 128, (rows, D), generator=g, device="cuda", dtype=torch.int8), 0.001 * torch.rand(rows, generator=g, device="cuda")
    offsets = torch.sort(torch.randint(0, rows + 1, (E + 1,), generator=g, device="cuda"))[0].to(torch.int32)
    offsets[0], offsets[E] = 0, rows
    a, b = ops.I8Weights(E, 2 * F, D, w1.data_ptr(), s1.data_ptr()), ops.I8Weights(E, D, F, w2.data_ptr(), s2.data_ptr())
    first = None
    for i in range(20):
        h, y = (torch.full(z, float(i), dtype=S.dtype(y_type), device="cuda") for z in ((rows, F), (rows, D)))
        hc, hs = I.buffers(rows, F)
        ops.i8_gate_up_device(a, c.data_ptr(), s.data_ptr(), rows, offsets.data_ptr(), h.data_ptr(), TYPES[y_type])
        ops.i8_quantize_rows_device(h.data_ptr(), TYPES[y_type], rows, F, hc.data_ptr(), hs.data_ptr(), rows)
        ops.i8_product_device(b, hc.data_ptr(), hs.data_ptr(), rows, offsets.data_ptr(), y.data_ptr(), TYPES[y_type])
        if first is None:
            first = h, hc, hs, y
            assert torch.isfinite(y).all() and (y != 0).any()
        assert all(torch.equal(p, q) for p, q in zip(first, (h, hc, hs, y)))
    ops.status()

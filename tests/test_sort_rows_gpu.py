"""On a B200: rows sorted by expert, the gradients of that and of the combine, and of the routing's weights, against the definitions in 64 bits."""
import numpy as np
import pytest

import more_ops_common as M
import ops_common as R
from c0ven_b200 import MoEError, _lib, ops

pytestmark = pytest.mark.gpu
TYPES = {"f32": ops.F32, "f16": ops.F16, "bf16": ops.BF16}
U = 2.0 ** -24  # half a step of f32


def dtype(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def dev(a, type=None):
    import torch

    t = torch.from_numpy(np.ascontiguousarray(a))
    return (t if type is None else t.to(dtype(type))).cuda()


def host(t):
    return t.double().cpu().numpy()


def places(rng, T, n, R, dropped=0.1):
    """Distinct places of 0 .. R - 1 for most assignments, the rest -1, R or further."""
    inv = rng.permutation(max(R, T * n))[:T * n].reshape(T, n).astype(np.int32)
    out = rng.random((T, n)) < dropped
    inv[out] = rng.choice([-1, R, R + 5, 2 ** 31 - 1, -2 ** 31], out.sum())
    return inv


SHAPES = [(1, 1, 8), (1, 16, 2560), (3, 2, 16), (7, 3, 4104), (300, 10, 64), (13, 8, 2560), (33, 5, 24), (21, 4, 264), (2, 6, 2056), (65, 16, 1024), (1001, 7, 520), (5, 2, 65536),
          # Long steps: a warp a row, 64 and 128 threads a row, a CTA; rows that leave the last CTA half empty.
          (1203, 3, 2560), (1100, 16, 1032), (1024, 5, 2880), (1501, 2, 3088), (1027, 12, 264), (2050, 8, 64)]


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T, n, D", SHAPES)
def test_sort_rows(T, n, D, type):
    import torch

    rng = np.random.default_rng(T * D + n)
    rows = max(1, T * n - T * n // 7)
    inv = places(rng, T, n, rows)
    wide = dev(rng.standard_normal((T, D + 8)).astype(np.float32), type)
    w = rng.standard_normal((T, n)).astype(np.float32)
    di, dw = dev(inv), dev(w)
    for x, stride in ((wide[:, :D].contiguous(), 0), (wide, D + 8)):
        for weights in (None, dw):
            xs = torch.full((rows + 1, D), 7.0, dtype=dtype(type), device="cuda")
            ops.sort_rows_device(x.data_ptr(), TYPES[type], T, n, D, di.data_ptr(), rows, xs.data_ptr(), stride=stride, w_ptr=None if weights is None else dw.data_ptr())
            # x times w in f32, then rounded to the type: to the bit.
            v = M.sort(x.float().cpu().numpy()[:, :D], inv, None if weights is None else w, np.full((rows, D), 7.0, np.float32))
            assert torch.equal(xs[:rows].cpu(), torch.from_numpy(v).to(dtype(type))) and (xs[rows] == 7.0).all()


def test_sort_rows_keeps_bits():
    """Without weights rows move as they are: NaN payloads, infinities, -0 and denormals among them."""
    import torch

    rng = np.random.default_rng(3)
    bits = dev(rng.integers(-2 ** 15, 2 ** 15, (40, 96)).astype(np.int16))
    inv = places(rng, 40, 3, 120, 0.0)
    di = dev(inv)
    for type in ("f16", "bf16"):
        out = torch.zeros((120, 96), dtype=torch.int16, device="cuda")
        ops.sort_rows_device(bits.data_ptr(), TYPES[type], 40, 3, 96, di.data_ptr(), 120, out.data_ptr())
        for k in range(3):
            assert torch.equal(out[di[:, k].long()], bits)


def chain(D):
    """Additions after one another in a sum over D columns: a thread's share, and the exchanges after it."""
    octets = D // 8
    log2 = min(8, max(0, (octets - 1).bit_length()))
    return 8 * -(-octets // (1 << log2)) + log2 + 8


def near(got, want, size, type, additions):
    """Within `additions` half steps of f32 of the terms' sizes, then half a step of the type (or of its least numbers)."""
    off = np.abs(got - want)
    bound = additions * U * size
    least = {"f32": 2.0 ** -149, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}[type]
    assert (off <= bound + R.HALF_STEP[type] * (np.abs(want) + bound) + least).all(), (off - bound).max()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T, n, D", SHAPES)
def test_sort_rows_grad(T, n, D, type):
    import torch

    rng = np.random.default_rng(T * D + n + 1)
    rows = max(1, T * n - T * n // 7)
    inv = places(rng, T, n, rows)
    wide, dxs = (dev(rng.standard_normal(s).astype(np.float32), type) for s in ((T, D + 8), (rows, D)))
    add = dev(rng.standard_normal((T, D)).astype(np.float32), type)
    w = rng.standard_normal((T, n)).astype(np.float32)
    di, dw = dev(inv), dev(w)
    v, ones = M.gathered(host(dxs), inv), np.ones((T, n))
    for weights in (None, w):
        f = (ones if weights is None else w.astype(np.float64))[..., None]
        for added in (False, True):
            for with_dw in (False, True):
                for with_dx in ((True, False) if with_dw and not added else (True,)):
                    dx = add.clone() if added else torch.full((T, D), 7.0, dtype=dtype(type), device="cuda")  # in place: dx is add
                    got = torch.full((T, n), 7.0, device="cuda")
                    ops.sort_rows_grad_device(dxs.data_ptr(), TYPES[type], rows, di.data_ptr(), T, n, D, dx_ptr=dx.data_ptr() if with_dx else None,
                                              w_ptr=None if weights is None else dw.data_ptr(), x_ptr=wide.data_ptr() if with_dw else None, stride=D + 8,
                                              add_ptr=dx.data_ptr() if added else None, dw_ptr=got.data_ptr() if with_dw else None)
                    if with_dx:
                        a = host(add) if added else 0.0
                        near(host(dx), (f * v).sum(1) + a, (np.abs(f * v)).sum(1) + np.abs(a), type, n + 2)
                    else:
                        assert (dx == 7.0).all()
                    if with_dw:
                        terms = host(wide)[:, None, :D] * v
                        near(host(got), terms.sum(2), np.abs(terms).sum(2), "f32", chain(D))
                    else:
                        assert (got == 7.0).all()


@pytest.mark.parametrize("dout_type, type", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("T, n, D", SHAPES)
def test_combine_rows_grad(T, n, D, dout_type, type):
    import torch

    rng = np.random.default_rng(T * D + n + 2)
    rows = max(1, T * n - T * n // 7)
    inv = places(rng, T, n, rows)
    dout, y = dev(rng.standard_normal((T, D)).astype(np.float32), dout_type), dev(rng.standard_normal((rows, D)).astype(np.float32), type)
    w = rng.standard_normal((T, n)).astype(np.float32)
    di, wd = dev(inv), dev(w)
    terms = host(dout)[:, None, :] * M.gathered(host(y), inv)
    for with_dy, with_dw, in_place in ((True, True, False), (True, True, True), (True, False, False), (False, True, False)):
        dy = y.clone() if in_place else torch.full((rows, D), 7.0, dtype=dtype(type), device="cuda")
        dw = torch.full((T, n), 7.0, device="cuda")
        before = dy.float().cpu().numpy()
        from_y = (dy if in_place else y).data_ptr() if with_dw else None
        ops.combine_rows_grad_device(dout.data_ptr(), TYPES[dout_type], from_y, TYPES[type], rows, di.data_ptr(), wd.data_ptr() if with_dy else None, T, n, D,
                                     dy_ptr=dy.data_ptr() if with_dy else None, dw_ptr=dw.data_ptr() if with_dw else None)
        want = M.sort(dout.float().cpu().numpy(), inv, w, before) if with_dy else before
        assert torch.equal(dy.cpu(), torch.from_numpy(want).to(dtype(type)))
        if with_dw:
            near(host(dw), terms.sum(2), np.abs(terms).sum(2), "f32", chain(D))
        else:
            assert (dw == 7.0).all()


def test_no_rows_to_gather():
    """R 0: nothing is read of the rows, dx is add or zeros, dw zeros."""
    import torch

    inv = dev(np.array([[0, -1, 5], [1, 2, 3]], np.int32))
    x, add, w = torch.ones((2, 16), device="cuda"), torch.full((2, 16), 3.0, device="cuda"), torch.ones((2, 3), device="cuda")
    dx, dw = torch.full((2, 16), 7.0, device="cuda"), torch.full((2, 3), 7.0, device="cuda")
    for a, value in ((None, 0.0), (add.data_ptr(), 3.0)):
        ops.sort_rows_grad_device(None, ops.F32, 0, inv.data_ptr(), 2, 3, 16, dx_ptr=dx.data_ptr(), x_ptr=x.data_ptr(), add_ptr=a, dw_ptr=dw.data_ptr())
        assert (dx == value).all() and (dw == 0).all()
    dw[:] = 7.0
    ops.combine_rows_grad_device(x.data_ptr(), ops.F32, None, ops.F32, 0, inv.data_ptr(), w.data_ptr(), 2, 3, 16, dw_ptr=dw.data_ptr())
    assert (dw == 0).all()


def test_infinities_and_nans_stay_where_they_belong():
    """What lies in rows that no entry names reaches nothing; what lies in a named one, its own results alone."""
    import torch

    inv = dev(np.array([[0, -1], [2, 9]], np.int32))
    dxs = torch.ones((4, 8), device="cuda")
    dxs[1], dxs[3], dxs[2, 5] = float("nan"), float("inf"), float("inf")
    x, w = torch.ones((2, 8), device="cuda"), torch.tensor([[2.0, float("nan")], [3.0, float("inf")]], device="cuda")
    dx, dw = torch.empty((2, 8), device="cuda"), torch.empty((2, 2), device="cuda")
    ops.sort_rows_grad_device(dxs.data_ptr(), ops.F32, 4, inv.data_ptr(), 2, 2, 8, dx_ptr=dx.data_ptr(), w_ptr=w.data_ptr(), x_ptr=x.data_ptr(), dw_ptr=dw.data_ptr())
    assert (dx[0] == 2).all() and dx[1, 5] == float("inf") and (dx[1, :5] == 3).all() and (dx[1, 6:] == 3).all()
    assert dw.tolist() == [[8.0, 0.0], [float("inf"), 0.0]]
    dy = torch.full((4, 8), 7.0, device="cuda")
    ops.combine_rows_grad_device(x.data_ptr(), ops.F32, dxs.data_ptr(), ops.F32, 4, inv.data_ptr(), w.data_ptr(), 2, 2, 8, dy_ptr=dy.data_ptr(), dw_ptr=dw.data_ptr())
    assert (dy[0] == 2).all() and (dy[1] == 7).all() and (dy[2] == 3).all() and (dy[3] == 7).all() and dw.tolist() == [[8.0, 0.0], [float("inf"), 0.0]]


def test_offsets_past_32_bits():
    """Rows whose places do not fit 32 bits: the last ones are right."""
    import torch

    rng = np.random.default_rng(5)
    rows, D = 66000, 65536  # 8.6 GB of bf16
    xs = torch.zeros((rows, D), dtype=torch.bfloat16, device="cuda")
    x = dev(rng.standard_normal((2, D)).astype(np.float32), "bf16")
    inv = dev(np.array([[rows - 1, 0], [rows - 2, 1]], np.int32))
    ops.sort_rows_device(x.data_ptr(), ops.BF16, 2, 2, D, inv.data_ptr(), rows, xs.data_ptr())
    assert torch.equal(xs[-1], x[0]) and torch.equal(xs[-2], x[1]) and torch.equal(xs[:2], x) and (xs[2:-2] == 0).all()
    dx = torch.empty((2, D), dtype=torch.bfloat16, device="cuda")
    ops.sort_rows_grad_device(xs.data_ptr(), ops.BF16, rows, inv.data_ptr(), 2, 2, D, dx_ptr=dx.data_ptr())
    assert torch.equal(dx, (2 * x.float()).bfloat16())
    dw, w = torch.empty((2, 2), device="cuda"), dev(np.array([[0.5, 2], [4, 0.25]], np.float32))
    ops.combine_rows_grad_device(x.data_ptr(), ops.BF16, xs.data_ptr(), ops.BF16, rows, inv.data_ptr(), w.data_ptr(), 2, 2, D, dy_ptr=xs.data_ptr(), dw_ptr=dw.data_ptr())
    assert torch.equal(xs[-1], 0.5 * x[0]) and torch.equal(xs[-2], 4 * x[1]) and torch.equal(xs[0], 2 * x[0])
    sq = (host(x) ** 2).sum(1, keepdims=True)
    near(host(dw), np.repeat(sq, 2, 1), np.repeat(sq, 2, 1), "f32", chain(D))
    # As many columns as rows of x: a step's rows past 2^32 values.
    T = rows * D // 64
    many = xs.view(T, 64)
    inv = torch.full((T, 1), -1, dtype=torch.int32, device="cuda")
    inv[-3:, 0] = torch.tensor([2, 0, 1], dtype=torch.int32)
    out = torch.zeros((3, 64), dtype=torch.bfloat16, device="cuda")
    many[-3:] = dev(rng.standard_normal((3, 64)).astype(np.float32), "bf16")
    ops.sort_rows_device(many.data_ptr(), ops.BF16, T, 1, 64, inv.data_ptr(), 3, out.data_ptr())
    assert torch.equal(out[[2, 0, 1]], many[-3:])


def route_case(rng, T, E, n, type, spread=1.0):
    """Logits of a type and the experts that the framework chooses of them."""
    import torch

    l = dev((spread * rng.standard_normal((T, E))).astype(np.float32), type)
    ids, w = torch.empty((T, n), dtype=torch.int32, device="cuda"), torch.empty((T, n), device="cuda")
    ops.route_logits_device(l.data_ptr(), TYPES[type], T, E, n, ids.data_ptr(), w.data_ptr())
    return l, ids


def check_route_grad(got, l, ids, dw, score, renorm, scale, type, known=None):
    want, size = known or M.route_grad(l, ids, dw.astype(np.float64), score, renorm, scale)
    # What a share p is off by: its exponential 2 ulp (4 U) and its argument's rounding, U of the largest difference in use, which for a sigmoid is the logit
    # itself; the sum over the row 21 U (16 a lane, 5 exchanges) with the terms' own; the division, and 1 - s likewise. The mean of d: those and 6 U more. Five products.
    finite = l[np.isfinite(l)]
    spread = min(200.0, float(finite.max() - finite.min()) if finite.size else 0.0) + (0.0 if score == "softmax" else min(90.0, float(np.abs(finite).max(initial=0.0))))
    bound = 2 * (2 * (4 + spread) + 21 + 12 + 5) * U * size
    least = {"f32": 2.0 ** -126, "f16": 2.0 ** -25, "bf16": 2.0 ** -126}[type] * (1 + abs(scale) * np.abs(dw).max(initial=0.0))
    off = np.abs(got - want)
    assert (off <= bound + R.HALF_STEP[type] * (np.abs(want) + bound) + least).all(), (off / (size + 1e-30)).max()


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T, E, n", [(1, 1, 1), (1, 512, 10), (9, 512, 16), (37, 160, 6), (13, 33, 4), (100, 8, 2), (5, 64, 8), (3, 255, 16), (700, 96, 1), (2, 16, 16),
                                     # More rows than warps that stay.
                                     (4001, 512, 10), (5003, 200, 8), (8005, 64, 4)])
def test_route_grad(T, E, n, score, renorm, type):
    import torch

    rng = np.random.default_rng(T * E + n)
    for spread in (1.0, 20.0):
        l, ids = route_case(rng, T, E, n, type, spread)
        if n > 1:
            ids[0, n // 2] = -1  # a place without an expert, whatever its weight's gradient
        dw = rng.standard_normal((T, n)).astype(np.float32)
        dd = dev(dw)
        dd[0, n // 2] = float("nan") if n > 1 else dd[0, 0]
        out = torch.full((T + 1, E + 3), 7.0, dtype=dtype(type), device="cuda")
        wide = torch.zeros((T, E + 5), dtype=dtype(type), device="cuda")
        wide[:, :E] = l
        known = M.route_grad(host(l), ids.cpu().numpy(), dw.astype(np.float64), score, renorm, 2.5)
        for src, stride, dst in ((l, 0, 0), (wide, E + 5, E + 3)):
            out[:] = 7.0
            ops.route_logits_grad_device(src.data_ptr(), TYPES[type], T, E, n, ids.data_ptr(), dd.data_ptr(), out.data_ptr(), score=TYPES_OF_SCORE[score], renorm=renorm,
                                         scale=2.5, stride=stride, dlogits_stride=dst)
            flat = out.view(-1)
            got = out[:T, :E] if dst else flat[:T * E].view(T, E)
            check_route_grad(host(got), host(l), ids.cpu().numpy(), dw, score, renorm, 2.5, type, known)
            assert (out[T] == 7.0).all() and (not dst or (out[:T, E:] == 7.0).all()) and (dst or (flat[T * E:] == 7.0).all())


TYPES_OF_SCORE = {"softmax": ops.SOFTMAX, "sigmoid": ops.SIGMOID}


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_grad_extremes(score, renorm):
    """Experts out by their logit or bias, rows of none, logits so small or large that scores vanish or are all one."""
    import torch

    rng = np.random.default_rng(8)
    T, E, n = 9, 48, 4
    l = rng.standard_normal((T, E)).astype(np.float32)
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    bias[5], bias[6] = -np.inf, np.nan
    l[0, 3], l[0, 9] = -np.inf, np.nan
    l[1] = -np.inf
    l[2] -= 100
    l[3] += 100
    l[4] = -1e30 * np.abs(l[4])
    l[5, :7], l[6] = np.finfo(np.float32).min, np.finfo(np.float32).min
    l[7] *= 60
    l[8, 20] = 1e30
    ids, w = torch.empty((T, n), dtype=torch.int32, device="cuda"), torch.empty((T, n), device="cuda")
    dl, db, dw = dev(l), dev(bias), rng.standard_normal((T, n)).astype(np.float32)
    dd, out = dev(dw), torch.full((T, E), 7.0, device="cuda")
    ops.route_logits_device(dl.data_ptr(), ops.F32, T, E, n, ids.data_ptr(), w.data_ptr(), score=TYPES_OF_SCORE[score], bias_ptr=db.data_ptr(), renorm=renorm)
    ops.route_logits_grad_device(dl.data_ptr(), ops.F32, T, E, n, ids.data_ptr(), dd.data_ptr(), out.data_ptr(), score=TYPES_OF_SCORE[score], bias_ptr=db.data_ptr(),
                                 renorm=renorm)
    l64 = l.astype(np.float64)
    l64[np.isnan(l64)] = -np.inf
    l64[:, 5:7] = -np.inf
    assert (ids[1] == -1).all() and (out[1] == 0).all() and (out[:, 5:7] == 0).all() and torch.isfinite(out).all()
    for t in range(T):  # a row's bound is its own spread's
        check_route_grad(host(out[t:t + 1]), l64[t:t + 1], ids[t:t + 1].cpu().numpy(), dw[t:t + 1], score, renorm, 1.0, "f32")


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_grad_against_differences(score, renorm):
    """Central differences of the weights in 64 bits: a step of 2^-14 leaves 2^-28 of the third derivative, below 4, times scale and dw."""
    import torch

    rng = np.random.default_rng(9)
    T, E, n, step = 12, 20, 4, 2.0 ** -14
    l, ids = route_case(rng, T, E, n, "f32")
    dw = rng.uniform(-1, 1, (T, n)).astype(np.float32)
    dd, out = dev(dw), torch.empty((T, E), device="cuda")
    ops.route_logits_grad_device(l.data_ptr(), ops.F32, T, E, n, ids.data_ptr(), dd.data_ptr(), out.data_ptr(), score=TYPES_OF_SCORE[score], renorm=renorm, scale=2.0)
    l64, i = host(l), ids.cpu().numpy()
    for e in range(E):
        hi, lo = l64.copy(), l64.copy()
        hi[:, e] += step
        lo[:, e] -= step
        d = (M.weights_by_logits(hi, i, score, renorm, 2.0) - M.weights_by_logits(lo, i, score, renorm, 2.0)) / (2 * step)
        # The f32 result is within some 60 half steps of terms of 2 at most.
        assert np.allclose((d * dw).sum(1), host(out)[:, e], rtol=0, atol=4 * n * 2 * step ** 2 + 120 * U)


@pytest.mark.parametrize("T, n, D", [(3, 4, 40), (50, 7, 264), (1300, 5, 2880)])
def test_gradients_are_the_linear_calls_transposes(T, n, D):
    """Sorting and the combine are linear in rows, results and weights: the change that a change of one of them makes, times a gradient, is that change times the
    gradient's. (Differences of linear calls are the calls of differences.) Sums in 64 bits of f32 results, each within a few half steps of its terms' sizes."""
    import torch

    rng = np.random.default_rng(T)
    rows = T * n
    inv = dev(rng.permutation(rows).reshape(T, n).astype(np.int32))
    f = lambda *s: dev(rng.standard_normal(s).astype(np.float32))  # noqa: E731
    x, v, g, w, u, dout = f(T, D), f(T, D), f(rows, D), f(T, n), f(T, n), f(T, D)
    y, z = f(rows, D), f(rows, D)
    out = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    dx, dw, dy, dw2, xs, xu, cz, cu = out(T, D), out(T, n), out(rows, D), out(T, n), out(rows, D), out(rows, D), out(T, D), out(T, D)
    p = lambda t: t.data_ptr()  # noqa: E731
    ops.sort_rows_grad_device(p(g), ops.F32, rows, p(inv), T, n, D, dx_ptr=p(dx), w_ptr=p(w), x_ptr=p(x), dw_ptr=p(dw))
    ops.sort_rows_device(p(v), ops.F32, T, n, D, p(inv), rows, p(xs), w_ptr=p(w))   # along v, the weights as they are
    ops.sort_rows_device(p(x), ops.F32, T, n, D, p(inv), rows, p(xu), w_ptr=p(u))   # along u, the rows as they are
    ops.combine_rows_grad_device(p(dout), ops.F32, p(y), ops.F32, rows, p(inv), p(w), T, n, D, dy_ptr=p(dy), dw_ptr=p(dw2))
    ops.combine_rows_device(p(z), ops.F32, rows, p(inv), p(w), T, n, D, p(cz))
    ops.combine_rows_device(p(y), ops.F32, rows, p(inv), p(u), T, n, D, p(cu))
    for a, b, c, d in ((xs, g, v, dx), (xu, g, u, dw), (cz, dout, z, dy), (cu, dout, u, dw2)):
        one, two = host(a) * host(b), host(c) * host(d)
        size = np.abs(host(g)).sum() * 8 if a is xs or a is xu else np.abs(host(dout)).sum() * 8 * n
        assert abs(one.sum() - two.sum()) <= (chain(D) + n + 4) * U * max(np.abs(one).sum(), np.abs(two).sum(), size)


def test_streams_and_captured_graphs():
    """On a stream of the caller's, and replayed from a captured graph with other inputs: the same bits as the plain call's."""
    import torch

    rng = np.random.default_rng(10)
    T, n, D, E = 130, 5, 264, 40
    rows = T * n
    inv = dev(places(rng, T, n, rows))
    x, dxs = (dev(rng.standard_normal(s).astype(np.float32), "bf16") for s in ((T, D), (rows, D)))
    dout, w = dev(rng.standard_normal((T, D)).astype(np.float32)), dev(rng.random((T, n)).astype(np.float32))
    l, ids = route_case(rng, T, E, n, "f32")
    out = {k: torch.zeros(s, dtype=t, device="cuda") for k, s, t in (("xs", (rows, D), torch.bfloat16), ("dx", (T, D), torch.bfloat16), ("dw", (T, n), torch.float32),
                                                                     ("dy", (rows, D), torch.bfloat16), ("dw2", (T, n), torch.float32), ("dl", (T, E), torch.float32))}

    def calls(st):
        p = {k: v.data_ptr() for k, v in out.items()}
        ops.sort_rows_device(x.data_ptr(), ops.BF16, T, n, D, inv.data_ptr(), rows, p["xs"], w_ptr=w.data_ptr(), stream=st)
        ops.combine_rows_grad_device(dout.data_ptr(), ops.F32, p["xs"], ops.BF16, rows, inv.data_ptr(), w.data_ptr(), T, n, D, dy_ptr=p["dy"], dw_ptr=p["dw2"], stream=st)
        ops.sort_rows_grad_device(p["dy"], ops.BF16, rows, inv.data_ptr(), T, n, D, dx_ptr=p["dx"], w_ptr=w.data_ptr(), x_ptr=x.data_ptr(), dw_ptr=p["dw"], stream=st)
        ops.route_logits_grad_device(l.data_ptr(), ops.F32, T, E, n, ids.data_ptr(), p["dw"], p["dl"], stream=st)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    calls(s.cuda_stream)
    s.synchronize()
    first = {k: v.clone() for k, v in out.items()}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(torch.cuda.current_stream().cuda_stream)
    for v in out.values():
        v.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out[k], first[k]) for k in out)
    x.neg_()
    graph.replay()
    torch.cuda.synchronize()
    got = {k: v.clone() for k, v in out.items()}
    calls(None)
    torch.cuda.synchronize()
    assert all(torch.equal(out[k], got[k]) for k in out) and torch.equal(got["xs"], -first["xs"])


def test_memory_refused():
    """Host memory, and addresses that are not aligned."""
    import torch

    d, h = torch.zeros(4096, device="cuda"), torch.zeros(4096)
    p, q = d.data_ptr(), h.data_ptr()
    for call in (lambda a, b: ops.sort_rows_device(a, ops.F32, 4, 2, 64, p, 8, b), lambda a, b: ops.sort_rows_grad_device(a, ops.F32, 8, p, 4, 2, 64, dx_ptr=b),
                 lambda a, b: ops.combine_rows_grad_device(a, ops.F32, p, ops.F32, 8, p, p, 4, 2, 64, dy_ptr=b),
                 lambda a, b: ops.route_logits_grad_device(a, ops.F32, 4, 64, 2, p, p, b)):
        for a, b, word in ((q, p, "not device memory"), (p, q, "not device memory"), (p + 2, p, "aligned"), (p, p + 2, "aligned"), (None, p, "required")):
            with pytest.raises(MoEError) as e:
                call(a, b)
            assert e.value.status == _lib.MOE_BAD_ARGUMENT and word in str(e.value)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [1, 29, 300])
def test_a_block_that_trains(T, score):
    """Routing, rows to expert order, the caller's own experts, the combine, and back: gradients of rows, router logits and experts against those of the block in
    64 bits, differentiated by torch."""
    import torch

    torch.manual_seed(T)
    E, n, D, F = 16, 3, 64, 32
    x, wr = torch.randn(T, D, device="cuda"), torch.randn(E, D, device="cuda") / 8
    w1, w2 = torch.randn(E, F, D, device="cuda") / 8, torch.randn(E, D, F, device="cuda") / 6
    dout = torch.randn(T, D, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    i32 = lambda *s: torch.empty(s, dtype=torch.int32, device="cuda")  # noqa: E731
    f32 = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    rows, code = T * n, TYPES_OF_SCORE[score]
    ids, w, offsets, inv, work = i32(T, n), f32(T, n), i32(E + 1), i32(T, n), torch.empty(ops.route_work_bytes(T, E), dtype=torch.uint8, device="cuda")
    logits = (x.double() @ wr.double().T).float()
    ops.route_logits_device(logits.data_ptr(), ops.F32, T, E, n, ids.data_ptr(), w.data_ptr(), score=code, offsets_ptr=offsets.data_ptr(), inv_ptr=inv.data_ptr(),
                            work_ptr=work.data_ptr(), work_bytes=work.numel(), scale=1.5, stream=st)
    xs, y, out = f32(rows, D), f32(rows, D), f32(T, D)
    ops.sort_rows_device(x.data_ptr(), ops.F32, T, n, D, inv.data_ptr(), rows, xs.data_ptr(), stream=st)
    # The caller's experts, in 64 bits so that what is off is the framework's.
    xe, m1, m2 = xs.double().requires_grad_(), w1.double().requires_grad_(), w2.double().requires_grad_()
    at = offsets.tolist()
    ye = torch.cat([torch.tanh(xe[at[e]:at[e + 1]] @ m1[e].T) @ m2[e].T for e in range(E)])
    y.copy_(ye.detach())
    ops.combine_rows_device(y.data_ptr(), ops.F32, rows, inv.data_ptr(), w.data_ptr(), T, n, D, out.data_ptr(), stream=st)
    dy, dw, dx, dl = f32(rows, D), f32(T, n), f32(T, D), f32(T, E)
    ops.combine_rows_grad_device(dout.data_ptr(), ops.F32, y.data_ptr(), ops.F32, rows, inv.data_ptr(), w.data_ptr(), T, n, D, dy_ptr=dy.data_ptr(), dw_ptr=dw.data_ptr(),
                                 stream=st)
    ye.backward(dy.double())
    dxs = xe.grad.float()
    ops.route_logits_grad_device(logits.data_ptr(), ops.F32, T, E, n, ids.data_ptr(), dw.data_ptr(), dl.data_ptr(), score=code, scale=1.5, stream=st)
    # dx: what came back through the router first, the experts' rows on top of it in place.
    dx.copy_(dl @ wr)
    ops.sort_rows_grad_device(dxs.data_ptr(), ops.F32, rows, inv.data_ptr(), T, n, D, dx_ptr=dx.data_ptr(), add_ptr=dx.data_ptr(), stream=st)

    X, WR, W1, W2 = (t.double().requires_grad_() for t in (x, wr, w1, w2))
    L = X @ WR.T
    s = torch.softmax(L, 1) if score == "softmax" else torch.sigmoid(L)
    g = s.gather(1, ids.long())
    g = g / g.sum(1, keepdim=True) * 1.5
    per = torch.einsum("edf,tef->ted", W2, torch.tanh(torch.einsum("efd,td->tef", W1, X)))
    want = (g.unsqueeze(2) * per.gather(1, ids.long().unsqueeze(2).expand(-1, -1, D))).sum(1)
    want.backward(dout.double())

    def close(a, b, rel):
        assert torch.linalg.vector_norm(a.double() - b) <= rel * torch.linalg.vector_norm(b)

    # Logits, rows, weights and sums are rounded to f32 a few times each, 2^-24 at a time; weights come within 2^-18.
    close(out, want.detach(), 2.0 ** -17)
    close(dx, X.grad, 2.0 ** -15)  # dl @ wr by torch in f32 among them
    close(dl.double().T @ x.double(), WR.grad, 2.0 ** -16)
    close(m1.grad, W1.grad, 2.0 ** -16)
    close(m2.grad, W2.grad, 2.0 ** -16)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
def test_odd_weights_gradients_reach_no_vanished_share(score, renorm):
    """Infinities and NaN in the weights' gradients of experts whose factor is 0 in f32 reach nothing; in the others what the formulas make of them."""
    import torch

    T, E, n = 6, 40, 3
    l = np.full((T, E), -300.0, np.float32)
    ids = np.tile(np.array([3, 17, 8], np.int32), (T, 1))
    l[:, 3] = [0.5, 0.5, 200, 200, -150, 0.5]    # by sigmoids 200 is 1 - s of 0
    l[:, 17] = [-200, 0.25, 0, 200, -152, 0.25]  # by softmax 200 apart is a share of 0
    l[:, 8] = [-200, 0, -200, 200, -400, -200]
    odd = np.array([[1, np.inf, np.nan], [1, np.inf, 2], [np.nan, 1, -np.inf], [np.inf, 1, 2], [1, 2, np.nan], [-1, 3, np.nan]], np.float32)
    dl, di, dd, out = dev(l), dev(ids), dev(odd), torch.full((T, E), 7.0, device="cuda")
    ops.route_logits_grad_device(dl.data_ptr(), ops.F32, T, E, n, di.data_ptr(), dd.data_ptr(), out.data_ptr(), score=TYPES_OF_SCORE[score], renorm=renorm)
    l64, d64, want = l.astype(np.float64), odd.astype(np.float64), np.zeros((T, E))
    small = 2.0 ** -150  # half of f32's least number: all factors here are far above it or below

    def share(p):
        return np.where(p < small, 0.0, p)

    for t in range(T):
        lc, factor, p = l64[t, ids[t]], np.ones(n), None
        if score == "softmax":
            of = lc if renorm else l64[t]
            p = share(np.exp(of - of.max()) / np.exp(of - of.max()).sum())
        else:
            factor = share(np.exp(-np.logaddexp(0, lc)))
            s = -np.logaddexp(0, -lc)
            p = share(np.exp(s - s.max()) / np.exp(s - s.max()).sum()) if renorm else share(np.exp(s))
        dense = score == "softmax" and not renorm
        d = np.zeros(E) if dense else d64[t]
        if dense:
            d[ids[t]] = d64[t]
        with np.errstate(invalid="ignore"):
            mean = np.where(p > 0, p * d, 0.0)[p > 0].sum() if score == "softmax" or renorm else 0.0
            v = np.where(p > 0, p, 0.0) * (factor if not dense else 1.0)
            v = np.where(v > 0, v * (d - mean), 0.0)
        want[t, slice(None) if dense else ids[t]] = v
    got = host(out)
    assert np.array_equal(np.isnan(got), np.isnan(want)), (got[:, [3, 17, 8]], want[:, [3, 17, 8]])
    assert np.allclose(got, want, rtol=2.0 ** -18, atol=2.0 ** -20, equal_nan=True)


def test_weights_gradients_as_large_as_f32_holds():
    """A softmax as it is: shares times gradients whose sum f32 does not hold before it is divided by the row's sum of exponentials."""
    import torch

    E = 64
    l, ids, dw = torch.zeros((2, E), device="cuda"), dev(np.array([[1, 2, 40], [0, 3, 63]], np.int32)), torch.full((2, 3), 3e38, device="cuda")
    dw[1, 1] = 1e38
    out = torch.empty((2, E), device="cuda")
    ops.route_logits_grad_device(l.data_ptr(), ops.F32, 2, E, 3, ids.data_ptr(), dw.data_ptr(), out.data_ptr(), renorm=False)
    want, _ = M.route_grad(host(l), ids.cpu().numpy(), dw.double().cpu().numpy(), "softmax", False, 1.0)
    assert np.allclose(host(out), want, rtol=2.0 ** -18, atol=0)


@pytest.mark.parametrize("shift", [0.0, 1000.0, -1000.0, 3e6])
def test_small_shares_by_one_rounding_of_their_exponents(shift):
    """Softmax weights as they are, f32, a chosen expert so far above the others that the row's sum is its exponential alone, and dw 1: a gradient is the share itself, off by
    its exponent's one rounding (in units of log 2, so half a step of numbers from 64 on), by log2(e)'s own to f32, 1.34e-8 of it, by two approximate exponentials of 2^-22, a
    quotient and a product. Of rows whose logits are all beyond 2^20 the difference itself is rounded first: half a step more."""
    import torch

    rng = np.random.default_rng(21)
    T, E = 128, 512
    l = (rng.uniform(-63, -46, (T, E)) + shift).astype(np.float32)
    top = rng.integers(0, E, T)
    l[np.arange(T), top] = (rng.uniform(0, 1, T) + shift).astype(np.float32)
    dl, di, dd, out = dev(l), dev(top.astype(np.int32)[:, None]), torch.ones((T, 1), device="cuda"), torch.empty((T, E), device="cuda")
    ops.route_logits_grad_device(dl.data_ptr(), ops.F32, T, E, 1, di.data_ptr(), dd.data_ptr(), out.data_ptr(), renorm=False)
    want, _ = M.route_grad(l.astype(np.float64), top[:, None], np.ones((T, 1)), "softmax", False, 1.0)
    rest = np.ones((T, E), bool)
    rest[np.arange(T), top] = False
    d = (l[np.arange(T), top].astype(np.float64)[:, None] - l)[rest]
    arg = d * np.log2(np.e)
    assert arg.min() > 65 and arg.max() < 127  # a step is 2^-17
    bound = np.log(2) * 2.0 ** -18 + 1.34e-8 * d + 2 * 2.0 ** -22 + 4 * U + (2.0 ** -19 if shift > 2 ** 20 else 0.0)
    off = np.abs(host(out)[rest] / want[rest] - 1)
    assert (off <= bound).all(), (off / bound).max()

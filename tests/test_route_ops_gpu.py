"""On a B200: moe_route_logits_device against the definition in 64 bits, row by row. Expert ids, offsets and places are compared
bit for bit, weights within what their arithmetic can be off by."""
import ctypes as C

import numpy as np
import pytest

import ops_common as R
from c0ven_b200 import MoEError, _lib, ops

pytestmark = pytest.mark.gpu

# The weights' arithmetic in f32: an exponential (2 ulp; the difference under it rounds by 2^-24 of itself, |l| and |d| at most some 20
# here: 20 steps), at most 16 sums, two divisions and the scale: under 64 half steps of 2^-24.
W_RTOL = 64 * 2.0 ** -24


def torch_rows(l, type):
    import torch

    t = torch.from_numpy(l.astype(np.float32)).to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[type])
    return t.cuda(), t.double().numpy()


def run(l_dev, T, E, k, type="f32", bias=None, lists=True, stride=0, stream=None, **kw):
    """ids, w, offsets, inv of a call; buffers are filled with what it must overwrite."""
    import torch

    ids, w = torch.full((T, k), -77, dtype=torch.int32, device="cuda"), torch.full((T, k), float("nan"), device="cuda")
    offsets, inv = torch.full((E + 1,), -77, dtype=torch.int32, device="cuda"), torch.full((T, k), -77, dtype=torch.int32, device="cuda")
    n = ops.route_work_bytes(T, E)
    work = torch.full((n + 64,), 0xAB, dtype=torch.uint8, device="cuda")
    b = None if bias is None else torch.from_numpy(bias).cuda()
    torch.cuda.synchronize()
    ops.route_logits_device(l_dev.data_ptr(), {"f32": ops.F32, "f16": ops.F16, "bf16": ops.BF16}[type], T, E, k, ids.data_ptr(), w.data_ptr(),
                            bias_ptr=None if b is None else b.data_ptr(), stride=stride, offsets_ptr=offsets.data_ptr() if lists else None,
                            inv_ptr=inv.data_ptr() if lists else None, work_ptr=work.data_ptr() if lists else None, work_bytes=n if lists else 0,
                            stream=stream, **kw)
    torch.cuda.synchronize()
    assert (work[n:] == 0xAB).all()
    return tuple(a.cpu().numpy() for a in (ids, w, offsets, inv))


def check(l, k, type="f32", bias=None, **kw):
    T, E = l.shape
    dev, exact = torch_rows(l, type)
    got = run(dev, T, E, k, type, bias, score=ops.SIGMOID if kw.get("score") == "sigmoid" else ops.SOFTMAX, **{a: v for a, v in kw.items() if a != "score"})
    want = R.route(exact, k, bias=bias, **kw)
    assert np.array_equal(got[0], want[0])
    assert np.allclose(got[1], want[1], rtol=W_RTOL, atol=1e-37, equal_nan=True)
    assert np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3])
    return got


@pytest.mark.parametrize("E, k", [(1, 1), (7, 3), (32, 16), (33, 4), (64, 6), (100, 16), (129, 2), (256, 8), (384, 9), (512, 10)])
@pytest.mark.parametrize("score, with_bias, renorm", [("softmax", False, True), ("softmax", True, False), ("sigmoid", False, False), ("sigmoid", True, True)])
def test_every_size(E, k, score, with_bias, renorm):
    rng = np.random.default_rng(E)
    for T in (1, 3, 37, 64, 65, 150):
        bias = (rng.standard_normal(E) * (0.1 if score == "sigmoid" else 0.5 / E)).astype(np.float32) if with_bias else None
        check(rng.standard_normal((T, E)) * 2, k, score=score, bias=bias, renorm=renorm, scale=2.5)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("E, G, used, k", [(256, 8, 4, 8), (16, 16, 5, 5), (96, 3, 1, 16), (64, 32, 3, 6), (500, 20, 7, 10), (512, 2, 1, 12)])
def test_groups(type, E, G, used, k):
    rng = np.random.default_rng(E + G)
    for T in (2, 70):
        for score, bias in (("sigmoid", (0.1 * rng.standard_normal(E)).astype(np.float32)), ("softmax", None), ("sigmoid", None), ("softmax", (rng.standard_normal(E) / E).astype(np.float32))):
            check(rng.standard_normal((T, E)), k, type, score=score, bias=bias, n_groups=G, n_groups_used=used)


def test_ties_go_to_the_lower_expert_and_zeros_have_no_sign():
    rng = np.random.default_rng(5)
    l = rng.integers(-2, 3, (90, 128)).astype(np.float64)
    l[rng.random(l.shape) < 0.1] = -0.0
    for kw in (dict(), dict(score="sigmoid", bias=np.zeros(128, np.float32)), dict(score="sigmoid", n_groups=8, n_groups_used=3),
               dict(bias=rng.integers(-1, 2, 128).astype(np.float32) / 128), dict(score="softmax", n_groups=4, n_groups_used=2, bias=np.full(128, 0.25, np.float32))):
        check(l, 9, **kw)
        check(np.zeros((3, 128)), 9, **kw)


def test_order_of_scores_that_vanish_or_come_to_one():
    """Without a bias the logits' order decides, where 64-bit scores are equal and ties leave many keys too."""
    E = 512
    for some in (31, 64, 200, 512):
        for k in (1, 8, 16):
            low = np.full((70, some), -2000.0)
            low[:, 0] = 0
            low[:, some - 6:some - 1] = -1000
            check(low, min(k, some), score="softmax")
            high = np.full((70, some), 50.0)
            high[:, some - 6:some - 1] = 60
            check(high, min(k, some), score="sigmoid")
    groups = np.full((70, E), 50.0)
    groups[:, 100:104] = 60
    check(groups, 10, score="sigmoid", n_groups=8, n_groups_used=3)


def test_keys_that_f32_cannot_tell_apart():
    """Scores next to one another, saturated ones and large biases: the order is the exact keys'."""
    rng = np.random.default_rng(6)
    T, E = 80, 96
    base = np.float32(1.25)
    l = base + rng.integers(0, 40, (T, E)) * np.spacing(base)     # neighbours in f32
    bias = (rng.integers(0, 3, E) * 2.0 ** -24).astype(np.float32)
    check(l, 12, score="sigmoid", bias=bias)
    check(l, 12, score="softmax", bias=bias)
    check(l, 12, score="sigmoid", bias=bias, n_groups=8, n_groups_used=3)
    check(l, 12, score="softmax", n_groups=8, n_groups_used=3)
    sat = rng.uniform(14, 30, (T, E))                              # sigmoids of 1 to f32
    check(sat, 12, score="sigmoid", bias=np.zeros(E, np.float32))
    check(sat, 12, score="sigmoid", bias=(rng.integers(-3, 4, E) * 1024.0).astype(np.float32), n_groups=6, n_groups_used=2)
    check(rng.uniform(-80, -20, (T, E)), 12, score="sigmoid", bias=(rng.standard_normal(E) * 1e-12).astype(np.float32))
    check(rng.standard_normal((T, E)) * 30, 12, score="softmax", bias=(rng.standard_normal(E) * 1e-9).astype(np.float32))


def test_masked_and_unusual_logits():
    """Experts out by -infinity or NaN, rows with too few or none left, the type's lowest and infinite values."""
    rng = np.random.default_rng(7)
    T, E, k = 100, 64, 8
    l = rng.standard_normal((T, E))
    l[rng.random((T, E)) < 0.5] = -np.inf
    l[rng.random((T, E)) < 0.1] = np.nan
    l[0] = -np.inf
    l[1] = np.nan
    l[2] = -np.inf
    l[2, 40] = 0.5
    l[3] = np.finfo(np.float32).min
    l[4] = np.finfo(np.float32).max
    l[5, 3] = l[5, 60] = np.inf
    l[6] = np.inf
    bias = (0.1 * rng.standard_normal(E)).astype(np.float32)
    bias[7], bias[9] = -np.inf, np.nan
    bias[11] = 1e30
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            got = check(l, k, score=score, renorm=renorm)
            assert (got[0][:2] == -1).all() and (got[1][:2] == 0).all() and (got[3][:2] == -1).all()
            check(l, k, score=score, renorm=renorm, bias=bias)
            check(l, k, score=score, renorm=renorm, n_groups=8, n_groups_used=2)
            check(l, k, score=score, renorm=renorm, bias=bias, n_groups=16, n_groups_used=3)
    lowest = np.full((2, E), float(np.finfo(np.float16).min))
    lowest[1, 5] = 0
    check(lowest, k, "f16", score="sigmoid")
    # Scores that vanish keep their proportions.
    check(rng.uniform(-200, -100, (5, E)), k, score="sigmoid", renorm=True)
    far = rng.uniform(-200, -150, (5, E))
    far[:, 0] = 10
    check(far, 4, score="softmax", bias=np.where(np.arange(E) == 0, -5, 0).astype(np.float32), renorm=True)


@pytest.mark.parametrize("type", ["f32", "f16", "bf16"])
def test_rows_apart_and_from_any_value(type):
    """Rows with a stride, starting anywhere the type allows, without lists."""
    import torch

    rng = np.random.default_rng(8)
    for T, E, stride, first in ((5, 60, 77, 3), (90, 130, 131, 1)):
        dev, exact = torch_rows(rng.standard_normal((1, first + T * stride)), type)
        view = torch.as_strided(dev, (T, E), (stride, 1), first)
        ids, w, offsets, inv = run(view, T, E, 5, type, lists=False, stride=stride)
        want = R.route(np.lib.stride_tricks.as_strided(exact[0, first:], (T, E), (stride * 8, 8)), 5)
        assert np.array_equal(ids, want[0]) and np.allclose(w, want[1], rtol=W_RTOL)
        assert (offsets == -77).all() and (inv == -77).all()


def test_no_rows_and_many():
    import torch

    offsets, inv = torch.full((65,), 9, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.route_logits_device(None, ops.F32, 0, 64, 4, None, None, offsets_ptr=offsets.data_ptr(), inv_ptr=inv.data_ptr())
    torch.cuda.synchronize()
    assert (offsets == 0).all()
    # Long steps: ids against a vectorised form (the sort's order), lists by their definition.
    for T, E, k in ((5000, 512, 10), (40001, 40, 16)):
        g = torch.Generator(device="cuda").manual_seed(T)
        l = torch.randn((T, E), generator=g, device="cuda")
        b = 0.1 * torch.randn(E, generator=g, device="cuda")
        ids, w, offs, inv = run(l, T, E, k, bias=b.cpu().numpy(), score=ops.SIGMOID)
        key = torch.sigmoid(l.double()) + b.double()
        want = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :k].cpu().numpy()
        assert np.array_equal(ids, want)
        s = torch.sigmoid(l.double()).gather(1, torch.from_numpy(want).cuda())
        assert np.allclose(w, (s / s.sum(1, keepdim=True)).cpu().numpy(), rtol=W_RTOL, atol=0)
        order = np.argsort(ids.reshape(-1), kind="stable")
        place = np.empty(T * k, np.int64)
        place[order] = np.arange(T * k)
        assert np.array_equal(inv.reshape(-1), place)
        assert np.array_equal(offs, np.concatenate([[0], np.cumsum(np.bincount(ids.reshape(-1), minlength=E))]))


def test_streams_and_captured_graphs():
    """On a stream of the caller's, and twice from one captured graph with other logits; two graphs that share the work buffer, one after the other."""
    import torch

    rng = np.random.default_rng(9)
    T, E, k = 200, 128, 6
    l, first = torch_rows(rng.standard_normal((T, E)), "f32")
    st = torch.cuda.Stream()
    got = run(l, T, E, k, stream=st.cuda_stream)
    assert all(np.array_equal(a, b) for a, b in zip((got[0], got[2], got[3]), np.array(R.route(first, k), object)[[0, 2, 3]]))
    work = torch.empty(ops.route_work_bytes(T, E), dtype=torch.uint8, device="cuda")
    graphs = []
    for _ in range(2):
        out = [torch.empty(s, dtype=d, device="cuda") for s, d in (((T, k), torch.int32), ((T, k), torch.float32), ((E + 1,), torch.int32), ((T, k), torch.int32))]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.route_logits_device(l.data_ptr(), ops.F32, T, E, k, out[0].data_ptr(), out[1].data_ptr(), offsets_ptr=out[2].data_ptr(),
                                    inv_ptr=out[3].data_ptr(), work_ptr=work.data_ptr(), work_bytes=work.numel(), stream=torch.cuda.current_stream().cuda_stream)
        graphs.append((graph, out))
    for seed in (1, 2):
        new, exact = torch_rows(np.random.default_rng(seed).standard_normal((T, E)), "f32")
        l.copy_(new)
        want = R.route(exact, k)
        for graph, out in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(np.array_equal(out[i].cpu().numpy(), want[i]) for i in (0, 2, 3))


def test_memory_that_is_not_the_devices_is_refused():
    import torch

    host = torch.zeros(4096)
    pinned = torch.zeros(4096).pin_memory()
    dev = torch.zeros(4096, device="cuda")
    for bad in (host, pinned):
        with pytest.raises(MoEError) as e:
            ops.route_logits_device(bad.data_ptr(), ops.F32, 4, 64, 4, dev.data_ptr(), dev.data_ptr())
        assert e.value.status == _lib.MOE_BAD_ARGUMENT and "logits is not device memory" in str(e.value)
    with pytest.raises(MoEError) as e:
        ops.route_logits_device(dev.data_ptr() + 2, ops.F32, 4, 64, 4, dev.data_ptr(), dev.data_ptr())
    assert "aligned" in str(e.value)
    with pytest.raises(MoEError) as e:
        ops.route_logits_device(dev.data_ptr(), ops.F32, 4, 64, 4, dev.data_ptr(), None)
    assert "w is required" in str(e.value)
    if torch.cuda.device_count() > 1:
        other = torch.zeros(4096, device="cuda:1")
        with pytest.raises(MoEError) as e:
            ops.route_logits_device(other.data_ptr(), ops.F32, 4, 64, 4, dev.data_ptr(), dev.data_ptr())
        assert "another device" in str(e.value)


def test_the_layers_own_router_agrees():
    """softmax without bias or groups is what moe_route_rows_static and the layer compute from the same logits."""
    import torch

    from c0ven_b200 import MoELayer, synth

    layer = synth.make_layer(n_embd=512, n_ff=256, n_experts=64, n_used=6, gate_type=synth.Q8_0, seed=3)
    gpu = MoELayer(layer, max_tokens=64)
    x = synth.make_input(40, 512, seed=4)
    gpu.forward(x)
    ids, w, inv, _ = gpu.route(40)
    logits, approximate, _, _ = gpu.logits(40)
    assert not approximate
    got = run(torch.from_numpy(logits).cuda(), 40, 64, 6)
    assert np.array_equal(got[0], ids) and np.array_equal(got[3].reshape(-1), inv)
    assert np.allclose(got[1], w, rtol=1e-5)
    gpu.close()
    assert C.sizeof(_lib.RouteConfig) == 32


def test_groups_whose_keys_sums_pass_f32():
    """Biases of the type's lowest value are no experts out: groups of them, whose sums f32 has no room for, stay as 64-bit sums order them."""
    rng = np.random.default_rng(10)
    E, G = 64, 8
    lowest = np.finfo(np.float32).min
    masked = np.full(E, lowest)
    masked[40:48] = 0.1 * rng.standard_normal(8)              # group 5 alone is not masked: the next to stay is group 0
    apart = masked.copy()
    apart[24:32] = lowest / 1.5                               # the sums of group 3's keys pass the lowest value too, but less far
    one = np.full(E, lowest)
    one[np.arange(E) % 8 == 3] = 0.0                          # a key a group that is not masked: no sum passes
    high = np.full(E, np.finfo(np.float32).max)
    high[:8] /= 4                                             # sums past the largest value, and group 0's below it
    for T in (3, 70):
        l = rng.standard_normal((T, E))
        for bias in (masked, apart, one, high):
            for used, k in ((2, 12), (3, 16), (8, 16)):
                for score in ("sigmoid", "softmax"):
                    got = check(l, k, score=score, bias=bias.astype(np.float32), n_groups=G, n_groups_used=used)
                    assert (got[0] >= 0).all()


def test_softmax_weights_over_the_whole_row():
    """Weights without renormalisation are divided by all experts' exponentials: many logits that lie alike, some 2 to 8 below the largest, whose
    errors would add up."""
    import torch

    rng = np.random.default_rng(11)
    T, E = 4096, 512
    top = rng.uniform(-4, 4, T).astype(np.float32)
    l = np.repeat((top - rng.uniform(2, 8, T).astype(np.float32))[:, None], E, 1)
    l[np.arange(T), rng.integers(0, E, T)] = top
    ids, w, _, _ = run(torch.from_numpy(l).cuda(), T, E, 2, lists=False, renorm=False)
    x = np.sort(l, 1)[:, ::-1].astype(np.float64)
    p = np.exp(x - x[:, :1])
    # Half steps of 2^-24: an exponential 4 (2 ulp) and 1 for what its argument's rounding left out; the sum is of 64 bits and rounded once, its reciprocal
    # and the product once each. The exponentials' errors are in the sum and in the weight alike, so that they count once at most.
    assert np.allclose(w, (p / p.sum(1, keepdims=True))[:, :2], rtol=8 * 2.0 ** -24, atol=0)
    assert np.array_equal(ids[:, 0], l.argmax(1))


@pytest.mark.parametrize("E, G, used, k", [(256, 8, 4, 8), (64, 32, 3, 6), (500, 20, 7, 10)])
def test_groups_in_long_steps(E, G, used, k):
    rng = np.random.default_rng(E)
    for T, score, with_bias in ((1500, "sigmoid", True), (901, "softmax", False)):
        check(rng.standard_normal((T, E)), k, score=score, bias=(0.1 * rng.standard_normal(E)).astype(np.float32) if with_bias else None, n_groups=G, n_groups_used=used)

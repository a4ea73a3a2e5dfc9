"""What the operators beside the MoE layer are measured on: routing of a step's logits, rows in microscaled 4-bit floating point
(MX: e2m1 codes, an e8m0 scale every 32 values), the experts' products over them, and the combine.

A case names its operator in "op":

- "route": expert ids, weights, expert offsets and each assignment's place in expert order, from a step's router logits;
- "quant": rows to MX, as they lie or scattered to expert order, and what the codes stand for;
- "product": MX rows times one matrix or the experts' matrices, each row with its own expert's;
- "ffn": gate and up with SwiGLU, its result as MX rows, then the down product;
- "combine": the weighted sum of each row's expert results.

With `own` false every operator is computed in its plain form, by elementary torch operations; with `own` true by the
framework's calls. All inputs come from the seed.
"""
import math

import numpy as np
import torch

own = False

F32, F16, BF16 = 0, 1, 30  # ggml's type numbers, as the framework's calls take them
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": F32, "f16": F16, "bf16": BF16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


# --- the cases -----------------------------------------------------------------------------------------------------

def _route(name, T, E, k, score, type, bias, groups, used, renorm, scale):
    return dict(name=name, op="route", T=T, E=E, k=k, score=score, type=type, bias=bias, groups=groups, used=used, renorm=renorm, scale=scale)


def _quant(name, T, K, k, type, out):
    return dict(name=name, op="quant", T=T, K=K, k=k, type=type, out=out)


def _product(name, E, T, k, N, K, y, zipf):
    return dict(name=name, op="product", E=E, T=T, k=k, N=N, K=K, y=y, zipf=zipf)


def _ffn(name, E, T, k, D, F, y, zipf, limit):
    return dict(name=name, op="ffn", E=E, T=T, k=k, D=D, F=F, y=y, zipf=zipf, limit=limit)


def _combine(name, T, k, D, y, residual):
    return dict(name=name, op="combine", T=T, k=k, D=D, y=y, residual=residual)


def listed():
    return [
        # One token's routing over the benchmark layer's 512 experts: the decode step, all latency.
        _route("route_1x512_softmax", 1, 512, 10, "softmax", "f32", False, 1, 1, True, 1.0),
        # A decode batch of odd size under a router with sigmoid scores, a balance bias and expert groups, bf16 logits.
        _route("route_37x256_sigmoid_groups", 37, 256, 8, "sigmoid", "bf16", True, 8, 4, True, 2.5),
        # The benchmark's long prompt, routed by sigmoid scores with a balance bias.
        _route("route_32768x512_sigmoid", 32768, 512, 10, "sigmoid", "f32", True, 1, 1, True, 1.0),
        # A few decode rows quantised straight into expert order.
        _quant("quant_13x2560_scatter8", 13, 2560, 8, "f32", "f32"),
        # The benchmark's long prompt as a model holds it between layers, in bf16, for a dense product.
        _quant("quant_32768x2048_bf16", 32768, 2048, 1, "bf16", "bf16"),
        # One dense matrix (a shared expert's down) on a ragged batch of rows, sizes that fill no tile.
        _product("product_dense_777x2080x1440", 1, 777, 1, 2080, 1440, "f16", 0.0),
        # Experts' down product of a packed ragged batch with skewed routing.
        _product("product_64x3521_zipf", 64, 3521, 4, 1024, 512, "bf16", 1.1),
        # One token through ten of 512 experts: weights read once, all latency.
        _ffn("ffn_512x1", 512, 1, 10, 2048, 512, "f16", 0.0, 0.0),
        # A decode batch: one or two rows an expert, weights of every expert read once.
        _ffn("ffn_512x100", 512, 100, 10, 2048, 512, "f16", 0.0, 0.0),
        # A long prompt through wide experts, skewed, with a SwiGLU limit: tensor-core work.
        _ffn("ffn_128x8192_zipf", 128, 8192, 8, 2560, 768, "bf16", 0.6, 7.0),
        # One token's results summed onto its residual row.
        _combine("combine_1x2560", 1, 8, 2560, "f16", True),
        # The benchmark's long prompt's results summed.
        _combine("combine_32768x2048", 32768, 10, 2048, "bf16", False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["route", "quant", "product", "ffn", "combine"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8, 16])
        E = groups * _log(rng, max(2, 8 // groups), 512 // groups)
        k = rng.randint(1, min(16, E))
        used = min(groups, max(-(-k * groups // E), rng.randint(1, groups)))
        bias = rng.random() < 0.6
        return dict(op=op, T=_log(rng, 1, 32768), E=E, k=k, score=rng.choice(["softmax", "sigmoid"]), type=rng.choice(["f32", "f16", "bf16"]), bias=bias,
                    groups=groups, used=used, renorm=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]))
    if op == "quant":
        K, k = 32 * _log(rng, 2, 256), rng.choice([1, 1, rng.randint(2, 10)])
        return dict(op=op, T=_log(rng, 1, max(2, 32768 * 2048 // (K * k))), K=K, k=k, type=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f32", "bf16"]))
    if op == "product":
        E = rng.choice([1, _log(rng, 2, 128)])
        k = 1 if E == 1 else rng.randint(1, min(8, E))
        N, K = 32 * _log(rng, 2, 96), 32 * _log(rng, 2, 96)
        return dict(op=op, E=E, T=_log(rng, 1, 4096), k=k, N=N, K=K, y=rng.choice(["f16", "bf16"]), zipf=rng.choice([0.0, 1.1]))
    if op == "ffn":
        E = _log(rng, 2, 128)
        return dict(op=op, E=E, T=_log(rng, 1, 4096), k=rng.randint(1, min(8, E)), D=32 * _log(rng, 4, 80), F=32 * _log(rng, 2, 24), y=rng.choice(["f16", "bf16"]),
                    zipf=rng.choice([0.0, 1.1]), limit=rng.choice([0.0, 7.0]))
    k, D = rng.randint(1, 16), 32 * _log(rng, 2, 128)
    return dict(op=op, T=_log(rng, 1, max(2, 32768 * 2048 * 10 // (k * D))), k=k, D=D, y=rng.choice(["f16", "bf16"]), residual=rng.random() < 0.5)


def work(case):
    c = case
    if c["op"] == "route":
        return dict(bytes=c["T"] * c["E"] * SIZE[c["type"]] + c["T"] * c["k"] * 12 + 4 * (c["E"] + 1), flops=4 * c["T"] * c["E"])
    if c["op"] == "quant":  # rows in, codes and scales out; then those in and their values out
        n = c["T"] * c["K"]
        return dict(bytes=n * SIZE[c["type"]] + 2 * c["k"] * n * 17 / 32 + c["k"] * n * SIZE[c["out"]], flops=4 * n * c["k"])
    if c["op"] == "combine":
        n = c["T"] * c["D"]
        return dict(bytes=c["k"] * n * SIZE[c["y"]] + 4 * n * (2 if c["residual"] else 1) + 8 * c["T"] * c["k"], flops=2 * c["k"] * n)
    # Experts that no row went to are not read.
    R, hit = c["T"] * c["k"], int((_counts(c, 0) > 0).sum())
    if c["op"] == "product":
        return dict(bytes=(hit * c["N"] + R) * c["K"] * 17 / 32 + R * c["N"] * SIZE[c["y"]], flops=2 * R * c["N"] * c["K"])
    D, F = c["D"], c["F"]
    return dict(bytes=hit * 3 * F * D * 17 / 32 + R * (D + 2 * F) * 17 / 32 + R * D * SIZE[c["y"]], flops=6 * R * F * D)


# --- inputs --------------------------------------------------------------------------------------------------------

def _counts(c, seed):
    """Rows each expert gets: every token's k distinct experts, drawn evenly or by a Zipf law."""
    return np.bincount(_ids(c, seed).reshape(-1), minlength=c["E"])


def _ids(c, seed):
    rng = np.random.default_rng(seed)
    p = -c["zipf"] * np.log(1.0 + rng.permutation(c["E"]))
    g = p + rng.gumbel(size=(c["T"], c["E"]))  # the k largest: k draws without replacement
    return np.argsort(-g, axis=1)[:, :c["k"]]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _weights(g, E, N, K):
    """Matrices in MX: codes uniform, scales over three powers of two, sized so that a row's products are of the order of one."""
    e0 = 127 - round(math.log2(3.0 * math.sqrt(K)))
    return (torch.randint(0, 256, (E, N, K // 2), generator=g, device="cuda", dtype=torch.uint8),
            torch.randint(e0 - 1, e0 + 2, (E, N, _stride(K)), generator=g, device="cuda", dtype=torch.uint8))


def _stride(K):
    return (K // 32 + 3) // 4 * 4  # bytes of a row's scales: whole words


def prepare(case, seed):
    c, g, s = case, _gen(seed), {}
    s["case"] = c
    if c["op"] == "route":
        T, E, k = c["T"], c["E"], c["k"]
        s["logits"] = _randn(g, (T, E), TORCH[c["type"]])
        s["bias"] = (0.1 if c["score"] == "sigmoid" else 0.5 / E) * _randn(g, (E,)) if c["bias"] else None
        s["ids"], s["w"] = torch.empty((T, k), dtype=torch.int32, device="cuda"), torch.empty((T, k), device="cuda")
        s["offsets"], s["inv"] = torch.empty(E + 1, dtype=torch.int32, device="cuda"), torch.empty((T, k), dtype=torch.int32, device="cuda")
        s["work"] = torch.empty(4 * E * (-(-T // 32) + 1), dtype=torch.uint8, device="cuda")
        return s
    if c["op"] == "quant":
        T, K, k = c["T"], c["K"], c["k"]
        s["x"] = _randn(g, (T, K), TORCH[c["type"]])
        s["inv"] = torch.randperm(T * k, generator=g, device="cuda").to(torch.int32).reshape(T, k) if k > 1 else None
        s["codes"], s["scales"] = _mx_rows(T * k, K)
        s["out"] = torch.empty((T * k, K), dtype=TORCH[c["out"]], device="cuda")
        return s
    T, k = c["T"], c["k"]
    R = T * k
    if c["op"] == "combine":
        s["y"] = _randn(g, (R, c["D"]), TORCH[c["y"]])
        s["inv"] = torch.randperm(R, generator=g, device="cuda").to(torch.int32).reshape(T, k)
        w = torch.rand((T, k), generator=g, device="cuda")
        s["w"] = w / w.sum(1, keepdim=True)
        s["residual"] = _randn(g, (T, c["D"])) if c["residual"] else None
        s["out"] = torch.empty((T, c["D"]), device="cuda")
        return s
    n = _counts(c, seed)
    s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(n)]).astype(np.int32)).cuda()
    # What the plain form's padded batch needs: the experts hit, the most rows one has, every row's place in it.
    hit = np.flatnonzero(n)
    s["hit"], s["most"] = torch.from_numpy(hit).cuda(), int(n.max())
    s["place"] = torch.from_numpy(np.concatenate([i * s["most"] + np.arange(n[e]) for i, e in enumerate(hit)])).cuda()
    D = c["K"] if c["op"] == "product" else c["D"]
    s["codes"], s["scales"] = _quantize(_randn(g, (R, D)))
    if c["op"] == "product":
        s["w"] = _weights(g, c["E"], c["N"], D)
        s["y"] = torch.empty((R, c["N"]), dtype=TORCH[c["y"]], device="cuda")
    else:
        s["w"], s["w2"] = _weights(g, c["E"], 2 * c["F"], D), _weights(g, c["E"], D, c["F"])
        s["h"] = _mx_rows(R, c["F"])
        s["y"] = torch.empty((R, D), dtype=TORCH[c["y"]], device="cuda")
    return s


def _mx_rows(R, K):
    return torch.empty((R, K // 2), dtype=torch.uint8, device="cuda"), torch.zeros((R, _stride(K)), dtype=torch.uint8, device="cuda")


# --- the plain forms -----------------------------------------------------------------------------------------------

def _pow2(n):
    """2^n exactly, in 64 bits."""
    return (n.long() + 1023 << 52).view(torch.float64)


def _quantize(x):
    """Codes two a byte (the even value's in the low half), scales with their rows filled up to whole words."""
    b = x.float().reshape(x.shape[0], -1, 32).double()
    _, e = torch.frexp(b.abs().amax(2))
    e = torch.where(b.abs().amax(2) > 0, e - 3, -127).clamp(-127, 127)
    v = b * _pow2(-e).unsqueeze(2)
    a = v.abs()
    code = ((a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5) + 8 * (v < 0)).to(torch.uint8).reshape(x.shape[0], -1)
    scales = torch.zeros((x.shape[0], _stride(x.shape[1])), dtype=torch.uint8, device=x.device)
    scales[:, :e.shape[1]] = (e + 127).to(torch.uint8)
    return code[:, 0::2] | code[:, 1::2] << 4, scales


def _values(codes, scales, dtype=torch.float32):
    """What MX rows stand for."""
    table = torch.tensor(VALUES, dtype=dtype, device=codes.device)
    v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    s = _pow2(scales[..., :v.shape[-1] // 32].long() - 127).to(dtype)
    return (v.unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)


def _by_expert(s, x, w):
    """x [R][K], sorted by expert, times each row's expert's matrix, in a batch padded to the fullest expert."""
    H, most = s["hit"].numel(), s["most"]
    b = torch.zeros((H * most, x.shape[1]), dtype=x.dtype, device=x.device)
    b[s["place"]] = x
    m = _values(w[0][s["hit"]], w[1][s["hit"]])
    return torch.bmm(b.view(H, most, -1), m.transpose(1, 2)).reshape(H * most, -1)[s["place"]]


def _swiglu(v, limit):
    g, u = v.chunk(2, 1)
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g / (1 + torch.exp(-g)) * u


def _route_plain(s):
    """In 64 bits: which experts are chosen hangs on sums of scores and biases that lie close together."""
    c, l = s["case"], s["logits"].double()
    E, k, G = c["E"], c["k"], c["groups"]
    e = torch.exp(l - l.amax(1, keepdim=True))
    score = e / e.sum(1, keepdim=True) if c["score"] == "softmax" else 1 / (1 + torch.exp(-l))
    # Without a bias the scores' order is the logits'.
    key = score + s["bias"].double() if s["bias"] is not None else l
    if G > 1:
        group = (score + (s["bias"].double() if s["bias"] is not None else 0)).view(-1, G, E // G)
        best = torch.sort(group, 2, descending=True)[0][:, :, :2].sum(2)
        stay = torch.sort(best, dim=1, descending=True, stable=True)[1][:, :c["used"]]
        kept = torch.zeros_like(best, dtype=torch.bool).scatter_(1, stay, True)
        key = torch.where(kept.repeat_interleave(E // G, 1), key, -math.inf)
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :k]
    w = score.gather(1, ids)
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True)
    order = torch.sort(ids.reshape(-1), stable=True)[1]
    inv = torch.empty_like(order)
    inv[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.zeros(E, dtype=torch.int64, device=ids.device).scatter_add_(0, ids.reshape(-1), torch.ones_like(order))
    offsets = torch.cat((counts.new_zeros(1), counts.cumsum(0)))
    return {"ids": ids.int(), "w": (w * c["scale"]).float(), "offsets": offsets.int(), "inv": inv.int().view(-1, k)}


def _plain(s):
    c = s["case"]
    if c["op"] == "route":
        return _route_plain(s)
    if c["op"] == "quant":
        codes, scales = _quantize(s["x"])
        v = _values(codes, scales)
        if s["inv"] is not None:
            rows = torch.empty((c["T"] * c["k"], c["K"]), device=v.device)
            rows[s["inv"].reshape(-1).long()] = v.repeat_interleave(c["k"], 0)
            v = rows
        return v.to(TORCH[c["out"]])
    if c["op"] == "combine":
        out = (s["y"].float()[s["inv"].long()] * s["w"].unsqueeze(2)).sum(1)
        return out + s["residual"] if s["residual"] is not None else out
    y = _by_expert(s, _values(s["codes"], s["scales"]), s["w"])
    if c["op"] == "ffn":
        y = _by_expert(s, _values(*_quantize(_swiglu(y, c["limit"]))), s["w2"])
    return y.to(TORCH[c["y"]])


# --- the framework's calls -----------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from c0ven_b200 import ops

    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    if c["op"] == "route":
        ops.route_logits_device(s["logits"].data_ptr(), GGML[c["type"]], c["T"], c["E"], c["k"], s["ids"].data_ptr(), s["w"].data_ptr(),
                                score=ops.SIGMOID if c["score"] == "sigmoid" else ops.SOFTMAX, bias_ptr=_ptr(s["bias"]), n_groups=c["groups"],
                                n_groups_used=c["used"], renorm=c["renorm"], scale=c["scale"], offsets_ptr=s["offsets"].data_ptr(),
                                inv_ptr=s["inv"].data_ptr(), work_ptr=s["work"].data_ptr(), work_bytes=s["work"].numel(), stream=st)
        return {"ids": s["ids"], "w": s["w"], "offsets": s["offsets"], "inv": s["inv"]}
    if c["op"] == "quant":
        R = c["T"] * c["k"]
        ops.mx4_quantize_rows_device(s["x"].data_ptr(), GGML[c["type"]], c["T"], c["K"], s["codes"].data_ptr(), s["scales"].data_ptr(), R,
                                     inv_ptr=_ptr(s["inv"]), n_used=c["k"], stream=st)
        ops.mx4_dequantize_rows_device(s["codes"].data_ptr(), s["scales"].data_ptr(), R, c["K"], s["out"].data_ptr(), GGML[c["out"]], stream=st)
        return s["out"]
    if c["op"] == "combine":
        ops.combine_rows_device(s["y"].data_ptr(), GGML[c["y"]], c["T"] * c["k"], s["inv"].data_ptr(), s["w"].data_ptr(), c["T"], c["k"], c["D"],
                                s["out"].data_ptr(), residual_ptr=_ptr(s["residual"]), stream=st)
        return s["out"]
    R, at = c["T"] * c["k"], s["offsets"].data_ptr()
    if c["op"] == "product":
        w = ops.Mx4Weights(c["E"], c["N"], c["K"], s["w"][0].data_ptr(), s["w"][1].data_ptr())
        ops.mx4_product_device(w, s["codes"].data_ptr(), s["scales"].data_ptr(), R, at, s["y"].data_ptr(), GGML[c["y"]], stream=st)
        return s["y"]
    w, w2 = (ops.Mx4Weights(c["E"], n, k, m[0].data_ptr(), m[1].data_ptr()) for n, k, m in ((2 * c["F"], c["D"], s["w"]), (c["D"], c["F"], s["w2"])))
    hc, hs = s["h"][0].data_ptr(), s["h"][1].data_ptr()
    ops.mx4_gate_up_device(w, s["codes"].data_ptr(), s["scales"].data_ptr(), R, at, hc, hs, swiglu_limit=c["limit"], stream=st)
    ops.mx4_product_device(w2, hc, hs, R, at, s["y"].data_ptr(), GGML[c["y"]], stream=st)
    return s["y"]


def run(state):
    return _own(state) if own else _plain(state)


# --- the definition in 64 bits, apart from the plain forms ------------------------------------------------------------

def _mx64(x):
    """What the MX form of rows x (64 bits) stands for: each value to the nearest of the sixteen, ties to the one with an even code."""
    b = x.reshape(x.shape[0], -1, 32)
    top = b.abs().amax(2, keepdim=True)
    s = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)))) - 2, -127, 127))
    s = torch.where(s * 4 > top, s / 2, torch.where(s * 8 <= top, s * 2, s))  # should the logarithm have rounded over a power of two
    a = (b / s).abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)).double()
    return (torch.sign(b) * torch.clamp(torch.round(a / step) * step, max=6.0) * s).reshape(x.shape)


def _rows64(codes, scales):
    v = torch.empty((codes.shape[0], codes.shape[1] * 2), dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        n = (codes >> 4 * half & 15).long()
        m, e = n & 1, n >> 1 & 3
        v[:, half::2] = torch.where(e == 0, m * 0.5, (1 + m * 0.5) * torch.pow(2.0, (e - 1).double())) * (1 - 2 * (n >> 3))
    return v * torch.pow(2.0, scales[:, :v.shape[1] // 32].double() - 127).repeat_interleave(32, 1)


def _ffn64(x, w, n):
    out, at = [], 0
    for e in np.flatnonzero(n):
        out.append(x[at:at + n[e]] @ _rows64(w[0][e], w[1][e]).T)
        at += n[e]
    return torch.cat(out)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "route":
        l = s["logits"].double()
        lse = torch.logsumexp(l, 1, keepdim=True)
        score = torch.exp(l - lse) if c["score"] == "softmax" else torch.special.expit(l)
        key = score + (s["bias"].double() if s["bias"] is not None else 0)
        if c["groups"] > 1:
            per = key.reshape(c["T"], c["groups"], -1)
            rank = torch.topk(per, min(2, per.shape[2]), 2)[0].sum(2)
            out = torch.sort(rank, dim=1, descending=True, stable=True)[1][:, c["used"]:]
            key = per.scatter(1, out.unsqueeze(2).expand(-1, -1, per.shape[2]), -math.inf).reshape(c["T"], -1)
        at = torch.topk(key, c["k"], 1)[1]
        w = score.gather(1, at)
        w = torch.exp(torch.log(w) - torch.log(w.sum(1, keepdim=True))) if c["renorm"] else w
        return {"ids": None, "w": w * c["scale"], "offsets": None, "inv": None}
    if c["op"] == "quant":
        v = _mx64(s["x"].double())
        if s["inv"] is None:
            return v
        rows = torch.empty((c["T"] * c["k"], c["K"]), dtype=torch.float64, device=v.device)
        for j in range(c["k"]):
            rows[s["inv"][:, j].long()] = v
        return rows
    if c["op"] == "combine":
        out = s["residual"].double() if s["residual"] is not None else torch.zeros((c["T"], c["D"]), dtype=torch.float64, device="cuda")
        for j in range(c["k"]):
            out = out + s["w"][:, j:j + 1].double() * s["y"][s["inv"][:, j].long()].double()
        return out
    n = _counts(c, seed)
    y = _ffn64(_rows64(s["codes"], s["scales"]), s["w"], n)
    if c["op"] == "ffn":
        g, u = y[:, :c["F"]], y[:, c["F"]:]
        if c["limit"] > 0:
            g, u = torch.minimum(g, torch.full_like(g, c["limit"])), torch.clamp(u, -c["limit"], c["limit"])
        y = _ffn64(_mx64(g * torch.special.expit(g) * u), s["w2"], n)
    return y

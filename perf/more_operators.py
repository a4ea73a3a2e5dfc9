"""What more operators beside the MoE layer are measured on: rows sorted by expert, the gradients of that, of the combine and of the routing's
weights, rows in 8-bit integers with a scale each, and the experts' products over them.

A case names its operator in "op":

- "sort": rows to expert order, each times its routing weights or as it is;
- "sort_grad": the gradient of that: of the rows, and of the weights where there are any;
- "combine_grad": the gradient of the weighted sum of each row's expert results: of the results and of the weights;
- "route_grad": the gradient of the routing's weights with respect to the logits;
- "quant": rows to 8-bit integers, as they lie or scattered to expert order, and what the codes stand for;
- "product": 8-bit rows times one matrix or the experts' matrices, each row with its own expert's;
- "ffn": gate and up with SwiGLU, its result in 8-bit rows, then the down product.

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


# --- the cases -----------------------------------------------------------------------------------------------------

def _sort(name, T, k, D, type, weighted, dropped):
    return dict(name=name, op="sort", T=T, k=k, D=D, type=type, weighted=weighted, dropped=dropped)


def _sort_grad(name, T, k, D, type, weighted, dropped):
    return dict(name=name, op="sort_grad", T=T, k=k, D=D, type=type, weighted=weighted, dropped=dropped)


def _combine_grad(name, T, k, D, type, dout, dropped):
    return dict(name=name, op="combine_grad", T=T, k=k, D=D, type=type, dout=dout, dropped=dropped)


def _route_grad(name, T, E, k, score, type, renorm, scale):
    return dict(name=name, op="route_grad", T=T, E=E, k=k, score=score, type=type, renorm=renorm, scale=scale)


def _quant(name, T, K, k, type, out):
    return dict(name=name, op="quant", T=T, K=K, k=k, type=type, out=out)


def _product(name, E, T, k, N, K, y, zipf):
    return dict(name=name, op="product", E=E, T=T, k=k, N=N, K=K, y=y, zipf=zipf)


def _ffn(name, E, T, k, D, F, y, zipf, limit):
    return dict(name=name, op="ffn", E=E, T=T, k=k, D=D, F=F, y=y, zipf=zipf, limit=limit)


def listed():
    return [
        # A few decode rows to expert order, in f32 as the layer's own rows are: all latency.
        _sort("sort_13x2560_f32", 13, 8, 2560, "f32", False, 0.0),
        # The benchmark's long prompt as a model holds it between layers, for experts of the caller's own.
        _sort("sort_32768x2048_bf16", 32768, 10, 2048, "bf16", False, 0.0),
        # A packed ragged batch under weights applied before the experts, an eighth of the assignments on another GPU: both gradients.
        _sort_grad("sort_grad_3521x2560_weighted", 3521, 8, 2560, "f16", True, 0.125),
        # The long prompt as a training batch: what comes back from the sum of every row's results.
        _combine_grad("combine_grad_16384x2048", 16384, 10, 2048, "bf16", "f32", 0.0),
        # A small batch of odd size under a sigmoid router, bf16 logits.
        _route_grad("route_grad_77x160_sigmoid", 77, 160, 6, "sigmoid", "bf16", True, 2.5),
        # The long prompt's router by softmax weights as they are: every expert's logit has a gradient.
        _route_grad("route_grad_32768x512_softmax", 32768, 512, 10, "softmax", "f32", False, 1.0),
        # A few decode rows straight into expert order.
        _quant("quant_13x2560_scatter8", 13, 2560, 8, "f32", "f32"),
        # The long prompt in bf16, for a dense product.
        _quant("quant_32768x2048_bf16", 32768, 2048, 1, "bf16", "bf16"),
        # One dense matrix (a shared expert's down) on a ragged batch of rows, sizes that fill no tile.
        _product("product_dense_777x2080x1440", 1, 777, 1, 2080, 1440, "f16", 0.0),
        # One token through ten of 512 experts: weights read once, all latency.
        _ffn("ffn_512x1", 512, 1, 10, 2048, 512, "f16", 0.0, 0.0),
        # A decode batch: one or two rows an expert, weights of every expert read once.
        _ffn("ffn_512x100", 512, 100, 10, 2048, 512, "f16", 0.0, 0.0),
        # A long prompt through wide experts, skewed, with a SwiGLU limit: tensor-core work.
        _ffn("ffn_128x8192_zipf", 128, 8192, 8, 2560, 768, "bf16", 0.6, 7.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["sort", "sort_grad", "combine_grad", "route_grad", "quant", "product", "ffn"])
    if op in ("sort", "sort_grad", "combine_grad"):
        k, D, type = rng.randint(1, 16), 8 * _log(rng, 1, 512), rng.choice(["f32", "f16", "bf16"])
        T = _log(rng, 1, max(2, min(32768, 32768 * 10 * 2048 // (k * D * SIZE[type]))))
        c = dict(op=op, T=T, k=k, D=D, type=type, dropped=rng.choice([0.0, 0.0, 0.125, 0.5]))
        return dict(c, dout=rng.choice(["f32", type])) if op == "combine_grad" else dict(c, weighted=rng.random() < 0.5)
    if op == "route_grad":
        E = _log(rng, 2, 512)
        return dict(op=op, T=_log(rng, 1, 32768), E=E, k=rng.randint(1, min(16, E)), score=rng.choice(["softmax", "sigmoid"]), type=rng.choice(["f32", "f16", "bf16"]),
                    renorm=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]))
    if op == "quant":
        K, k = 32 * _log(rng, 2, 256), rng.choice([1, 1, rng.randint(2, 10)])
        return dict(op=op, T=_log(rng, 1, max(2, 32768 * 2048 // (K * k))), K=K, k=k, type=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f32", "bf16"]))
    if op == "product":
        E = rng.choice([1, _log(rng, 2, 128)])
        k = 1 if E == 1 else rng.randint(1, min(8, E))
        return dict(op=op, E=E, T=_log(rng, 1, 4096), k=k, N=32 * _log(rng, 2, 100), K=32 * _log(rng, 2, 100), y=rng.choice(["f16", "bf16"]), zipf=rng.choice([0.0, 1.1]))
    E = _log(rng, 2, 128)
    return dict(op=op, E=E, T=_log(rng, 1, 4096), k=rng.randint(1, min(8, E)), D=32 * _log(rng, 4, 80), F=32 * _log(rng, 2, 24), y=rng.choice(["f16", "bf16"]),
                zipf=rng.choice([0.0, 1.1]), limit=rng.choice([0.0, 7.0]))


def work(case):
    c = case
    if c["op"] in ("sort", "sort_grad", "combine_grad"):
        # Assignments that are elsewhere move nothing but their entries of the lists.
        T, k, n, R = c["T"], c["k"], c["T"] * c["D"], _rows(c)
        moved, lists = R * c["D"] * SIZE[c["type"]], 4 * T * k
        if c["op"] == "combine_grad":  # results and the sums' gradient in, results' gradient out; lists of places, weights, weights' gradient
            return dict(bytes=n * SIZE[c["dout"]] + 2 * moved + 3 * lists, flops=3 * R * c["D"])
        # One side of the rows, one of their copies; with weights the lists of those, and for their gradient the rows and one list more.
        both = c["weighted"] and c["op"] == "sort_grad"
        return dict(bytes=n * SIZE[c["type"]] * (2 if both else 1) + moved + lists * (1 + c["weighted"] + both), flops=R * c["D"] * (4 if both else 1))
    if c["op"] == "route_grad":
        n, chosen = c["T"] * c["E"] * SIZE[c["type"]], c["T"] * c["k"]
        dense = c["score"] == "softmax" and not c["renorm"]  # every logit counts; else the chosen ones
        return dict(bytes=n + (n if dense else chosen * SIZE[c["type"]]) + 8 * chosen, flops=4 * (c["T"] * c["E"] if dense else chosen))
    if c["op"] == "quant":  # rows in, codes and scales out; then those in and their values out
        n = c["T"] * c["K"]
        return dict(bytes=n * SIZE[c["type"]] + 2 * c["k"] * (n + 4 * c["T"]) + c["k"] * n * SIZE[c["out"]], flops=4 * n * c["k"])
    # Experts that no row went to are not read.
    R, hit = c["T"] * c["k"], int((_counts(c, 0) > 0).sum())
    if c["op"] == "product":
        return dict(bytes=(hit * c["N"] + R) * (c["K"] + 4) + R * c["N"] * SIZE[c["y"]], flops=2 * R * c["N"] * c["K"])
    D, F = c["D"], c["F"]
    return dict(bytes=hit * (3 * F * D + 4 * (2 * F + D)) + R * (D + 4) + R * D * SIZE[c["y"]], flops=6 * R * F * D)


# --- inputs --------------------------------------------------------------------------------------------------------

def _rows(c):
    """Assignments that are here: the rows of expert order."""
    return c["T"] * c["k"] - int(c["dropped"] * c["T"] * c["k"])


def _counts(c, seed):
    """Rows each expert gets: every token's k distinct experts, drawn evenly or by a Zipf law."""
    rng = np.random.default_rng(seed)
    p = -c["zipf"] * np.log(1.0 + rng.permutation(c["E"]))
    g = p + rng.gumbel(size=(c["T"], c["E"]))  # the k largest: k draws without replacement
    return np.bincount(np.argsort(-g, axis=1)[:, :c["k"]].reshape(-1), minlength=c["E"])


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _empty(shape, type):
    return torch.empty(shape, dtype=TORCH[type], device="cuda")


def _weights(g, E, N, K):
    """Matrices as their rows' rounding leaves them: codes of a bell curve, a scale a row, sized so that a row's products are of the order of one."""
    codes = torch.empty((E, N, K), dtype=torch.int8, device="cuda")
    for e in range(0, E, 64):
        m = codes[e:e + 64]
        m.copy_((30 * torch.randn(m.shape, generator=g, device="cuda")).round_().clamp_(-127, 127))
    return codes, (0.5 + torch.rand((E, N), generator=g, device="cuda")) / (30 * math.sqrt(K))


def prepare(case, seed):
    c, g, s = case, _gen(seed), {}
    s["case"] = c
    T, k = c["T"], c.get("k", 1)
    if c["op"] in ("sort", "sort_grad", "combine_grad"):
        D, R = c["D"], _rows(c)
        place = torch.randperm(T * k, generator=g, device="cuda")
        s["inv"] = torch.where(place < R, place, -1).to(torch.int32).reshape(T, k)
        w = torch.rand((T, k), generator=g, device="cuda")
        s["w"] = w / w.sum(1, keepdim=True) if c.get("weighted", True) else None
        s["dw"] = torch.empty((T, k), device="cuda")
        if c["op"] == "combine_grad":
            s["dout"], s["y"], s["dy"] = _randn(g, (T, D), TORCH[c["dout"]]), _randn(g, (R, D), TORCH[c["type"]]), _empty((R, D), c["type"])
        else:
            s["x"] = _randn(g, (T, D), TORCH[c["type"]])
            s["xs" if c["op"] == "sort" else "dx"] = _empty((R if c["op"] == "sort" else T, D), c["type"])
            if c["op"] == "sort_grad":
                s["dxs"] = _randn(g, (R, D), TORCH[c["type"]])
        return s
    if c["op"] == "route_grad":
        s["logits"] = _randn(g, (T, c["E"]), TORCH[c["type"]])
        s["ids"] = torch.topk(s["logits"].float(), k, 1)[1].to(torch.int32)
        s["dw"], s["dlogits"] = _randn(g, (T, k)), _empty((T, c["E"]), c["type"])
        return s
    R = T * k
    if c["op"] == "quant":
        K = c["K"]
        s["x"] = _randn(g, (T, K), TORCH[c["type"]])
        s["inv"] = torch.randperm(R, generator=g, device="cuda").to(torch.int32).reshape(T, k) if k > 1 else None
        s["codes"], s["scales"] = _i8_rows(R, K)
        s["out"] = _empty((R, K), c["out"])
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
        s["y"] = _empty((R, c["N"]), c["y"])
    else:
        s["w"], s["w2"] = _weights(g, c["E"], 2 * c["F"], D), _weights(g, c["E"], D, c["F"])
        s["h"], s["hq"] = _empty((R, c["F"]), c["y"]), _i8_rows(R, c["F"])
        s["y"] = _empty((R, D), c["y"])
    return s


def _i8_rows(R, K):
    return torch.empty((R, K), dtype=torch.int8, device="cuda"), torch.empty(R, device="cuda")


# --- the plain forms -----------------------------------------------------------------------------------------------

def _quantize(x):
    """Codes by 64 bits, so that none hangs on a rounding at a border; scales rounded to 32."""
    x = x.double()
    top = x.abs().amax(1, keepdim=True)
    codes = torch.round(x * 127 / torch.where(top > 0, top, 1.0))
    return codes.to(torch.int8), (top / torch.full_like(top, 127)).float().squeeze(1)


def _values(codes, scales):
    return codes.float() * scales.unsqueeze(-1)


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


def _gathered(rows, inv):
    """rows[inv], zeros where an entry names none: [T][k][D] in 32 bits."""
    return rows.float()[inv.long().clamp(min=0)] * (inv >= 0).unsqueeze(2)


def _scattered(inv, v, R):
    """Row inv[t][k] of R is v[t][k]; entries that name none go to a row behind them."""
    out = torch.empty((R + 1, v.shape[2]), dtype=v.dtype, device=v.device)
    out[torch.where(inv >= 0, inv, R).long().reshape(-1)] = v.reshape(-1, v.shape[2])
    return out[:R]


def _route_grad_plain(s):
    c, l, ids, dw = s["case"], s["logits"].float(), s["ids"].long(), s["dw"]
    chosen = l.gather(1, ids)
    if c["score"] == "softmax":
        e = torch.exp(l - l.amax(1, keepdim=True))
        picked = e.gather(1, ids)
        total = picked.sum(1, keepdim=True) if c["renorm"] else e.sum(1, keepdim=True)
        p = picked / total
        mean = (p * dw).sum(1, keepdim=True)
        if c["renorm"]:
            out = torch.zeros_like(l).scatter_(1, ids, p * (dw - mean))
        else:
            out = (e / total * -mean).scatter_(1, ids, p * (dw - mean))
    else:
        q = 1 / (1 + torch.exp(chosen))  # 1 - s
        score = 1 / (1 + torch.exp(-chosen))
        if c["renorm"]:
            p = score / score.sum(1, keepdim=True)
            d = p * q * (dw - (p * dw).sum(1, keepdim=True))
        else:
            d = score * q * dw
        out = torch.zeros_like(l).scatter_(1, ids, d)
    return (out * c["scale"]).to(TORCH[c["type"]])


def _plain(s):
    c = s["case"]
    type = TORCH[c["type"]] if "type" in c else None
    if c["op"] == "sort":
        v = s["x"].unsqueeze(1).expand(-1, c["k"], -1)
        v = (v.float() * s["w"].unsqueeze(2)).to(type) if s["w"] is not None else v
        return _scattered(s["inv"], v, _rows(c))
    if c["op"] == "sort_grad":
        d = _gathered(s["dxs"], s["inv"])
        if s["w"] is None:
            return {"dx": d.sum(1).to(type)}
        return {"dx": (d * s["w"].unsqueeze(2)).sum(1).to(type), "dw": (d * s["x"].float().unsqueeze(1)).sum(2)}
    if c["op"] == "combine_grad":
        dout = s["dout"].float().unsqueeze(1)
        dy = _scattered(s["inv"], (dout * s["w"].unsqueeze(2)).to(type), _rows(c))
        return {"dy": dy, "dw": (_gathered(s["y"], s["inv"]) * dout).sum(2)}
    if c["op"] == "route_grad":
        return _route_grad_plain(s)
    if c["op"] == "quant":
        v = _values(*_quantize(s["x"]))
        if s["inv"] is not None:
            v = _scattered(s["inv"], v.unsqueeze(1).expand(-1, c["k"], -1), c["T"] * c["k"])
        return v.to(TORCH[c["out"]])
    y = _by_expert(s, _values(s["codes"], s["scales"]), s["w"])
    if c["op"] == "ffn":
        y = _by_expert(s, _values(*_quantize(_swiglu(y, c["limit"]).to(TORCH[c["y"]]))), s["w2"])
    return y.to(TORCH[c["y"]])


# --- the framework's calls -----------------------------------------------------------------------------------------

def _ptr(t):
    return None if t is None else t.data_ptr()


def _own(s):
    from c0ven_b200 import ops

    c, st = s["case"], torch.cuda.current_stream().cuda_stream
    T, k = c["T"], c.get("k", 1)
    if c["op"] == "sort":
        ops.sort_rows_device(s["x"].data_ptr(), GGML[c["type"]], T, k, c["D"], s["inv"].data_ptr(), _rows(c), s["xs"].data_ptr(), w_ptr=_ptr(s["w"]), stream=st)
        return s["xs"]
    if c["op"] == "sort_grad":
        weighted = s["w"] is not None
        ops.sort_rows_grad_device(s["dxs"].data_ptr(), GGML[c["type"]], _rows(c), s["inv"].data_ptr(), T, k, c["D"], dx_ptr=s["dx"].data_ptr(), w_ptr=_ptr(s["w"]),
                                  x_ptr=s["x"].data_ptr() if weighted else None, dw_ptr=s["dw"].data_ptr() if weighted else None, stream=st)
        return {"dx": s["dx"], "dw": s["dw"]} if weighted else {"dx": s["dx"]}
    if c["op"] == "combine_grad":
        ops.combine_rows_grad_device(s["dout"].data_ptr(), GGML[c["dout"]], s["y"].data_ptr(), GGML[c["type"]], _rows(c), s["inv"].data_ptr(), s["w"].data_ptr(), T, k,
                                     c["D"], dy_ptr=s["dy"].data_ptr(), dw_ptr=s["dw"].data_ptr(), stream=st)
        return {"dy": s["dy"], "dw": s["dw"]}
    if c["op"] == "route_grad":
        ops.route_logits_grad_device(s["logits"].data_ptr(), GGML[c["type"]], T, c["E"], k, s["ids"].data_ptr(), s["dw"].data_ptr(), s["dlogits"].data_ptr(),
                                     score=ops.SIGMOID if c["score"] == "sigmoid" else ops.SOFTMAX, renorm=c["renorm"], scale=c["scale"], stream=st)
        return s["dlogits"]
    R = T * k
    if c["op"] == "quant":
        ops.i8_quantize_rows_device(s["x"].data_ptr(), GGML[c["type"]], T, c["K"], s["codes"].data_ptr(), s["scales"].data_ptr(), R, inv_ptr=_ptr(s["inv"]), n_used=k,
                                    stream=st)
        ops.i8_dequantize_rows_device(s["codes"].data_ptr(), s["scales"].data_ptr(), R, c["K"], s["out"].data_ptr(), GGML[c["out"]], stream=st)
        return s["out"]
    at = s["offsets"].data_ptr()
    if c["op"] == "product":
        w = ops.I8Weights(c["E"], c["N"], c["K"], s["w"][0].data_ptr(), s["w"][1].data_ptr())
        ops.i8_product_device(w, s["codes"].data_ptr(), s["scales"].data_ptr(), R, at, s["y"].data_ptr(), GGML[c["y"]], stream=st)
        return s["y"]
    F = c["F"]
    w, w2 = (ops.I8Weights(c["E"], n, m, t[0].data_ptr(), t[1].data_ptr()) for n, m, t in ((2 * F, c["D"], s["w"]), (c["D"], F, s["w2"])))
    h, hc, hs = s["h"].data_ptr(), s["hq"][0].data_ptr(), s["hq"][1].data_ptr()
    ops.i8_gate_up_device(w, s["codes"].data_ptr(), s["scales"].data_ptr(), R, at, h, GGML[c["y"]], swiglu_limit=c["limit"], stream=st)
    ops.i8_quantize_rows_device(h, GGML[c["y"]], R, F, hc, hs, R, stream=st)
    ops.i8_product_device(w2, hc, hs, R, at, s["y"].data_ptr(), GGML[c["y"]], stream=st)
    return s["y"]


def run(state):
    return _own(state) if own else _plain(state)


# --- the definition in 64 bits, apart from the plain forms ------------------------------------------------------------

def _i8_64(x):
    """What rows x (64 bits) in 8-bit integers stand for: of the two whole numbers around a quotient the nearer, the even one where both are."""
    top = x.abs().max(1)[0]
    q = (x * 127) / torch.where(top == 0, torch.ones_like(top), top)[:, None]
    lo = torch.floor(q)
    up = (q - lo > 0.5) | ((q - lo == 0.5) & (torch.remainder(lo, 2) == 1))
    return (lo + up) * torch.div(top, torch.full_like(top, 127.0)).to(torch.float32).double()[:, None]


def _by_expert64(x, w, n):
    out, at = [], 0
    for e in np.flatnonzero(n):
        out.append(x[at:at + n[e]] @ (w[0][e].double() * w[1][e].double()[:, None]).T)
        at += n[e]
    return torch.cat(out)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] in ("sort", "sort_grad", "combine_grad"):
        R, w = _rows(c), torch.ones((c["T"], c["k"]), dtype=torch.float64, device="cuda") if s["w"] is None else s["w"].double()
        rows = torch.zeros((R, c["D"]), dtype=torch.float64, device="cuda")
        dx, dw = torch.zeros((c["T"], c["D"]), dtype=torch.float64, device="cuda"), torch.zeros((c["T"], c["k"]), dtype=torch.float64, device="cuda")
        for j in range(c["k"]):
            t = torch.nonzero(s["inv"][:, j] >= 0)[:, 0]
            r = s["inv"][t, j].long()
            if c["op"] == "sort":
                rows[r] = w[t, j, None] * s["x"][t].double()
            elif c["op"] == "sort_grad":
                dx[t] += w[t, j, None] * s["dxs"][r].double()
                dw[t, j] = torch.einsum("td,td->t", s["x"][t].double(), s["dxs"][r].double())
            else:
                rows[r] = w[t, j, None] * s["dout"][t].double()
                dw[t, j] = torch.einsum("td,td->t", s["dout"][t].double(), s["y"][r].double())
        if c["op"] == "sort":
            return rows
        if c["op"] == "sort_grad":
            return {"dx": dx, "dw": dw} if s["w"] is not None else {"dx": dx}
        return {"dy": rows, "dw": dw}
    if c["op"] == "route_grad":
        l = s["logits"].double().requires_grad_(True)
        score = torch.softmax(l, 1) if c["score"] == "softmax" else torch.sigmoid(l)
        w = score.gather(1, s["ids"].long())
        w = w / w.sum(1, keepdim=True) if c["renorm"] else w
        return torch.autograd.grad(w * c["scale"], l, s["dw"].double())[0]
    if c["op"] == "quant":
        v = _i8_64(s["x"].double())
        if s["inv"] is None:
            return v
        rows = torch.empty((c["T"] * c["k"], c["K"]), dtype=torch.float64, device=v.device)
        for j in range(c["k"]):
            rows[s["inv"][:, j].long()] = v
        return rows
    n = _counts(c, seed)
    y = _by_expert64(s["codes"].double() * s["scales"].double()[:, None], s["w"], n)
    if c["op"] == "ffn":
        g, u = y[:, :c["F"]], y[:, c["F"]:]
        if c["limit"] > 0:
            g, u = torch.minimum(g, torch.full_like(g, c["limit"])), torch.clamp(u, -c["limit"], c["limit"])
        y = _by_expert64(_i8_64((g * torch.special.expit(g) * u).to(TORCH[c["y"]]).double()), s["w2"], n)
    return y

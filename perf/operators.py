"""Cases of the layer-level operators for language-model blocks, in plain torch and as calls of the library.

Three operators of include/qcnn.h: products with 4-bit weights (qcnn_op_matvec_w4), products grouped by expert
(qcnn_op_grouped_matmul) and the two ends of a residual block (qcnn_op_norm_res).  `own` selects the library's calls;
otherwise the same formulas run as elementary torch operations in 32 bits (64 for the integer sums).
"""
import ctypes
import math

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


# ---- cases ---------------------------------------------------------------------------------------------
def _w4(name, rows, n, k, group, type, zeros, bias):
    return {"name": name, "op": "w4", "rows": rows, "n": n, "k": k, "group": group, "type": type, "zeros": zeros, "bias": bias}


def _grouped(name, experts, rows, n, k, type, otype, skew, gather, scaled, bias, act, behind):
    return {"name": name, "op": "grouped", "experts": experts, "rows": rows, "n": n, "k": k, "type": type, "otype": otype, "skew": skew,
            "gather": gather, "scaled": scaled, "bias": bias, "act": act, "behind": behind}


def _norm(name, rows, d, type, wtype, post, pre, gate, act, parts, beta):
    return {"name": name, "op": "norm", "rows": rows, "d": d, "type": type, "wtype": wtype, "post": post, "pre": pre, "gate": gate, "act": act,
            "parts": parts, "beta": beta}


def listed():
    return [
        # one token through a square projection: the smallest call of a decoding loop, latency and 8 MB of weights
        _w4("w4_token_bf16", 1, 4096, 4096, 128, "bf16", False, False),
        # sixteen sequences decoded together through a wide projection: 64 MB of weights with zero points
        _w4("w4_batch_f16", 16, 16384, 8192, 64, "f16", True, False),
        # odd sizes in the library's float32 configuration: a row that ends inside a byte, a short last group
        _w4("w4_odd_f32", 5, 1001, 2047, 32, "f32", True, True),
        # eight tokens decoded, eight experts of 64 each: one or two rows an expert, some experts with none
        _grouped("grouped_decode_bf16", 64, 64, 1024, 2048, "bf16", "bf16", 0.3, True, False, False, 2, 0),
        # a long prompt: 16384 rows over 16 experts of unequal load, rows scaled by their routing weights
        _grouped("grouped_prefill_bf16", 16, 16384, 4096, 2048, "bf16", "bf16", 0.5, True, True, False, 0, 0),
        # the network's 1x1 layer (48 -> 32 channels) over the pixels of eight 416x240 frames of the four QPs' models
        _grouped("grouped_frames_i8", 4, 8 * 416 * 240, 32, 48, "i8", "f32", 0.0, False, False, True, 1, 0),
        # int8 experts with a scale for each row and each output, rows behind the last expert left alone
        _grouped("grouped_prefill_i8", 8, 8192, 4096, 4096, "i8", "bf16", 0.5, False, True, True, 0, 37),
        # odd sizes in the float32 configuration
        _grouped("grouped_odd_f32", 7, 333, 129, 515, "f32", "f32", 1.0, True, True, True, 1, 5),
        # one token between two blocks: a latency call
        _norm("norm_token_bf16", 1, 4096, "bf16", "bf16", "rms", "rms", 0, 0, 0, 1.0),
        # a long prompt between two blocks, a gate value for each element
        _norm("norm_prefill_bf16", 16384, 4096, "bf16", "f32", "rms", "rms", 1, 1, 0, 1.0),
        # the end of an expert block: eight experts' rows added up for each token
        _norm("norm_combine_f16", 4096, 2048, "f16", "f16", "none", "rms", 0, 0, 8, 1.0),
        # layer norms of odd rows in the float32 configuration, one gate row for 100 rows (a sample's condition)
        _norm("norm_odd_f32", 517, 1001, "f32", "f32", "layer", "layer", 100, 2, 0, 0.7),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return min(hi, max(lo, v))


def draw(rng):
    op = rng.choice(("w4", "grouped", "norm"))
    if op == "w4":
        while True:
            c = _w4("", _log(rng, 1, 64), _log(rng, 64, 16384), _log(rng, 64, 16384), rng.choice((32, 64, 128)), rng.choice(("f32", "f16", "bf16")),
                    rng.random() < 0.5, rng.random() < 0.5)
            if rng.random() < 0.5:  # half of the shapes are the even ones of a model
                c["n"], c["k"] = (c["n"] + 63) // 64 * 64, (c["k"] + 63) // 64 * 64
            if c["n"] * c["k"] <= 16384 * 8192 and c["rows"] * c["n"] * c["k"] <= 16 * 16384 * 8192:
                break
    elif op == "grouped":
        while True:
            t = rng.choice(("f32", "f16", "bf16", "i8"))
            ot = t if t != "i8" else rng.choice(("f32", "f16", "bf16"))
            c = _grouped("", _log(rng, 1, 128), _log(rng, 1, 16384), _log(rng, 32, 4096), _log(rng, 32, 4096), t, ot, rng.choice((0.0, 0.5, 1.0)),
                         rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.5, rng.choice((0, 1, 2)), rng.choice((0, 0, 3, 100)))
            if rng.random() < 0.5:
                c["n"], c["k"] = (c["n"] + 63) // 64 * 64, (c["k"] + 63) // 64 * 64
            work = c["rows"] * c["n"] * c["k"]
            if work <= 16384 * 4096 * 2048 and c["experts"] * c["n"] * c["k"] <= 1 << 28 and (t != "f32" or work <= 1 << 34):
                break
    else:
        while True:
            c = _norm("", _log(rng, 1, 16384), _log(rng, 16, 16384), rng.choice(("f32", "f16", "bf16")), "f32", rng.choice(("none", "rms", "layer")),
                      rng.choice(("none", "rms", "layer")), rng.choice((0, 1, 7, 1024)), rng.choice((0, 1, 2, 3)), rng.choice((0, 0, 2, 5, 8)),
                      rng.choice((1.0, 0.5)))
            c["wtype"] = rng.choice(("f32", c["type"]))
            if rng.random() < 0.5:
                c["d"] = (c["d"] + 63) // 64 * 64
            if c["rows"] * c["d"] * max(1, c["parts"]) <= 1 << 26 and (c["type"] != "f32" or c["rows"] * c["d"] <= 1 << 25):
                break
    del c["name"]
    return c


# ---- inputs --------------------------------------------------------------------------------------------
def _sizes(case, seed):
    """Rows of each expert: Zipf-like loads of a router, permuted; small calls leave experts empty."""
    g = torch.Generator().manual_seed(seed + 7)
    e = case["experts"]
    p = (1.0 / torch.arange(1, e + 1, dtype=torch.float64)) ** case["skew"]
    p = p[torch.randperm(e, generator=g)]
    pick = torch.multinomial(p / p.sum(), case["rows"], replacement=True, generator=g)
    return torch.bincount(pick, minlength=e).tolist()


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV)

    s = dict(case)
    if case["op"] == "w4":
        rows, n, k, ng = case["rows"], case["n"], case["k"], -(-case["k"] // case["group"])
        x = normal(rows, k) * (1 + 9 * (torch.rand(k, generator=g, device=DEV) < 0.01))  # a few strong channels
        s["x"] = x.to(t)
        s["q"] = torch.randint(0, 256, (n, (k + 1) // 2), generator=g, device=DEV, dtype=torch.uint8)  # two weights a byte, the even k low
        s["scale"] = ((0.5 + torch.rand(ng, n, generator=g, device=DEV)) / (4.6 * math.sqrt(k))).to(t)
        s["zero"] = torch.randint(4, 12, (ng, n), generator=g, device=DEV, dtype=torch.uint8) if case["zeros"] else None
        s["b"] = normal(n) if case["bias"] else None
        s["y"] = torch.empty(rows, n, device=DEV, dtype=t)
    elif case["op"] == "grouped":
        e, rows, n, k = case["experts"], case["rows"], case["n"], case["k"]
        sizes = _sizes(case, seed)
        total = rows + case["behind"]
        s["sizes"] = sizes
        s["offsets"] = torch.tensor([0] + sizes).cumsum(0).to(torch.int32).to(DEV)
        xrows = max(1, -(-rows // 8)) if case["gather"] else rows  # a token goes to up to eight experts
        if case["type"] == "i8":
            s["x"] = (normal(xrows, k) * 40).round().clamp(-127, 127).to(torch.int8)
            s["w"] = (normal(e, n, k) * 40).round().clamp(-127, 127).to(torch.int8)
            s["xs"] = (0.5 + torch.rand(xrows, generator=g, device=DEV)) / 40
            s["ws"] = (0.5 + torch.rand(e, n, generator=g, device=DEV)) / (40 * math.sqrt(k))
        else:
            s["x"] = normal(xrows, k).to(t)
            s["w"] = (normal(e, n, k) / math.sqrt(k)).to(t)
            s["xs"] = s["ws"] = None
        s["src"] = (torch.randperm(rows, generator=g, device=DEV) % xrows).to(torch.int32) if case["gather"] else None
        s["rs"] = torch.rand(total, generator=g, device=DEV) if case["scaled"] else None
        s["b"] = normal(e, n) if case["bias"] else None
        s["xrows"], s["total"] = xrows, total
        s["y"] = torch.zeros(total, n, device=DEV, dtype=TYPES[case["otype"]])
    else:
        rows, d, parts = case["rows"], case["d"], case["parts"]
        wt = TYPES[case["wtype"]]
        yrows = rows * max(1, parts)
        s["x"] = (normal(rows, d) * (1 + 19 * (torch.rand(d, generator=g, device=DEV) < 0.005))).to(t)
        s["v"] = normal(yrows, d).to(t)
        s["index"] = torch.randperm(yrows, generator=g, device=DEV).to(torch.int32).view(rows, parts) if parts else None
        s["g"] = normal(-(-rows // case["gate"]), d).to(t) if case["gate"] else None
        for at in ("post", "pre"):
            s[at + "_w"] = (1 + 0.2 * normal(d)).to(wt) if case[at] != "none" else None
            s[at + "_b"] = (0.2 * normal(d)).to(wt) if case[at] == "layer" else None
        s["yrows"], s["alpha"] = yrows, 0.8
        s["h"] = torch.empty(rows, d, device=DEV, dtype=t)
        s["n"] = torch.empty(rows, d, device=DEV, dtype=t)
    return s


# ---- one pass ------------------------------------------------------------------------------------------
def _nibbles(q, k):
    return torch.stack((q & 15, q >> 4), -1).view(q.shape[0], -1)[:, :k]


def _act(v, act):
    return torch.relu(v) if act == 1 else v / (1 + torch.exp(-v)) if act == 2 else v


def _plain_w4(s):
    rows, n, k, grp = s["rows"], s["n"], s["k"], s["group"]
    ng = s["scale"].shape[0]
    q = _nibbles(s["q"], k).float()
    if ng * grp > k:
        q = torch.cat((q, q.new_zeros(n, ng * grp - k)), 1)
    zero = s["zero"].t().float().unsqueeze(2) if s["zero"] is not None else 8.0
    w = ((q.view(n, ng, grp) - zero) * s["scale"].t().float().unsqueeze(2)).view(n, ng * grp)[:, :k]
    y = s["x"].float() @ w.t()
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(s["x"].dtype)


def _plain_grouped(s):
    wide = torch.float64 if s["type"] == "i8" else torch.float32  # int8 sums pass 2^24
    x = s["x"][s["src"].long()] if s["src"] is not None else s["x"]
    xs = s["xs"][s["src"].long()] if s["xs"] is not None and s["src"] is not None else s["xs"]
    out, at = torch.zeros(s["total"], s["n"], device=DEV, dtype=s["y"].dtype), 0
    for e, c in enumerate(s["sizes"]):
        if c:
            v = (x[at:at + c].to(wide) @ s["w"][e].to(wide).t())
            if xs is not None:
                v = v * s["ws"][e] * xs[at:at + c, None]
            v = v.float()
            if s["b"] is not None:
                v = v + s["b"][e]
            v = _act(v, s["act"])
            if s["rs"] is not None:
                v = v * s["rs"][at:at + c, None]
            out[at:at + c] = v.to(out.dtype)
            at += c
    return out


def _plain_norm_of(v, kind, w, b, eps):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(-1, keepdim=True) + eps) * w.float()
    return v + b.float() if b is not None else v


def _plain_norm(s):
    v = s["v"].float()
    if s["index"] is not None:
        v = v[s["index"].long()].sum(1)
    u = _plain_norm_of(v, s["post"], s["post_w"], s["post_b"], 1e-6)
    if s["g"] is not None:
        g = s["g"].float()
        g = torch.sigmoid(g) if s["act"] == 1 else torch.tanh(g) if s["act"] == 2 else g * torch.sigmoid(g) if s["act"] == 3 else g
        u = u * g.repeat_interleave(s["gate"], 0)[: s["rows"]]
    h = s["beta"] * s["x"].float() + s["alpha"] * u
    n = _plain_norm_of(h, s["pre"], s["pre_w"], s["pre_b"], 1e-6)
    return h.to(s["x"].dtype), n.to(s["x"].dtype)


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _own(s):
    from qcnn_gpu_amd import capi
    lib, stream = capi.load(), torch.cuda.current_stream().cuda_stream
    kind = {"f32": capi.F32, "f16": capi.F16, "bf16": capi.BF16, "i8": capi.I8}
    if s["op"] == "w4":
        a = capi.MatvecW4(x=_ptr(s["x"]), y=_ptr(s["y"]), w=_ptr(s["q"]), scale=_ptr(s["scale"]), zero=_ptr(s["zero"]), bias=_ptr(s["b"]),
                          ldx=s["k"], ldy=s["n"], ldw=(s["k"] + 1) // 2, rows=s["rows"], n=s["n"], k=s["k"], group=s["group"],
                          type=kind[s["type"]], scale_type=kind[s["type"]], out_type=kind[s["type"]])
        capi.check(lib.qcnn_op_matvec_w4(ctypes.byref(a), stream))
        return s["y"]
    if s["op"] == "grouped":
        a = capi.GroupedMatmul(x=_ptr(s["x"]), y=_ptr(s["y"]), w=_ptr(s["w"]), offsets=_ptr(s["offsets"]), src=_ptr(s["src"]),
                               x_scale=_ptr(s["xs"]), w_scale=_ptr(s["ws"]), bias=_ptr(s["b"]), row_scale=_ptr(s["rs"]),
                               ldx=s["k"], ldy=s["n"], ldw=s["k"], w_stride=s["n"] * s["k"], rows=s["total"], x_rows=s["xrows"],
                               experts=s["experts"], n=s["n"], k=s["k"], type=kind[s["type"]], out_type=kind[s["otype"]], act=s["act"])
        capi.check(lib.qcnn_op_grouped_matmul(ctypes.byref(a), stream))
        return s["y"]
    norm = {"none": capi.NORM_NONE, "rms": capi.NORM_RMS, "layer": capi.NORM_LAYER}
    d = s["d"]
    a = capi.NormRes(x=_ptr(s["x"]), y=_ptr(s["v"]), index=_ptr(s["index"]), gate=_ptr(s["g"]), post_w=_ptr(s["post_w"]), post_b=_ptr(s["post_b"]),
                     pre_w=_ptr(s["pre_w"]), pre_b=_ptr(s["pre_b"]), h=_ptr(s["h"]), n=_ptr(s["n"]), ldx=d, ldy=d, ldg=d, ldh=d, ldn=d,
                     rows=s["rows"], y_rows=s["yrows"], d=d, parts=max(1, s["parts"]), gate_rows=max(1, s["gate"]), type=kind[s["type"]],
                     w_type=kind[s["wtype"]], post=norm[s["post"]], pre=norm[s["pre"]], act=s["act"], alpha=s["alpha"], beta=s["beta"],
                     post_eps=1e-6, pre_eps=1e-6)
    capi.check(lib.qcnn_op_norm_res(ctypes.byref(a), stream))
    return s["h"], s["n"]


def run(state):
    if own:
        return _own(state)
    return {"w4": _plain_w4, "grouped": _plain_grouped, "norm": _plain_norm}[state["op"]](state)


# ---- what a pass cannot do without ---------------------------------------------------------------------
def work(case):
    sz = SIZE[case["type"]]
    if case["op"] == "w4":
        rows, n, k, ng = case["rows"], case["n"], case["k"], -(-case["k"] // case["group"])
        return {"bytes": n * ((k + 1) // 2) + ng * n * (sz + (1 if case["zeros"] else 0)) + rows * (k + n) * sz + (4 * n if case["bias"] else 0),
                "flops": 2 * rows * n * k}
    if case["op"] == "grouped":
        e, rows, n, k = case["experts"], case["rows"], case["n"], case["k"]
        used = sum(c > 0 for c in _sizes(case, 0))
        xrows = max(1, -(-rows // 8)) if case["gather"] else rows
        per_expert = n * k * sz + (4 * n if case["bias"] else 0) + (4 * n if case["type"] == "i8" else 0)
        per_row = n * SIZE[case["otype"]] + (4 if case["gather"] else 0) + (4 if case["scaled"] else 0)
        return {"bytes": used * per_expert + xrows * (k * sz + (4 if case["type"] == "i8" else 0)) + rows * per_row + 4 * (e + 1),
                "flops": 2 * rows * n * k}
    rows, d, parts = case["rows"], case["d"], case["parts"]
    gate = -(-rows // case["gate"]) * d * sz if case["gate"] else 0
    weights = sum({"none": 0, "rms": 1, "layer": 2}[case[at]] for at in ("post", "pre")) * d * SIZE[case["wtype"]]
    return {"bytes": rows * d * sz * (3 + max(1, parts)) + gate + weights + 4 * rows * parts, "flops": rows * d * (12 + max(1, parts))}


# ---- the definitions in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "w4":
        n, k, grp = case["n"], case["k"], case["group"]
        at = torch.arange(k, device=DEV)
        byte = s["q"][:, at // 2].to(torch.int32)
        code = torch.where((at % 2 == 0)[None], byte % 16, byte // 16).to(f8)
        of = at // grp
        z = s["zero"].to(f8)[of].t() if s["zero"] is not None else torch.full((n, k), 8.0, device=DEV, dtype=f8)
        y = torch.matmul(s["x"].to(f8), ((code - z) * s["scale"].to(f8)[of].t()).t().contiguous())
        return y + s["b"].to(f8) if s["b"] is not None else y
    if case["op"] == "grouped":
        y = torch.zeros(s["total"], case["n"], device=DEV, dtype=f8)
        ends = s["offsets"].tolist()
        rows = s["src"].long() if s["src"] is not None else torch.arange(case["rows"], device=DEV)
        for e in range(case["experts"]):
            lo, hi = ends[e], ends[e + 1]
            if hi > lo:
                r = rows[lo:hi]
                v = torch.matmul(s["x"][r].to(f8), s["w"][e].to(f8).t().contiguous())
                if s["ws"] is not None:
                    v *= s["ws"][e].to(f8)[None, :] * s["xs"][r].to(f8)[:, None]
                if s["b"] is not None:
                    v += s["b"][e].to(f8)
                if case["act"] == 1:
                    v = v.clamp_min(0)
                elif case["act"] == 2:
                    v = v * torch.sigmoid(v)
                y[lo:hi] = v * s["rs"][lo:hi].to(f8)[:, None] if s["rs"] is not None else v
        return y

    def norm(v, at):
        if case[at] == "none":
            return v
        w = s[at + "_w"].to(f8)
        if case[at] == "rms":
            return v * w * torch.rsqrt(v.pow(2).mean(1, keepdim=True) + 1e-6)
        m = v.mean(1, keepdim=True)
        return (v - m) * w * torch.rsqrt(v.var(1, unbiased=False, keepdim=True) + 1e-6) + s[at + "_b"].to(f8)

    rows, parts = case["rows"], case["parts"]
    if parts:
        y = torch.zeros(rows, case["d"], device=DEV, dtype=f8)
        for j in range(parts):
            y += s["v"][s["index"][:, j].long()].to(f8)
    else:
        y = s["v"].to(f8)
    y = norm(y, "post")
    if case["gate"]:
        g = s["g"].to(f8)[torch.arange(rows, device=DEV) // case["gate"]]
        y = y * {0: lambda v: v, 1: torch.sigmoid, 2: torch.tanh, 3: lambda v: v * torch.sigmoid(v)}[case["act"]](g)
    h = s["x"].to(f8) * case["beta"] + 0.8 * y
    return h, norm(h, "pre")

"""What is timed of the 4-bit Linear layer, the root-mean-square norm and their 8-bit activations.

    linear   y[b][o] = act(bias[o] + sum_g s[o][g] * sum_{k in g} (n[o][k] - z[o][g]) * x[b][k])
    linear8  the same with x[b][k] = xs[b][k / xgroup] * q[b][k], q signed 8-bit codes
    norm     h = x + res;  sum = h;  y = h * w / sqrt(mean(h * h) + eps)
    norm8    the same with y in 8 bits: scale = max|y| / 127 over a row or a group of columns, q = rint(y / scale)
    rows8    8 bits without the norm: y = x

Codes n have 4 bits (two in a byte, even k in the low half), a group of `group` weights of a row shares a scale and a zero
point z (8 where none are given); group 0 is the whole row.  What is held in 8 bits is compared as the values it stands for.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
CODE = {"fp32": 0, "fp16": 1, "bf16": 2}
EPS = 1e-5


def _linear(name, dtype, B, nin, nout, group, zeros, bias, act):
    return dict(name=name, op="linear", dtype=dtype, B=B, nin=nin, nout=nout, group=group, zeros=zeros, bias=bias, act=act)


def _linear8(name, dtype, B, nin, nout, group, zeros, bias, act, xgroup):
    return dict(_linear(name, dtype, B, nin, nout, group, zeros, bias, act), op="linear8", xgroup=xgroup)


def _rows(name, op, dtype, rows, cols, res, group=0):
    return dict(name=name, op=op, dtype=dtype, rows=rows, cols=cols, res=res, group=group)


def listed():
    return [
        # the norm in front of a layer while one token is produced: nothing but latency
        _rows("norm_token", "norm", "bf16", 1, 4096, True),
        # a handful of rows of an odd length, in the engine's default type, without a residual
        _rows("norm_odd", "norm", "fp32", 333, 5003, False),
        # the norm over a long prompt
        _rows("norm_prompt", "norm", "bf16", 16384, 8192, True),
        # the same norms where the Linear layer behind takes 8-bit activations
        _rows("norm8_tokens", "norm8", "fp16", 8, 4096, True),
        _rows("norm8_prompt", "norm8", "bf16", 8192, 4096, True, 128),
        # activations between two Linear layers, on their way into the second
        _rows("rows8_batch", "rows8", "fp16", 700, 9216, False),
        # the first Linear of VGG-16 for one image on the fp32 engine
        _linear("linear_image", "fp32", 1, 25088, 4096, 128, False, True, True),
        # a classifier for a ragged batch, small groups with zero points, a length that no vector divides
        _linear("linear_ragged", "fp16", 33, 4090, 1000, 32, True, True, False),
        # one token through a wide layer: as fast as the codes come from memory
        _linear("linear_token", "bf16", 1, 8192, 32768, 128, False, False, False),
        # a prompt through a square layer: as fast as the matrix cores multiply
        _linear("linear_prompt", "bf16", 4096, 8192, 8192, 128, False, False, False),
        # the same two ends with 8-bit activations
        _linear8("linear8_token", "fp16", 1, 4096, 16384, 128, False, True, True, 0),
        _linear8("linear8_prompt", "bf16", 1024, 8192, 8192, 128, True, False, False, 128),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "norm8", "rows8", "linear", "linear", "linear8", "linear8"])
    if op in ("norm", "norm8", "rows8"):
        cols = _log(rng, 64, 16384)
        if rng.random() < 0.5:
            cols = max(64, cols // 64 * 64)
        rows = _log(rng, 1, min(32768, 16384 * 8192 // cols))
        # (8-bit values of an fp32 tensor are not compared here: a value next to a border may fall on either side)
        dtype = rng.choice(["fp32", "fp16", "bf16"] if op == "norm" else ["fp16", "bf16"])
        group = rng.choice([0, 32, 64, 128, 256]) if op != "norm" else 0
        return dict(op=op, dtype=dtype, rows=rows, cols=cols, res=op != "rows8" and rng.random() < 0.7, group=group)
    nin, nout = _log(rng, 256, 25088), _log(rng, 256, 32768)
    if rng.random() < 0.7:
        nin = max(256, nin // 128 * 128)
    nout = min(nout, 8192 * 32768 // nin)
    B = _log(rng, 1, 4096)
    B = max(1, min(B, 4096 * 8192 * 8192 // 2 // (nin * nout)))
    case = dict(op=op, dtype=rng.choice(["fp32", "fp16", "bf16"]), B=B, nin=nin, nout=nout, group=rng.choice([0, 32, 64, 128, 128, 256]),
                zeros=rng.random() < 0.4, bias=rng.random() < 0.5, act=rng.random() < 0.5)
    if op == "linear8":
        case["xgroup"] = rng.choice([0, case["group"]])
    return case


def _groups(n, group):
    return 1 if group == 0 else -(-n // group)


def _made(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    g = _made(seed)
    dt = DTYPES[case["dtype"]]
    s = dict(case)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    if case["op"] in ("norm", "norm8", "rows8"):
        rows, cols = case["rows"], case["cols"]
        # a few columns are much larger than the rest, as in the residual stream of a deep network
        gain = 1 + 9 * (torch.rand(cols, generator=g, device="cuda") < 0.01).float()
        s["x"] = (normal(rows, cols) * gain).to(dt)
        s["r"] = normal(rows, cols).to(dt) if case["res"] else None
        s["w"] = 1 + 0.1 * normal(cols) if case["op"] != "rows8" else None
        s["sum"] = torch.empty_like(s["x"]) if case["res"] else None
        s["y"] = torch.empty_like(s["x"])
        if case["op"] != "norm":
            s["q"] = torch.empty((rows, cols), device="cuda", dtype=torch.int8)
            s["scale"] = torch.empty((rows, _groups(cols, case["group"])), device="cuda", dtype=torch.float32)
    else:
        B, nin, nout, group = case["B"], case["nin"], case["nout"], case["group"]
        n = _groups(nin, group)
        # codes of weights that are normally distributed: 8 is zero, three steps one standard deviation
        step = 4096 * 4096 // nin + 1
        s["codes"] = torch.empty((nout, (nin + 1) // 2), device="cuda", dtype=torch.uint8)
        for at in range(0, nout, step):
            c = (normal(min(step, nout - at), s["codes"].shape[1], 2) * 3 + 8).round_().clamp_(0, 15).to(torch.uint8)
            s["codes"][at:at + step] = c[..., 0] | (c[..., 1] << 4)
        s["scales"] = ((0.5 + torch.rand((nout, n), generator=g, device="cuda")) / (3 * math.sqrt(nin))).to(dt)
        s["zeros"] = torch.randint(5, 12, (nout, n), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        s["bias"] = 0.1 * normal(nout) if case["bias"] else None
        s["y"] = torch.empty((B, nout), device="cuda", dtype=dt)
        if case["op"] == "linear":
            s["x"] = normal(B, nin).to(dt)
        else:
            m = _groups(nin, case["xgroup"])
            s["q"] = (normal(B, nin) * 32).round_().clamp_(-127, 127).to(torch.int8)
            s["xs"] = (0.5 + torch.rand((B, m), generator=g, device="cuda")) / 32
    if own:
        _own_prepare(s)
    return s


def _own_prepare(s):
    """What a program keeps of the framework: the library, and a layer's weights in the order the kernels read them."""
    from thnets_amd import api
    s["lib"] = lib = api.load_library()
    s["ptr"] = p = {k: (s[k].data_ptr() if s.get(k) is not None else None)
                    for k in ("x", "r", "w", "sum", "y", "q", "scale", "codes", "scales", "zeros", "bias", "xs")}
    if s["op"] in ("linear", "linear8"):
        shape = (s["nout"], s["nin"], s["group"], CODE[s["dtype"]], 1 if s["zeros"] is not None else 0)
        s["packed"] = torch.empty(lib.thhip_w4_packed_bytes(*shape), device="cuda", dtype=torch.uint8)
        p["packed"] = s["packed"].data_ptr()
        if lib.thhip_w4_pack(p["codes"], p["scales"], p["zeros"], p["packed"], *shape[:4]) != 0:
            raise RuntimeError("thhip_w4_pack refused the layer")
        lib.thhip_sync()


def _own_run(s):
    lib, p, dt = s["lib"], s["ptr"], CODE[s["dtype"]]
    op = s["op"]
    if op == "linear":
        rc = lib.thhip_linear_w4(p["x"], s["nin"], p["packed"], p["bias"], p["y"], s["nout"], s["B"], s["nin"], s["nout"],
                                 s["group"], 1 if s["zeros"] is not None else 0, 1 if s["act"] else 0, 0.0, 0.0, dt)
    elif op == "linear8":
        rc = lib.thhip_linear_w4_i8(p["q"], s["nin"], p["xs"], s["xgroup"], p["packed"], p["bias"], p["y"], s["nout"], s["B"],
                                    s["nin"], s["nout"], s["group"], 1 if s["zeros"] is not None else 0, 1 if s["act"] else 0,
                                    0.0, 0.0, dt)
    elif op == "norm":
        c = s["cols"]
        rc = lib.thhip_rmsnorm(p["x"], c, p["r"], c, p["w"], EPS, p["sum"], c, p["y"], c, s["rows"], c, dt)
    else:
        c = s["cols"]
        if op == "norm8":
            rc = lib.thhip_rmsnorm_i8(p["x"], c, p["r"], c, p["w"], EPS, p["sum"], c, p["q"], c, p["scale"], s["group"], s["rows"], c, dt)
        else:
            rc = lib.thhip_quantize_rows(p["x"], c, p["q"], c, p["scale"], s["group"], s["rows"], c, dt)
        rc = rc or lib.thhip_dequantize_rows(p["q"], c, p["scale"], s["group"], p["y"], c, s["rows"], c, dt)
    if rc != 0:
        raise RuntimeError("the call was refused")
    return _outputs(s, s["y"], s.get("sum"), s.get("scale"))


def _outputs(s, y, total, scale):
    out = {"y": y}
    if total is not None:
        out["sum"] = total
    if scale is not None:
        out["scale"] = scale
    return out


def _spread(v, n, group):
    """A value a group -> a value a column."""
    return v.expand(v.shape[0], n) if group == 0 else v.repeat_interleave(group, 1)[:, :n]


def _weights(s, kind):
    """The layer's weights as numbers, [nOut][nIn]."""
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).reshape(s["nout"], -1)[:, :s["nin"]].to(kind)
    z = _spread(s["zeros"].to(kind), s["nin"], s["group"]) if s["zeros"] is not None else 8
    return (codes - z) * _spread(s["scales"].to(kind), s["nin"], s["group"])


def run(s):
    if own:
        return _own_run(s)
    dt, op = DTYPES[s["dtype"]], s["op"]
    if op in ("linear", "linear8"):
        x = s["x"].float() if op == "linear" else s["q"].float() * _spread(s["xs"], s["nin"], s["xgroup"])
        y = x @ _weights(s, torch.float32).T
        if s["bias"] is not None:
            y = y + s["bias"]
        if s["act"]:
            y = torch.where(y > 0, y, 0.0)
        return _outputs(s, y.to(dt), None, None)
    h = s["x"].float()
    if s["r"] is not None:
        h = h + s["r"].float()
    total = h.to(dt) if s["r"] is not None else None
    y = h if op == "rows8" else h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["w"]
    if op == "norm":
        return _outputs(s, y.to(dt), total, None)
    cols, group = s["cols"], s["group"]
    if group == 0:
        scale = y.abs().amax(1, keepdim=True) / 127
    else:
        n = _groups(cols, group)
        scale = torch.nn.functional.pad(y.abs(), (0, n * group - cols)).view(s["rows"], n, group).amax(2) / 127
    wide = _spread(scale, cols, group)
    return _outputs(s, (torch.round(y / wide) * wide).to(dt), total, scale)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("linear", "linear8"):
        B, nin, nout = case["B"], case["nin"], case["nout"]
        n = _groups(nin, case["group"])
        layer = nout * ((nin + 1) // 2) + nout * n * (size + (1 if case["zeros"] else 0)) + (4 * nout if case["bias"] else 0)
        x = B * nin * size if case["op"] == "linear" else B * nin + 4 * B * _groups(nin, case["xgroup"])
        return {"bytes": layer + x + B * nout * size, "flops": 2 * B * nin * nout}
    rows, cols = case["rows"], case["cols"]
    moved = rows * cols * size * (3 if case["res"] else 1) + (4 * cols if case["op"] != "rows8" else 0)
    if case["op"] == "norm":
        moved += rows * cols * size
    else:
        moved += rows * cols + 4 * rows * _groups(cols, case["group"])
    return {"bytes": moved, "flops": (6 if case["op"] != "rows8" else 3) * rows * cols}


def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    kind = torch.float64
    if case["op"] in ("linear", "linear8"):
        B, nin, nout, group = case["B"], case["nin"], case["nout"], case["group"]
        step = group or nin
        y = torch.zeros((B, nout), device="cuda", dtype=kind)
        if s["bias"] is not None:
            y += s["bias"].to(kind)
        for i in range(_groups(nin, group)):
            # group by group: the codes of its columns, their products, then the group's scale
            a, b = i * step, min(nin, (i + 1) * step)
            k = torch.arange(a, b, device="cuda")
            n = ((s["codes"][:, k // 2] >> (4 * (k % 2)).to(torch.uint8)) & 15).to(kind)
            n -= s["zeros"][:, i:i + 1].to(kind) if s["zeros"] is not None else 8
            if case["op"] == "linear":
                x = s["x"][:, a:b].to(kind)
            else:
                at = i if case["xgroup"] else 0
                x = s["q"][:, a:b].to(kind) * s["xs"][:, at:at + 1].to(kind)
            y += torch.mm(x, n.t().contiguous()) * s["scales"][:, i].to(kind)
        return {"y": y.clamp_(min=0) if case["act"] else y}
    rows, cols, group = case["rows"], case["cols"], case["group"]
    y = torch.empty((rows, cols), device="cuda", dtype=kind)
    total = torch.empty_like(y) if case["res"] else None
    scale = torch.empty((rows, _groups(cols, group)), device="cuda", dtype=kind) if case["op"] != "norm" else None
    some = max(1, (1 << 25) // cols)
    for at in range(0, rows, some):
        h = s["x"][at:at + some].to(kind)
        if s["r"] is not None:
            h = h + s["r"][at:at + some].to(kind)
            total[at:at + some] = h
        if case["op"] != "rows8":
            h = h / ((h.square().sum(1) / cols + EPS).sqrt())[:, None] * s["w"].to(kind)
        if scale is not None:
            for i, a in enumerate(range(0, cols, group or cols)):
                part = h[:, a:a + (group or cols)]
                top = torch.maximum(part.max(1)[0], -part.min(1)[0]) / 127
                scale[at:at + some, i] = top
                part.copy_((part / top[:, None]).round() * top[:, None])
        y[at:at + some] = h
    return _outputs(s, y, total, scale)

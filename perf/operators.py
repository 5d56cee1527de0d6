"""The operators over groups of rows and over 4-bit tables whose speed is measured.

A case is one call a user of this package makes on data in device memory:

* ``group``     rows sorted by the router they were sent to (``extension.group_rows``);
* ``grouped``   every row times the matrix of its group (``extension.project_grouped``),
                with ``train`` the gradients of rows and matrices too;
* ``quantize``  vectors to 4-bit blocks and back (``extension.quantize_fp4``,
                ``extension.dequantize_fp4``);
* ``scores``    queries times a 4-bit table, dense or one table per group
                (``extension.project_fp4``).

Sizes follow the package's own collections (96, 200 and 768 dimensions, routers of 32 x 32
and 64 x 64, batches of 1024, 16384 and 65536 queries) and go on to what a trained
encoder with one matrix per group multiplies.  Rows of a group are contiguous; how many
each group has is drawn from the seed, evenly or with a few groups that take most of them.
The tables are what a program quantises once and keeps; queries are quantised in the call.
"""
import math

import torch

own = False
DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
#: values per block scale
BLOCK = {"mxfp4": 32, "nvfp4": 16}
#: what the codes 0..7 stand for, and the borders between them (a tie goes to the even code)
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_FLOPS = 1.5e12          # of a drawn case
MOST_BYTES = 1.5e9


def _group(name, rows, groups, skew=0.0):
    return {"name": name, "op": "group", "rows": rows, "groups": groups, "skew": skew}


def _grouped(name, dtype, rows, groups, d, d_out, train=False, skew=0.0):
    return {"name": name, "op": "grouped", "dtype": dtype, "rows": rows, "groups": groups,
            "d": d, "d_out": d_out, "train": train, "skew": skew}


def _quantize(name, method, dtype, rows, d):
    return {"name": name, "op": "quantize", "method": method, "dtype": dtype, "rows": rows, "d": d}


def _scores(name, method, dtype, rows, d, d_out, out, groups=0, skew=0.0):
    return {"name": name, "op": "scores", "method": method, "dtype": dtype, "rows": rows, "d": d,
            "d_out": d_out, "out": out, "groups": groups, "skew": skew}


def listed():
    return [
        # the router of 64 x 64 has sent a batch of 1024 queries: latency is all that counts
        _group("group_1024", 1024, 64),
        # a collection of a million vectors put into its lists
        _group("group_million", 1_000_000, 1024, 1.0),
        # a batch of queries against the 64 leaves of each one's router, reduced space
        _grouped("leaves_f32", "f32", 1024, 64, 128, 64),
        # serving with a matrix per group, two rows a group: the matrices are read once
        _grouped("serve_bf16", "bf16", 128, 64, 2048, 1024),
        # a training step at odd sizes: 200 dimensions, rows of 333 values, ragged groups
        _grouped("train_odd_f16", "f16", 4099, 13, 200, 333, True, 0.5),
        # a training step of a 768-dimensional encoder with 32 groups, a few of them popular
        _grouped("train_bf16", "bf16", 16384, 32, 768, 2048, True, 1.0),
        # the largest training step: 65536 rows, 64 groups
        _grouped("train_large_bf16", "bf16", 65536, 64, 2048, 1792, True, 0.5),
        # queries of a batch to 4-bit blocks
        _quantize("quantize_batch", "mxfp4", "f32", 1024, 768),
        # a table of a quarter million vectors to 4-bit blocks
        _quantize("quantize_table", "nvfp4", "bf16", 262_144, 768),
        # one query against a 4-bit table that is read once
        _scores("scores_one", "mxfp4", "f32", 1, 768, 524_288, "f32"),
        # grouped 4-bit matrices, ragged and odd
        _scores("scores_grouped", "nvfp4", "bf16", 9973, 776, 1500, "bf16", 48, 0.5),
        # a large batch against a large 4-bit matrix
        _scores("scores_large", "mxfp4", "bf16", 16384, 4096, 8192, "bf16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    while True:
        op = rng.choice(["group", "grouped", "grouped", "quantize", "scores", "scores"])
        skew = rng.choice([0.0, 0.5, 1.0])
        if op == "group":
            case = _group("", _log(rng, 16, 1_000_000), _log(rng, 8, 1024), skew)
        elif op == "grouped":
            dtype = rng.choice(["bf16", "f16", "f32"])
            case = _grouped("", dtype, _log(rng, 1, 65536), _log(rng, 1, 128), _log(rng, 16, 4096),
                            _log(rng, 16, 4096), rng.random() < 0.5, skew)
            if rng.random() < 0.5:      # as models have it: multiples of eight
                case["d"], case["d_out"] = (-(-case[k] // 8) * 8 for k in ("d", "d_out"))
            if dtype == "f32" and work(case)["flops"] > MOST_FLOPS / 16:
                continue
        elif op == "quantize":
            case = _quantize("", rng.choice(list(BLOCK)), rng.choice(list(DTYPES)),
                             _log(rng, 1, 262_144), _log(rng, 16, 4096))
        else:
            groups = rng.choice([0, 0, _log(rng, 2, 64)])
            case = _scores("", rng.choice(list(BLOCK)), rng.choice(list(DTYPES)),
                           _log(rng, 1, 16384), _log(rng, 16, 4096),
                           _log(rng, 16, 4096 if groups else 262_144),
                           rng.choice(["f32", "bf16", "f16"]), groups, skew if groups else 0.0)
        cost = work(case)
        if cost["flops"] <= MOST_FLOPS and cost["bytes"] <= MOST_BYTES:
            del case["name"]
            return case


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "group":
        return {"bytes": 16 * rows + 8 * case["groups"], "flops": 0}
    d = case["d"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if op == "quantize":            # in; codes and scales out, in again; values out
        code = 0.5 + 1.0 / BLOCK[case["method"]]
        return {"bytes": rows * d * (size[case["dtype"]] + 2 * code + 4), "flops": 0}
    groups = max(1, case["groups"])
    used = groups * (1 - (1 - 1 / groups) ** rows)      # groups that have rows, on average
    if op == "grouped":
        s, w = size[case["dtype"]], used * d * case["d_out"]
        x, y = rows * d, rows * case["d_out"]
        flops = 2.0 * rows * d * case["d_out"]
        if not case["train"]:
            return {"bytes": s * (x + y + w), "flops": flops}
        # y; then dy, rows and matrices again, both gradients (of every group) out
        return {"bytes": s * (3 * x + 2 * y + 2 * w + groups * d * case["d_out"]), "flops": 3 * flops}
    code = 0.5 + 1.0 / BLOCK[case["method"]]
    return {"bytes": rows * d * size[case["dtype"]] + used * d * case["d_out"] * code
            + rows * case["d_out"] * size[case["out"]], "flops": 2.0 * rows * d * case["d_out"]}


# ---- inputs ------------------------------------------------------------------------
def _router_ids(g, rows, groups, skew):
    """A router id per row: group r is chosen with a weight of (r + 1) ** -skew, the
    popular ones spread over the ids."""
    weight = torch.arange(1, groups + 1, device=DEVICE, dtype=torch.float64) ** -skew
    weight = weight[torch.randperm(groups, generator=g, device=DEVICE)]
    edge = torch.cumsum(weight / weight.sum(), 0)
    u = torch.rand(rows, generator=g, device=DEVICE, dtype=torch.float64)
    return torch.searchsorted(edge, u).clamp_(max=groups - 1)


def _offsets(ids, groups):
    count = torch.bincount(ids, minlength=groups)
    return torch.cat([torch.zeros(1, dtype=torch.int64, device=DEVICE), torch.cumsum(count, 0)])


def _vectors(g, rows, d, dtype):
    """Embedding-like rows: a spectrum that falls as one over the dimension, unit norm times the
    root of their length, so that values are of order one."""
    scale = torch.arange(1, d + 1, device=DEVICE, dtype=torch.float32) ** -0.5
    scale = scale[torch.randperm(d, generator=g, device=DEVICE)]
    x = torch.randn(rows, d, generator=g, device=DEVICE) * scale
    return (x * (math.sqrt(d) / x.norm(dim=1, keepdim=True).clamp_min(1e-6))).to(DTYPES[dtype])


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))
    op, rows = case["op"], case["rows"]
    state = {"case": dict(case)}
    if op == "group":
        state["ids"] = _router_ids(g, rows, case["groups"], case["skew"])
        return state
    d = case["d"]
    x = _vectors(g, rows, d, case["dtype"])
    state["x"] = x
    if op == "quantize":
        return state
    groups, d_out = case["groups"], case["d_out"]
    if groups:
        ids = _router_ids(g, rows, groups, case["skew"])
        state["offsets"] = _offsets(ids, groups)
        # the most rows a group has: what a program that pads its groups allocates by
        state["most"] = int((state["offsets"][1:] - state["offsets"][:-1]).max())
    if op == "grouped":
        w = torch.randn(groups, d_out, d, generator=g, device=DEVICE) / math.sqrt(d)
        state["w"] = w.to(DTYPES[case["dtype"]])
        if case["train"]:
            state["dy"] = torch.randn(rows, d_out, generator=g, device=DEVICE).to(x.dtype)
            state["x"].requires_grad_(True)
            state["w"].requires_grad_(True)
        return state
    n = max(1, groups) * d_out          # the table, quantised once, in parts
    parts = [_quantize_plain(_vectors(g, min(n - at, 65536), d, "f32"), case["method"])
             for at in range(0, n, 65536)]
    codes, scales, row_scale = (torch.cat(p) if p[0] is not None else None for p in zip(*parts))
    shape = (groups, d_out) if groups else (d_out,)
    state["codes"] = codes.view(*shape, -1)
    state["scales"] = scales.view(*shape, -1)
    state["row_scale"] = None if row_scale is None else row_scale.view(*shape)
    return state


# ---- 4-bit blocks, plain ------------------------------------------------------------
def _fields(x, method):
    """Values of blocks [rows, blocks, size] as (codes 0..15, scale bytes, row scale): what a
    block format holds."""
    rows, d = x.shape
    size = BLOCK[method]
    x = torch.nn.functional.pad(x.float(), (0, -d % 32)).view(rows, -1, size)
    top = x.abs().amax(-1)
    row_scale = None
    if method == "mxfp4":
        exponent = (top.view(torch.int32) >> 23)
        byte = (exponent - 2).clamp_min(0)
        value = x * ((254 - byte) << 23).view(torch.float32).unsqueeze(-1)
        byte = torch.where(exponent == 255, exponent, byte)     # NaN or infinity: no scale
    else:
        # the least power of two that brings the row's largest value to 6 * 448 = 1.3125 * 2 ** 11
        most = top.amax(-1).view(torch.int32)
        power = (most >> 23) - 127 - 11 + ((most & 0x7fffff) > 0x280000).int()
        row_scale = ((power.clamp_min(-126) + 127) << 23).view(torch.float32)
        row_scale = torch.where((most >> 23) == 255, float("nan"), row_scale)
        ratio = (top / row_scale.unsqueeze(-1) / 6.0).clamp(max=448.0)
        block = ratio.to(torch.float8_e4m3fn)
        byte = block.view(torch.uint8)
        step = (block.float() * row_scale.unsqueeze(-1)).unsqueeze(-1)
        value = torch.where(step > 0, x / step, 0.0)
    a = value.abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int()
            + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int())
    return code + 8 * value.signbit().int(), byte.to(torch.uint8), row_scale


def _quantize_plain(x, method):
    """Codes two a byte (the even value in the low half), rows padded to whole blocks of 32."""
    code, byte, row_scale = _fields(x, method)
    code = code.view(x.size(0), -1).to(torch.uint8)
    return code[:, 0::2] | (code[:, 1::2] << 4), byte, row_scale


def _values_plain(codes, scales, row_scale, method, d):
    """What packed codes stand for, [rows, d] in 32 bits."""
    rows = codes.size(0)
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=codes.device)
    code = torch.stack([codes & 15, codes >> 4], dim=-1).view(rows, -1)
    value = level[code.int()].view(rows, scales.size(1), -1)
    if method == "mxfp4":
        e = scales.int()
        scale = torch.where(e > 0, (e << 23), 1 << 22).view(torch.float32)  # 2 ** -127 is subnormal
        scale = torch.where(e == 255, float("nan"), scale)
        value = value * scale.unsqueeze(-1)
    else:
        value = value * scales.view(torch.float8_e4m3fn).float().unsqueeze(-1)
        value = value * row_scale.view(-1, 1, 1)
    return value.reshape(rows, -1)[:, :d]


# ---- plain forms ----------------------------------------------------------------------
def _places(rows, offsets):
    """Group of each row and its place in the group."""
    at = torch.arange(rows, device=DEVICE)
    group = torch.searchsorted(offsets[1:], at, right=True)
    return group, at - offsets[group]


def _padded(x, group, place, groups, most):
    out = torch.zeros(groups, most, x.size(1), device=x.device)
    out[group, place] = x.float()
    return out


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "group":
        ids = state["ids"]
        order = torch.sort(ids, stable=True)[1]
        return {"order": order, "offsets": _offsets(ids, case["groups"])}
    x = state["x"].detach()
    rows, d = x.shape
    if op == "quantize":
        parts = _quantize_plain(x, case["method"])
        return {"values": _values_plain(*parts, case["method"], d)}
    if op == "grouped":
        w = state["w"].detach().float()
        groups = w.size(0)
        group, place = _places(rows, state["offsets"])
        xs = _padded(x, group, place, groups, state["most"])
        out = {"y": torch.bmm(xs, w.transpose(1, 2))[group, place].to(x.dtype)}
        if case["train"]:
            dys = _padded(state["dy"], group, place, groups, state["most"])
            out["dx"] = torch.bmm(dys, w)[group, place].to(x.dtype)
            out["dw"] = torch.bmm(dys.transpose(1, 2), xs).to(x.dtype)
        return out
    method = case["method"]
    values = _values_plain(*_quantize_plain(x, method), method, d)
    codes, scales, row_scale = state["codes"], state["scales"], state["row_scale"]
    table = _values_plain(codes.view(-1, codes.size(-1)), scales.view(-1, scales.size(-1)),
                          row_scale, method, d)
    if not case["groups"]:
        return {"scores": (values @ table.T).to(DTYPES[case["out"]])}
    group, place = _places(rows, state["offsets"])
    xs = _padded(values, group, place, case["groups"], state["most"])
    table = table.view(case["groups"], -1, d)
    return {"scores": torch.bmm(xs, table.transpose(1, 2))[group, place].to(DTYPES[case["out"]])}


def _framework(state):
    from pilotann_b200 import extension
    case = state["case"]
    op = case["op"]
    if op == "group":
        order, offsets = extension.group_rows(state["ids"], case["groups"])
        return {"order": order, "offsets": offsets}
    x = state["x"]
    if op == "quantize":
        return {"values": extension.dequantize_fp4(extension.quantize_fp4(x, case["method"]))}
    if op == "grouped":
        w = state["w"]
        y = extension.project_grouped(x, w, state["offsets"])
        if not case["train"]:
            return {"y": y}
        dx, dw = torch.autograd.grad(y, (x, w), state["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    table = extension.Fp4Table(state["codes"], state["scales"], state["row_scale"], case["d"],
                               case["method"])
    return {"scores": extension.project_fp4(x, table, state.get("offsets"),
                                            dtype=DTYPES[case["out"]])}


def run(state):
    return _framework(state) if own else _plain(state)


# ---- the definition in 64 bits ----------------------------------------------------------
def _two_to(power):
    """Powers of two, by their bits (a library's exponential may be off in the last place)."""
    return ((power.long() + 1023) << 52).view(torch.float64)


def _fp4_exact(x, method):
    """What the nearest 4-bit block values of x [rows, d] stand for."""
    rows, d = x.shape
    size = BLOCK[method]
    level = torch.tensor(LEVELS, device=x.device, dtype=torch.float64)
    out = torch.empty(rows, d, device=x.device, dtype=torch.float64)
    for at in range(0, rows, 16384):
        part = x[at:at + 16384].double()
        n = part.size(0)
        blocks = torch.nn.functional.pad(part, (0, -d % size)).view(n, -1, size)
        top = blocks.abs().amax(-1, keepdim=True)
        if method == "mxfp4":
            power = torch.frexp(top)[1] - 1                     # of the leading bit
            step = _two_to(torch.where(top > 0, power, -125).clamp(min=-125) - 2)
        else:
            part, power = torch.frexp(top.amax(1, keepdim=True) / 2688.0)
            row = _two_to((power - (part == 0.5).int()).clamp(min=-126))
            ratio = (top / (6.0 * row)).clamp(max=448.0)
            step = ratio.float().to(torch.float8_e4m3fn).double() * row
        value = (blocks / step).nan_to_num(0.0)
        # nearest level; of two at the same distance the one with the even index
        far = (value.abs().clamp(max=6.0).unsqueeze(-1) - level).abs()
        far = far + torch.tensor([0.0, 1e-12] * 4, device=x.device, dtype=torch.float64)
        near = level[far.argmin(-1)]
        out[at:at + n] = (near.copysign(value) * step).view(n, -1)[:, :d]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "group":
        ids = state["ids"].cpu()
        order = torch.argsort(ids * case["rows"] + torch.arange(case["rows"]))
        edges = [int((ids < r).sum()) for r in range(case["groups"] + 1)]
        return {"order": order, "offsets": torch.tensor(edges)}
    x = state["x"].detach()
    d = x.size(1)
    if op == "quantize":
        return {"values": _fp4_exact(x, case["method"])}
    if op == "grouped":
        w = state["w"].detach()
        y = torch.empty(x.size(0), case["d_out"], device=DEVICE, dtype=torch.float64)
        dx = torch.empty(x.size(0), d, device=DEVICE, dtype=torch.float64)
        dw = torch.zeros(w.shape, device=DEVICE, dtype=torch.float64)
        edges = state["offsets"].tolist()
        for r, (lo, hi) in enumerate(zip(edges, edges[1:])):
            mine, weight = x[lo:hi].double(), w[r].double()
            y[lo:hi] = mine @ weight.T
            if case["train"]:
                dy = state["dy"][lo:hi].double()
                dx[lo:hi] = dy @ weight
                dw[r] = dy.T @ mine
        return {"y": y, "dx": dx, "dw": dw} if case["train"] else {"y": y}
    method = case["method"]
    size = BLOCK[method]
    values = _fp4_exact(x, method)
    level = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device=DEVICE, dtype=torch.float64)

    def table(codes, scales, row_scale):
        code = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(1).long()
        if method == "mxfp4":
            scale = _two_to(scales.long() - 127)
        else:
            scale = scales.view(torch.float8_e4m3fn).double() * row_scale.double().unsqueeze(1)
        return (level[code] * scale.repeat_interleave(size, 1))[:, :d]

    codes, scales, row_scale = state["codes"], state["scales"], state["row_scale"]
    out = torch.empty(x.size(0), case["d_out"], device=DEVICE, dtype=torch.float64)
    if not case["groups"]:
        for at in range(0, case["d_out"], 32768):
            part = slice(at, at + 32768)
            out[:, part] = values @ table(codes[part], scales[part],
                                          None if row_scale is None else row_scale[part]).T
        return {"scores": out}
    edges = state["offsets"].tolist()
    for r, (lo, hi) in enumerate(zip(edges, edges[1:])):
        out[lo:hi] = values[lo:hi] @ table(codes[r], scales[r],
                                           None if row_scale is None else row_scale[r]).T
    return {"scores": out}

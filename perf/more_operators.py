"""Gated feed-forward blocks and products in 8-bit floating point: the workloads by which their speed is judged.

A case is one pass through operators of ``cumpsgemm_b200.experts`` on row-major torch CUDA tensors: rows
(tokens) sorted by the expert they go to, ``group_ends`` (int32, on the device) holding the running total of rows
after each expert.  gate_up is (groups, 2 * hidden, width): an expert's rows of the gate, then those of the
projection that it gates; down is (groups, width, hidden).

Fields of a case
  op       "gated"     h = act(x gate_e^T) * (x up_e^T) for the rows of each expert e: ``gated_matmul``
           "block"     y = h down_e^T, and from the gradient of y those of x, gate_up and down:
                       ``gated_feed_forward``, as a training step runs it
           "f8"        rows brought to 8-bit floating point with a scale for each 128 values, then the product
                       with 8-bit weights (groups, hidden, width) that have a scale for each 128 x 128:
                       ``quantize_blocks``, ``f8_matmul``
           "f8_block"  the whole block with such operands: ``quantize_blocks``, ``f8_gated_matmul``,
                       ``f8_matmul``
  dtype    of x, the weights, the gradients ("f8", "f8_block": of x; the output is bfloat16)
  rows, width, hidden, groups   x is (rows, width); spare = rows behind the last expert's, which belong to none
           and whose results are zero
  activation  "silu", "gelu", "gelu_tanh" or "relu"
  skew     0: every expert gets about as many rows; the larger, the more of them go to a few
  mode     how FP32 operands are multiplied
  magnitude  of the gradient of y
  topk     "f8", "f8_block": 0: row r of x is used as row r; > 0: x has rows / topk tokens, each used by that
           many experts through a row index

Sizes are those of the sweep, the example and the tests of this repository, and generic ones.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST_FLOPS = {"gated": 4.0 * 32768 * 4096 * 4096, "block": 18.0 * 16384 * 4096 * 4096,
               "f8": 2.0 * 8192 ** 3, "f8_block": 6.0 * 32764 * 2048 * 4096}
_MOST_WEIGHTS = 1 << 30  # elements
_TOP = 448.0             # largest magnitude of e4m3

_handle = None


def _get_handle():
    """The one handle a program creates and keeps."""
    global _handle
    if _handle is None:
        from cumpsgemm_b200 import api

        _handle = api.Handle()
        _handle.use_current_torch_stream()
    return _handle


def _case(op, rows, width, hidden, groups=1, dtype="bf16", activation="silu", spare=0, skew=0.0, mode="FP16TCEC",
          magnitude=1.0, topk=0, name=None):
    c = dict(op=op, rows=rows, width=width, hidden=hidden, groups=groups, dtype=dtype, activation=activation,
             spare=spare, skew=skew, mode=mode, magnitude=magnitude, topk=topk)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # the gated half of a dense block for one token: latency, and the weights' way from memory
        _case("gated", 1, 4096, 4096, name="gated_one_row"),
        # decoding a batch: a few rows for each of many experts
        _case("gated", 256, 2048, 2048, 64, dtype="fp16", activation="gelu", skew=0.5, name="gated_decode"),
        # a long prompt: the largest of this kind
        _case("gated", 32768, 4096, 4096, 16, skew=0.5, name="gated_prompt"),
        # a training step of a small layer: seven products of a few microseconds each
        _case("block", 512, 1024, 1024, 8, skew=0.5, magnitude=0.01, name="block_small"),
        # a training step of a large layer: the largest of all
        _case("block", 16384, 4096, 4096, 16, skew=0.5, magnitude=0.01, name="block_train"),
        # rows that fill no tile, most of them in a few experts, a buffer with room to spare
        _case("block", 4099, 1000, 1496, 32, dtype="fp16", activation="gelu_tanh", skew=1.5, spare=29,
              magnitude=0.01, name="block_ragged"),
        # FP32 master copies whose gradients need scaling, nothing a multiple of anything
        _case("block", 1999, 777, 1501, 6, dtype="fp32", skew=0.5, magnitude=1e-6, mode="FP16TCEC_SCALING",
              name="block_fp32_ragged"),
        # one token through one linear layer with 8-bit weights
        _case("f8", 1, 4096, 4096, name="f8_one_row"),
        # a linear layer with 8-bit weights over a long prompt: the largest product
        _case("f8", 8192, 8192, 8192, name="f8_prompt"),
        # experts with 8-bit weights, sizes that end inside a block of 128, tokens in float16
        _case("f8", 3996, 2777, 3001, 12, dtype="fp16", skew=1.5, topk=4, name="f8_ragged"),
        # decoding a batch through gated experts with 8-bit weights
        _case("f8_block", 256, 4096, 2048, 32, skew=0.5, topk=4, name="f8_block_decode"),
        # gated experts with 8-bit weights over a long prompt
        _case("f8_block", 32764, 2048, 4096, 16, skew=0.5, topk=4, name="f8_block_prompt"),
    ]


def _log_size(rng, lo, hi):
    """Spread over the logarithm; half of them left as they come, half rounded to a multiple of 32."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    return v if rng.random() < 0.5 else max(lo, (v + 16) // 32 * 32)


def draw(rng):
    op = rng.choice(["gated", "block", "f8", "f8_block"])
    rows = _log_size(rng, 1, 32768)
    width, hidden = _log_size(rng, 64, 8192), _log_size(rng, 64, 8192)
    groups = max(1, int(round(64 ** rng.random())))
    topk = 0
    if op in ("f8", "f8_block"):
        if rng.random() < 0.4:
            groups = 1
        else:
            topk = rng.choice([1, 2, 4, 8])
            rows = (rows + topk - 1) // topk * topk
    dtype = rng.choice(["bf16", "bf16", "fp16"] if op in ("f8", "f8_block") else ["bf16", "bf16", "fp16", "fp32"])
    c = _case(op, rows, width, hidden, groups, dtype=dtype,
              activation=rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]),
              spare=0 if op in ("f8", "f8_block") else rng.choice([0, 0, 7, 64]), skew=rng.choice([0.0, 0.5, 1.5]),
              mode=rng.choice(["FP16TCEC", "FP16TCEC_SCALING"]) if dtype == "fp32" else "FP16TCEC",
              magnitude=0.01 if op == "block" else 1.0, topk=topk)
    per = {"gated": 2, "block": 3, "f8": 1, "f8_block": 3}[op] * width * hidden
    while c["groups"] * per > _MOST_WEIGHTS:
        c["groups"] = max(1, c["groups"] // 2)
    while work(c)["flops"] > _MOST_FLOPS[op] / (4 if dtype == "fp32" else 1):
        c["rows"] = max(1, c["rows"] // 2 // max(1, topk)) * max(1, topk)
    return c


def _counts(case):
    """Rows of each expert, largest first: shares that fall off as a power of the rank."""
    e, rows = case["groups"], case["rows"]
    r = random.Random("%d %d %s" % (rows, e, case["skew"]))
    share = [(i + 1.0) ** -case["skew"] * r.uniform(0.7, 1.3) for i in range(e)]
    whole, at, counts, before = sum(share), 0.0, [], 0
    for s in share:
        at += s / whole
        upto = rows if len(counts) == e - 1 else min(rows, int(round(at * rows)))
        counts.append(upto - before)
        before = upto
    return counts


def _blocks(v):
    return (v + 127) // 128


def work(case):
    rows, w, h, e = case["rows"], case["width"], case["hidden"], case["groups"]
    size = _DTYPES[case["dtype"]].itemsize
    used = sum(c > 0 for c in _counts(case))
    total = rows + case["spare"]
    if case["op"] == "gated":  # x, gate_up; h
        return {"bytes": (rows * w + used * 2 * h * w + total * h) * size, "flops": 4.0 * rows * w * h}
    if case["op"] == "block":  # x, dy, the weights of experts with rows; y, dx, all weight gradients
        moved = rows * 2 * w + used * 3 * h * w + total * 2 * w + e * 3 * h * w
        return {"bytes": moved * size, "flops": 18.0 * rows * w * h}
    tokens = rows // max(1, case["topk"])
    read = tokens * w * size + (rows * 4 if case["topk"] else 0)
    if case["op"] == "f8":
        read += used * (h * w + 4 * _blocks(h) * _blocks(w))
        return {"bytes": read + rows * h * 2 + rows * _blocks(w) * 4, "flops": 2.0 * rows * w * h}
    read += used * (3 * h * w + 4 * (_blocks(2 * h) * _blocks(w) + _blocks(w) * _blocks(h)))
    return {"bytes": read + rows * w * 2, "flops": 6.0 * rows * w * h}


def _block_weights(w):
    """8-bit weights with a scale for each 128 x 128, as a checkpoint holds them."""
    n, k = w.shape
    nb, kb = _blocks(n), _blocks(k)
    t = torch.zeros(nb * 128, kb * 128, device=w.device)
    t[:n, :k] = w
    t = t.view(nb, 128, kb, 128)
    scale = t.abs().amax((1, 3)) / _TOP
    q = (t / scale[:, None, :, None].clamp(min=1e-30)).clamp(-_TOP, _TOP).reshape(nb * 128, kb * 128)[:n, :k]
    return q.to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, w, h, e = case["rows"], case["width"], case["hidden"], case["groups"]
    dtype, total = _DTYPES[case["dtype"]], case["rows"] + case["spare"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale)

    counts = _counts(case)
    random.Random(seed).shuffle(counts)  # which expert is the busy one changes
    s = dict(case=dict(case), counts=counts, ends=torch.tensor(counts).cumsum(0).to(torch.int32).cuda())
    if case["op"] in ("f8", "f8_block"):
        tokens = rows // max(1, case["topk"])
        x = normal(tokens, w)
        x[:, torch.randperm(w, generator=g, device="cuda")[: max(1, w // 128)]] *= 20.0  # channels with outliers
        s["x"] = x.to(dtype)
        if case["topk"]:
            s["index"] = (torch.randperm(rows, generator=g, device="cuda") // case["topk"]).to(torch.int32)
        shapes = {"w": (h, w)} if case["op"] == "f8" else {"gate_up": (2 * h, w), "down": (w, h)}
        for name, (n, k) in shapes.items():
            q = torch.empty(e, n, k, dtype=torch.float8_e4m3fn, device="cuda")
            scale = torch.empty(e, _blocks(n), _blocks(k), device="cuda")
            for i in range(e):
                q[i], scale[i] = _block_weights(normal(n, k, scale=k ** -0.5))
            s[name], s[name + "_scale"] = q, scale
        return s
    s["x"] = normal(total, w).to(dtype)
    s["gate_up"] = torch.empty(e, 2 * h, w, dtype=dtype, device="cuda")
    for i in range(e):
        s["gate_up"][i] = normal(2 * h, w, scale=w ** -0.5)
    if case["op"] == "block":
        s["down"] = torch.empty(e, w, h, dtype=dtype, device="cuda")
        for i in range(e):
            s["down"][i] = normal(w, h, scale=h ** -0.5)
        s["dy"] = normal(total, w, scale=case["magnitude"]).to(dtype)
    return s


def _run_own(s):
    from cumpsgemm_b200 import api, experts

    c, handle = s["case"], _get_handle()
    how = dict(activation=c["activation"])
    if c["op"] in ("f8", "f8_block"):
        ends = s["ends"] if c["topk"] else None
        q, scale = experts.quantize_blocks(handle, s["x"], row_index=s.get("index"))
        if c["op"] == "f8":
            return {"y": experts.f8_matmul(handle, q, scale, s["w"], s["w_scale"], ends), "x_scale": scale}
        q, scale = experts.f8_gated_matmul(handle, q, scale, s["gate_up"], s["gate_up_scale"], ends, **how)
        return {"y": experts.f8_matmul(handle, q, scale, s["down"], s["down_scale"], ends)}
    how["mode"] = api.ComputeMode[c["mode"]]
    if c["op"] == "gated":
        return experts.gated_matmul(handle, s["x"], s["gate_up"], s["ends"], **how)
    x, gate_up, down = (s[n].detach().requires_grad_() for n in ("x", "gate_up", "down"))
    y = experts.gated_feed_forward(handle, x, gate_up, down, s["ends"], **how)
    dx, dgate_up, ddown = torch.autograd.grad(y, (x, gate_up, down), s["dy"])
    return {"y": y.detach(), "dx": dx, "dgate_up": dgate_up, "ddown": ddown}


def _padded(s):
    """(experts, most rows of one) row numbers, and which of them are rows of that expert."""
    ends = s["ends"].long()
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    at = starts[:, None] + torch.arange(max(s["counts"]), device=ends.device)
    return at, at < ends[:, None]


def _side_by_side(s, x):
    """(experts, most rows of one, columns): the rows of each expert in 32 bits, zeros behind them."""
    at, real = _padded(s)
    return torch.where(real[..., None], x[at.clamp(max=x.shape[0] - 1)].float(), 0.0)


def _back(s, y, total):
    """Such rows in their places, zeros where a row belongs to no expert."""
    at, real = _padded(s)
    out = y.new_zeros(total, y.shape[2])
    out[at[real]] = y[real]
    return out


def _act(name, v):
    """The activation and its derivative."""
    if name == "relu":
        return v.clamp(min=0.0), (v > 0).to(v.dtype)
    if name == "silu":
        p = 1.0 / (1.0 + torch.exp(-v))
        return v * p, p * (1.0 + v * (1.0 - p))
    if name == "gelu":
        p = 0.5 * (1.0 + torch.erf(v * math.sqrt(0.5)))
        return v * p, p + v * torch.exp(-0.5 * v * v) * (2.0 * math.pi) ** -0.5
    r = math.sqrt(2.0 / math.pi)
    t = torch.tanh(r * (v + 0.044715 * v * v * v))
    return 0.5 * v * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * r * (1.0 + 3 * 0.044715 * v * v)


def _quantised(x):
    """Rows as the 8-bit values stand for, divided by their scales, and the scales; columns filled up to 128."""
    rows, k = x.shape
    t = torch.nn.functional.pad(x, (0, _blocks(k) * 128 - k)).view(rows, _blocks(k), 128)
    top = t.abs().amax(2, keepdim=True)
    q = torch.where(top > 0, t * _TOP / top, t)
    return q.to(torch.float8_e4m3fn).float(), top[..., 0] / _TOP


def _plain_f8(s, q, scale, w, w_scale):
    """Rows of each expert in 32 bits times its weights, each with its scales."""
    rows = (q * scale[..., None]).flatten(1)
    e, n, k = w.shape
    spread = w_scale.repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :n, :k]
    return _back(s, torch.bmm(_side_by_side(s, rows[:, :k]), (w.float() * spread).transpose(1, 2)), rows.shape[0])


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    dtype, total, h = _DTYPES[c["dtype"]], c["rows"] + c["spare"], c["hidden"]
    if c["op"] in ("f8", "f8_block"):
        q, scale = _quantised(s["x"].float())
        if c["topk"]:
            q, scale = q[s["index"].long()], scale[s["index"].long()]
        if c["op"] == "f8":
            return {"y": _plain_f8(s, q, scale, s["w"], s["w_scale"]).to(torch.bfloat16), "x_scale": scale}
        pre = _plain_f8(s, q, scale, s["gate_up"], s["gate_up_scale"])
        q, scale = _quantised(_act(c["activation"], pre[:, :h])[0] * pre[:, h:])
        return {"y": _plain_f8(s, q, scale, s["down"], s["down_scale"]).to(torch.bfloat16)}
    gate_up = s["gate_up"].float()
    x = _side_by_side(s, s["x"])
    pre = torch.bmm(x, gate_up.transpose(1, 2))
    act, slope = _act(c["activation"], pre[..., :h])
    hid = act * pre[..., h:]
    if c["op"] == "gated":
        return _back(s, hid, total).to(dtype)
    down, dy = s["down"].float(), _side_by_side(s, s["dy"])
    y = torch.bmm(hid, down.transpose(1, 2))
    dhid = torch.bmm(dy, down)
    dpre = torch.cat([dhid * pre[..., h:] * slope, dhid * act], 2)
    return {"y": _back(s, y, total).to(dtype), "dx": _back(s, torch.bmm(dpre, gate_up), total).to(dtype),
            "dgate_up": torch.bmm(dpre.transpose(1, 2), x).to(dtype),
            "ddown": torch.bmm(dy.transpose(1, 2), hid).to(dtype)}


def _exact_act(name, v):
    f = torch.nn.functional
    return {"silu": f.silu, "gelu": f.gelu, "relu": f.relu,
            "gelu_tanh": lambda t: f.gelu(t, approximate="tanh")}[name](v)


def _exact_rounded(x):
    """What rows stand for when they have been brought to 8 bits, and the scales, by blocks of columns."""
    values, scales = [], []
    for part in x.split(128, 1):
        step = part.abs().amax(1, keepdim=True) / _TOP
        q = torch.where(step > 0, part / step, part)
        values.append(q.float().to(torch.float8_e4m3fn).double() * step)
        scales.append(step)
    return torch.cat(values, 1), torch.cat(scales, 1)


def _exact_weights(q, scale):
    n, k = q.shape
    rows, cols = torch.arange(n, device=q.device) // 128, torch.arange(k, device=q.device) // 128
    return q.double() * scale.double()[rows][:, cols]


def exact(case, seed):
    s = prepare(case, seed)
    total, h = case["rows"] + case["spare"], case["hidden"]
    ends = s["ends"].tolist()
    spans = list(zip([0] + ends[:-1], ends))
    x = s["x"].double()
    if case["op"] in ("f8", "f8_block"):
        x, scale = _exact_rounded(x)
        if case["topk"]:
            x, scale = x[s["index"].long()], scale[s["index"].long()]
        y = x.new_zeros(total, h if case["op"] == "f8" else case["width"])
        for i, (a, b) in enumerate(spans):
            if case["op"] == "f8":
                y[a:b] = x[a:b] @ _exact_weights(s["w"][i], s["w_scale"][i]).t()
                continue
            pre = x[a:b] @ _exact_weights(s["gate_up"][i], s["gate_up_scale"][i]).t()
            hid = _exact_rounded(_exact_act(case["activation"], pre[:, :h]) * pre[:, h:])[0]
            y[a:b] = hid @ _exact_weights(s["down"][i], s["down_scale"][i]).t()
        return {"y": y, "x_scale": scale} if case["op"] == "f8" else {"y": y}
    if case["op"] == "gated":
        hid = x.new_zeros(total, h)
        for i, (a, b) in enumerate(spans):
            gate, up = s["gate_up"][i].double().split(h)
            hid[a:b] = _exact_act(case["activation"], x[a:b] @ gate.t()) * (x[a:b] @ up.t())
        return hid
    dy = s["dy"].double()
    y, dx, dgate_up, ddown = torch.zeros_like(x), torch.zeros_like(x), [], []
    for i, (a, b) in enumerate(spans):
        leaves = [t.double().detach().requires_grad_() for t in (x[a:b], s["gate_up"][i], s["down"][i])]
        gate, up = leaves[1].split(h)
        out = (_exact_act(case["activation"], leaves[0] @ gate.t()) * (leaves[0] @ up.t())) @ leaves[2].t()
        grads = torch.autograd.grad(out, leaves, dy[a:b])
        y[a:b], dx[a:b] = out.detach(), grads[0]
        dgate_up.append(grads[1])
        ddown.append(grads[2])
    return {"y": y, "dx": dx, "dgate_up": torch.stack(dgate_up), "ddown": torch.stack(ddown)}

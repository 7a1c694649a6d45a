"""Products of a mixture-of-experts layer: the workloads by which their speed is judged.

A case is one pass through one operator of ``cumpsgemm_b200.experts`` on row-major torch CUDA
tensors: rows (tokens) sorted by the expert they go to, ``group_ends`` (int32, on the device)
holding the running total of rows after each expert.

Fields of a case
  op       "matmul"  y = x w_e for the rows of each expert e: ``grouped_matmul``
           "wgrad"   dw_e = x_e^T dy_e, the gradient of the weights: ``grouped_matmul_wgrad``
           "i8"      rows brought to 8-bit integers with a scale each, then the integer product
                     with 8-bit weights that have a scale for each output channel:
                     ``quantize_rows``, ``i8_matmul``
  dtype    of x, w, dy ("i8": of x; the output is bfloat16)
  rows, n, k, groups   x is (rows, k), y (rows, n), w (groups, k, n), or (groups, n, k) where
           transpose_w is true ("i8": always); spare = rows behind the last expert's, which
           belong to none and whose output is zero
  skew     0: every expert gets about as many rows; the larger, the more of them go to a few
  mode     how FP32 operands are multiplied
  magnitude  of x, and of dy: activations are of order one, gradients are not
  topk     "i8": 0: row r of x is used as row r (one expert, a plain linear layer); > 0: x has
           rows / topk tokens, each used by that many experts through a row index

Sizes are those of the sweep and the tests of this repository, and generic ones.
"""
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_MOST_FLOPS = 2 * 32768 * 4096 * 4096  # of the largest listed cases
_MOST_WEIGHTS = 1 << 29                # elements

_handle = None


def _get_handle():
    """The one handle a program creates and keeps."""
    global _handle
    if _handle is None:
        from cumpsgemm_b200 import api

        _handle = api.Handle()
        _handle.use_current_torch_stream()
    return _handle


def _case(op, rows, n, k, groups=1, dtype="bf16", transpose_w=False, spare=0, skew=0.0,
          mode="FP16TCEC", magnitude=1.0, topk=0, name=None):
    c = dict(op=op, rows=rows, n=n, k=k, groups=groups, dtype=dtype, transpose_w=transpose_w,
             spare=spare, skew=skew, mode=mode, magnitude=magnitude, topk=topk)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one step of a few sequences through a small layer: launch and latency
        _case("matmul", 16, 1024, 1024, 8, transpose_w=True, skew=0.5, name="matmul_few_rows"),
        # decoding a batch: a few rows for each of many experts, the weights are the traffic
        _case("matmul", 256, 2048, 4096, 64, skew=0.5, name="matmul_decode"),
        # a long prompt, or the forward pass of training: the largest
        _case("matmul", 32768, 4096, 4096, 16, skew=0.5, name="matmul_prompt"),
        # gradient of a layer's input, rows that fill no tile, a buffer with room to spare
        _case("matmul", 8191, 2048, 8192, 32, dtype="fp16", transpose_w=True, skew=1.0, spare=100,
              magnitude=0.01, name="matmul_input_grad"),
        # FP32 master copies, nothing a multiple of anything
        _case("matmul", 1999, 3001, 2777, 6, dtype="fp32", skew=0.5, mode="FP16TCEC_SCALING",
              name="matmul_fp32_ragged"),
        # gradient of the weights of the largest layer
        _case("wgrad", 32768, 4096, 4096, 16, skew=0.5, magnitude=0.01, name="wgrad_prompt"),
        # many experts, most of the rows in a few of them and none in others
        _case("wgrad", 4099, 2000, 1000, 64, dtype="fp16", skew=1.5, transpose_w=True, spare=29,
              magnitude=0.01, name="wgrad_ragged"),
        # FP32 gradients whose magnitude needs the operands scaled
        _case("wgrad", 2048, 1024, 1024, 8, dtype="fp32", skew=0.5, mode="FP16TCEC_SCALING",
              magnitude=1e-6, name="wgrad_fp32"),
        # one token through one quantised linear layer
        _case("i8", 1, 4096, 4096, name="i8_one_row"),
        # decoding a batch through quantised experts
        _case("i8", 256, 2048, 4096, 32, topk=4, skew=0.5, name="i8_decode"),
        # a quantised linear layer over a long prompt: the largest
        _case("i8", 8192, 8192, 8192, name="i8_prompt"),
        # quantised experts over a long prompt
        _case("i8", 32764, 4096, 2048, 16, topk=4, skew=0.5, name="i8_experts_prompt"),
    ]


def _log_size(rng, lo, hi):
    """Spread over the logarithm; half of them left as they come, half rounded to a multiple of 32."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    return v if rng.random() < 0.5 else max(lo, (v + 16) // 32 * 32)


def draw(rng):
    op = rng.choice(["matmul", "matmul", "wgrad", "wgrad", "i8"])
    rows = _log_size(rng, 1, 32768)
    n, k = _log_size(rng, 64, 8192), _log_size(rng, 64, 8192)
    groups = max(1, int(round(64 ** rng.random())))
    topk = 0
    if op == "i8":
        if rng.random() < 0.4:
            groups = 1
        else:
            topk = rng.choice([1, 2, 4, 8])
            rows = (rows + topk - 1) // topk * topk
    while groups * n * k > _MOST_WEIGHTS:
        groups = max(1, groups // 2)
    while 2 * rows * n * k > _MOST_FLOPS:
        rows = max(1, rows // 2 // max(1, topk)) * max(1, topk)
    dtype = "bf16" if op == "i8" else rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if dtype == "fp32":
        rows = min(rows, 8192)
    return _case(op, rows, n, k, groups, dtype=dtype, transpose_w=rng.random() < 0.5,
                 spare=0 if op == "i8" else rng.choice([0, 0, 7, 64]),
                 skew=rng.choice([0.0, 0.5, 1.5]),
                 mode=rng.choice(["FP16TCEC", "FP16TCEC_SCALING"]) if dtype == "fp32" else "FP16TCEC",
                 magnitude=0.01 if op == "wgrad" else 1.0, topk=topk)


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


def work(case):
    rows, n, k, e = case["rows"], case["n"], case["k"], case["groups"]
    size = _DTYPES[case["dtype"]].itemsize
    used = sum(c > 0 for c in _counts(case))
    flops = 2.0 * rows * n * k
    if case["op"] == "i8":
        tokens = rows // max(1, case["topk"])
        read = tokens * k * size + (rows * 4 if case["topk"] else 0) + used * (n * k + n * 4)
        return {"bytes": read + rows * n * 2 + rows * 4, "flops": flops}
    if case["op"] == "wgrad":
        return {"bytes": (rows * (n + k) + e * n * k) * size, "flops": flops}
    return {"bytes": (rows * k + used * n * k + (rows + case["spare"]) * n) * size, "flops": flops}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rows, n, k, e = case["rows"], case["n"], case["k"], case["groups"]
    dtype, total = _DTYPES[case["dtype"]], case["rows"] + case["spare"]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda").mul_(scale)

    counts = _counts(case)
    random.Random(seed).shuffle(counts)  # which expert is the busy one changes
    ends = torch.tensor(counts).cumsum(0).to(torch.int32).cuda()
    s = dict(case=dict(case), counts=counts, ends=ends)
    if case["op"] == "i8":
        tokens = rows // max(1, case["topk"])
        x = normal(tokens, k)
        x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 128)]] *= 20.0  # channels with outliers
        s["x"] = x.to(dtype)
        if case["topk"]:
            s["index"] = (torch.randperm(rows, generator=g, device="cuda") // case["topk"]).to(torch.int32)
        s["wq"] = torch.empty(e, n, k, dtype=torch.int8, device="cuda")
        s["w_scale"] = torch.empty(e, n, device="cuda")
        for i in range(e):  # as a checkpoint holds them
            w = normal(n, k, scale=k ** -0.5)
            s["w_scale"][i] = w.abs().amax(1) / 127.0
            s["wq"][i] = torch.round(w / s["w_scale"][i][:, None]).clamp_(-127, 127).to(torch.int8)
        return s
    s["x"] = normal(total, k, scale=1.0 if case["op"] == "wgrad" else case["magnitude"]).to(dtype)
    if case["op"] == "wgrad":
        s["dy"] = normal(total, n, scale=case["magnitude"]).to(dtype)
    else:
        shape = (n, k) if case["transpose_w"] else (k, n)
        s["w"] = torch.empty(e, *shape, dtype=dtype, device="cuda")
        for i in range(e):
            s["w"][i] = normal(*shape, scale=k ** -0.5)
    return s


def _padded(s):
    """(experts, most rows of one) row numbers, and which of them are rows of that expert."""
    ends = s["ends"].long()
    starts = torch.cat([ends.new_zeros(1), ends[:-1]])
    at = starts[:, None] + torch.arange(max(s["counts"]), device=ends.device)
    return at, at < ends[:, None]


def _plain_matmul(s, x, w, total):
    """Rows of each expert side by side, one batched product, the rows back to their places."""
    at, real = _padded(s)
    y = torch.bmm(x[at.clamp(max=x.shape[0] - 1)].float(), w)
    out = y.new_zeros(total, w.shape[2])
    out[at[real]] = y[real]
    return out


def run(s):
    c = s["case"]
    if own:
        from cumpsgemm_b200 import api, experts

        h = _get_handle()
        if c["op"] == "i8":
            q, scale = experts.quantize_rows(h, s["x"], row_index=s.get("index"))
            y = experts.i8_matmul(h, q, scale, s["wq"], s["w_scale"], s["ends"] if c["topk"] else None)
            return {"y": y, "x_scale": scale}
        mode = api.ComputeMode[c["mode"]]
        if c["op"] == "wgrad":
            return experts.grouped_matmul_wgrad(h, s["x"], s["dy"], s["ends"],
                                                transpose_w=c["transpose_w"], mode=mode)
        return experts.grouped_matmul(h, s["x"], s["w"], s["ends"], transpose_w=c["transpose_w"],
                                      mode=mode)
    dtype, total = _DTYPES[c["dtype"]], c["rows"] + c["spare"]
    if c["op"] == "i8":
        x = s["x"].float()
        top = x.abs().amax(1, keepdim=True)
        q = torch.round(x * torch.where(top > 0, torch.full_like(top, 127.0) / top, top))
        scale = (top / 127.0)[:, 0]
        if c["topk"]:
            q, scale = q[s["index"].long()], scale[s["index"].long()]
        y = _plain_matmul(s, q, s["wq"].float().transpose(1, 2), total)
        at, real = _padded(s)
        expert = torch.arange(c["groups"], device=q.device)[:, None].expand_as(at)[real]
        return {"y": (y * scale[:, None] * s["w_scale"][expert]).to(torch.bfloat16), "x_scale": scale}
    if c["op"] == "wgrad":
        at, real = _padded(s)
        at = at.clamp(max=total - 1)
        x = torch.where(real[..., None], s["x"][at].float(), 0.0)
        dy = torch.where(real[..., None], s["dy"][at].float(), 0.0)
        dw = torch.bmm(dy.transpose(1, 2), x) if c["transpose_w"] else torch.bmm(x.transpose(1, 2), dy)
        return dw.to(dtype)
    w = s["w"].float()
    return _plain_matmul(s, s["x"], w.transpose(1, 2) if c["transpose_w"] else w, total).to(dtype)


def exact(case, seed):
    s = prepare(case, seed)
    total, n, k = case["rows"] + case["spare"], case["n"], case["k"]
    x = s["x"].double()
    ends = s["ends"].tolist()
    spans = list(zip([0] + ends[:-1], ends))
    if case["op"] == "wgrad":
        dy = s["dy"].double()
        parts = [x[a:b].t() @ dy[a:b] for a, b in spans]
        return torch.stack([p.t().contiguous() if case["transpose_w"] else p for p in parts])
    y = torch.zeros(total, n, dtype=torch.float64, device="cuda")
    if case["op"] == "i8":
        if case["topk"]:
            x = x[s["index"].long()]
        step = x.abs().amax(1) / 127
        q = (x / step.clamp(min=1e-300)[:, None]).round()
        for i, (a, b) in enumerate(spans):
            y[a:b] = (q[a:b] @ s["wq"][i].double().t()) * s["w_scale"][i].double() * step[a:b, None]
        return {"y": y, "x_scale": step}
    for i, (a, b) in enumerate(spans):
        w = s["w"][i].double()
        y[a:b] = x[a:b] @ (w.t() if case["transpose_w"] else w)
    return y

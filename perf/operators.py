"""Cases of the operators around the MoE block that a training step and a serving step need: layer norm, tokens sorted by
expert and back, and the orthogonalised update of stacked expert weights.

``run`` computes them either in plain torch operations (``own = False``) or through ``bibo_b200.functional`` (``own = True``).
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def listed():
    return [
        # one decoding step of eight sequences at the block's hidden size
        dict(name="norm_decode", op="norm", rows=8, hidden=2048, type="bf16", wtype="bf16", train=False, bias=True, pad=0),
        # the training batch of the benchmark configuration: forward and backward, norm weights kept in fp32
        dict(name="norm_train", op="norm", rows=32768, hidden=2048, type="bf16", wtype="fp32", train=True, bias=True, pad=0),
        # an odd hidden size read out of a wider tensor, fp32, weight without bias
        dict(name="norm_ragged", op="norm", rows=4097, hidden=1531, type="fp32", wtype="fp32", train=True, bias=False, pad=5),
        # eight decoding tokens through router output, expert order and back
        dict(name="route_decode", op="route", tokens=8, hidden=2048, experts=64, top_k=6, type="bf16", train=False, empty=0.0,
             align=1, skew=0.3),
        # the training batch of the benchmark configuration, both directions
        dict(name="route_train", op="route", tokens=32768, hidden=2048, experts=64, top_k=6, type="bf16", train=True, empty=0.0,
             align=1, skew=0.0),
        # a skewed router, slots dropped by a capacity limit, odd sizes, fp32
        dict(name="route_dropped", op="route", tokens=5003, hidden=1153, experts=40, top_k=3, type="fp32", train=True, empty=0.3,
             align=1, skew=1.0),
        # a prompt through many small experts, groups padded to the row tile of a grouped product
        dict(name="route_prefill", op="route", tokens=16384, hidden=1024, experts=256, top_k=8, type="bf16", train=False,
             empty=0.0, align=128, skew=0.5),
        # the router's own weight
        dict(name="ortho_router", op="ortho", batch=1, m=64, n=2048, type="fp32", steps=5),
        # odd sizes, a few matrices, taller than wide
        dict(name="ortho_odd", op="ortho", batch=3, m=1030, n=777, type="fp32", steps=5),
        # a dense layer's projection of the ten-layer model
        dict(name="ortho_dense", op="ortho", batch=1, m=4096, n=1024, type="bf16", steps=5),
        # down projections of all experts of the benchmark configuration
        dict(name="ortho_down", op="ortho", batch=64, m=2048, n=512, type="bf16", steps=5),
        # gate and up projections of all experts of the benchmark configuration
        dict(name="ortho_gate_up", op="ortho", batch=64, m=1024, n=2048, type="bf16", steps=5),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "route", "ortho"])
    dtype = rng.choice(["bf16", "fp32"])
    if op == "norm":
        hidden = _log(rng, 48, 16384)
        rows = _log(rng, 1, max(1, min(65536, (1 << 25) // hidden)))
        return dict(op=op, rows=rows, hidden=hidden, type=dtype, wtype=rng.choice([dtype, "fp32"]), train=rng.random() < 0.6,
                    bias=rng.random() < 0.7, pad=rng.choice([0, 0, 8, 3]))
    if op == "route":
        hidden, top_k = _log(rng, 48, 8192), rng.randint(1, 8)
        experts = _log(rng, max(8, top_k), 256)
        tokens = _log(rng, 1, max(1, min(65536, (1 << 27) // (hidden * top_k))))
        return dict(op=op, tokens=tokens, hidden=hidden, experts=experts, top_k=top_k, type=dtype, train=rng.random() < 0.6,
                    empty=rng.choice([0.0, 0.0, 0.2, 0.875]), align=rng.choice([1, 1, 16, 128]), skew=rng.choice([0.0, 0.5, 1.5]))
    m, n = _log(rng, 16, 4096), _log(rng, 16, 4096)
    most = (1 << 36) // (m * n * min(m, n))
    return dict(op=op, batch=_log(rng, 1, max(1, min(64, most))), m=m, n=n, type=dtype, steps=5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = _TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    state = dict(case)
    if case["op"] == "norm":
        rows, hidden = case["rows"], case["hidden"]
        # a residual stream: an offset per channel, and a few channels much larger than the rest
        gain = 1.0 + 20.0 * (torch.rand(hidden, generator=g, device="cuda") > 0.99)
        wide = torch.zeros(rows, hidden + case["pad"], device="cuda", dtype=dtype)
        wide[:, :hidden] = ((normal(rows, hidden) + 0.5 * normal(hidden)) * gain).to(dtype)
        wtype = _TYPES[case["wtype"]]
        state["x"] = wide[:, :hidden]
        state["weight"] = (1.0 + 0.2 * normal(hidden)).to(wtype)
        state["shift"] = (0.2 * normal(hidden)).to(wtype) if case["bias"] else None
        state["dy"] = (1e-2 * normal(rows, hidden)).to(dtype) if case["train"] else None
    elif case["op"] == "route":
        tokens, hidden, experts, top_k = case["tokens"], case["hidden"], case["experts"], case["top_k"]
        logits = normal(tokens, experts) - case["skew"] * torch.log1p(torch.arange(experts, device="cuda"))
        idx = torch.topk(logits, top_k, dim=1).indices.sort(dim=1).values
        weight = torch.sigmoid(torch.gather(logits, 1, idx))
        weight = weight / weight.sum(1, keepdim=True)
        if case["empty"]:
            idx = torch.where(torch.rand(tokens, top_k, generator=g, device="cuda") < case["empty"], -1, idx)
        rows = _rows_cap(case)
        state["idx"], state["weight"] = idx.to(torch.int32), weight
        state["x"] = normal(tokens, hidden).to(dtype)
        state["ys"] = normal(rows, hidden).to(dtype)          # the experts' results, in expert order
        if case["train"]:
            state["dout"] = (1e-2 * normal(tokens, hidden)).to(dtype)
            state["dxs"] = (1e-2 * normal(rows, hidden)).to(dtype)   # the experts' input gradients
    else:
        batch, m, n = case["batch"], case["m"], case["n"]
        # momentum of a weight gradient: a few strong directions with decaying strength over a broad floor
        r = min(16, m, n)
        strength = 1.0 / torch.arange(1, r + 1, device="cuda")
        update = torch.matmul(normal(batch, m, r) * strength, normal(batch, r, n))
        update += 0.1 * normal(batch, m, n)
        state["update"] = (1e-3 * update).to(dtype)
    return state


def _rows_cap(case):
    slots, align = case["tokens"] * case["top_k"], case["align"]
    rows = slots + min(slots, case["experts"]) * (align - 1)
    return (rows + align - 1) // align * align


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from bibo_b200 import functional as Fn
    if s["op"] == "norm":
        if not s["train"]:
            return {"y": Fn.layernorm_forward(s["x"], s["weight"], s["shift"], 1e-5)}
        y, saved = Fn.layernorm_forward(s["x"], s["weight"], s["shift"], 1e-5, keep=True)
        dx, dweight, dshift = Fn.layernorm_backward(s["dy"], s["x"], s["weight"], saved, has_bias=s["shift"] is not None)
        got = {"y": y, "dx": dx, "dweight": dweight}
        if dshift is not None:
            got["dshift"] = dshift
        return got
    if s["op"] == "route":
        plan = Fn.dispatch_plan(s["idx"], s["experts"], align=s["align"])
        got = {"offsets": plan.offsets, "slot_row": plan.slot_row, "xs": Fn.dispatch_forward(s["x"], plan),
               "out": Fn.combine_forward(s["ys"], s["weight"], plan)}
        if s["train"]:
            got["dys"], got["dweight"] = Fn.combine_backward(s["dout"], s["ys"], s["weight"], plan)
            got["dx"] = Fn.dispatch_backward(s["dxs"], plan)
        return got
    return {"update": Fn.orthogonalize(s["update"], steps=s["steps"])}


def _run_plain(s):
    if s["op"] == "norm":
        x, w = s["x"].float(), s["weight"].float()
        mean = x.mean(1, keepdim=True)
        centred = x - mean
        rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + 1e-5)
        xhat = centred * rstd
        y = xhat * w if s["shift"] is None else xhat * w + s["shift"].float()
        got = {"y": y.to(s["x"].dtype)}
        if s["train"]:
            dy = s["dy"].float()
            dxhat = dy * w
            dx = rstd * (dxhat - dxhat.mean(1, keepdim=True) - xhat * (dxhat * xhat).mean(1, keepdim=True))
            got["dx"] = dx.to(s["x"].dtype)
            got["dweight"] = (dy * xhat).sum(0).to(s["weight"].dtype)
            if s["shift"] is not None:
                got["dshift"] = dy.sum(0).to(s["shift"].dtype)
        return got
    if s["op"] == "route":
        tokens, top_k = s["idx"].shape
        experts, align, dtype = s["experts"], s["align"], s["x"].dtype
        slots, rows = tokens * top_k, s["ys"].shape[0]
        key = s["idx"].reshape(-1).long()
        key = torch.where(key < 0, experts, key)                      # empty slots sort behind the last expert
        key, order = torch.sort(key, stable=True)
        counts = torch.bincount(key, minlength=experts + 1)
        start = torch.cumsum(counts, 0) - counts
        padded = (counts[:experts] + align - 1) // align * align
        offsets = torch.cumsum(padded, 0) - padded
        row = torch.cat([offsets, offsets.new_zeros(1)])[key] + torch.arange(slots, device=key.device) - start[key]
        row = torch.where(key < experts, row, rows)                    # one row too many takes what no expert gets
        slot_row = torch.empty_like(row)
        slot_row[order] = row
        row_token = torch.full((rows + 1,), -1, device=key.device)
        row_token[row] = order // top_k
        used = (row_token[:rows] >= 0)[:, None]
        x = s["x"].float()
        ys = torch.cat([s["ys"].float(), x.new_zeros(1, x.shape[1])])
        w = torch.where(s["idx"] >= 0, s["weight"], 0.0)
        picked = ys[slot_row].view(tokens, top_k, -1)
        got = {"offsets": torch.cat([offsets, padded.sum()[None]]).int(),
               "slot_row": torch.where(slot_row < rows, slot_row, -1).int().view(tokens, top_k),
               "xs": torch.where(used, x[row_token[:rows].clamp_min(0)], 0.0).to(dtype),
               "out": (picked * w[:, :, None]).sum(1).to(dtype)}
        if s["train"]:
            dout = s["dout"].float()
            got["dweight"] = torch.where(s["idx"] >= 0, (picked * dout[:, None]).sum(2), 0.0)
            dys = x.new_zeros(rows + 1, x.shape[1])
            dys[slot_row] = (dout[:, None] * w[:, :, None]).view(slots, -1)
            got["dys"] = dys[:rows].to(dtype)
            dxs = torch.cat([s["dxs"].float(), x.new_zeros(1, x.shape[1])])
            got["dx"] = dxs[slot_row].view(tokens, top_k, -1).sum(1).to(dtype)
        return got
    u = s["update"].float()
    tall = u.shape[1] > u.shape[2]
    x = u.transpose(1, 2) if tall else u
    x = x / (torch.sqrt((x * x).sum((1, 2), keepdim=True)) + 1e-7)
    a, b, c = _COEFFICIENTS
    for _ in range(s["steps"]):
        gram = torch.matmul(x, x.transpose(1, 2))
        x = a * x + torch.matmul(b * gram + c * torch.matmul(gram, gram), x)
    return {"update": (x.transpose(1, 2) if tall else x).to(torch.bfloat16).contiguous()}


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["op"] == "norm":
        n, wsize = case["rows"] * case["hidden"], 2 if case["wtype"] == "bf16" else 4
        vectors = 1 + case["bias"]
        return {"bytes": n * size * (4 if case["train"] else 2) + case["hidden"] * wsize * vectors * (2 if case["train"] else 1),
                "flops": n * (24 if case["train"] else 8)}
    if case["op"] == "route":
        tokens, hidden, top_k = case["tokens"], case["hidden"], case["top_k"]
        slots, rows = tokens * top_k, _rows_cap(case)
        filled = slots * (1.0 - case["empty"])
        # forward: x, the filled rows of ys, indices, weights -> xs (all rows), out, slot rows
        moved = hidden * size * (tokens + filled + rows + tokens) + slots * 12 + case["experts"] * 4
        flops = 2 * filled * hidden
        if case["train"]:
            # backward: dout, the filled rows of dxs -> dys (all rows), dx, dweight
            moved += hidden * size * (tokens + filled + rows + tokens) + slots * 4
            flops += 4 * filled * hidden
        return {"bytes": moved, "flops": flops}
    m, n = min(case["m"], case["n"]), max(case["m"], case["n"])
    # a step: the Gram matrix and its square are symmetric, so half of their products determine them
    step = m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n
    return {"bytes": case["batch"] * m * n * (size + 2), "flops": case["batch"] * case["steps"] * step}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w = s["x"].double(), s["weight"].double()
        b = 0.0 if s["shift"] is None else s["shift"].double()
        h = x.shape[1]
        mean = x.sum(1) / h
        var = (x * x).sum(1) / h - mean * mean
        scale = 1.0 / torch.sqrt(var + 1e-5)
        z = (x - mean[:, None]) * scale[:, None]
        got = {"y": torch.addcmul(torch.zeros_like(z) + b, z, w)}
        if case["train"]:
            # the Jacobian of z applied to the incoming gradient, as projections off the constant vector and off z
            dy = s["dy"].double()
            v = dy * w
            along_one = torch.einsum("rh->r", v) / h
            along_z = torch.einsum("rh,rh->r", v, z) / h
            got["dx"] = (v - along_one[:, None] - z * along_z[:, None]) * scale[:, None]
            got["dweight"] = torch.einsum("rh,rh->h", dy, z)
            if s["shift"] is not None:
                got["dshift"] = torch.einsum("rh->h", dy)
        return got
    if case["op"] == "route":
        # by rank: a slot's row is its expert's first row plus the number of earlier slots of that expert
        tokens, top_k = s["idx"].shape
        rows, align = s["ys"].shape[0], case["align"]
        flat = s["idx"].reshape(-1)
        slot_row = torch.full((tokens * top_k,), -1, dtype=torch.long, device=flat.device)
        offsets, at = [], 0
        for e in range(case["experts"]):
            mine = (flat == e).nonzero()[:, 0]
            offsets.append(at)
            slot_row[mine] = at + torch.arange(mine.numel(), device=flat.device)
            at += -(-mine.numel() // align) * align
        offsets.append(at)
        filled = (slot_row >= 0).nonzero()[:, 0]
        to, token = slot_row[filled], filled // top_k
        x, ys, w = s["x"].double(), s["ys"].double(), s["weight"].double().reshape(-1)[filled]
        xs = x.new_zeros(rows, x.shape[1])
        xs[to] = x[token]
        out = torch.zeros_like(x).index_add_(0, token, ys[to] * w[:, None])
        got = {"offsets": torch.tensor(offsets, dtype=torch.int32), "slot_row": slot_row.int().view(tokens, top_k), "xs": xs, "out": out}
        if case["train"]:
            dout = s["dout"].double()
            dw = x.new_zeros(tokens * top_k)
            dw[filled] = torch.einsum("sh,sh->s", ys[to], dout[token])
            dys = torch.zeros_like(ys)
            dys[to] = dout[token] * w[:, None]
            got["dweight"], got["dys"] = dw.view(tokens, top_k), dys
            got["dx"] = torch.zeros_like(x).index_add_(0, token, s["dxs"].double()[to])
        return got
    # the steps as one polynomial of the first Gram matrix: x_k = p_k x_0 and gram_k = p_k gram_0 p_k, all of which commute
    x = s["update"].double()
    left = x.shape[1] <= x.shape[2]
    x = x / (torch.linalg.vector_norm(x, dim=(1, 2), keepdim=True) + 1e-7)
    gram = torch.matmul(x, x.mT) if left else torch.matmul(x.mT, x)
    a, b, c = _COEFFICIENTS
    one = torch.eye(gram.shape[1], dtype=x.dtype, device=x.device)
    total = one
    for _ in range(case["steps"]):
        factor = a * one + torch.matmul(gram, b * one + c * gram)
        total = torch.matmul(factor, total)
        gram = torch.matmul(torch.matmul(factor, gram), factor)
    return {"update": torch.matmul(total, x) if left else torch.matmul(x, total)}
